"""How near the paged operators come to their definitions: roundings that are part of the contract, to the bit, and bounds
that name every rounding of the kernels.

Bounds, fixed beforehand. u = 2^-8 is half a unit of bf16. Rounding to bf16 moves a value by up to u of itself and, over many
values, by r = 2^-8 / sqrt(3) / sqrt(3 / (2 ln 2)) = 1.53e-3 of their 2-norm (errors uniform in a spacing, logarithms of the
values uniform in a binade). Attention rounds its output (r) and, before the product with V, its probabilities: to bf16 (r of
the sum of their contributions, which for random V is the output's own norm: sqrt(2) r = 2.2e-3 together) or, over an e4m3
cache with few rows, to f16 (three bits more: 1.5e-3). K and V scales are applied in fp32. So, over outputs of several
thousand values: 2.7e-3 and 1.9e-3. Scales rounded into the tiles would give 3.4e-3.
Per element, with A = sum_j p_j |v_j|: u |o| for the output, u A or 2^-11 A for the probabilities, and (exp(2 e) - 1) A for scores
off by e = 2^-16 max_j scale sum_d |q_d k_jd|.
"""
import math

import pytest
import torch

import model as M
from test_paged_gpu import D, DEV, U, attend64, cumulative, ints, make_cache, ops

pytestmark = pytest.mark.gpu


def check(got, want, A, reach, p_bits):
    bound = U * want.abs() + 2.0 ** -p_bits * A + torch.expm1(2 * 2.0 ** -16 * reach) * A + 1e-30
    err = (got.double() - want).abs()
    assert not got.isnan().any() and (err / bound).max().item() <= 1, (err / bound).max().item()
    return (err.norm() / want.norm()).item()


SIZES = {   # new tokens, lengths, n_q, n_kv, page
    "decode": ([1] * 5, [700, 33, 2500, 1025, 4096], 32, 8, 32),
    "few_tokens": ([4, 3, 2], [500, 1000, 65], 32, 8, 16),
    "chunk": ([200], [1500], 16, 4, 64),
    "chunks": ([64, 33, 129], [900, 2000, 129], 32, 8, 16),
}


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("name", SIZES)
def test_attention_rounds_only_probabilities_and_outputs(name, fp8):
    n, lens, n_q, n_kv, page = SIZES[name]
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(len(name))
    c, rows = make_cache(lens, n_kv, page, fp8, g)
    q = (torch.randn(sum(n), n_q, D, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    out, cu = torch.empty_like(q), cumulative(n)
    k.paged_attention(q, ints(cu), ints(lens), c["table"], c["k"], c["v"], out, D ** -0.5, max(n), k_scale=c["ks"], v_scale=c["vs"])
    few = fp8 and max(n) * n_q // n_kv <= 16
    want = [attend64(q[a:b].double(), *rows[i], lens[i] - n[i], D ** -0.5) for i, (a, b) in enumerate(zip(cu, cu[1:]))]
    rel = check(out, *(torch.cat(x) for x in zip(*want)), 11 if few else 8)
    assert rel < (1.9e-3 if few else 2.7e-3), rel


@pytest.mark.parametrize("name", ["decode", "few_tokens"])
def test_few_rows_over_bf16_pages_keep_their_probabilities(name):
    """P goes to the bf16 products in two parts, its rounding and what that leaves (2^-16 of it at most is lost): the
    output's own rounding is all that counts, as in the contiguous cache's attention."""
    n, lens, n_q, n_kv, page = SIZES[name]
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(len(name))
    c, rows = make_cache(lens, n_kv, page, False, g)
    q = (torch.randn(sum(n), n_q, D, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    out, cu = torch.empty_like(q), cumulative(n)
    k.paged_attention(q, ints(cu), ints(lens), c["table"], c["k"], c["v"], out, D ** -0.5, max(n))
    want = [attend64(q[a:b].double(), *rows[i], lens[i] - n[i], D ** -0.5) for i, (a, b) in enumerate(zip(cu, cu[1:]))]
    rel = check(out, *(torch.cat(x) for x in zip(*want)), 16)
    assert rel < 1.9e-3, rel


def set_rows(c, table, page, pos, K=None, V=None):
    """Overwrite positions of sequence 0; returns the rows as the cache holds them, in 64 bits."""
    pg, slot = table[0, pos // page].long(), pos % page
    held = []
    for x, pool, sc in ((K, "k", "ks"), (V, "v", "vs")):
        if c[sc] is None:
            c[pool][pg, :, slot] = x
            held.append(x.double())
        else:
            q8, s = M.quantize_kv_rows(x)
            c[pool][pg, :, slot] = q8.view(torch.uint8)
            c[sc][pg, :, slot] = s
            held.append(q8.float().double() * s.double()[..., None])
    return held


@pytest.mark.parametrize("n", [1, 4, 70])
@pytest.mark.parametrize("big", ["first", "middle", "last", "scattered"])
def test_value_rows_of_very_different_size(n, big):
    """e4m3 value rows 2^45 times the others', whose own weights are nearly zero (2^-60 and less): what the others give must
    not be lost beside them."""
    k = ops()
    L, n_kv, n_q, page = 700, 2, 8, 32
    g = torch.Generator(device=DEV).manual_seed(n)
    c, _ = make_cache([L], n_kv, page, True, g)
    K, V = (torch.randn(L, n_kv, D, generator=g, device=DEV) for _ in range(2))
    K[:, :, 0] = 3.0
    at = {"first": [0], "middle": [333], "last": [L - n], "scattered": [5, 130, 131, 400, 601]}[big]
    V[at] *= 2.0 ** 45
    K[at, :, 0] = -3.0
    pos = torch.arange(L, device=DEV)
    K, V = set_rows(c, c["table"], page, pos, K.to(torch.bfloat16), V.to(torch.bfloat16))
    q = torch.randn(n, n_q, D, generator=g, device=DEV)
    q[:, :, 0] = 90.0                                # 6 x 90 / sqrt(128) = 47.7, a factor of 2^-68 before the rest's few
    q = q.to(torch.bfloat16)
    out = torch.empty_like(q)
    k.paged_attention(q, ints([0, n]), ints([L]), c["table"], c["k"], c["v"], out, D ** -0.5, n, k_scale=c["ks"], v_scale=c["vs"])
    want, A, reach = attend64(q.double(), K, V, L - n, D ** -0.5)
    assert (want.abs() / 2.0 ** 30).max() < 1        # (the large rows are not what the answer is)
    check(out, want, A, reach, 11 if n * n_q // n_kv <= 16 else 8)


@pytest.mark.parametrize("n", [1, 4, 70])
def test_weights_and_value_rows_that_balance(n):
    """Scores that rise by 40 in steps while the value rows fall by as much: every step counts alike in the output."""
    k = ops()
    L, n_kv, n_q, page = 700, 2, 8, 64
    g = torch.Generator(device=DEV).manual_seed(10 + n)
    c, _ = make_cache([L], n_kv, page, True, g)
    K, V = (torch.randn(L, n_kv, D, generator=g, device=DEV) for _ in range(2))
    steps = torch.linspace(0, 1, L, device=DEV)[:, None, None]
    K[:, :, :1] = 10 * steps - 5
    V *= torch.exp(-40 * steps)
    pos = torch.arange(L, device=DEV)
    K, V = set_rows(c, c["table"], page, pos, K.to(torch.bfloat16), V.to(torch.bfloat16))
    q = torch.randn(n, n_q, D, generator=g, device=DEV)
    q[:, :, 0] = 4 * math.sqrt(D)
    q = q.to(torch.bfloat16)
    out = torch.empty_like(q)
    k.paged_attention(q, ints([0, n]), ints([L]), c["table"], c["k"], c["v"], out, D ** -0.5, n, k_scale=c["ks"], v_scale=c["vs"])
    check(out, *attend64(q.double(), K, V, L - n, D ** -0.5), 11 if n * n_q // n_kv <= 16 else 8)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 4, 200])
def test_large_values_under_rising_scores(n, fp8):
    """Values of 2^100 while the running maximum rises by 2^26 in weight a tile: sums stay finite."""
    k = ops()
    L, n_kv, n_q, page = 1500, 2, 8, 64
    g = torch.Generator(device=DEV).manual_seed(n)
    c, _ = make_cache([L], n_kv, page, fp8, g)
    K, V = (torch.randn(L, n_kv, D, generator=g, device=DEV) for _ in range(2))
    K[:, :, 0] = torch.linspace(-40, 40, L, device=DEV)[:, None]
    pos = torch.arange(L, device=DEV)
    K, V = set_rows(c, c["table"], page, pos, K.to(torch.bfloat16), (V * 2.0 ** 100).to(torch.bfloat16))
    q = torch.randn(n, n_q, D, generator=g, device=DEV)
    q[:, :, 0] = 30
    q = q.to(torch.bfloat16)
    out = torch.empty_like(q)
    k.paged_attention(q, ints([0, n]), ints([L]), c["table"], c["k"], c["v"], out, D ** -0.5, n, k_scale=c["ks"], v_scale=c["vs"])
    check(out, *attend64(q.double(), K, V, L - n, D ** -0.5), 11 if fp8 and n * n_q // n_kv <= 16 else 8)
    if not fp8:
        q, kk, v = (x.to(torch.bfloat16) for x in (q.expand(n, -1, -1), K[:n].contiguous(), V[:n].contiguous()))
        k.packed_attention(q, kk, v, ints([0, n]), out, D ** -0.5, n)
        check(out, *attend64(q.double(), kk.double(), v.double(), 0, D ** -0.5), 8)


@pytest.mark.parametrize("amax", ["normal", "multiples of 7", "tiny", "huge"])
def test_e4m3_rows_are_the_rounded_quotients(amax):
    """Stored rows to the bit: s = max|x| / 448 and q = e4m3(x / s), each rounded once from fp32 quotients. bf16 rows lie on
    ties of e4m3 often (a maximum of 7, 14, 21, ... makes s a short number), where a quotient that is off by an ulp
    lands on the other neighbour."""
    k = ops()
    g = torch.Generator().manual_seed(len(amax))
    T, n_kv, page = 512, 4, 16
    x = torch.randn(T, n_kv, D, generator=g)
    if amax == "multiples of 7":
        x[:, :, 0] = 7.0 * torch.randint(1, 37, (T, n_kv), generator=g)
        x[:, :, 1:] = torch.randint(-40, 41, (T, n_kv, D - 1), generator=g) / 8
    x = (x * {"tiny": 1e-30, "huge": 1e37}.get(amax, 1.0)).to(torch.bfloat16)
    if amax == "tiny":
        x[::2] = (x[::2].float() * 1e-8).to(torch.bfloat16)     # down to subnormals
        x[0], x[1, :, 1:] = 0, 0
    qkv = torch.zeros(T, 6 * n_kv * D, dtype=torch.bfloat16, device=DEV)
    qkv[:, 5 * n_kv * D:] = x.flatten(1).to(DEV)
    c, _ = make_cache([T], n_kv, page, True, torch.Generator(device=DEV).manual_seed(1))
    cos, sin = M.rope_angles(T, 128, 1e6, DEV)
    q_out = torch.empty(T, 4 * n_kv, D, dtype=torch.bfloat16, device=DEV)
    k.paged_qkv(qkv, ints([0, T]), ints([T]), c["table"], c["k"], c["v"], q_out, cos, sin, k_scale=c["ks"], v_scale=c["vs"])
    pos = torch.arange(T, device=DEV)
    pg, slot = c["table"][0, pos // page].long(), pos % page
    # (the reference in 64 bits: a quotient of two fp32 numbers rounds to fp32 alike from its 64-bit value)
    s = (x.double().abs().amax(-1) / 448).float()
    want = torch.where(s[..., None] > 0, (x.double() / s.clamp(min=1e-300).double()[..., None]), 0.0).float()
    want = want.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(c["vs"][pg, :, slot].cpu(), s)
    assert torch.equal(c["v"][pg, :, slot].cpu(), want)

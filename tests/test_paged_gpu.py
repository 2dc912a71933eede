"""The paged-serving operators (csrc/paged.cuh and the ragged attention) against plain implementations in 64 bits, at
the sizes and masks where they can go wrong.

Bounds, fixed beforehand (u = 2^-8, half a unit of bf16, which has 8 significant bits):
* paged_qkv: q and bf16 rows: one rounding, |err| <= u |x| plus fp32 noise 2^-18 of the head's largest value (a norm's
  sum, two products). e4m3 rows: s within 2^-20 relative, x within half an e4m3 step (2^-4 |x|, at least s 2^-10).
* paged_kv_read: bf16 rows bit for bit; dequantised rows u |x|.
* attention, per element, with A = sum_j p_j |v_j|: the output's rounding u |o|, the probabilities' rounding to bf16
  u A, and scores off by at most e give a relative change of each weight below exp(2 e) - 1. e = 2^-16 max_j scale
  sum_d |q_d k_jd| (fp32 sums of 128 products, the exponential). An e4m3 cache may be multiplied by its scales and
  rounded to bf16 first: u more of A for V, and e = (u + 2^-16) max_j scale sum_d |q_d k_jd|.
  Over a whole output the roundings are independent: relative 2-norm below 4e-3 (bf16), 6e-3 (e4m3).
"""
import math

import pytest
import torch

import model as M

pytestmark = pytest.mark.gpu
D, U, DEV = 128, 2.0 ** -8, "cuda"


def ops():
    from kernels import ops as o
    return o()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def cumulative(n):
    c = [0]
    for x in n:
        c.append(c[-1] + x)
    return c


def make_cache(lens, n_kv, page, fp8, g, spare=2, poison=True, width=None):
    """Pages with the given lengths' rows; every other slot holds NaN (e4m3: NaN scales too). Returns the call's
    tensors and the rows in 64 bits, [len, n_kv, D] per sequence."""
    per = [-(-n // page) for n in lens]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((max(len(lens), 1), width or max(per + [1])), -7, dtype=torch.int32, device=DEV)
    k = torch.full((pages, n_kv, page, D), math.nan, dtype=torch.bfloat16, device=DEV)
    v = k.clone()
    ks = vs = None
    if fp8:
        k, v = (torch.full((pages, n_kv, page, D), 0x7F, dtype=torch.uint8, device=DEV) for _ in range(2))
        ks, vs = (torch.full((pages, n_kv, page), math.nan, device=DEV) for _ in range(2))
    rows, at = [], 0
    for b, n in enumerate(lens):
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
        pos = torch.arange(n, device=DEV)
        pg, slot = table[b, pos // page].long(), pos % page
        both = []
        for pool, sc in ((k, ks), (v, vs)):
            x = torch.randn(n, n_kv, D, generator=g, device=DEV).to(torch.bfloat16)
            if fp8:
                q, s = M.quantize_kv_rows(x)
                pool[pg, :, slot] = q.view(torch.uint8)
                sc[pg, :, slot] = s
                both.append(q.float().double() * s.double()[..., None])
            else:
                pool[pg, :, slot] = x
                both.append(x.double())
        rows.append(both)
    return dict(k=k, v=v, ks=ks, vs=vs, table=table), rows


def attend64(q, K, V, first, scale):
    """q [n, n_q, D], K/V [L, n_kv, D] in 64 bits; row i sees keys 0 .. first + i. Returns (out, A, reach) where reach =
    max over visible keys of scale sum |q k|."""
    n, n_q, _ = q.shape
    L, n_kv, _ = K.shape
    G = n_q // n_kv
    out, A, reach = (torch.zeros(n, n_q, D, dtype=torch.float64, device=DEV) for _ in range(3))
    hidden = torch.arange(L, device=DEV)[None, :] > (first + torch.arange(n, device=DEV))[:, None]
    for h in range(n_q):
        if not L:
            continue
        s = (q[:, h] @ K[:, h // G].T * scale).masked_fill(hidden, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = (s - m.masked_fill(m == -math.inf, 0)).exp()
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        out[:, h], A[:, h] = p @ V[:, h // G], p @ V[:, h // G].abs()
        r = (q[:, h].abs() @ K[:, h // G].abs().T * scale).masked_fill(hidden, 0)
        reach[:, h] = r.amax(-1, keepdim=True)
    return out, A, reach


def check_attention(got, want, A, reach, fp8):
    u = U if fp8 else 0.0
    bound = U * want.abs() + (U + u) * A + torch.expm1(2 * (u + 2.0 ** -16) * reach) * A + 1e-30
    err = (got.double() - want).abs()
    assert not got.isnan().any()
    worst = (err / bound).max().item() if err.numel() else 0
    assert worst <= 1, worst
    if want.norm() > 0:
        rel = (err.norm() / want.norm()).item()
        assert rel < (6e-3 if fp8 else 4e-3), rel


# name: (new tokens, lengths, n_q, n_kv, page)
PAGED = {
    "one_key": ([1], [1], 32, 8, 16),
    "short": ([1], [17], 32, 8, 16),
    "page_ends": ([1] * 9, [15, 16, 17, 63, 64, 65, 127, 128, 129], 32, 8, 64),
    "page_128": ([1] * 4, [1, 127, 128, 300], 16, 4, 128),
    "ragged_decode": ([1] * 7, [700, 1, 2500, 64, 33, 1025, 4096], 32, 8, 32),
    "few_tokens": ([2, 8, 5, 1, 3], [2, 500, 64, 65, 1000], 32, 8, 16),
    "few_to_many": ([7, 8, 9, 10, 16, 17], [900, 128, 9, 64, 129, 17], 32, 8, 64),
    "no_tokens": ([1, 0, 3, 0], [50, 40, 3, 0], 32, 8, 16),
    "more_tokens_than_keys": ([5, 1, 40], [2, 0, 33], 32, 8, 16),
    "chunk": ([128], [1000], 32, 8, 64),
    "chunk_odd": ([129, 1, 61], [129, 777, 2000], 32, 8, 32),
    "chunks": ([200, 64, 65, 33], [1500, 64, 129, 4000], 32, 8, 16),
    "mixed": ([300, 1, 1, 1, 1, 4], [2300, 5, 800, 1500, 128, 640], 32, 8, 64),
    "mha": ([1, 40, 130], [300, 100, 130], 8, 8, 16),
    "group_3": ([1, 9, 90], [300, 100, 257], 12, 4, 32),
    "group_5": ([1, 7, 55], [300, 100, 257], 10, 2, 64),
    "group_7": ([1, 4, 5, 77], [129, 640, 100, 257], 28, 4, 128),
    "group_16": ([1, 2, 3, 33], [129, 640, 100, 257], 16, 1, 16),
    "group_32": ([1, 2, 20], [129, 640, 100], 32, 1, 64),
    "long": ([1, 20], [20000, 9000], 8, 2, 64),
    "many": ([1] * 100 + [3] * 40, list(range(1, 141)), 4, 1, 16),
    "many_mixed": ([1, 30, 0] * 15, [40 + 37 * i for i in range(45)], 8, 2, 16),
}


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("name", PAGED)
def test_paged_attention(name, fp8):
    n, lens, n_q, n_kv, page = PAGED[name]
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(sum(lens) + n_q)
    c, rows = make_cache(lens, n_kv, page, fp8, g)
    T = sum(n)
    q = (torch.randn(T, n_q, D, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    cu = ints(cumulative(n))
    args = (q, cu, ints(lens), c["table"], c["k"], c["v"])
    k.paged_attention(*args, out, D ** -0.5, max(n), k_scale=c["ks"], v_scale=c["vs"])
    again = torch.empty_like(out)
    k.paged_attention(*args, again, D ** -0.5, max(n), k_scale=c["ks"], v_scale=c["vs"])
    torch.cuda.synchronize()
    assert k.device_error() == 0
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))     # no order of additions that changes
    at = 0
    for b in range(len(n)):
        want, A, reach = attend64(q[at:at + n[b]].double(), *rows[b], lens[b] - n[b], D ** -0.5)
        check_attention(out[at:at + n[b]], want, A, reach, fp8)
        at += n[b]


@pytest.mark.parametrize("lens", [[1], [127], [128], [129], [300], [1, 1, 1], [5, 0, 64, 65], [0, 0, 7], [513, 31, 256],
                                  [2000, 1, 77], list(range(0, 71))], ids=str)
@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (12, 4), (10, 2), (28, 4), (16, 1)], ids=str)
def test_packed_attention(lens, heads):
    n_q, n_kv = heads
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(sum(lens) + n_q)
    T = sum(lens)
    x = (torch.randn(T, n_q + 2 * n_kv, D, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    q, kk, v = x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]
    out = torch.full((T, n_q, D), 7.0, dtype=torch.bfloat16, device=DEV)
    k.packed_attention(q, kk, v, ints(cumulative(lens)), out, D ** -0.5, max(lens))
    again = torch.empty_like(out)
    k.packed_attention(q, kk, v, ints(cumulative(lens)), again, D ** -0.5, max(lens))
    torch.cuda.synchronize()
    assert k.device_error() == 0
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    at = 0
    for n in lens:
        r = slice(at, at + n)
        want, A, reach = attend64(q[r].double(), kk[r].double(), v[r].double(), 0, D ** -0.5)
        check_attention(out[r], want, A, reach, False)
        at += n


def test_packed_prompts_do_not_touch_each_other():
    """NaN and infinite rows of one prompt leave its neighbours as they are, and rows past cu[B] are not written."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(5)
    lens = [70, 130, 40, 300]
    cu = cumulative(lens)
    T = cu[-1] + 9
    q, kk, v = (torch.randn(T, h, D, generator=g, device=DEV).to(torch.bfloat16) for h in (32, 8, 8))
    for bad in (math.nan, math.inf):
        for t in (kk, v):
            t[cu[1]:cu[2]] = bad
            t[cu[4]:] = bad
        out = torch.full((T, 32, D), 7.0, dtype=torch.bfloat16, device=DEV)
        k.packed_attention(q, kk, v, ints(cu), out, D ** -0.5, max(lens))
        assert bool((out[cu[4]:] == 7).all())
        for b in (0, 2, 3):
            r = slice(cu[b], cu[b + 1])
            check_attention(out[r], *attend64(q[r].double(), kk[r].double(), v[r].double(), 0, D ** -0.5), False)
        assert bool(out[cu[1]:cu[2]].isnan().all())
    assert k.device_error() == 0


@pytest.mark.parametrize("n", [1, 100])
def test_large_scores(n):
    """Scores of several hundred: the running maximum keeps the exponentials finite and the small weights exact."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(n)
    c, rows = make_cache([1000], 8, 64, False, g)
    q = (torch.randn(n, 32, D, generator=g, device=DEV) * 200).to(torch.bfloat16)
    out = torch.empty_like(q)
    k.paged_attention(q, ints([0, n]), ints([1000]), c["table"], c["k"], c["v"], out, D ** -0.5, n)
    want, A, reach = attend64(q.double(), *rows[0], 1000 - n, D ** -0.5)
    check_attention(out, want, A, reach, False)


def test_rising_scores_rescale_the_sums():
    """Keys ordered so that the running maximum rises in every tile."""
    k = ops()
    L, n_kv, page = 1500, 2, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    c, rows = make_cache([L], n_kv, page, False, g)
    K = torch.randn(L, n_kv, D, generator=g, device=DEV)
    K[:, :, 0] = torch.linspace(-40, 40, L, device=DEV)[:, None]
    K = K.to(torch.bfloat16)
    pos = torch.arange(L, device=DEV)
    c["k"][c["table"][0, pos // page].long(), :, pos % page] = K
    for n in (1, 6, 200):
        q = torch.randn(n, 8, D, generator=g, device=DEV)
        q[:, :, 0] = 30
        q = q.to(torch.bfloat16)
        out = torch.empty_like(q)
        k.paged_attention(q, ints([0, n]), ints([L]), c["table"], c["k"], c["v"], out, D ** -0.5, n)
        check_attention(out, *attend64(q.double(), K.double(), rows[0][1], L - n, D ** -0.5), False)


@pytest.mark.parametrize("group", [3, 4])
def test_a_row_depends_on_its_own_tokens_only(group):
    """The same prompt and chunk beside neighbours of ordinary, huge and NaN values: the same bits."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(group)
    n_kv, n = 2, 50
    q, kk, v = (torch.randn(n, h, D, generator=g, device=DEV).to(torch.bfloat16) for h in (n_kv * group, n_kv, n_kv))
    c, _ = make_cache([n + 400], n_kv, 16, False, g)
    seen = []
    for other in (1.0, 1e4, math.nan):
        def beside(x):
            return torch.cat([x, torch.randn(n, x.shape[1], D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16) * other])
        qb, kb, vb = beside(q), beside(kk), beside(v)
        a, b = torch.empty_like(qb), torch.empty_like(qb)
        k.packed_attention(qb, kb, vb, ints([0, n, 2 * n]), a, D ** -0.5, n)
        table = c["table"].expand(2, -1).contiguous()
        k.paged_attention(qb, ints([0, n, 2 * n]), ints([n + 400, 300]), table, c["k"], c["v"], b, D ** -0.5, n)
        seen.append((a[:n].clone(), b[:n].clone()))
    for a, b in seen[1:]:
        assert torch.equal(a.view(torch.int16), seen[0][0].view(torch.int16)) and torch.equal(b.view(torch.int16), seen[0][1].view(torch.int16))
    assert k.device_error() == 0


@pytest.mark.parametrize("n", [1, 64])
def test_strides_streams_and_padding(n):
    """q and out inside wider tensors, a table wider than it is read, rows past cu[B], a stream of its own."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(3)
    lens, n_q, n_kv = [200, 333], 16, 4
    c, rows = make_cache(lens, n_kv, 16, False, g, width=64)
    T = 2 * n + 3
    wide = torch.randn(T, n_q + 2, 2 * D, generator=g, device=DEV).to(torch.bfloat16)
    q = wide[:, 1:n_q + 1, D:]
    out_wide = torch.full((n_q, T, D + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    out = out_wide.transpose(0, 1)[:, :, :D]
    cu, sl = ints([0, n, 2 * n]), ints(lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k.paged_attention(q, cu, sl, c["table"], c["k"], c["v"], out, D ** -0.5, n)
    torch.cuda.current_stream().wait_stream(side)
    assert bool((out[2 * n:] == 7).all()) and bool((out_wide[:, :, D:] == 7).all())
    for b in range(2):
        r = slice(b * n, (b + 1) * n)
        check_attention(out[r], *attend64(q[r].double(), *rows[b], lens[b] - n, D ** -0.5), False)
    assert k.device_error() == 0


def test_pool_past_32_bit_offsets():
    """Pages whose byte offsets pass 2^32: the last of 6 GiB pools."""
    k = ops()
    n_kv, page = 8, 128
    pages = 6 * (1 << 30) // (n_kv * page * D * 2)
    g = torch.Generator(device=DEV).manual_seed(9)
    kp, vp = (torch.empty(pages, n_kv, page, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    used = [pages - 1, 3, pages - 2]
    for t in (kp, vp):
        t[used] = torch.randn(3, n_kv, page, D, generator=g, device=DEV).to(torch.bfloat16)
    table, L = ints([used]), 3 * page - 5
    K, V = (t[used].transpose(1, 2).reshape(-1, n_kv, D)[:L].double() for t in (kp, vp))
    for n in (1, 40):
        q = torch.randn(n, 32, D, generator=g, device=DEV).to(torch.bfloat16)
        out = torch.empty_like(q)
        k.paged_attention(q, ints([0, n]), ints([L]), table, kp, vp, out, D ** -0.5, n)
        check_attention(out, *attend64(q.double(), K, V, L - n, D ** -0.5), False)
    ko, vo = (torch.empty(L, n_kv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k.paged_kv_read(ints([0, L]), table, kp, vp, ko, vo)
    assert torch.equal(ko.double(), K) and torch.equal(vo.double(), V)
    assert k.device_error() == 0


def test_attention_in_a_graph_follows_the_lengths():
    """A captured decode step replayed with other lengths and tables."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(4)
    c, rows = make_cache([1500, 900, 40], 8, 64, False, g)
    q = torch.randn(3, 32, D, generator=g, device=DEV).to(torch.bfloat16)
    out = torch.empty_like(q)
    cu, lens, ws = ints([0, 1, 2, 3]), ints([3, 3, 3]), k.attention_workspace(DEV)

    def step():
        k.paged_attention(q, cu, lens, c["table"], c["k"], c["v"], out, D ** -0.5, 1, workspace=ws)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for now in ([1500, 900, 40], [1, 64, 39], [700, 899, 2]):
        lens.copy_(ints(now))
        graph.replay()
        for b in range(3):
            want = attend64(q[b:b + 1].double(), rows[b][0][:now[b]], rows[b][1][:now[b]], now[b] - 1, D ** -0.5)
            check_attention(out[b:b + 1], *want, False)
    assert k.device_error() == 0


def test_capture_needs_a_workspace_of_the_callers():
    k = ops()
    c, _ = make_cache([40], 8, 16, False, torch.Generator(device=DEV).manual_seed(1))
    q = torch.zeros(1, 32, D, dtype=torch.bfloat16, device=DEV)
    cu, lens = ints([0, 1]), ints([40])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k._scratch.pop(("ragged", q.get_device(), torch.cuda.current_stream().cuda_stream), None)
        with pytest.raises(RuntimeError, match="before the capture"):
            k.paged_attention(q, cu, lens, c["table"], c["k"], c["v"], q, 0.1, 1)


# ---- the cache's rows ----------------------------------------------------------------------------------------
def rotate64(x, cos, sin, interleaved):
    x = x.clone()
    h = cos.shape[-1]
    a = torch.arange(h, device=DEV) * 2 if interleaved else torch.arange(h, device=DEV)
    b = a + (1 if interleaved else h)
    lo, hi = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = lo * cos - hi * sin, hi * cos + lo * sin
    return x


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("rot,interleaved,norm,page,n_q,n_kv", [
    (128, False, True, 64, 32, 8), (128, True, False, 16, 8, 2), (64, False, False, 32, 4, 1), (64, True, True, 128, 16, 4),
    (96, False, True, 16, 12, 4), (16, True, True, 16, 10, 2), (32, False, False, 64, 3, 3)])
def test_paged_qkv(rot, interleaved, norm, page, n_q, n_kv, fp8):
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(rot + n_q)
    n, lens = [1, 0, 40, 3, 130], [77, 12, 40, 1000, 131]
    c, _ = make_cache(lens, n_kv, page, fp8, g)
    T = sum(n)
    wide = torch.randn(T + 2, (n_q + 2 * n_kv) * D + 8, generator=g, device=DEV).to(torch.bfloat16)
    wide[2, n_q * D:(n_q + 1) * D] = 0                                    # a zero key row
    qkv = wide[:, :(n_q + 2 * n_kv) * D]
    cos, sin = M.rope_angles(1000, rot, 1e6, DEV, {"type": "yarn", "factor": 4.0, "original_max_position": 200})
    qn, kn = ((torch.randn(D, generator=g, device=DEV) * 0.2 + 1).to(torch.bfloat16) if norm else None for _ in range(2))
    q_out = torch.full((T + 2, n_q, D), 7.0, dtype=torch.bfloat16, device=DEV)
    k_out = torch.full((T + 2, n_kv, D), 7.0, dtype=torch.bfloat16, device=DEV)
    before = {x: c[x].clone() for x in ("k", "v")}
    cu = ints(cumulative(n))
    k.paged_qkv(qkv, cu, ints(lens), c["table"], c["k"], c["v"], q_out, cos, sin, q_norm=qn, k_norm=kn, eps=1e-6,
                interleaved=interleaved, k_scale=c["ks"], v_scale=c["vs"], k_out=k_out)
    torch.cuda.synchronize()
    assert k.device_error() == 0
    assert bool((q_out[T:] == 7).all()) and bool((k_out[T:] == 7).all())
    touched = torch.zeros(c["k"].shape[:1] + c["k"].shape[2:3], dtype=torch.bool, device=DEV)
    at = 0
    for b in range(len(n)):
        pos = torch.arange(lens[b] - n[b], lens[b], device=DEV)
        pg, slot = c["table"][b, pos // page].long(), pos % page
        touched[pg, slot] = True
        x = qkv[at:at + n[b]].double().view(n[b], n_q + 2 * n_kv, D)
        cs, sn = cos[pos].double()[:, None], sin[pos].double()[:, None]

        def turned(y, w):
            if w is not None:
                y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            return rotate64(y, cs, sn, interleaved)

        q64, k64, v64 = turned(x[:, :n_q], qn), turned(x[:, n_q:n_q + n_kv], kn), x[:, n_q + n_kv:]

        def near(got, want):
            err = (got.double() - want).abs()
            return bool((err <= U * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True)).all())

        assert near(q_out[at:at + n[b]], q64) and near(k_out[at:at + n[b]], k64)
        for name, want in (("k", k64), ("v", v64)):
            if not fp8:
                assert near(c[name][pg, :, slot], want)
                continue
            s = c[name + "s"][pg, :, slot].double()
            assert bool(((s - want.abs().amax(-1) / 448).abs() <= 2.0 ** -20 * s).all())
            got = c[name][pg, :, slot].view(torch.float8_e4m3fn).float().double() * s[..., None]
            # half a step of e4m3 (3 mantissa bits), with the scale's and the quotient's fp32 error beside it
            assert bool(((got - want).abs() <= (2.0 ** -4 + 2.0 ** -18) * want.abs() + 1.001 * 2.0 ** -10 * s[..., None]).all())
        at += n[b]
    for x in ("k", "v"):                                                  # no other byte of the pools
        same = (c[x].view(torch.uint8) == before[x].view(torch.uint8)).flatten(3).all(-1).all(1)
        assert bool((same | touched).all())


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("lens,page,n_kv", [([1], 16, 8), ([0, 5, 64, 0, 65], 64, 8), ([300, 17], 32, 3), ([129], 128, 1)])
def test_paged_kv_read(lens, page, n_kv, fp8):
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(page)
    c, rows = make_cache(lens, n_kv, page, fp8, g)
    T = sum(lens)
    # into a contiguous cache's layout [n_kv, max_seq, 128]
    ko, vo = (torch.full((n_kv, T + 4, D), 7.0, dtype=torch.bfloat16, device=DEV).transpose(0, 1) for _ in range(2))
    k.paged_kv_read(ints(cumulative(lens)), c["table"], c["k"], c["v"], ko, vo, k_scale=c["ks"], v_scale=c["vs"])
    for out, i in ((ko, 0), (vo, 1)):
        want = torch.cat([r[i] for r in rows])
        err = (out[:T].double() - want).abs()
        assert bool((err <= (U * want.abs() if fp8 else 0)).all())
        assert bool((out[T:] == 7).all())
    starts = [n // 3 for n in lens]                                       # the rest of each sequence
    part = [n - s for n, s in zip(lens, starts)]
    ko, vo = (torch.empty(sum(part), n_kv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k.paged_kv_read(ints(cumulative(part)), c["table"], c["k"], c["v"], ko, vo, k_scale=c["ks"], v_scale=c["vs"],
                    starts=ints(starts))
    want = torch.cat([r[0][s:] for r, s in zip(rows, starts)])
    assert bool(((ko.double() - want).abs() <= (U * want.abs() if fp8 else 0)).all())
    assert k.device_error() == 0


def test_written_rows_read_back():
    """What paged_qkv wrote comes out of paged_kv_read: k_out bit for bit (bf16), within half a step of e4m3."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(6)
    cos, sin = M.rope_angles(256, 128, 1e6, DEV)
    n = [100, 7, 64]
    for fp8 in (False, True):
        c, _ = make_cache(n, 8, 16, fp8, g)
        T, cu = sum(n), ints(cumulative(n))
        qkv = torch.randn(T, 48 * D, generator=g, device=DEV).to(torch.bfloat16)
        q, ko, kr, vr = (torch.empty(T, h, D, dtype=torch.bfloat16, device=DEV) for h in (32, 8, 8, 8))
        k.paged_qkv(qkv, cu, ints(n), c["table"], c["k"], c["v"], q, cos, sin, k_scale=c["ks"], v_scale=c["vs"], k_out=ko)
        k.paged_kv_read(cu, c["table"], c["k"], c["v"], kr, vr, k_scale=c["ks"], v_scale=c["vs"])
        v = qkv[:, 40 * D:].view(T, 8, D)
        if not fp8:
            assert torch.equal(kr, ko) and torch.equal(vr, v)
        for got, want in ((kr, ko), (vr, v)):
            step = want.float().abs().amax(-1, keepdim=True) / 448
            assert bool(((got.float() - want.float()).abs() <= 0.0725 * want.float().abs() + step * 2.0 ** -9).all())


def test_non_finite_rows_stay_themselves():
    """A key or value row with a NaN or an infinity reads back as NaN from an e4m3 cache, its neighbours do not."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(8)
    cos, sin = M.rope_angles(64, 128, 1e6, DEV)
    c, _ = make_cache([20], 8, 16, True, g)
    qkv = torch.randn(20, 48 * D, generator=g, device=DEV).to(torch.bfloat16)
    qkv[3, 41 * D + 5] = math.nan
    qkv[9, 41 * D + 5] = math.inf
    q, kr, vr = (torch.empty(20, h, D, dtype=torch.bfloat16, device=DEV) for h in (32, 8, 8))
    cu = ints([0, 20])
    k.paged_qkv(qkv, cu, ints([20]), c["table"], c["k"], c["v"], q, cos, sin, k_scale=c["ks"], v_scale=c["vs"])
    k.paged_kv_read(cu, c["table"], c["k"], c["v"], kr, vr, k_scale=c["ks"], v_scale=c["vs"])
    bad = vr.isnan().any(-1)
    assert bad[3, 1] and bad[9, 1] and int(bad.sum()) == 2 and not kr.isnan().any()


def test_empty_batches():
    k = ops()
    c, _ = make_cache([20], 8, 16, False, torch.Generator(device=DEV).manual_seed(1))
    none, x = ints([0]), torch.empty(0, 32, D, dtype=torch.bfloat16, device=DEV)
    kv = x[:, :8]
    cos, sin = M.rope_angles(16, 128, 1e6, DEV)
    for cu, lens, table in ((none, ints([]), c["table"][:0]), (ints([0, 0]), ints([20]), c["table"])):
        k.paged_attention(x, cu, lens, table, c["k"], c["v"], x, 0.1, 1)
        k.packed_attention(x, kv, kv, cu, x, 0.1, 1)
        k.paged_kv_read(cu, table, c["k"], c["v"], kv, kv)
        k.paged_qkv(torch.empty(0, 48 * D, dtype=torch.bfloat16, device=DEV), cu, lens, table, c["k"], c["v"], x, cos, sin)
    torch.cuda.synchronize()
    assert k.device_error() == 0


# ---- refusals ------------------------------------------------------------------------------------------------
def test_refusals():
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(2)
    c, _ = make_cache([40], 8, 16, False, g)
    q = torch.randn(1, 32, D, generator=g, device=DEV).to(torch.bfloat16)
    out = torch.empty_like(q)
    good = dict(q=q, cu=ints([0, 1]), seq_lens=ints([40]), block_table=c["table"], k_pages=c["k"], v_pages=c["v"], out=out,
                scale=0.1, max_q=1)
    k.paged_attention(**good)
    wide = torch.empty(1, 32, D + 4, dtype=torch.bfloat16, device=DEV)
    for bad in (dict(q=q.float()), dict(q=q[..., :64]), dict(q=q.cpu()), dict(out=out[:, :16]), dict(cu=ints([0, 1]).long()),
                dict(cu=ints([0, 1, 1])), dict(seq_lens=ints([40, 40])), dict(seq_lens=ints([40]).float()),
                dict(block_table=c["table"].long()), dict(k_pages=c["k"].float()), dict(k_pages=c["k"][:, :4]),
                dict(k_pages=c["k"].transpose(0, 1)), dict(k_scale=torch.ones(1, device=DEV)), dict(scale=0.0),
                dict(scale=float("nan")), dict(max_q=0), dict(q=wide[..., :D], out=wide[..., :D]),
                dict(q=q[:, :12].contiguous(), out=out[:, :12].contiguous()),
                dict(workspace=torch.zeros(16, dtype=torch.uint8, device=DEV)),
                dict(k_pages=c["k"].view(torch.uint8)[..., :D].contiguous(), v_pages=c["v"].view(torch.uint8)[..., :D].contiguous())):
        with pytest.raises(RuntimeError):
            k.paged_attention(**{**good, **bad})
    odd = torch.zeros(4, 8, 24, D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="page_size"):
        k.paged_attention(**{**good, "k_pages": odd, "v_pages": odd})
    x = torch.zeros(4, 48, D, dtype=torch.bfloat16, device=DEV)
    packed = dict(q=x[:, :32], k=x[:, 32:40], v=x[:, 40:], cu=ints([0, 4]), out=torch.empty(4, 32, D, dtype=torch.bfloat16, device=DEV),
                  scale=0.1, max_q=4)
    k.packed_attention(**packed)
    for bad in (dict(k=x[:2, 32:40]), dict(v=x[:, 40:46]), dict(v=x[:, 40:].contiguous()), dict(cu=ints([0, 4]).cpu()),
                dict(out=x[:, :16]), dict(k=x[:, 32:39], v=x[:, 40:47]), dict(scale=-1.0)):
        with pytest.raises(RuntimeError):
            k.packed_attention(**{**packed, **bad})
    cos, sin = M.rope_angles(64, 128, 1e6, DEV)
    qkv = torch.zeros(1, 48 * D, dtype=torch.bfloat16, device=DEV)
    write = dict(qkv=qkv, cu=ints([0, 1]), seq_lens=ints([40]), block_table=c["table"], k_pages=c["k"], v_pages=c["v"], q_out=out,
                 cos=cos, sin=sin)
    k.paged_qkv(**write)
    for bad in (dict(qkv=qkv[:, :40 * D]), dict(qkv=qkv.float()), dict(cos=cos.double(), sin=sin.double()), dict(cos=cos[:32]),
                dict(cos=cos[:, :5].contiguous(), sin=sin[:, :5].contiguous()),
                dict(q_norm=torch.ones(D, dtype=torch.bfloat16, device=DEV)), dict(k_out=out)):
        with pytest.raises(RuntimeError):
            k.paged_qkv(**{**write, **bad})
    read = dict(cu=ints([0, 4]), block_table=c["table"], k_pages=c["k"], v_pages=c["v"], k_out=x[:, :8], v_out=x[:, 8:16])
    k.paged_kv_read(**read)
    for bad in (dict(k_out=x[:, :7]), dict(v_out=x[:, 8:16].contiguous()), dict(starts=ints([0, 0]))):
        with pytest.raises(RuntimeError):
            k.paged_kv_read(**{**read, **bad})
    torch.cuda.synchronize()
    assert k.device_error() == 0


def test_positions_outside_the_cache_set_the_error_word():
    """A length past the block table, a page id outside the pool: the row is not written, the error word says so."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(2)
    cos, sin = M.rope_angles(64, 128, 1e6, DEV)
    for table, length in (([[0, 1]], 33), ([[0, 99]], 20), ([[0, -1]], 20), ([[0, 1]], 0)):
        c, _ = make_cache([32], 8, 16, False, g)
        before = c["k"].clone()
        qkv = torch.randn(1, 48 * D, generator=g, device=DEV).to(torch.bfloat16)
        q = torch.empty(1, 32, D, dtype=torch.bfloat16, device=DEV)
        k.paged_qkv(qkv, ints([0, 1]), ints([length]), ints(table), c["k"], c["v"], q, cos, sin)
        torch.cuda.synchronize()
        assert k.device_error() == 2
        assert torch.equal(c["k"].view(torch.int16), before.view(torch.int16))
    for n in (1, 20):
        c, _ = make_cache([32], 8, 16, False, g)
        q = torch.randn(n, 32, D, generator=g, device=DEV).to(torch.bfloat16)
        k.paged_attention(q, ints([0, n]), ints([30]), ints([[0, 99]]), c["k"], c["v"], torch.empty_like(q), 0.1, n)
        torch.cuda.synchronize()
        assert k.device_error() == 2

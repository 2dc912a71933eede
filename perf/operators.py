"""The paged-serving operators and the cases they are measured on.

Four operators, each in a plain form (elementary torch operations in 32 bits, rounded once at the end) and, with
`own` set, through the framework's entry points (`kernels.ops()`):

  paged_qkv         the qkv projection's rows: per-head RMSNorm, rotary positions, K and V (quantised or not) into the
                    pages of their sequences, q to a tensor of its own
  paged_kv_read     the K and V rows of whole sequences back out of the pages, dequantised
  paged_attention   causal attention of each sequence's new tokens (one, a few, or a chunk) over its paged cache
  packed_attention  causal attention of whole prompts of different lengths, packed without padding

Sequence b of a call has its tokens in rows cu[b] .. cu[b+1] - 1; its last new token sits at position
seq_lens[b] - 1. Position p of a sequence lies in slot p % page_size of page block_table[b][p // page_size]; a page
holds [kv_heads][page_size][128] values, and for an 8-bit cache [kv_heads][page_size] fp32 row scales beside them.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128          # the framework's head size
EPS = 1e-6
E4M3_MAX = 448.0


# ---- the cases ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step's rows for a batch of 16: a launch of a few microseconds
        dict(name="qkv_decode_bf16", op="paged_qkv", batch=16, q_max=1, ctx_max=4096, n_q=32, n_kv=8, page=64, fp8=False,
             rot=128, interleaved=False, yarn=False, norm=True, lens=1),
        # the rows of many prompts at once into an 8-bit cache, positions scaled for long contexts
        dict(name="qkv_prompts_fp8", op="paged_qkv", batch=16, q_max=1024, ctx_max=0, n_q=32, n_kv=8, page=64, fp8=True,
             rot=128, interleaved=False, yarn=True, norm=True, lens=0),
        # ragged chunks, half of each head rotated in the interleaved layout, no head norm, small pages
        dict(name="qkv_ragged_fp8", op="paged_qkv", batch=7, q_max=383, ctx_max=1500, n_q=16, n_kv=4, page=16, fp8=True,
             rot=64, interleaved=True, yarn=False, norm=False, lens=3),
        # a preempted sequence leaves the pages
        dict(name="read_one_bf16", op="paged_kv_read", batch=1, ctx_max=777, n_q=32, n_kv=8, page=16, fp8=False, lens=0),
        # a whole batch at long contexts, out of an 8-bit cache
        dict(name="read_batch_fp8", op="paged_kv_read", batch=16, ctx_max=16384, n_q=32, n_kv=8, page=64, fp8=True, lens=5),
        # one sequence's decode step at a short context: latency
        dict(name="decode_one_bf16", op="paged_attention", batch=1, q_max=1, ctx_max=777, n_q=32, n_kv=8, page=16,
             fp8=False, lens=0),
        # the batch-16 decode step at contexts up to 32k, both cache types
        dict(name="decode_16_bf16", op="paged_attention", batch=16, q_max=1, ctx_max=32768, n_q=32, n_kv=8, page=64,
             fp8=False, lens=7),
        dict(name="decode_16_fp8", op="paged_attention", batch=16, q_max=1, ctx_max=32768, n_q=32, n_kv=8, page=64,
             fp8=True, lens=7),
        # one step of a server that prefills in chunks: a chunk beside sequences that decode
        dict(name="mixed_chunk_bf16", op="paged_attention", batch=9, q_max=448, ctx_max=8192, n_q=32, n_kv=8, page=32,
             fp8=False, lens=-1),
        # chunks of several sequences over an 8-bit cache
        dict(name="chunks_fp8", op="paged_attention", batch=4, q_max=509, ctx_max=8192, n_q=32, n_kv=8, page=64, fp8=True,
             lens=9),
        # one long prompt
        dict(name="prompt_8192", op="packed_attention", batch=1, q_max=8192, n_q=32, n_kv=8, lens=0),
        # the prompts that arrived together, of one token up to 2048
        dict(name="prompts_ragged", op="packed_attention", batch=9, q_max=2048, n_q=32, n_kv=8, lens=11),
    ]


HEADS = ((32, 8), (16, 4), (8, 2), (4, 1), (8, 8), (12, 4), (10, 2), (16, 1), (28, 4))


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("paged_qkv", "paged_kv_read", "paged_attention", "paged_attention", "packed_attention"))
    n_q, n_kv = rng.choice(HEADS)
    c = dict(op=op, n_q=n_q, n_kv=n_kv, lens=rng.randrange(12, 1 << 20))
    if op != "packed_attention":
        c.update(page=rng.choice((16, 32, 64, 128)), fp8=rng.random() < 0.5)
    if op == "paged_qkv":
        c.update(batch=_log(rng, 1, 64), rot=rng.choice((32, 64, 96, 128)), interleaved=rng.random() < 0.5,
                 yarn=rng.random() < 0.5, norm=rng.random() < 0.7)
        c.update(q_max=_log(rng, 1, 16384 // c["batch"]), ctx_max=_log(rng, 1, 4096))
    elif op == "paged_kv_read":
        c.update(batch=_log(rng, 1, 64))
        c.update(ctx_max=_log(rng, 16, 262144 // c["batch"]))
    elif op == "paged_attention":
        c.update(batch=_log(rng, 1, 64))
        top = min(32768, 524288 // c["batch"])
        c.update(q_max=rng.choice((1, 1, rng.randrange(2, 9), _log(rng, 8, 512))))
        c.update(ctx_max=_log(rng, c["q_max"] + 16, max(c["q_max"] + 32, min(top, 50_000_000 // (c["batch"] * c["q_max"])))))
    else:
        c.update(batch=_log(rng, 1, 32))
        c.update(q_max=_log(rng, 16, int(8192 / math.sqrt(c["batch"]))))
    return c


def _lengths(c):
    """(new tokens, cached keys with them) of each sequence. lens = 0: all at their largest; -1: one chunk, the others
    decode; else the seed of ragged lengths, of which one is the largest and, in a packed batch, one is 1."""
    B, q_max, ctx = c["batch"], c.get("q_max", 0), c.get("ctx_max", 0)
    rng = random.Random(c["lens"])
    if c["op"] == "paged_kv_read":
        k = [ctx] * B if c["lens"] == 0 else [ctx] + [rng.randint(1, ctx) for _ in range(B - 1)]
        return k, k
    if c["lens"] == 0:
        q = [q_max] * B
    elif c["lens"] == -1:
        q = [q_max] + [1] * (B - 1)
    else:
        q = [q_max] + [rng.randint(1, q_max) for _ in range(B - 1)]
    if c["op"] == "packed_attention":
        if B > 2:
            q[1] = 1
        return q, q
    if c["op"] == "paged_qkv":   # ctx_max counts what is cached before
        return q, [n + (rng.randint(0, ctx) if ctx else 0) for n in q]
    return q, [max(n, ctx if i == 0 or c["lens"] <= 0 else rng.randint(1, ctx)) for i, n in enumerate(q)]


def work(case):
    c = case
    q, k = _lengths(c)
    T, keys = sum(q), sum(k)
    n_q, n_kv = c["n_q"], c["n_kv"]
    row = n_kv * (D + 4 if c.get("fp8") else 2 * D)          # one position's K (or V) in the cache
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(q, k))   # (query, visible key) pairs
    if c["op"] == "paged_qkv":
        return dict(bytes=T * ((n_q + 2 * n_kv) * D * 2 + n_q * D * 2 + 2 * row + c["rot"] * 4),
                    flops=T * ((n_q + n_kv) * (4 * D * c["norm"] + 3 * c["rot"]) + (4 * n_kv * D if c["fp8"] else 0)))
    if c["op"] == "paged_kv_read":
        return dict(bytes=T * (2 * row + 2 * n_kv * D * 2), flops=T * 2 * n_kv * D if c["fp8"] else 0)
    if c["op"] == "paged_attention":
        return dict(bytes=2 * T * n_q * D * 2 + 2 * keys * row, flops=4 * D * n_q * pairs)
    return dict(bytes=2 * T * (n_q + n_kv) * D * 2, flops=4 * D * n_q * pairs)


# ---- what a caller has in hand -----------------------------------------------------------------------------
def _rope_tables(max_pos, rot, yarn):
    """fp32 cos and sin [max_pos, rot / 2]; with yarn, frequencies scaled by parts for 4 times the trained length."""
    base, trained, factor = 1_000_000.0, 32768, 4.0
    i = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64)
    inv = base ** (-i / rot)
    mul = 1.0
    if yarn:
        turns = trained * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)
        mul = 0.1 * math.log(factor) + 1.0
    a = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * inv[None]
    return (a.cos() * mul).float(), (a.sin() * mul).float()


def _quantise(x):
    """fp32 rows [..., D] -> e4m3 values [..., D] and fp32 scales [...]: s = max|x| / 448, e4m3(x / s), a zero row zeros."""
    s = x.abs().amax(-1) / E4M3_MAX
    q = torch.where(s[..., None] > 0, x / s[..., None], torch.zeros_like(x))
    return q.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    c = case
    q_lens, k_lens = _lengths(c)
    B, T, n_q, n_kv = len(q_lens), sum(q_lens), c["n_q"], c["n_kv"]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    s = dict(c=c, cu=ints(cu), seq_lens=ints(k_lens), max_q=max(q_lens), max_k=max(k_lens), scale=D ** -0.5)
    if c["op"] == "packed_attention":
        # q, k and v as views of one projection's rows, as a model has them
        rows = normal(T, n_q + 2 * n_kv, D)
        s.update(q=rows[:, :n_q], k=rows[:, n_q:n_q + n_kv], v=rows[:, n_q + n_kv:],
                 out=torch.empty(T, n_q, D, dtype=torch.bfloat16, device="cuda"))
        return s
    P = c["page"]
    per = [-(-n // P) for n in k_lens]
    width, pages = max(per), sum(per) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")   # entries past a sequence's end mean nothing
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    s["block_table"] = table
    for name in ("k", "v"):
        pool = normal(pages, n_kv, P, D)
        if c["fp8"]:
            q8, sc = [], []
            for part in pool.split(1024):
                a, b = _quantise(part.float())
                q8.append(a)
                sc.append(b)
            s[name + "_pages"], s[name + "_scale"] = torch.cat(q8), torch.cat(sc)
        else:
            s[name + "_pages"], s[name + "_scale"] = pool, None
    if c["op"] == "paged_qkv":
        s["qkv"] = normal(T, (n_q + 2 * n_kv) * D)
        s["q_out"] = torch.empty(T, n_q, D, dtype=torch.bfloat16, device="cuda")
        s["cos"], s["sin"] = _rope_tables(max(k_lens), c["rot"], c["yarn"])
        s["q_norm"] = (1 + 0.1 * normal(D)) if c["norm"] else None
        s["k_norm"] = (1 + 0.1 * normal(D)) if c["norm"] else None
    elif c["op"] == "paged_kv_read":
        s["k_out"] = torch.empty(T, n_kv, D, dtype=torch.bfloat16, device="cuda")
        s["v_out"] = torch.empty(T, n_kv, D, dtype=torch.bfloat16, device="cuda")
    else:
        s["q"] = normal(T, n_q, D)
        s["out"] = torch.empty(T, n_q, D, dtype=torch.bfloat16, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------------------
def run(state):
    s, op = state, state["c"]["op"]
    if own:
        k = _ops()
        if op == "paged_qkv":
            k.paged_qkv(s["qkv"], s["cu"], s["seq_lens"], s["block_table"], s["k_pages"], s["v_pages"], s["q_out"],
                        s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                        interleaved=s["c"]["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
            return _cache_out(s, s["q_out"])
        if op == "paged_kv_read":
            k.paged_kv_read(s["cu"], s["block_table"], s["k_pages"], s["v_pages"], s["k_out"], s["v_out"],
                            k_scale=s["k_scale"], v_scale=s["v_scale"])
            return dict(k=s["k_out"], v=s["v_out"])
        if op == "paged_attention":
            k.paged_attention(s["q"], s["cu"], s["seq_lens"], s["block_table"], s["k_pages"], s["v_pages"], s["out"],
                              s["scale"], s["max_q"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        else:
            k.packed_attention(s["q"], s["k"], s["v"], s["cu"], s["out"], s["scale"], s["max_q"])
        return s["out"]
    return {"paged_qkv": _plain_qkv, "paged_kv_read": _plain_read, "paged_attention": _plain_paged,
            "packed_attention": _plain_packed}[op](s)


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inferencekit-engines_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from kernels import ops
    return ops()


def _cache_out(s, q):
    """The call's outputs: q, and the whole cache (every page, written or not)."""
    out = dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])
    if s["k_scale"] is not None:
        out.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
    return out


def _rows(cu, T):
    """The sequence of each of T rows, and the row's place in it."""
    r = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    return b, r - cu[b]


def _norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _rotate(x, cos, sin, interleaved):
    """x [T, heads, D] with its first 2 * cos.shape[1] dims rotated by the row's angles; the others as they are."""
    h = cos.shape[1]
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    c, s = cos[:, None], sin[:, None]
    lo, hi = a * c - b * s, b * c + a * s
    turned = torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1)
    return torch.cat((turned, x[..., 2 * h:]), -1)


def _plain_qkv(s):
    c = s["c"]
    n_q, n_kv, P = c["n_q"], c["n_kv"], c["page"]
    T = s["qkv"].shape[0]
    b, i = _rows(s["cu"], T)
    pos = s["seq_lens"][b] - (s["cu"][b + 1] - s["cu"][b]) + i
    x = s["qkv"].float().view(T, n_q + 2 * n_kv, D)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(_norm(x[:, :n_q], s["q_norm"]), cos, sin, c["interleaved"])
    k = _rotate(_norm(x[:, n_q:n_q + n_kv], s["k_norm"]), cos, sin, c["interleaved"])
    page, slot = s["block_table"][b, pos // P].long(), (pos % P).long()
    if c["fp8"]:
        k8, ks = _quantise(k)
        v8, vs = _quantise(x[:, n_q + n_kv:])
        s["k_pages"].view(torch.uint8)[page, :, slot] = k8.view(torch.uint8)
        s["v_pages"].view(torch.uint8)[page, :, slot] = v8.view(torch.uint8)
        s["k_scale"][page, :, slot] = ks
        s["v_scale"][page, :, slot] = vs
    else:
        s["k_pages"][page, :, slot] = k.bfloat16()
        s["v_pages"][page, :, slot] = x[:, n_q + n_kv:].bfloat16()
    return _cache_out(s, q.bfloat16())


def _plain_read(s):
    c = s["c"]
    P, T = c["page"], s["k_out"].shape[0]
    b, i = _rows(s["cu"], T)
    page, slot = s["block_table"][b, i // P].long(), i % P

    def rows(pages, scale):
        if scale is None:
            return pages[page, :, slot]
        return (pages.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float() * scale[page, :, slot][..., None]).bfloat16()

    return dict(k=rows(s["k_pages"], s["k_scale"]), v=rows(s["v_pages"], s["v_scale"]))


def _attend(q, k, v, cu, seq_lens, max_q, scale):
    """q [T, n_q, D] packed; k, v fp32 [B, n_kv, L, D] padded to the longest. Returns bf16 [T, n_q, D]."""
    T, n_q, _ = q.shape
    B, n_kv, L, _ = k.shape
    b, i = _rows(cu, T)
    n = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + torch.arange(max_q, device=q.device)).clamp(max=T - 1)
    qp = q.float()[at].view(B, max_q, n_kv, n_q // n_kv, D).permute(0, 2, 1, 3, 4).reshape(B, n_kv, -1, D)
    p = (qp @ k.transpose(-1, -2)).view(B, n_kv, max_q, n_q // n_kv, L).mul_(scale)
    last = (seq_lens - n)[:, None] + torch.arange(max_q, device=q.device)            # the last visible position
    p.masked_fill_((torch.arange(L, device=q.device) > last[..., None])[:, None, :, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    p = p.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(B, n_kv, -1, L) @ v).view(B, n_kv, max_q, n_q // n_kv, D) / l.masked_fill(l == 0, 1.0)
    return o.permute(0, 2, 1, 3, 4).reshape(B, max_q, n_q, D)[b, i].bfloat16()


def _plain_paged(s):
    B, width = s["block_table"].shape
    at = s["block_table"].clamp(min=0).long()
    inside = torch.arange(width * s["c"]["page"], device=at.device) < s["seq_lens"][:, None]

    def rows(pages, scale):
        x = pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scale[at][..., None] if scale is not None else pages[at].float()
        x = x.transpose(1, 2).reshape(B, pages.shape[1], -1, D)                      # [B, n_kv, width * page, D]
        return x.masked_fill_(~inside[:, None, :, None], 0.0)

    return _attend(s["q"], rows(s["k_pages"], s["k_scale"]), rows(s["v_pages"], s["v_scale"]), s["cu"], s["seq_lens"],
                   s["max_q"], s["scale"])


def _plain_packed(s):
    T = s["q"].shape[0]
    at = (s["cu"][:-1, None] + torch.arange(s["max_q"], device=s["q"].device)).clamp(max=T - 1)
    return _attend(s["q"], s["k"].float()[at].transpose(1, 2), s["v"].float()[at].transpose(1, 2), s["cu"],
                   s["seq_lens"], s["max_q"], s["scale"])


# ---- the definitions in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    q_lens, k_lens = _lengths(c)
    n_q, n_kv = c["n_q"], c["n_kv"]
    G = n_q // n_kv

    def position(b, p):
        """Page and slot of positions p (a tensor) of sequence b."""
        P = c["page"]
        return s["block_table"][b].long()[p // P], p % P

    def cached(name, b, n):
        """The first n rows of sequence b: [n, n_kv, D] in 64 bits."""
        page, slot = position(b, torch.arange(n, device="cuda"))
        if s[name + "_scale"] is None:
            return s[name + "_pages"][page, :, slot].double()
        r = s[name + "_pages"].view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn)
        return r.float().double() * s[name + "_scale"][page, :, slot].double().unsqueeze(-1)

    if c["op"] == "paged_qkv":
        out = _cache_out(s, torch.zeros(s["q_out"].shape, dtype=torch.float64, device="cuda"))
        for name in ("k_pages", "v_pages", "k_scale", "v_scale"):
            if name in out:
                out[name] = (out[name].float() if c["fp8"] else out[name]).double()
        half = c["rot"] // 2
        even = torch.arange(half, device="cuda") * 2 if c["interleaved"] else torch.arange(half, device="cuda")
        odd = even + (1 if c["interleaved"] else half)
        row = 0
        for b, (n, length) in enumerate(zip(q_lens, k_lens)):
            pos = torch.arange(length - n, length, device="cuda")
            page, slot = position(b, pos)
            x = s["qkv"][row:row + n].double().view(n, -1, D)
            angle = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            for first, heads, w in ((0, n_q, s["q_norm"]), (n_q, n_kv, s["k_norm"]), (n_q + n_kv, n_kv, None)):
                y = x[:, first:first + heads].clone()
                if first < n_q + n_kv:
                    if w is not None:
                        y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
                    z = torch.complex(y[..., even], y[..., odd]) * angle
                    y[..., even], y[..., odd] = z.real, z.imag
                if first == 0:
                    out["q"][row:row + n] = y
                    continue
                name = "k" if first == n_q else "v"
                if c["fp8"]:
                    sc = y.abs().max(-1).values / E4M3_MAX
                    y = (y / sc.clamp(min=1e-300).unsqueeze(-1)).to(torch.float8_e4m3fn).double()
                    out[name + "_scale"][page, :, slot] = sc
                out[name + "_pages"][page, :, slot] = y
            row += n
        return out
    if c["op"] == "paged_kv_read":
        return dict(k=torch.cat([cached("k", b, n) for b, n in enumerate(k_lens)]),
                    v=torch.cat([cached("v", b, n) for b, n in enumerate(k_lens)]))
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, length) in enumerate(zip(q_lens, k_lens)):
        if c["op"] == "packed_attention":
            K, V = s["k"][row:row + n].double(), s["v"][row:row + n].double()
        else:
            K, V = cached("k", b, length), cached("v", b, length)
        hidden = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
        for h in range(n_q):
            w = s["q"][row:row + n, h].double() @ K[:, h // G].T * s["scale"]
            w = torch.softmax(w.masked_fill_(hidden, -math.inf), -1)
            out[row:row + n, h] = w @ V[:, h // G]
        row += n
    return out

"""The operators for sequences that share pages (beams, samples of one prompt, requests behind one system prompt), and the
cases they are measured on.

Four operators, each in a plain form (elementary torch operations, rounded once at the end) and, with `own` set, through the
framework's entry points (`kernels.ops()`):

  paged_plan        the pass of a batch, from its lengths: free pages into the block tables, row offsets, the slot and the
                    position of every token row, and how many leading positions the sequences of a group share
  paged_fork        the reordering of states: each row continues a parent row; whole pages are shared by count, a partly
                    filled last page is copied for all but one of a parent's children
  beam_select       the best k continuations of each request over its beams and the vocabulary
  shared_attention  causal attention over a paged cache whose sequences share their first positions in groups

Sequence b of a pass has its tokens in rows cu[b] .. cu[b+1] - 1; its last new token sits at position seq_lens[b] - 1. Position p
of a sequence lies in slot p % page_size of page block_table[b][p // page_size]; refs counts the sequences that hold a page,
0 for a free one. A page holds [kv_heads][page_size][128] values, and for an 8-bit cache fp32 row scales beside them.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 128          # the framework's head size
E4M3_MAX = 448.0


# ---- the cases ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a batch of 16: every sequence grows by a token, some of them into a new page
        dict(name="plan_decode", op="paged_plan", batch=16, members=4, ctx_max=4096, new_max=1, page=64, lens=1),
        # a server's pass: many prompts and decoding sequences at once, small pages, a large pool
        dict(name="plan_prompts", op="paged_plan", batch=700, members=7, ctx_max=1500, new_max=127, page=16, lens=2),
        # the four beams of one request change places
        dict(name="fork_beams4", op="paged_fork", requests=1, beams=4, ctx_max=777, page=16, fp8=False, layers=36, n_kv=8, lens=0),
        # many requests' beams at once over an 8-bit cache, requests that ended among them
        dict(name="fork_batch_fp8", op="paged_fork", requests=8, beams=8, ctx_max=600, page=64, fp8=True, layers=36, n_kv=8, lens=3),
        # one request with four beams: latency
        dict(name="select_4_bf16", op="beam_select", requests=1, beams=4, vocab=151936, k=8, fp32=False, lens=0),
        # a batch of requests, twice as many candidates as beams
        dict(name="select_128_bf16", op="beam_select", requests=16, beams=8, vocab=151936, k=16, fp32=False, lens=0),
        # requests with different numbers of beams, fp32 logits of an odd vocabulary, excluded tokens, the largest k
        dict(name="select_ragged_f32", op="beam_select", requests=9, beams=31, vocab=32003, k=64, fp32=True, lens=4),
        # the decode step of four beams behind a short prompt: latency
        dict(name="shared_beams4", op="shared_attention", groups=1, members=4, prefix=704, own=45, q_max=1, n_q=32, n_kv=8,
             page=16, fp8=False, lens=0),
        # 64 requests behind one long system prompt
        dict(name="shared_64_bf16", op="shared_attention", groups=1, members=64, prefix=8192, own=500, q_max=1, n_q=32, n_kv=8,
             page=64, fp8=False, lens=5),
        # the beams of eight requests with prompts of different lengths, an 8-bit cache
        dict(name="shared_groups_fp8", op="shared_attention", groups=8, members=8, prefix=16384, own=200, q_max=1, n_q=32, n_kv=8,
             page=64, fp8=True, lens=6),
        # several tokens a sequence (a draft to be judged) behind shared prompts
        dict(name="shared_drafts_bf16", op="shared_attention", groups=3, members=13, prefix=4096, own=333, q_max=7, n_q=32, n_kv=8,
             page=32, fp8=False, lens=8),
    ]


HEADS = ((32, 8), (16, 4), (8, 2), (4, 1), (8, 8), (12, 4), (10, 2), (16, 1), (28, 4))


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("paged_plan", "paged_fork", "beam_select", "shared_attention", "shared_attention"))
    c = dict(op=op, lens=rng.randrange(12, 1 << 20))
    if op == "paged_plan":
        c.update(batch=_log(rng, 1, 700), members=rng.randrange(1, 9), page=rng.choice((16, 32, 64, 128)))
        c.update(ctx_max=_log(rng, 1, min(16384, 1_000_000 // c["batch"])), new_max=_log(rng, 1, min(2048, 80_000 // c["batch"])))
    elif op == "paged_fork":
        c.update(requests=_log(rng, 1, 16), page=rng.choice((16, 32, 64, 128)), fp8=rng.random() < 0.5, layers=rng.choice((1, 2, 36)),
                 n_kv=rng.choice((1, 2, 4, 8)))
        c.update(beams=_log(rng, 1, 64 // c["requests"]))
        c.update(ctx_max=_log(rng, 1, min(4096, 4000 // c["requests"])))
        heads = c["requests"] * c["beams"] * c["page"] * c["n_kv"] * (1 if c["fp8"] else 2)
        c["layers"] = max(1, min(c["layers"], 64 * 64 * 8 * 36 // heads))
    elif op == "beam_select":
        c.update(requests=_log(rng, 1, 16), fp32=rng.random() < 0.5, vocab=_log(rng, 100, 151936), k=rng.randrange(1, 65))
        c.update(beams=_log(rng, 1, min(32, 128 // c["requests"])))
    else:
        n_q, n_kv = rng.choice(HEADS)
        c.update(n_q=n_q, n_kv=n_kv, page=rng.choice((16, 32, 64, 128)), fp8=rng.random() < 0.5, groups=_log(rng, 1, 8))
        c.update(members=_log(rng, 1, 64 // c["groups"]), q_max=rng.choice((1, 1, rng.randrange(2, 9), _log(rng, 8, 64))))
        c.update(prefix=_log(rng, 64, min(16384, 500_000 // (c["groups"] * c["members"] * c["q_max"]) + 64)), own=_log(rng, c["q_max"], 600))
    return c


def _ragged(rng, n, top, low=1):
    """n whole numbers from `low` to `top`, the first of them the largest."""
    return [top] + [rng.randint(low, top) for _ in range(n - 1)]


def _sizes(c):
    """The case's lengths, from its `lens` alone (0: all at their largest)."""
    rng = random.Random(c["lens"])
    flat = c["lens"] == 0
    if c["op"] == "paged_plan":
        B = c["batch"]
        lens = [rng.randint(0, c["ctx_max"]) for _ in range(B)]
        new = [c["new_max"]] + [rng.choice((1, c["new_max"], rng.randint(0, c["new_max"]))) for _ in range(B - 1)]
        if c["new_max"] == 1:
            new = [1] * B
        return lens, new
    if c["op"] == "paged_fork":
        R = c["requests"]
        lens = [c["ctx_max"]] * R if flat else _ragged(rng, R, c["ctx_max"])
        ended = [False] * R if flat else [False] + [rng.random() < 0.15 for _ in range(R - 1)]
        return lens, ended
    if c["op"] == "beam_select":
        return [c["beams"]] * c["requests"] if flat else _ragged(rng, c["requests"], c["beams"])
    G, P = c["groups"], c["page"]
    members = [c["members"]] * G if flat else _ragged(rng, G, c["members"])
    prefix = [n // P * P for n in ([c["prefix"]] * G if flat else _ragged(rng, G, c["prefix"]))]
    B = sum(members)
    new = [c["q_max"]] * B if flat else _ragged(rng, B, c["q_max"])
    tail = [c["own"]] * B if flat else [max(n, rng.randint(1, c["own"])) for n in new]
    return members, prefix, new, tail


def _parents(c):
    """paged_fork's parents: beams of the same request, good ones more often; -1 for a request that ended."""
    lens, ended = _sizes(c)
    rng = random.Random(c["lens"] + 1)
    W = c["beams"]
    return [-1 if ended[r] else r * W + min(int(rng.expovariate(0.5)), W - 1) for r in range(c["requests"]) for _ in range(W)]


def work(case):
    c = case
    if c["op"] == "paged_plan":
        lens, new = _sizes(c)
        B, (pages, width) = c["batch"], _plan_pool(c)
        return dict(bytes=4 * (2 * pages + 2 * B * width + 4 * B + 2 * sum(new)), flops=pages + B + 4 * sum(new))
    if c["op"] == "paged_fork":
        lens, ended = _sizes(c)
        P, W, parents = c["page"], c["beams"], _parents(c)
        row = c["n_kv"] * 2 * (D + 4 if c["fp8"] else 2 * D) * c["layers"]     # one position's K and V in every layer
        copies = sum((lens[r] % P) * (W - len(set(parents[r * W:(r + 1) * W]))) for r in range(len(lens)) if not ended[r])
        entries = sum(-(-n // P) * W for n in lens)
        return dict(bytes=2 * copies * row + 4 * (4 * entries + 3 * W * len(lens)), flops=2 * entries)
    if c["op"] == "beam_select":
        rows = sum(_sizes(c))
        return dict(bytes=rows * c["vocab"] * (4 if c["fp32"] else 2) + 4 * rows + 12 * c["requests"] * c["k"], flops=4 * rows * c["vocab"])
    members, prefix, new, tail = _sizes(c)
    row = c["n_kv"] * (D + 4 if c["fp8"] else 2 * D)
    first = [p for m, p in zip(members, prefix) for _ in range(m)]
    pairs = sum(n * (p + t) - n * (n - 1) // 2 for p, n, t in zip(first, new, tail))
    return dict(bytes=2 * sum(new) * c["n_q"] * D * 2 + 2 * row * (sum(prefix) + sum(tail)), flops=4 * D * c["n_q"] * pairs)


# ---- what a caller has in hand -----------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(n):
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    return cu


def _plan_pool(c):
    """Pages of paged_plan's pool and the tables' width: what the batch can need, and a quarter more."""
    lens, new = _sizes(c)
    need = [-(-(a + b) // c["page"]) for a, b in zip(lens, new)]
    return sum(need) * 5 // 4 + 8, max(need) + 1


def _quantise(x):
    """fp32 rows [..., D] -> e4m3 values [..., D] and fp32 scales [...]: s = max|x| / 448, e4m3(x / s), a zero row zeros."""
    s = x.abs().amax(-1) / E4M3_MAX
    q = torch.where(s[..., None] > 0, x / s[..., None], torch.zeros_like(x))
    return q.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), s


def _pools(g, shape, fp8, s):
    """K and V pages of N(0, 1) rows, [..., D] of `shape` [.., pages, n_kv, page], into the state."""
    for name in ("k", "v"):
        if not fp8:
            s[name + "_pages"], s[name + "_scale"] = torch.randn(*shape, D, generator=g, device="cuda", dtype=torch.bfloat16), None
            continue
        flat = math.prod(shape[:-2]), shape[-2], shape[-1]
        q8 = torch.empty(*flat, D, device="cuda", dtype=torch.float8_e4m3fn)
        sc = torch.empty(flat, device="cuda")
        for i in range(0, flat[0], 2048):
            n = min(2048, flat[0] - i)
            q8[i:i + n], sc[i:i + n] = _quantise(torch.randn(n, *flat[1:], D, generator=g, device="cuda"))
        s[name + "_pages"], s[name + "_scale"] = q8.view(*shape, D), sc.view(*shape)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    s = dict(c=c)
    if c["op"] == "paged_plan":
        lens, new = _sizes(c)
        P, M = c["page"], c["members"]
        pages, width = _plan_pool(c)
        order = rng.sample(range(pages), pages)
        table, refs = [[-1] * width for _ in lens], [0] * pages
        for b, n in enumerate(lens):
            head = b // M * M
            joint = min(lens[head:head + M]) // P // 2      # whole pages that the sequences of a group share
            for j in range(-(-n // P)):
                p = table[head][j] if j < joint and b != head else order.pop()
                table[b][j] = p
                refs[p] += 1
        groups = list(range(0, len(lens), M)) + [len(lens)]
        T = sum(new)
        s.update(refs=_ints(refs), table=_ints(table), lens=_ints(lens), new=_ints(new), groups=_ints(groups), T=T,
                 refs_out=_ints(refs), table_out=_ints(table), cu=_ints([0] * (len(lens) + 1)), seq_lens=_ints(lens),
                 slots=_ints([0] * T), positions=_ints([0] * T), shared=_ints([0] * (len(groups) - 1)), info=_ints([0, 0]))
    elif c["op"] == "paged_fork":
        lens, ended = _sizes(c)
        P, W, R = c["page"], c["beams"], c["requests"]
        width = -(-max(lens) // P) + 1
        joint = [max(0, n // P - 2) for n in lens]      # whole pages that a request's beams share: its prompt
        pages = sum(j + W * (-(-n // P) - j) for n, j in zip(lens, joint)) + R * W + 5
        order = rng.sample(range(pages), pages)
        table, refs = [[-1] * width for _ in range(R * W)], [0] * pages
        for r, n in enumerate(lens):
            for w in range(W):
                for j in range(-(-n // P)):
                    p = table[r * W][j] if j < joint[r] and w else order.pop()
                    table[r * W + w][j] = p
                    refs[p] += 1
        s.update(refs=_ints(refs), table=_ints(table), lens=_ints([n for n in lens for _ in range(W)]), parents=_ints(_parents(c)),
                 refs_out=_ints(refs), table_out=_ints(table), lens_out=_ints([0] * (R * W)), info=_ints([0, 0]))
        _pools(g, (c["layers"], pages, c["n_kv"], P), c["fp8"], s)
    elif c["op"] == "beam_select":
        beams = _sizes(c)
        rows, k = sum(beams), c["k"]
        x = torch.randn(rows, c["vocab"], generator=g, device="cuda").mul_(2.5)
        if c["fp32"]:                               # tokens that a grammar excludes
            x.masked_fill_(torch.rand(c["vocab"], generator=g, device="cuda") < 0.3, -math.inf)
        s.update(logits=x if c["fp32"] else x.bfloat16(), scores=torch.randn(rows, generator=g, device="cuda") * 2 - 20,
                 cu=_ints(_offsets(beams)), beams=max(beams), out_scores=torch.zeros(len(beams), k, device="cuda"),
                 out_parents=_ints([[0] * k] * len(beams)), out_tokens=_ints([[0] * k] * len(beams)))
    else:
        members, prefix, new, tail = _sizes(c)
        P, n_q, n_kv = c["page"], c["n_q"], c["n_kv"]
        B, T, groups = sum(members), sum(new), _offsets(members)
        of = [i for i, m in enumerate(members) for _ in range(m)]
        seq_lens = [prefix[of[b]] + tail[b] for b in range(B)]
        pages = sum(prefix) // P + sum(-(-t // P) for t in tail) + 3
        order = rng.sample(range(pages), pages)
        width = max(-(-n // P) for n in seq_lens)
        table = [[-1] * width for _ in range(B)]
        for b in range(B):
            for j in range(-(-seq_lens[b] // P)):
                table[b][j] = table[groups[of[b]]][j] if j < prefix[of[b]] // P and b != groups[of[b]] else order.pop()
        s.update(table=_ints(table), cu=_ints(_offsets(new)), seq_lens=_ints(seq_lens), groups=_ints(groups), shared=_ints(prefix),
                 max_q=max(new), scale=D ** -0.5, q=torch.randn(T, n_q, D, generator=g, device="cuda", dtype=torch.bfloat16),
                 out=torch.empty(T, n_q, D, dtype=torch.bfloat16, device="cuda"))
        _pools(g, (pages, n_kv, P), c["fp8"], s)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["c"]
    op = c["op"]
    if own:
        k = _ops()
        if op == "paged_plan":
            k.paged_plan(s["refs"], s["lens"], s["new"], s["table"], s["cu"], s["seq_lens"], c["page"], refs_out=s["refs_out"],
                         table_out=s["table_out"], slots=s["slots"], positions=s["positions"], groups=s["groups"], shared=s["shared"],
                         info=s["info"])
            return {n: s[n] for n in ("cu", "seq_lens", "refs_out", "table_out", "slots", "positions", "shared", "info")}
        if op == "paged_fork":
            k.paged_fork(s["refs"], s["lens"], s["parents"], s["table"], s["table_out"], s["lens_out"], s["k_pages"], s["v_pages"],
                         k_scale=s["k_scale"], v_scale=s["v_scale"], refs_out=s["refs_out"], info=s["info"])
            return _fork_out(s)
        if op == "beam_select":
            k.beam_select(s["logits"], s["scores"], s["cu"], s["out_scores"], s["out_parents"], s["out_tokens"])
            return dict(scores=s["out_scores"], parents=s["out_parents"], tokens=s["out_tokens"])
        k.shared_attention(s["q"], s["cu"], s["seq_lens"], s["table"], s["groups"], s["shared"], s["k_pages"], s["v_pages"], s["out"],
                           s["scale"], s["max_q"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return s["out"]
    return {"paged_plan": _plain_plan, "paged_fork": _plain_fork, "beam_select": _plain_select, "shared_attention": _plain_shared}[op](s)


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inferencekit-engines_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from kernels import ops
    return ops()


def _fork_out(s):
    out = {n: s[n] for n in ("refs_out", "table_out", "lens_out", "info", "k_pages", "v_pages")}
    if s["k_scale"] is not None:
        out.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
    return out


def _rows(cu, T):
    """The sequence of each of T rows, and the row's place in it."""
    r = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    return b, r - cu[b]


def _exclusive(n):
    return torch.cumsum(n, 0) - n


def _plain_plan(s):
    P, refs, table, lens, new = s["c"]["page"], s["refs"], s["table"], s["lens"], s["new"]
    B, width = table.shape
    have, want = (lens + P - 1) // P, (lens + new + P - 1) // P
    total, free = (want - have).sum(), (refs == 0).sum()
    fits = total <= free
    order = torch.argsort((refs != 0).to(torch.int32), stable=True).to(torch.int32)      # free pages first, in order
    j = torch.arange(width, device=table.device)
    at = _exclusive(want - have)[:, None] + j - have[:, None]
    grown = (j >= have[:, None]) & (j < want[:, None]) & fits
    s["table_out"].copy_(torch.where(grown, order[at.clamp(0, refs.numel() - 1)], table))
    s["refs_out"].copy_(refs + ((refs == 0) & (torch.cumsum((refs == 0).int(), 0) <= total) & fits))
    s["cu"].copy_(torch.cat((torch.zeros_like(new[:1]), torch.cumsum(new, 0))) * fits)
    s["seq_lens"].copy_(lens + new * fits)
    b, i = _rows(s["cu"], s["T"])
    pos = lens[b] + i
    s["positions"].copy_(pos)
    s["slots"].copy_(s["table_out"][b, pos // P] * P + pos % P)
    # leading entries that every sequence of a group has in the same page, and positions that all of them have
    g, _ = _rows(s["groups"], B)
    head = s["groups"][g].long()
    same = torch.cumprod(((table == table[head]) & (table >= 0) & (j < want[:, None])).int(), 1).sum(1) * P
    n = torch.minimum(same, lens).to(torch.int32)
    s["shared"].copy_(torch.full_like(s["shared"], 1 << 30).scatter_reduce_(0, g, n, "amin"))
    s["info"].copy_(torch.stack(((total - free).clamp(min=0), free - total * fits)))
    return {n: s[n] for n in ("cu", "seq_lens", "refs_out", "table_out", "slots", "positions", "shared", "info")}


def _plain_fork(s):
    P, refs, table, lens, parents = s["c"]["page"], s["refs"], s["table"], s["lens"], s["parents"].long()
    B, width = table.shape
    j = torch.arange(width, device=table.device)
    up = parents.clamp(min=0)
    n = torch.where(parents < 0, 0, lens[up]).to(torch.int32)
    held, taken = j < ((lens + P - 1) // P)[:, None], j < ((n + P - 1) // P)[:, None]
    first = ~((parents[:, None] == parents) & (torch.arange(len(parents), device=up.device)[:, None] > torch.arange(len(parents), device=up.device))).any(1)
    copied = (parents >= 0) & (n % P > 0) & ~first                                  # rows whose last page is a copy
    last = (n // P).long()
    rows = table[up]
    kept = taken & ~(copied[:, None] & (j == last[:, None]))
    count = refs.long() - torch.zeros_like(refs).long().scatter_add_(0, table.clamp(min=0).long().flatten(), held.long().flatten())
    count.scatter_add_(0, rows.clamp(min=0).long().flatten(), kept.long().flatten())
    order = torch.argsort((count != 0).to(torch.int32), stable=True)
    fresh = order[_exclusive(copied.long()).clamp(max=refs.numel() - 1)]
    out = torch.where(taken, torch.where(kept, rows, fresh[:, None].to(torch.int32)), -1)
    s["table_out"].copy_(out)
    s["lens_out"].copy_(n)
    count.scatter_add_(0, fresh, copied.long())
    s["refs_out"].copy_(count)
    s["info"].copy_(torch.stack((torch.zeros_like(count[0]), (count == 0).sum())))
    src = rows.gather(1, last[:, None]).clamp(min=0)[:, 0].long()
    dst = torch.where(copied, out.gather(1, last[:, None])[:, 0].long(), src)       # (rows without a copy: onto itself)
    filled = (torch.arange(P, device=up.device) < (n % P)[:, None])[None, :, None]
    for pages in (s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]):
        if pages is not None:
            v = pages.view(torch.uint8) if pages.dtype == torch.float8_e4m3fn else pages
            m = filled if v.dim() == 4 else filled[..., None]
            v[:, dst] = torch.where(m, v[:, src], v[:, dst])
    return _fork_out(s)


def _plain_select(s):
    logits, cu, W, k = s["logits"], s["cu"].long(), s["beams"], s["c"]["k"]
    x = logits.double()
    x = s["scores"].double()[:, None] + (x - torch.logsumexp(x, 1, keepdim=True))
    V = x.shape[1]
    at = cu[:-1, None] + torch.arange(W, device=cu.device)
    inside = at < cu[1:, None]
    x = x[at.clamp(max=len(logits) - 1)].masked_fill(~inside[..., None], -math.inf).flatten(1)
    best, i = torch.sort(x, dim=1, descending=True, stable=True)                    # ties: the lowest index
    best, i = best[:, :k], i[:, :k]
    if best.shape[1] < k:
        best = torch.nn.functional.pad(best, (0, k - best.shape[1]), value=-math.inf)
        i = torch.nn.functional.pad(i, (0, k - i.shape[1]))
    none = best == -math.inf
    s["out_scores"].copy_(best)
    s["out_parents"].copy_((cu[:-1, None] + i // V).masked_fill(none, -1))
    s["out_tokens"].copy_((i % V).masked_fill(none, -1))
    return dict(scores=s["out_scores"], parents=s["out_parents"], tokens=s["out_tokens"])


def _plain_shared(s):
    P, q, cu, seq_lens, max_q = s["c"]["page"], s["q"], s["cu"], s["seq_lens"], s["max_q"]
    T, n_q, _ = q.shape
    B, width = s["table"].shape
    n_kv, L = s["c"]["n_kv"], width * P
    at = s["table"].clamp(min=0).long()
    inside = torch.arange(L, device=q.device) < seq_lens[:, None]

    def rows(pages, scale):
        x = pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scale[at][..., None] if scale is not None else pages[at].float()
        return x.transpose(1, 2).reshape(B, n_kv, L, D).masked_fill_(~inside[:, None, :, None], 0.0)

    b, i = _rows(cu, T)
    n = cu[1:] - cu[:-1]
    take = (cu[:-1, None] + torch.arange(max_q, device=q.device)).clamp(max=T - 1)
    qp = q.float()[take].view(B, max_q, n_kv, n_q // n_kv, D).permute(0, 2, 1, 3, 4).reshape(B, n_kv, -1, D)
    p = (qp @ rows(s["k_pages"], s["k_scale"]).transpose(-1, -2)).view(B, n_kv, max_q, n_q // n_kv, L).mul_(s["scale"])
    last = (seq_lens - n)[:, None] + torch.arange(max_q, device=q.device)            # the last visible position
    p.masked_fill_((torch.arange(L, device=q.device) > last[..., None])[:, None, :, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    p = p.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(B, n_kv, -1, L) @ rows(s["v_pages"], s["v_scale"])).view(B, n_kv, max_q, n_q // n_kv, D) / l.masked_fill(l == 0, 1.0)
    s["out"].copy_(o.permute(0, 2, 1, 3, 4).reshape(B, max_q, n_q, D)[b, i])
    return s["out"]


# ---- the definitions in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    c = case
    if c["op"] in ("paged_plan", "paged_fork"):     # whole numbers and copies
        return None
    s = prepare(case, seed)
    if c["op"] == "beam_select":
        k, cu = c["k"], s["cu"].tolist()
        out = dict(scores=np.full((len(cu) - 1, k), -np.inf), parents=np.full((len(cu) - 1, k), -1), tokens=np.full((len(cu) - 1, k), -1))
        x = s["logits"].double().cpu().numpy()
        base = s["scores"].double().cpu().numpy()
        for b in range(len(cu) - 1):
            found = []
            for r in range(cu[b], cu[b + 1]):
                top = x[r].max()
                if top == -np.inf:
                    continue
                lse = top + math.log(math.fsum(np.exp(x[r] - top)))
                border = np.partition(x[r], -min(k, x.shape[1]))[-min(k, x.shape[1])]
                found += [(-(base[r] + (x[r, v] - lse)), r, int(v)) for v in np.flatnonzero((x[r] >= border) & (x[r] > -np.inf))]
            for i, (score, r, v) in enumerate(sorted(found)[:k]):
                out["scores"][b, i], out["parents"][b, i], out["tokens"][b, i] = -score, r, v
        return {n: torch.from_numpy(v).cuda() if n == "scores" else torch.from_numpy(v).to("cuda", torch.int32) for n, v in out.items()}
    P, G = c["page"], c["n_q"] // c["n_kv"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    cu, seq_lens = s["cu"].tolist(), s["seq_lens"].tolist()
    for b, length in enumerate(seq_lens):
        lo, hi = cu[b], cu[b + 1]
        p = torch.arange(length, device="cuda")
        page, slot = s["table"][b].long()[p // P], p % P

        def cached(name):
            if s[name + "_scale"] is None:
                return s[name + "_pages"][page, :, slot].double().transpose(0, 1)
            r = s[name + "_pages"].view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn)
            return (r.float().double() * s[name + "_scale"][page, :, slot].double().unsqueeze(-1)).transpose(0, 1)

        n = hi - lo
        hidden = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
        q = s["q"][lo:hi].double().view(n, c["n_kv"], G, D)
        w = torch.einsum("nhgd,hkd->hgnk", q, cached("k")) * s["scale"]
        w = torch.softmax(w.masked_fill_(hidden, -math.inf), -1)
        out[lo:hi] = torch.einsum("hgnk,hkd->nhgd", w, cached("v")).reshape(n, c["n_q"], D)
    return out

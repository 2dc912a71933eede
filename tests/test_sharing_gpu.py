"""The operators for sequences that share pages: plans and forks against a simulation in Python, the beam selection and the
attention with shared prefixes against plain implementations in 64 bits.

Bounds, fixed beforehand:
* Tables, counts, slots and copies: equal.
* beam_select: a score is rounded to fp32 (2^-24 |s|), and a row's sum of exponentials is off by at most 2^-17 of itself: a
  term by 2^-22 (exp2's two ulps) and 2^-23 (its argument, weighted by the term), a sum of 64 terms and some 12 steps of a tree
  by 100 half ulps of 2^-24 (2^-17.4). Scores are ordered in 64 bits: whatever is taken at rank i has, exactly, the i-th best
  score within twice that bound; in one row the larger logit comes first, equal ones by token.
* shared_attention: as paged_attention's (test_paged_gpu.py, the kernels' roundings are the same).
"""
import math
import random

import pytest
import torch

from test_paged_gpu import D, DEV, attend64, check_attention, cumulative, ints, make_cache, ops

pytestmark = pytest.mark.gpu


# ---- paged_plan --------------------------------------------------------------------------------------------
def plan(refs, table, lens, new, P, groups, rows):
    """What a plan leaves, by the definition; lists in, lists out (None: nothing is taken)."""
    width, refs, table = len(table[0]) if table else 0, list(refs), [list(r) for r in table]
    use = [n if ln >= 0 and n >= 0 and ln + n <= width * P else 0 for ln, n in zip(lens, new)]
    free = [p for p, r in enumerate(refs) if r == 0]
    need = [-(-(ln + n) // P) - -(-ln // P) if n else 0 for ln, n in zip(lens, use)]
    shared = []
    for a, b in zip(groups, groups[1:]):
        n = min([max(ln, 0) for ln in lens[a:b]] or [0])
        for j in range(-(-n // P)):
            if len({table[i][j] for i in range(a, b)}) > 1 or table[a][j] < 0:
                n = min(n, j * P)
        shared.append(n)
    if sum(need) > len(free) or sum(use) > rows:
        return dict(cu=[0] * (len(lens) + 1), seq_lens=list(lens), refs=refs, table=table, slots=[], positions=[], shared=shared,
                    info=[max(0, sum(need) - len(free)), len(free)])
    slots, positions = [], []
    for b, (ln, n) in enumerate(zip(lens, use)):
        for j in range(need[b]):
            p = free.pop(0)
            refs[p] = 1
            table[b][-(-ln // P) + j] = p
        for pos in range(ln, ln + n):
            positions.append(pos)
            slots.append(table[b][pos // P] * P + pos % P)
    return dict(cu=cumulative(use), seq_lens=[ln + n for ln, n in zip(lens, use)], refs=refs, table=table, slots=slots,
                positions=positions, shared=shared, info=[0, len(free)])


def random_state(rng, lens, P, pages, width, groups=()):
    """refs and tables of sequences with these lengths (entries behind them: junk); groups share a random number of pages."""
    free, refs, table = rng.sample(range(pages), pages), [0] * pages, [[rng.choice((-5, 0, 7)) for _ in range(width)] for _ in lens]
    head, joint = list(range(len(lens))), [0] * len(lens)
    for a, b in zip(groups, groups[1:]):
        n = rng.randint(0, min([-(-max(x, 0) // P) for x in lens[a:b]] or [0]))
        for i in range(a, b):
            head[i], joint[i] = a, n
    for b, n in enumerate(lens):
        for j in range(-(-max(n, 0) // P)):
            table[b][j] = table[head[b]][j] if head[b] != b and j < joint[b] else free.pop()
            refs[table[b][j]] += 1
    return refs, table


PLANS = {   # lens, new, page, free pages, groups
    "one": ([0], [1], 16, 3, [0, 1]),
    "page_ends": ([15, 16, 17, 0, 31], [1, 1, 1, 0, 2], 16, 9, [0, 5]),
    "prompts": ([0, 0, 0], [300, 1, 77], 32, 40, [0, 1, 3]),
    "exactly_enough": ([16, 16, 16], [1, 16, 17], 16, 4, [0, 3]),
    "one_too_few": ([16, 16, 16], [1, 16, 17], 16, 3, [0, 1, 3]),
    "none_free_none_needed": ([1, 5], [15, 3], 16, 0, [0, 2]),
    "sits_out": ([100, 64, 1], [0, 0, 0], 64, 5, [0, 0, 3]),
    "mixed": ([1000, 0, 127, 128, 129, 5], [1, 700, 1, 1, 1, 0], 128, 60, [0, 2, 6]),
    "many": ([37 * i % 500 for i in range(1500)], [i % 3 for i in range(1500)], 64, 1600, list(range(0, 1501, 5))),
    "large_pool": ([40, 50], [5000, 3000], 16, 100_000, [0, 2]),
    "most_sequences": ([i % 40 for i in range(16384)], [1] * 16384, 16, 2000, [0, 16384]),
    "9000_sequences": ([i % 7 for i in range(9000)], [i % 2 for i in range(9000)], 16, 3000, [0, 3, 9000]),
}


@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in_place"])
@pytest.mark.parametrize("name", PLANS)
def test_plan(name, in_place):
    lens, new, P, spare, groups = PLANS[name]
    rng = random.Random(len(name))
    width = max(-(-(a + b) // P) for a, b in zip(lens, new)) + 2
    refs, table = random_state(rng, lens, P, sum(-(-n // P) for n in lens) + spare, width, groups)
    extra = sum(r == 0 for r in refs) - spare       # pages that sharing saved: someone else's
    for p in [p for p, r in enumerate(refs) if r == 0][:extra]:
        refs[p] = 3
    T = sum(new) + 3
    want = plan(refs, table, lens, new, P, groups, T)
    r, t = ints(refs), ints(table)
    ro, to = (r, t) if in_place else (torch.full_like(r, -9), torch.full((len(lens), width + 5), -9, dtype=torch.int32, device=DEV)[:, :width])
    cu, sl, slots, pos = (torch.full((n,), -9, dtype=torch.int32, device=DEV) for n in (len(lens) + 1, len(lens), T, T))
    sh, info = torch.full((len(groups) - 1,), -9, dtype=torch.int32, device=DEV), ints([-9, -9])
    k = ops()
    k.device_error()
    k.paged_plan(r, ints(lens), ints(new), t, cu, sl, P, refs_out=None if in_place else ro, table_out=None if in_place else to, slots=slots,
                 positions=pos, groups=ints(groups), shared=sh, info=info)
    assert k.device_error() == (8 if name == "one_too_few" else 0)
    for got, key in ((cu, "cu"), (sl, "seq_lens"), (ro, "refs"), (to, "table"), (sh, "shared"), (info, "info")):
        assert got.tolist() == want[key], key
    n = len(want["slots"])
    assert slots.tolist() == want["slots"] + [-9] * (T - n) and pos.tolist() == want["positions"] + [-9] * (T - n)
    if not in_place:
        assert r.tolist() == refs and t.tolist() == table


def test_plan_with_bad_lengths_and_too_few_rows():
    k, P = ops(), 16
    lens, new, refs, table = [-1, 5, 30, 20], [4, -2, 5, 3], [0, 0, 1, 1, 0, 1, 1], [[0, 0], [2, 0], [3, 5], [6, 3]]
    for rows, err in ((3, 2), (2, 2)):
        want = plan(refs, table, lens, new, P, [0, 4], rows)
        if rows == 2:
            assert want["cu"] == [0] * 5
        r, t, cu, sl, info = ints(refs), ints(table), ints([-9] * 5), ints([-9] * 4), ints([-9, -9])
        slots, sh = ints([-9] * rows), ints([-9])
        k.device_error()
        k.paged_plan(r, ints(lens), ints(new), t, cu, sl, P, slots=slots, groups=ints([0, 4]), shared=sh, info=info)
        assert k.device_error() == err
        assert (cu.tolist(), sl.tolist(), r.tolist(), t.tolist(), info.tolist()) == (want["cu"], want["seq_lens"], want["refs"], want["table"], want["info"])
        assert slots.tolist() == (want["slots"] + [-9] * rows)[:rows]
    # a page outside the pool in an old entry, and groups outside the batch
    t, cu, sl, slots, sh = ints([[9, 0]]), ints([-9] * 2), ints([-9]), ints([-9]), ints([-9, -9])
    k.paged_plan(ints([0, 0]), ints([3]), ints([1]), t, cu, sl, P, slots=slots, groups=ints([0, 1, 2]), shared=sh)
    assert k.device_error() == 2 and slots.tolist() == [-1] and sh.tolist() == [3, 0]


def test_plan_of_nothing():
    k, z = ops(), torch.zeros(0, dtype=torch.int32, device=DEV)
    cu, info = ints([-9]), ints([-9, -9])
    k.paged_plan(ints([0, 1, 0]), z, z, torch.zeros(0, 4, dtype=torch.int32, device=DEV), cu, z, 16, groups=ints([0]), shared=z, info=info)
    assert cu.tolist() == [0] and info.tolist() == [0, 2] and k.device_error() == 0


# ---- paged_fork --------------------------------------------------------------------------------------------
def fork(refs, table, lens, parents, P):
    """(refs, table, lens, info, copies [(row, from, to, filled rows)]) by the definition."""
    width, old = len(table[0]), list(refs)
    refs = list(refs)
    for b, n in enumerate(lens):
        for j in range(-(-n // P)):
            refs[table[b][j]] -= 1
    seen, copy = set(), []
    for b in parents:
        part = b >= 0 and lens[b] % P
        copy.append(bool(part and (b in seen or refs[table[b][lens[b] // P]])))
        seen.add(b)
    after = list(refs)
    for b, c in zip(parents, copy):
        for j in range(-(-lens[b] // P) - c if b >= 0 else 0):
            after[table[b][j]] += 1
    free = [p for p, r in enumerate(after) if r == 0]
    if sum(copy) > len(free):
        return old, [[-1] * width for _ in parents], [0] * len(parents), [sum(copy) - len(free), sum(r == 0 for r in old)], []
    rows, copies = [], []
    for i, (b, c) in enumerate(zip(parents, copy)):
        n = lens[b] if b >= 0 else 0
        row = table[b][:-(-n // P)] if b >= 0 else []
        if c:
            p = free.pop(0)
            after[p] = 1
            copies.append((i, row[-1], p, n % P))
            row = row[:-1] + [p]
        rows.append(row + [-1] * (width - len(row)))
    return after, rows, [lens[b] if b >= 0 else 0 for b in parents], [0, len(free)], copies


FORKS = {   # lens, parents, page, spare pages, groups of sequences that share
    "stay": ([20, 33, 16], [0, 1, 2], 16, 3, [0, 3]),
    "spread": ([77], [0] * 5, 16, 9, [0, 1]),
    "spread_whole_pages": ([64], [0] * 4, 32, 0, [0, 1]),
    "beams": ([100] * 4, [2, 0, 2, 2], 64, 5, [0, 4]),
    "exactly_enough": ([20, 20], [0, 0, 0], 16, 0, [0, 1, 2]),
    "one_too_few": ([20, 20], [0, 0, 0, 1], 16, 1, [0, 1, 2]),
    "end": ([20, 90, 5], [-1, -1, -1], 16, 2, [0, 3]),
    "swap": ([20, 90, 5], [2, 1, 0, -1], 128, 2, [0, 1, 3]),
    "empty_sequences": ([0, 1, 0], [0, 0, 1, 1, 2], 16, 2, [0, 3]),
    "many": ([37 * (i // 8) % 500 for i in range(800)], [i // 8 * 8 + (i * i) % 8 for i in range(800)], 32, 900, list(range(0, 801, 8))),
    "large_pool": ([100, 40], [1, 0, 0, 1], 16, 60_000, [0, 2]),
    "most_rows": ([i % 20 for i in range(16384)], [i ^ 1 if i % 3 else i for i in range(16384)], 16, 9000, [0, 16384]),
    "6000_rows": ([3] * 6000, list(range(6000)), 16, 10, [0, 6000]),
}


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "layers"])
@pytest.mark.parametrize("name", FORKS)
def test_fork(name, kind):
    lens, parents, P, spare, groups = FORKS[name]
    rng = random.Random(len(name))
    width = max(-(-n // P) for n in lens) + 2
    pages = sum(-(-n // P) for n in lens) + spare
    refs, table = random_state(rng, lens, P, pages, width, groups)
    # what a group shares are whole pages: a partly filled one belongs to its sequence
    for b, n in enumerate(lens):
        if n % P and refs[table[b][n // P]] > 1:
            old, free = table[b][n // P], [p for p, r in enumerate(refs) if r == 0]
            refs[old] -= 1
            table[b][n // P] = free[-1]
            refs[free[-1]] = 1
    for p in [p for p, r in enumerate(refs) if r == 0][spare:]:
        refs[p] = 2
    want = fork(refs, table, lens, parents, P)
    g = torch.Generator(device=DEV).manual_seed(5)
    fp8, n_kv = kind == "e4m3", 3
    lead = (3, pages) if kind != "bf16" else (pages,)
    if fp8:
        pools = [torch.randint(0, 255, (*lead, n_kv, P, D), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2)]
        scales = [torch.rand(*lead, n_kv, P, generator=g, device=DEV) for _ in range(2)]
    else:
        pools = [torch.randn(*lead, n_kv, P, D, generator=g, device=DEV).bfloat16() for _ in range(2)]
        scales = [None, None]
    expect = [x if x is None else x.clone() for x in (*pools, *scales)]
    for x in expect:
        for _, a, b, n in want[4] if x is not None else ():
            y = x if kind != "bf16" else x[None]
            y[:, b, :, :n] = y[:, a, :, :n]
    r, t, ro = ints(refs), ints(table), torch.full((pages,), -9, dtype=torch.int32, device=DEV)
    to = torch.full((len(parents), width + 3), -9, dtype=torch.int32, device=DEV)[:, :width]
    lo, info = torch.full((len(parents),), -9, dtype=torch.int32, device=DEV), ints([-9, -9])
    k = ops()
    k.device_error()
    k.paged_fork(r, ints(lens), ints(parents), t, to, lo, *pools, *scales, refs_out=ro, info=info)
    assert k.device_error() == (8 if name == "one_too_few" else 0)
    assert (ro.tolist(), to.tolist(), lo.tolist(), info.tolist()) == (want[0], want[1], want[2], want[3])
    for got, x in zip((*pools, *scales), expect):
        assert x is None or torch.equal(got.view(torch.uint8), x.view(torch.uint8))
    assert r.tolist() == refs and t.tolist() == table
    k.paged_fork(r, ints(lens), ints(parents), t, to, lo, *pools, *scales)            # the counts in place
    assert r.tolist() == want[0] and to.tolist() == want[1]
    k.device_error()


def test_fork_copies_what_a_sequence_outside_holds():
    """A partly filled page that someone else holds too is nobody's to keep."""
    k, P = ops(), 16
    pool = torch.randn(4, 1, P, D, device=DEV).bfloat16()
    refs, to, lo = ints([2, 0, 0, 1]), ints([[-9, -9]]), ints([-9])
    k.paged_fork(refs, ints([5]), ints([0]), ints([[0, 0]]), to, lo, pool, pool.clone())
    assert refs.tolist() == [1, 1, 0, 1] and to.tolist() == [[1, -1]] and torch.equal(pool[1, :, :5], pool[0, :, :5])


def test_fork_with_bad_inputs():
    """Lengths past the table, pages outside the pool and parents that are none set the error word; nothing else is touched."""
    k, P = ops(), 16
    pool = torch.randn(4, 1, P, D, device=DEV).bfloat16()
    before = pool.clone()
    refs, to, lo = ints([1, 1, 0, 0]), ints([[-9, -9]] * 4), ints([-9] * 4)
    k.device_error()
    k.paged_fork(refs, ints([99, 20]), ints([0, 1, 7, -2]), ints([[0, 1], [0, 44]]), to, lo, pool, pool.clone())
    assert k.device_error() == 2
    assert lo.tolist() == [0, 20, 0, 0] and to.tolist()[0] == [-1, -1] and to.tolist()[2:] == [[-1, -1]] * 2 and torch.equal(pool, before)


# ---- beam_select -------------------------------------------------------------------------------------------
def check_select(logits, scores, cu, k, got):
    """The bounds above, for (scores, parents, tokens) as lists."""
    V = logits.shape[1]
    x = logits.double()
    lp = scores.double()[:, None] + (x - torch.logsumexp(x, 1, keepdim=True))
    lp = lp.masked_fill((x == -math.inf) | (scores == -math.inf)[:, None], -math.inf)
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        s, parent, token = (g[b] for g in got)
        best = lp[lo:hi].flatten().topk(min(k, (hi - lo) * V)).values.tolist() if hi > lo else []
        best = [v for v in best if v > -math.inf]
        assert [p >= 0 for p in parent] == [i < len(best) for i in range(k)], b
        assert len(set(zip(parent, token))) >= len(best)
        for i in range(k):
            if i >= len(best):
                assert (s[i], parent[i], token[i]) == (-math.inf, -1, -1)
                continue
            assert lo <= parent[i] < hi and 0 <= token[i] < V
            e = lp[parent[i], token[i]].item()
            tol = abs(e) * 2.0 ** -24 + 2.0 ** -17
            assert abs(s[i] - e) <= tol and abs(e - best[i]) <= 2 * tol, (b, i, s[i], e, best[i])
        for r in range(lo, hi):                     # in a row: by logit, then by token, and none left out
            mine = [t for p, t in zip(parent, token) if p == r]
            order = torch.sort(x[r], descending=True, stable=True).indices[:len(mine)].tolist()
            assert mine == order, (b, r, mine, order)


def select(logits, scores, cu, k, **kw):
    B = len(cu) - 1
    out = torch.full((B, k), 7.0, device=DEV), torch.full((B, k), 7, dtype=torch.int32, device=DEV), torch.full((B, k), 7, dtype=torch.int32, device=DEV)
    o = ops()
    o.device_error()
    o.beam_select(logits, scores, ints(cu), *out, **kw)
    return o.device_error(), tuple(t.tolist() for t in out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cu,V,k", [([0, 1], 1, 1), ([0, 1], 5, 8), ([0, 4], 151936, 8), ([0, 3, 3, 10], 32003, 64), ([0, 1, 2, 3], 16384, 1),
                                    ([0, 128], 257, 33), ([0, 2], 16377, 16), ([0, 31, 32], 8193, 17), ([0, 1], 1048576, 64)], ids=str)
def test_select(cu, V, k, dtype):
    g = torch.Generator(device=DEV).manual_seed(V + k)
    logits = (torch.randn(cu[-1] + 2, V, generator=g, device=DEV) * 3).to(dtype)
    scores = torch.randn(cu[-1] + 2, generator=g, device=DEV) * 2 - 15
    err, got = select(logits, scores, cu, k)
    assert err == 0
    check_select(logits, scores, cu, k, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two_values", "few_left", "one_hot", "zeros_of_both_signs", "best_in_one_thread"])
def test_select_ties_and_orders(kind, dtype):
    V, k, rows = 40000, 50, 3
    x = torch.zeros(rows, V, device=DEV)
    if kind == "rising":
        x += torch.arange(V, device=DEV) / V * 20
    elif kind == "falling":
        x -= torch.arange(V, device=DEV) / V * 20
    elif kind == "two_values":
        x[:, ::3] = 1
    elif kind == "few_left":
        x.fill_(-math.inf)
        x[:, 39998:] = 1.0
        x[1, 5] = 2.0
    elif kind == "one_hot":
        x.fill_(-40)
        x[:, 77] = 60
    elif kind == "zeros_of_both_signs":
        x[:, ::2] = -0.0
    elif kind == "best_in_one_thread":
        x[:, 8:16] = 5
        x[:, 2048 + 8:2048 + 16] = 5
        x[:, 4096 + 8:4096 + 16] = 6
    logits, scores = x.to(dtype), torch.tensor([-1.0, -1.0, -7.5], device=DEV)
    err, got = select(logits, scores, [0, rows], k)
    assert err == 0
    check_select(logits, scores, [0, rows], k, got)
    if kind == "equal":                             # exact ties: by row, then token
        assert got[1][0] == [0] * k and got[2][0] == list(range(k))


def test_select_first_step_and_dead_beams():
    """Beams with a score of -inf give nothing, whatever lies in their rows; a request of only such beams is empty."""
    g = torch.Generator(device=DEV).manual_seed(1)
    logits = torch.randn(8, 1000, generator=g, device=DEV).bfloat16()
    scores = torch.tensor([0.0] + [-math.inf] * 7, device=DEV)
    logits[1] = math.nan
    err, got = select(logits, scores, [0, 4, 8], 6)
    assert err == 0 and got[1][0] == [0] * 6 and got[1][1] == [-1] * 6 and got[0][1] == [-math.inf] * 6
    check_select(logits[:1], scores[:1], [0, 1], 6, ([got[0][0]], [got[1][0]], [got[2][0]]))


def test_select_reports_rows_that_are_not_numbers():
    g = torch.Generator(device=DEV).manual_seed(2)
    for what in ("nan", "inf", "score_nan", "score_inf", "all_excluded"):
        logits, scores = torch.randn(3, 5000, generator=g, device=DEV), torch.zeros(3, device=DEV)
        if what == "nan":
            logits[1, 4321] = math.nan
        elif what == "inf":
            logits[1, 17] = math.inf
        elif what == "all_excluded":
            logits[1] = -math.inf
        else:
            scores[1] = math.nan if what == "score_nan" else math.inf
        err, got = select(logits, scores, [0, 3], 9)
        assert err == (0 if what == "all_excluded" else 2)
        assert set(got[1][0]) == {0, 2}
        keep = torch.tensor([0, 2], device=DEV)
        check_select(logits[keep], scores[keep], [0, 2], 9, ([got[0][0]], [[{0: 0, 2: 1}[p] for p in got[1][0]]], [got[2][0]]))


def test_select_strides_and_alignment():
    """Rows that begin anywhere, a view of a larger tensor: nothing outside it is looked at."""
    g = torch.Generator(device=DEV).manual_seed(3)
    for dtype in (torch.bfloat16, torch.float32):
        for first in (0, 1, 3, 7):
            big = torch.full((5, 3333), math.nan, device=DEV, dtype=dtype)
            big[1:4, first:first + 3001] = torch.randn(3, 3001, generator=g, device=DEV).to(dtype)
            logits, scores = big[1:4, first:first + 3001], torch.zeros(3, device=DEV)
            err, got = select(logits, scores, [0, 2, 3], 20)
            assert err == 0
            check_select(logits, scores, [0, 2, 3], 20, got)


def test_select_offsets_that_are_none():
    """A request whose rows are not the call's is empty and sets the error word; the others are as they would be alone."""
    g = torch.Generator(device=DEV).manual_seed(4)
    logits, scores = torch.randn(4, 100, generator=g, device=DEV), torch.zeros(4, device=DEV)
    for cu, bad in (([0, 5], {0}), ([2, 1, 4], {0}), ([-1, 4], {0}), ([0, 4, 300], {1}), ([0, 2, 4], set())):
        err, got = select(logits, scores, cu, 3)
        assert err == (2 if bad else 0)
        for b in range(len(cu) - 1):
            one = [[t[b]] for t in got]
            if b in bad:
                assert one == [[[-math.inf] * 3], [[-1] * 3], [[-1] * 3]]
            else:
                lo, hi = cu[b], cu[b + 1]
                check_select(logits[lo:hi], scores[lo:hi], [0, hi - lo], 3, (one[0], [[v - lo for v in one[1][0]]], one[2]))


# ---- shared_attention --------------------------------------------------------------------------------------
SHARED = {   # members and prefix of each group (prefix None: its sequences are on their own); new tokens; own keys; n_q, n_kv, page
    "beams": ([(4, 640)], [1], [30], 32, 8, 16),
    "alone": ([(1, 256), (1, 0)], [1], [5, 300], 32, 8, 16),
    "no_prefix": ([(3, 0), (2, 16)], [1], [40, 7], 32, 8, 16),
    "short_prefix": ([(5, 64), (3, 128), (2, 48)], [1], [1, 2, 100], 32, 8, 16),
    "many": ([(40, 2048)], [1], [1, 64, 65, 300, 17], 32, 8, 64),
    "more_than_a_tile": ([(70, 1024), (33, 384)], [1], [9, 130], 32, 8, 128),
    "groups": ([(3, 512), (9, 1536), (2, 4096), (17, 128), (1, 900)], [1], [1, 33, 200], 16, 4, 32),
    "no_group": ([(4, 512), (3, None), (5, 256)], [1], [20, 150], 32, 8, 32),
    "drafts": ([(6, 1024), (3, 256)], [1, 5, 2, 8], [8, 60, 200], 32, 8, 16),
    "chunks": ([(3, 512), (2, 1024)], [130, 1, 40, 9], [140, 200], 32, 8, 64),
    "mha": ([(9, 512)], [1, 3], [4, 70], 8, 8, 16),
    "group_3": ([(7, 384), (2, 128)], [1, 4], [4, 70], 12, 4, 32),
    "group_5": ([(30, 640)], [1], [4, 70], 10, 2, 64),
    "group_7": ([(11, 640)], [1, 2], [4, 70], 28, 4, 128),
    "group_16": ([(5, 640), (20, 256)], [1], [4, 70], 16, 1, 16),
    "group_32": ([(5, 640)], [1, 2], [4, 70], 32, 1, 64),
    "long": ([(3, 20480), (2, 8192)], [1], [77, 1500], 8, 2, 64),
    "many_groups": ([(2, 128 * (i % 4)) for i in range(60)], [1], [5, 18, 140], 8, 2, 16),
    "no_tokens": ([(4, 512)], [1, 0], [20], 32, 8, 16),
    "two_quarters": ([(13, 512), (9, 256)], [1], [3, 90], 32, 8, 32),
    "large": ([(30, 1280), (2, 1024), (17, 2048)], [1], [33, 1], 32, 8, 64),
    "large_drafts": ([(20, 2048), (11, 3968)], [4, 1, 3], [33, 6], 32, 8, 32),
}


def shared_case(name, fp8, seed=0, way="as_it_is"):
    """The call's tensors, with their rows in 64 bits: groups' tables name the prefix's pages, other pages hold NaN. way "large": with a
    group of 90 more sequences, which alone saves enough reads for the launch of the large prefixes, so that every large one is read
    once. "tensor": also with so many empty groups that only prefixes of one block of rows are left to the warps."""
    spec, new, own, n_q, n_kv, page = SHARED[name]
    if way != "as_it_is":
        spec = spec + [(90, -(-240_001 // (89 * n_kv)) // 128 * 128 + 128)]
    g = torch.Generator(device=DEV).manual_seed(seed + len(name) + n_q)
    members = [m for m, _ in spec]
    of = [i for i, m in enumerate(members) for _ in range(m)]
    B = len(of)
    n = [new[b % len(new)] for b in range(B)]
    tail = [max(own[b % len(own)], n[b]) for b in range(B)]
    prefix = [(p or 0) // page * page for _, p in spec]
    heads = cumulative(members)
    # one cache row for each prefix, then one for each sequence's own part
    c, rows = make_cache(prefix + tail, n_kv, page, fp8, g)
    lens = [prefix[of[b]] + tail[b] for b in range(B)]
    table = torch.full((B, max(-(-x // page) for x in lens) + 1), -7, dtype=torch.int32, device=DEV)
    full = []
    for b in range(B):
        a, z = prefix[of[b]] // page, -(-tail[b] // page)
        table[b, :a] = c["table"][of[b], :a]
        table[b, a:a + z] = c["table"][len(spec) + b, :z]
        full.append([torch.cat((rows[of[b]][i], rows[len(spec) + b][i])) for i in range(2)])
    grouped = [i for i, (_, p) in enumerate(spec) if p is not None]
    groups, shared = [], []
    for i in range(len(spec)):                      # (groups are a run: one that is on its own is left out by shared 0)
        groups.append(heads[i])
        shared.append(prefix[i] if i in grouped else 0)
    groups.append(B)
    if way == "tensor":
        groups, shared = groups + [B] * 420, shared + [0] * 420
    q = (torch.randn(sum(n) + 2, n_q, D, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    return dict(c, table=table, q=q, n=n, lens=lens, cu=cumulative(n), groups=groups, shared=shared, rows=full, page=page)


@pytest.mark.parametrize("way", ["as_it_is", "large", "tensor"])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("name", SHARED)
def test_shared_attention(name, fp8, way):
    s = shared_case(name, fp8, way=way)
    out = torch.full_like(s["q"], 3.0)
    k = ops()
    k.device_error()
    k.shared_attention(s["q"], ints(s["cu"]), ints(s["lens"]), s["table"], ints(s["groups"]), ints(s["shared"]), s["k"], s["v"], out, D ** -0.5,
                       max(s["n"]), k_scale=s["ks"], v_scale=s["vs"])
    assert k.device_error() == 0
    assert (out[s["cu"][-1]:] == 3).all()           # rows past the last sequence are left alone
    parts = [attend64(s["q"][a:b].double(), *s["rows"][i], s["lens"][i] - s["n"][i], D ** -0.5) for i, (a, b) in enumerate(zip(s["cu"], s["cu"][1:]))]
    check_attention(out[:s["cu"][-1]], *(torch.cat(x) for x in zip(*parts)), fp8)

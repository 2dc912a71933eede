"""How the operators for sequences that share pages may be called: captured and replayed over new contents, on two streams at once,
one after another on one workspace, with strides, with inputs that are refused or set the error word. Bounds as in
test_sharing_gpu.py."""
import math
import threading

import pytest
import torch

from test_paged_gpu import D, DEV, attend64, check_attention, cumulative, ints, make_cache, ops
from test_sharing_gpu import check_select, fork, plan, shared_case

pytestmark = pytest.mark.gpu


def run_shared(s, out, ws=None, **kw):
    a = dict(q=s["q"], cu=ints(s["cu"]), seq_lens=ints(s["lens"]), block_table=s["table"], groups=ints(s["groups"]), shared=ints(s["shared"]),
             k_pages=s["k"], v_pages=s["v"], out=out, scale=D ** -0.5, max_q=max(s["n"]), k_scale=s["ks"], v_scale=s["vs"], workspace=ws)
    ops().shared_attention(**{**a, **kw})


def check_shared(s, out, fp8=False):
    parts = [attend64(s["q"][a:b].double(), *s["rows"][i], s["lens"][i] - s["n"][i], D ** -0.5) for i, (a, b) in enumerate(zip(s["cu"], s["cu"][1:]))]
    check_attention(out[:s["cu"][-1]], *(torch.cat(x) for x in zip(*parts)), fp8)


def test_shared_calls_of_different_shapes_on_one_workspace():
    """Large and small calls in turn, shared and not, on one workspace: none leaves anything to the next."""
    k = ops()
    ws = k.shared_workspace(DEV, 300, 32)
    cases = [(n, f) for n in ("large", "drafts", "mha", "many_groups", "chunks", "beams") for f in (False, True)]
    for rnd in range(2):
        for i, (name, fp8) in enumerate(cases):
            s = shared_case(name, fp8, seed=rnd, way=("as_it_is", "large", "tensor")[i % 3])
            if s["q"].shape[0] > 300:
                continue
            out = torch.zeros_like(s["q"])
            run_shared(s, out, ws)
            assert k.device_error() == 0
            check_shared(s, out, fp8)


@pytest.mark.parametrize("name", ["large", "large_drafts", "beams"])
def test_shared_graph_follows_its_inputs(name):
    """A captured call replayed over other rows, lengths and shared lengths of the same batch."""
    k = ops()
    a, b = shared_case(name, False, seed=1), shared_case(name, False, seed=2)
    ws = k.shared_workspace(DEV, *a["q"].shape[:2])
    names = ("q", "table", "k", "v")
    buf = {n: a[n].clone() for n in names}
    cu, lens, groups, shared = (ints(a[n]) for n in ("cu", "lens", "groups", "shared"))
    out = torch.zeros_like(a["q"])
    # pages of the two cases have their own numbers: equal shapes hold both
    assert all(a[n].shape == b[n].shape for n in names)

    def call():
        k.shared_attention(buf["q"], cu, lens, buf["table"], groups, shared, buf["k"], buf["v"], out, D ** -0.5, max(a["n"]), workspace=ws)

    with pytest.raises(RuntimeError, match="before the capture"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            k.shared_attention(buf["q"], cu, lens, buf["table"], groups, shared, buf["k"], buf["v"], out, D ** -0.5, max(a["n"]))
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for s in (b, a, b):
        for n in names:
            buf[n].copy_(s[n])
        shared.copy_(ints([x - x % 256 for x in s["shared"]] if s is a else s["shared"]))   # less than is in common will do
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert k.device_error() == 0
        check_shared(s, out)


def test_calls_on_two_streams():
    """Each stream's own workspaces: calls that run beside each other."""
    k = ops()
    cases = [shared_case("large", False, seed=i) for i in range(2)]
    g = torch.Generator(device=DEV).manual_seed(9)
    logits = [torch.randn(24, 20000, generator=g, device=DEV) for _ in range(2)]
    scores, cu = torch.zeros(24, device=DEV), ints([0, 8, 24])
    outs = [torch.zeros_like(c["q"]) for c in cases]
    sel = [(torch.zeros(2, 16, device=DEV), *(torch.zeros(2, 16, dtype=torch.int32, device=DEV) for _ in range(2))) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                run_shared(cases[i], outs[i])
                k.beam_select(logits[i], scores, cu, *sel[i])
    torch.cuda.synchronize()
    assert k.device_error() == 0
    for i in range(2):
        check_shared(cases[i], outs[i])
        check_select(logits[i], scores, [0, 8, 24], 16, [t.tolist() for t in sel[i]])


def test_host_threads_share_a_stream():
    """Calls from two threads on one stream, each of several launches, on the stream's own workspaces."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(10)
    logits = [torch.randn(12, 30000, generator=g, device=DEV) for _ in range(2)]
    scores, cu = torch.zeros(12, device=DEV), ints([0, 5, 12])
    want = []
    for x in logits:
        out = (torch.zeros(2, 16, device=DEV), *(torch.zeros(2, 16, dtype=torch.int32, device=DEV) for _ in range(2)))
        k.beam_select(x, scores, cu, *out)
        want.append([t.clone() for t in out])
    cases, outs = [shared_case("large", False, seed=i) for i in range(2)], []
    args = []
    for s in cases:
        out = torch.zeros_like(s["q"])
        run_shared(s, out)
        outs.append(out.clone())
        args.append((s["q"], ints(s["cu"]), ints(s["lens"]), s["table"], ints(s["groups"]), ints(s["shared"]), s["k"], s["v"]))
    torch.cuda.synchronize()
    failed = []
    stream = torch.cuda.current_stream()

    def work(i):
        with torch.cuda.stream(stream):
            res = [(torch.zeros(2, 16, device=DEV), *(torch.zeros(2, 16, dtype=torch.int32, device=DEV) for _ in range(2))) for _ in range(40)]
            att = [torch.zeros_like(cases[i]["q"]) for _ in range(10)]
            for n, out in enumerate(res):
                k.beam_select(logits[i], scores, cu, *out)
                if n % 4 == 0:
                    k.shared_attention(*args[i], att[n // 4], D ** -0.5, 1)
            stream.synchronize()
            failed.extend(n for n, out in enumerate(res) if not all(torch.equal(a, b) for a, b in zip(out, want[i])))
            failed.extend(n for n, a in enumerate(att) if not torch.equal(a, outs[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and k.device_error() == 0


def test_shared_strides():
    """q and out as views of wider rows, heads apart; rows and gaps outside them untouched."""
    s = shared_case("large", False)
    T, n_q, _ = s["q"].shape
    wide = torch.full((T, n_q + 3, D + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    q = wide[:, 1:n_q + 1, :D]
    q.copy_(s["q"])
    back = torch.full((n_q, T + 2, D), 5.0, dtype=torch.bfloat16, device=DEV)
    out = back[:, 1:T + 1].transpose(0, 1)
    run_shared(dict(s, q=q), out)
    assert ops().device_error() == 0
    check_shared(s, out)
    assert (back[:, 0] == 5).all() and (back[:, T + 1] == 5).all() and (out[s["cu"][-1]:] == 5).all()


@pytest.mark.parametrize("members,empty", [(4, 0), (7, 400), (14, 0), (14, 400), (40, 0)])
def test_shared_large_and_rising_scores(members, empty):
    """Scores whose maxima lie late in the prefix and far above the first ones (the running maximum has to move), for prefixes of
    the warps and, in four, two and one parts, of the tensor cores, and own keys far below or above them."""
    n_kv, n_q, page, prefix, own = 8, 32, 32, 6400, 40
    g = torch.Generator(device=DEV).manual_seed(members)
    c, rows = make_cache([prefix] + [own] * members, n_kv, page, False, g)
    pos = torch.arange(prefix, device=DEV)
    lift = (pos[:, None, None] / prefix * 12).bfloat16()             # keys that grow along the prefix
    k_pages = c["k"]
    base = rows[0][0].bfloat16()
    new = (base * (0.1 + lift)).bfloat16()
    k_pages[c["table"][0, pos // page].long(), :, pos % page] = new
    rows[0][0] = new.double()
    for b in range(members):
        mul = 0.01 if b % 2 else 15.0
        p = torch.arange(own, device=DEV)
        new = (rows[1 + b][0].bfloat16() * mul).bfloat16()
        k_pages[c["table"][1 + b, p // page].long(), :, p % page] = new
        rows[1 + b][0] = new.double()
    table = torch.cat((c["table"][:1, :prefix // page].expand(members, -1), c["table"][1:, :-(-own // page)]), 1).contiguous()
    q = torch.randn(members, n_q, D, generator=g, device=DEV).bfloat16()
    s = dict(q=q, n=[1] * members, cu=list(range(members + 1)), lens=[prefix + own] * members, table=table, k=c["k"], v=c["v"], ks=None, vs=None,
             groups=[0, members], shared=[prefix], rows=[[torch.cat((rows[0][i], rows[1 + b][i])) for i in range(2)] for b in range(members)])
    s["groups"], s["shared"] = s["groups"] + [members] * empty, s["shared"] + [0] * empty
    out = torch.zeros_like(q)
    run_shared(s, out)
    assert ops().device_error() == 0
    check_shared(s, out)


def test_a_row_depends_on_its_own_query_only():
    """Another member's query changes nothing in a row, to the bit."""
    for name in ("beams", "two_quarters", "large"):
        s = shared_case(name, False, way="tensor")
        a, b = torch.zeros_like(s["q"]), torch.zeros_like(s["q"])
        run_shared(s, a)
        q = s["q"].clone()
        q[1] *= 40
        run_shared(dict(s, q=q), b)
        keep = [i for i in range(s["cu"][-1]) if i != 1]
        assert torch.equal(a[keep], b[keep]) and not torch.equal(a[1], b[1])


def test_shared_inputs_that_are_wrong():
    """Groups and lengths that are none set the error word; every access stays inside, and the next call is as it would be."""
    k = ops()
    s = shared_case("large", False)
    B = len(s["n"])
    out = torch.zeros_like(s["q"])
    longer = [s["shared"][0] + 4096] + s["shared"][1:]
    for bad in (dict(groups=[0, B + 5], shared=[640]), dict(groups=[-3, 4], shared=[640]), dict(groups=[5, 2, B], shared=[640, 640]),
                dict(shared=[-1] + s["shared"][1:]), dict(shared=[1 << 30] + s["shared"][1:]), dict(shared=longer)):
        k.device_error()
        run_shared(dict(s, **bad), out)
        assert k.device_error() == 2, bad
    run_shared(s, out)
    assert k.device_error() == 0
    check_shared(s, out)
    with pytest.raises(RuntimeError, match="workspace"):
        run_shared(s, out, k.attention_workspace(DEV))
    with pytest.raises(RuntimeError, match="workspace"):
        run_shared(s, out, k.shared_workspace(DEV, 4, 8))
    with pytest.raises(RuntimeError, match="shared"):
        run_shared(s, out, shared=ints([1, 2]))
    with pytest.raises(RuntimeError, match="max_q|rows"):
        run_shared(s, out, max_q=0)


def test_more_tokens_than_max_q():
    """A sequence with more rows than max_q says sets the error word and keeps its old output."""
    s = shared_case("chunks", False)
    k = ops()
    out = torch.full_like(s["q"], 3.0)
    k.device_error()
    run_shared(s, out, max_q=1)
    assert k.device_error() == 2 and (out[:130] == 3).all()


def test_empty_calls():
    k, z = ops(), torch.zeros(0, dtype=torch.int32, device=DEV)
    pool = torch.zeros(4, 1, 16, D, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(0, 4, D, dtype=torch.bfloat16, device=DEV)
    k.shared_attention(q, ints([0]), z, torch.zeros(0, 2, dtype=torch.int32, device=DEV), ints([0]), z, pool, pool, q, 0.1, 1)
    s = shared_case("beams", False)
    out = torch.zeros_like(s["q"])
    run_shared(dict(s, groups=[0], shared=[]), out)                 # no groups: paged attention
    check_shared(s, out)
    # every sequence ends: a fork without rows
    refs, info = ints([1, 0, 2, 1]), ints([-9, -9])
    k.paged_fork(refs, ints([20, 5]), z, ints([[0, 2], [2, -1]]), torch.zeros(0, 2, dtype=torch.int32, device=DEV), z.clone(), pool, pool, info=info)
    assert refs.tolist() == [0, 0, 0, 1] and info.tolist() == [0, 3]
    # from nothing: rows without parents
    to, lo = ints([[-9, -9]] * 2), ints([-9, -9])
    k.paged_fork(refs, z, ints([-1, -1]), torch.zeros(0, 2, dtype=torch.int32, device=DEV), to, lo, pool, pool)
    assert to.tolist() == [[-1, -1]] * 2 and lo.tolist() == [0, 0]
    out = (torch.zeros(2, 3, device=DEV), *(torch.zeros(2, 3, dtype=torch.int32, device=DEV) for _ in range(2)))
    k.beam_select(torch.zeros(0, 50, device=DEV), torch.zeros(0, device=DEV), ints([0, 0, 0]), *out)
    assert out[0].tolist() == [[-math.inf] * 3] * 2 and out[1].tolist() == [[-1] * 3] * 2
    assert k.device_error() == 0


def test_plan_and_fork_in_graphs_follow_their_inputs():
    k, P = ops(), 16
    lens, new, parents = [5, 16, 40], [3, 1, 0], [0, 0, 2, -1]
    pool = torch.randn(30, 2, P, D, device=DEV).bfloat16()
    refs, table = [0] * 30, [[-1] * 5 for _ in range(3)]
    for b, n in enumerate(lens):
        for j in range(-(-n // P)):
            table[b][j] = 29 - 4 * b - j
            refs[29 - 4 * b - j] = 1
    r, t, ro, to = ints(refs), ints(table), ints([0] * 30), ints(table)
    ln, nw, pr, cu, sl, t2, l2, r2 = ints(lens), ints(new), ints(parents), ints([0] * 4), ints([0] * 3), ints([[0] * 5] * 4), ints([0] * 4), ints([0] * 30)

    def calls():
        k.paged_plan(r, ln, nw, t, cu, sl, P, refs_out=ro, table_out=to)
        k.paged_fork(ro, sl, pr, to, t2, l2, pool, pool.clone(), refs_out=r2)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        calls()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        calls()
    for lens2, new2, parents2 in ((lens, new, parents), ([4, 10, 33], [1, 30, 9], [2, 2, 1, 0]), (lens, [0, 0, 0], [-1, -1, -1, 1])):
        ln.copy_(ints(lens2)), nw.copy_(ints(new2)), pr.copy_(ints(parents2))
        g.replay()
        torch.cuda.synchronize()
        a = plan(refs, table, lens2, new2, P, [0], 1 << 20)
        b = fork(a["refs"], a["table"], a["seq_lens"], parents2, P)
        assert (cu.tolist(), sl.tolist(), to.tolist(), ro.tolist()) == (a["cu"], a["seq_lens"], a["table"], a["refs"])
        assert (r2.tolist(), t2.tolist(), l2.tolist()) == b[:3]
    assert k.device_error() == 0


def test_a_pool_of_pages_past_32_bit_bytes():
    """Pages whose copies lie past 2^32 bytes."""
    pages, n_kv, P = 36000, 8, 64
    k_pages = torch.empty(pages, n_kv, P, D, dtype=torch.bfloat16, device=DEV)       # 4.7 GB
    k_pages[pages - 1, :, :7] = 3.0
    refs, to, lo = torch.ones(pages, dtype=torch.int32, device=DEV), ints([[-9], [-9]]), ints([-9, -9])
    refs[pages - 2] = 0
    ops().paged_fork(refs, ints([7]), ints([0, 0]), ints([[pages - 1]]), to, lo, k_pages, k_pages.clone())
    assert to.tolist() == [[pages - 1], [pages - 2]]
    assert (k_pages[pages - 2, :, :7] == 3).all()


def test_refusals():
    k, P = ops(), 16
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)   # noqa: E731
    pool = torch.zeros(4, 1, P, D, dtype=torch.bfloat16, device=DEV)
    table = i(2, 3)
    for bad in (dict(refs=i(4).long()), dict(lens=i(2, 1)), dict(new=i(3)), dict(cu=i(2)), dict(seq_lens=i(3)), dict(page_size=24),
                dict(table_out=i(3, 3)), dict(slots=i(2, 2)), dict(positions=i(5), slots=i(4)), dict(info=i(3)), dict(groups=i(2)),
                dict(shared=i(1)), dict(groups=i(0), shared=i(0)), dict(block_table=i(3, 2).t()), dict(refs_out=i(5)), dict(lens=torch.zeros(2).int())):
        a = dict(refs=i(4), lens=i(2), new=i(2), block_table=table, cu=i(3), seq_lens=i(2), page_size=P)
        with pytest.raises(RuntimeError):
            k.paged_plan(**{**a, **bad})
    lens = i(2)
    with pytest.raises(RuntimeError, match="overlap"):
        k.paged_plan(i(4), lens, i(2), table, i(3), lens, P)
    for bad in (dict(parents=i(2).float()), dict(table_out=i(2, 4)), dict(lens_out=i(3)), dict(k_pages=pool[:, :, :8]), dict(k_scale=torch.zeros(4, 1, P, device=DEV)),
                dict(k_pages=pool.view(torch.uint8)[..., :D].contiguous(), v_pages=pool.view(torch.uint8)[..., :D].contiguous()), dict(refs=i(5)),
                dict(table_out=table), dict(v_pages=pool.float())):
        a = dict(refs=i(4), lens=i(2), parents=i(2), block_table=table, table_out=i(2, 3), lens_out=i(2), k_pages=pool, v_pages=pool)
        with pytest.raises(RuntimeError):
            k.paged_fork(**{**a, **bad})
    f = lambda *shape: torch.zeros(shape, device=DEV)   # noqa: E731
    for bad in (dict(logits=f(3, 9).half()), dict(scores=f(2)), dict(cu=i(2, 1)), dict(out_scores=f(1, 65)), dict(out_parents=i(1, 5)),
                dict(out_tokens=i(2, 4)), dict(logits=f(9, 3).t()), dict(out_scores=f(2, 4)), dict(workspace=f(4)),
                dict(workspace=torch.zeros(64, dtype=torch.uint8, device=DEV))):
        a = dict(logits=f(3, 9), scores=f(3), cu=i(2), out_scores=f(1, 4), out_parents=i(1, 4), out_tokens=i(1, 4))
        with pytest.raises(RuntimeError):
            k.beam_select(**{**a, **bad})
    with pytest.raises(RuntimeError, match="before the capture"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            k.beam_select(f(3, 9), f(3), i(2), f(1, 4), i(1, 4), i(1, 4))
    assert k.device_error() == 0

"""The paged operators on the GPU, called in ways of their own: shared tables, several host threads, captures, orders and
strides. Outputs are compared bit for bit with those of the ordinary call."""
import pytest
import torch

from test_paged_gpu import D, DEV, cumulative, ints, make_cache, ops

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_one_table_for_every_sequence(n, fp8):
    """An expanded table: several queries over one context, several ranges of one sequence."""
    k = ops()
    c, _ = make_cache([300], 4, 32, fp8, torch.Generator(device=DEV).manual_seed(n))
    B, lens = 3, [300, 190, n]
    q = torch.randn(B * n, 16, D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    cu = ints(cumulative([n] * B))
    got = []
    for table in (c["table"].expand(B, -1), c["table"].expand(B, -1).contiguous()):
        out = torch.empty_like(q)
        k.paged_attention(q, cu, ints(lens), table, c["k"], c["v"], out, D ** -0.5, n, k_scale=c["ks"], v_scale=c["vs"])
        ko, vo = (torch.empty(B * n, 4, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        k.paged_kv_read(cu, table, c["k"], c["v"], ko, vo, k_scale=c["ks"], v_scale=c["vs"], starts=ints([0, 100, 300 - n]))
        got.append((out, ko, vo))
    assert all(same(a, b) for a, b in zip(*got))
    assert k.device_error() == 0


def test_a_capture_needs_a_workspace_of_its_own():
    """Also on a stream that an earlier call has given one."""
    k = ops()
    c, _ = make_cache([40], 8, 16, False, torch.Generator(device=DEV).manual_seed(1))
    q, out = torch.zeros(1, 32, D, dtype=torch.bfloat16, device=DEV), torch.empty(1, 32, D, dtype=torch.bfloat16, device=DEV)
    call = (q, ints([0, 1]), ints([40]), c["table"], c["k"], c["v"], out, 0.1, 1)
    ws, side = k.attention_workspace(DEV), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k.paged_attention(*call)
        assert ("ragged", q.get_device(), side.cuda_stream) in k._scratch
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="before the capture"):
            k.paged_attention(*call)
        k.paged_attention(*call, workspace=ws)
    graph.replay()
    torch.cuda.synchronize()
    assert k.device_error() == 0


def test_host_threads_share_a_stream():
    """Mixed batches (two launches a call), packed prompts and decode steps from several threads on one stream and its one
    workspace: each call's output as from a call alone."""
    import threading
    k = ops()
    work = []
    for i in range(4):
        g = torch.Generator(device=DEV).manual_seed(i)
        n = [1, 30 + 17 * i, 1, 2]
        lens = [900 + 100 * i, 700, 50, 400]
        c, _ = make_cache(lens, 4, 32, i % 2 == 1, g)
        q = torch.randn(sum(n), 16, D, generator=g, device=DEV).to(torch.bfloat16)
        kv = torch.randn(2, sum(n), 4, D, generator=g, device=DEV).to(torch.bfloat16)
        work.append((q, kv, c, ints(cumulative(n)), ints(lens), max(n), ints(list(range(5)))))

    def calls(i, outs):
        q, kv, c, cu, lens, top, ones = work[i]
        for a, b, d in outs:
            k.paged_attention(q, cu, lens, c["table"], c["k"], c["v"], a, D ** -0.5, top, k_scale=c["ks"], v_scale=c["vs"])
            k.packed_attention(q, kv[0], kv[1], cu, b, D ** -0.5, top)
            k.paged_attention(q[:4], ones, lens, c["table"], c["k"], c["v"], d, D ** -0.5, 1, k_scale=c["ks"], v_scale=c["vs"])

    def outputs(i, n):
        q = work[i][0]
        return [(torch.empty_like(q), torch.empty_like(q), torch.empty_like(q[:4])) for _ in range(n)]

    want = [outputs(i, 1) for i in range(4)]
    for i in range(4):
        calls(i, want[i])
    torch.cuda.synchronize()
    got = [outputs(i, 50) for i in range(4)]
    threads = [threading.Thread(target=calls, args=(i, got[i])) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert k.device_error() == 0
    for i in range(4):
        for outs in got[i]:
            assert all(same(a, b) for a, b in zip(outs, want[i][0]))


def test_outputs_of_any_order():
    """Rows within heads, heads within rows, and the two laid between each other (rows 256 apart, heads 384): the same
    bits; expanded outputs are refused."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(3)
    lens, n_q, n_kv = [100], 8, 2
    c, _ = make_cache(lens, n_kv, 16, False, g)
    cu, sl = ints([0, 3]), ints(lens)
    q = torch.randn(3, n_q, D, generator=g, device=DEV).to(torch.bfloat16)
    kv = torch.randn(2, 3, n_kv, D, generator=g, device=DEV).to(torch.bfloat16)

    def run(out, ko, vo):
        k.paged_attention(q, cu, sl, c["table"], c["k"], c["v"], out, D ** -0.5, 3)
        k.paged_kv_read(cu, c["table"], c["k"], c["v"], ko, vo)
        both = torch.empty_like(q).copy_(out)
        k.packed_attention(q, kv[0], kv[1], cu, out, D ** -0.5, 3)
        return both, torch.empty_like(q).copy_(out), ko.contiguous(), vo.contiguous()

    def empty(heads, row, head):
        return torch.empty(3 * row + heads * head, dtype=torch.bfloat16, device=DEV).as_strided((3, heads, D), (row, head, 1))

    want = run(*(empty(h, h * D, D) for h in (n_q, n_kv, n_kv)))
    for row, head in ((D, 3 * D), (1200, D), (D, 400), (256, 384 * 2)):
        got = run(*(empty(h, row, head) for h in (n_q, n_kv, n_kv)))
        assert all(same(a, b) for a, b in zip(got, want))
    between = [torch.empty(4096, dtype=torch.bfloat16, device=DEV).as_strided((3, n_kv, D), (256, 384, 1)) for _ in range(2)]
    k.paged_kv_read(cu, c["table"], c["k"], c["v"], *between)
    assert all(same(a.contiguous(), b) for a, b in zip(between, want[2:]))
    with pytest.raises(RuntimeError, match="overlap"):
        k.paged_attention(q, cu, sl, c["table"], c["k"], c["v"], q[:1].expand(3, -1, -1), D ** -0.5, 3)
    with pytest.raises(RuntimeError, match="overlap"):
        k.packed_attention(q, kv[0], kv[1], cu, q[:, :1].expand(-1, n_q, -1), D ** -0.5, 3)
    assert k.device_error() == 0


@pytest.mark.parametrize("what", ["decode", "mixed", "packed", "linear"])
def test_a_call_may_be_a_threads_first(what):
    """A new host thread whose first use of the GPU is one of the calls that build tensor maps."""
    import threading
    import model as M
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(7)
    c, _ = make_cache([300], 2, 16, False, g)
    n = 1 if what == "decode" else 40
    q = torch.randn(n, 8, D, generator=g, device=DEV).to(torch.bfloat16)
    kv = torch.randn(2, n, 2, D, generator=g, device=DEV).to(torch.bfloat16)
    cu, lens, ws = ints([0, n]), ints([300]), k.attention_workspace(DEV)
    w = torch.randn(256, 256, generator=g, device=DEV).to(torch.float8_e4m3fn)
    scale, x = torch.ones(256, device=DEV), torch.randn(4, 256, generator=g, device=DEV).to(torch.bfloat16)

    def call(out):
        if what == "linear":
            k.fp8_gemm_rows(x, w, scale, out)
        elif what == "packed":
            k.packed_attention(q, kv[0], kv[1], cu, out, D ** -0.5, n, workspace=ws)
        else:
            k.paged_attention(q, cu, lens, c["table"], c["k"], c["v"], out, D ** -0.5, n, workspace=ws)

    want, got = (torch.zeros_like(x if what == "linear" else q) for _ in range(2))
    call(want)
    failed = []

    def first():
        try:
            call(got)
        except RuntimeError as e:
            failed.append(e)

    t = threading.Thread(target=first)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not failed and same(got, want) and k.device_error() == 0


@pytest.mark.parametrize("n_q,n,launches", [(8, 1, 1), (16, 1, 1), (8, 40, 2), (9, 2, 1), (16, 2, 1), (32, 1, 1), (32, 40, 1)])
def test_launches_of_a_call(n_q, n, launches):
    """One KV head. A mixed batch is two launches where some sequence can have few rows: one token has more than 8 of them
    from 9 query heads per KV head on."""
    import ctypes
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(n_q)
    c, _ = make_cache([300, 70], 1, 16, False, g)
    q = torch.randn(2 * n, n_q, D, generator=g, device=DEV).to(torch.bfloat16)
    out, cu, lens, ws = torch.empty_like(q), ints([0, n, 2 * n]), ints([300, 70]), k.attention_workspace(DEV)

    def call():
        k.paged_attention(q, cu, lens, c["table"], c["k"], c["v"], out, D ** -0.5, n, workspace=ws)

    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    nodes = ctypes.c_size_t(0)
    assert ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
    assert nodes.value == launches


def one_row(heads, row):
    """[1, heads, D] whose row stride means nothing (a transposed vector has 1)."""
    return torch.zeros(heads * D, dtype=torch.bfloat16, device=DEV).as_strided((1, heads, D), (row, D, 1))


@pytest.mark.parametrize("row", [1, 0, 4100])
def test_a_single_row_has_no_stride(row):
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(5)
    c, _ = make_cache([70], 2, 16, False, g)
    cos, sin = torch.rand(2, 128, 64, generator=g, device=DEV)
    x = torch.randn(12 * D, generator=g, device=DEV).to(torch.bfloat16)
    cu, lens = ints([0, 1]), ints([70])

    def run(row):
        q, ko, kr, vr, o, op = (one_row(h, r) for h, r in ((8, row), (2, row), (2, row), (2, row), (8, row), (8, row)))
        qkv = torch.empty_like(x).copy_(x).as_strided((1, 12 * D), (row, 1))
        k.paged_qkv(qkv, cu, lens, c["table"], c["k"], c["v"], q, cos, sin, k_out=ko)
        k.paged_kv_read(cu, c["table"], c["k"], c["v"], kr, vr, starts=ints([69]))
        k.paged_attention(q, cu, lens, c["table"], c["k"], c["v"], o, D ** -0.5, 1)
        k.packed_attention(q, ko, vr, cu, op, D ** -0.5, 1)
        return [t.flatten() for t in (q, ko, kr, vr, o, op)]

    want = run(12 * D)
    assert all(same(a, b) for a, b in zip(run(row), want))
    assert same(want[1], want[2]) and k.device_error() == 0


def test_broadcast_inputs():
    """Queries, keys and values expanded over rows or heads give what their copies give."""
    k = ops()
    g = torch.Generator(device=DEV).manual_seed(6)
    c, _ = make_cache([300], 4, 32, False, g)
    cu, lens = ints([0, 50]), ints([300])
    x = torch.randn(50, 8, D, generator=g, device=DEV).to(torch.bfloat16)
    rows, heads = x[:1].expand(50, -1, -1), x[:, :1].expand(-1, 8, -1)
    for q in (rows, heads):
        got = []
        for t in (q, q.contiguous()):
            out = torch.empty(50, 8, D, dtype=torch.bfloat16, device=DEV)
            k.paged_attention(t, cu, lens, c["table"], c["k"], c["v"], out, D ** -0.5, 50)
            got.append(out.clone())
        assert same(*got)
    for kv in (rows[:, :4], heads[:, :4]):
        got = []
        for t in (kv, kv.contiguous()):
            out = torch.empty(50, 8, D, dtype=torch.bfloat16, device=DEV)
            k.packed_attention(x, t, t, cu, out, D ** -0.5, 50)
            got.append(out)
        assert same(*got)
    assert k.device_error() == 0

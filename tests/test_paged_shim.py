"""What the paged operators' shim sends to the library, without a GPU: CPU tensors that say they are on device 0, and a
library that records its arguments."""
import weakref

import pytest
import torch


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on GPU `index`."""
    index = 0

    def get_device(self):
        return self.index


def gpu(t):
    return t.as_subclass(OnGpu)


class Library:
    """Stands in for the C library: every entry point unpacks its argument struct, records it and succeeds."""

    def __init__(self, kernels):
        self.calls = []
        for name, fmt in (("qk_paged_qkv", kernels._QKV_ARGS), ("qk_paged_kv_read", kernels._READ_ARGS),
                          ("qk_paged_attention", kernels._ATTENTION_ARGS), ("qk_packed_attention", kernels._ATTENTION_ARGS)):
            setattr(self, name, self.entry(name, fmt))

    def entry(self, name, fmt):
        def call(args, stream):
            self.calls.append((name, fmt.unpack(args)))
            return 0
        return call

    def qk_ragged_attention_workspace_bytes(self):
        return 512


@pytest.fixture
def shim(monkeypatch):
    import kernels
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 0x100)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    return kernels.DecodeOps(Library(kernels))


def ints(v):
    return gpu(torch.tensor(v, dtype=torch.int32))


def bf16(*shape):
    return gpu(torch.zeros(*shape, dtype=torch.bfloat16))


TABLE_STRIDE = 12   # the field of qk_paged_cache_t


def table_calls(shim, table, lens):
    """Each call that takes a block table, with one new row a sequence; the row strides that were sent."""
    B = len(lens)
    pages, cu = bf16(8, 2, 16, 128), ints(list(range(B + 1)))
    q, kv = bf16(B, 4, 128), bf16(B, 2, 128)
    tab = gpu(torch.zeros(64, 64))
    ws = gpu(torch.zeros(512, dtype=torch.uint8))
    shim.paged_attention(q, cu, ints(lens), table, pages, pages, q, 0.1, 1, workspace=ws)
    shim.paged_kv_read(cu, table, pages, pages, kv, kv)
    shim.paged_qkv(bf16(B, 8 * 128), cu, ints(lens), table, pages, pages, q, tab, tab)
    return [args[TABLE_STRIDE] for _, args in shim.lib.calls]


def test_a_table_is_sent_with_its_own_row_stride(shim):
    """One table for several ranges of a sequence is an expanded one: stride 0, not the width (rows past its end)."""
    row = torch.tensor([[1, 2, 3]], dtype=torch.int32)
    assert table_calls(shim, gpu(row.expand(3, -1)), [40, 41, 42]) == [0, 0, 0]
    shim.lib.calls.clear()
    wide = torch.zeros(4, 10, dtype=torch.int32)
    assert table_calls(shim, gpu(wide[:, :3]), [40] * 4) == [10] * 3
    shim.lib.calls.clear()
    overlapping = torch.zeros(8, dtype=torch.int32).as_strided((3, 3), (2, 1))   # the library refuses it
    assert table_calls(shim, gpu(overlapping), [40] * 3) == [2] * 3
    shim.lib.calls.clear()
    assert table_calls(shim, gpu(torch.zeros(8, dtype=torch.int32).as_strided((1, 3), (1, 1))), [40]) == [3] * 3


def test_the_library_takes_shared_tables_and_refuses_overlapping_ones():
    import os
    import kernels
    if not os.path.exists(kernels.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    lib = kernels.load_library()

    def read(batch, width, stride):   # no rows: the checks, and no launch
        return lib.qk_paged_kv_read(kernels._READ_ARGS.pack(256, 256, 0, 0, 256, 0, 256, batch, 8, 10, 16, width, stride, 0,
                                                            0, 256, 256, 0, 1024, 128), 0)

    assert read(3, 4, 0) == 0 and read(3, 4, 4) == 0 and read(3, 4, 9) == 0
    for stride in (1, 3, -1, -4):
        assert read(3, 4, stride) == 1 and b"table_stride" in lib.qk_last_error()


class Linears:
    """The batched linear's entry points: a scratch that grows with the rows, and the scratch pointers of the calls."""

    def __init__(self):
        self.seen = []

    def qk_fp8_gemm_rows_scratch_bytes(self, M, N, K):
        return 1024 * M

    def qk_fp8_gemm_rows(self, x, norm, M, K, w, ws, mode, N, eps, out, scratch, nbytes, stream):
        assert nbytes >= 1024 * M
        self.seen.append(scratch.value)
        return 0


@pytest.fixture
def linear(monkeypatch):
    import kernels
    monkeypatch.setattr(kernels, "_stream", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    k = kernels.DecodeOps(Linears())
    w = torch.zeros(128, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)

    def call(rows, **kw):
        x = torch.zeros(rows, 128, dtype=torch.bfloat16)
        k.fp8_gemm_rows(x, w, torch.zeros(128), x.clone(), **kw)
    return k, call


def test_a_scratch_that_a_graph_may_hold_outlives_a_larger_one(linear):
    k, call = linear
    call(4)
    held = weakref.ref(k._scratch[("gemm", 0)])
    call(128)
    call(4)
    first, second, third = k.lib.seen
    assert first != second and third == second and held() is not None and held().data_ptr() == first


def test_the_gemvs_scratch_outlives_a_larger_one(monkeypatch):
    import kernels
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    k = kernels.DecodeOps(Linears())
    held = [weakref.ref(t) for t in k.scratch(torch.device("cpu"), 64, 4)]
    assert [weakref.ref(t) for t in k.scratch(torch.device("cpu"), 32, 4)] == held
    k.scratch(torch.device("cpu"), 65, 4)
    assert all(r() is not None for r in held)


def test_a_scratch_of_the_callers(linear):
    k, call = linear
    own = k.gemm_scratch("cpu", 64, [(128, 128)])
    assert own.numel() == 64 * 1024 and not own.any()
    call(64, scratch=own)
    call(4, scratch=own)
    assert k.lib.seen == [own.data_ptr()] * 2 and not k._scratch
    for bad in (own.float(), own[::2]):
        with pytest.raises(RuntimeError, match="scratch"):
            call(4, scratch=bad)
    with pytest.raises(RuntimeError, match="scratch"):
        call(65, scratch=own)


def paged_calls(k, index):
    """Every paged operator with tensors of GPU `index`."""
    def on(t):
        t = gpu(t)
        t.index = index
        return t

    def zeros(*shape, dtype=torch.bfloat16):
        return on(torch.zeros(*shape, dtype=dtype))

    cu, lens, table = (on(torch.tensor(v, dtype=torch.int32)) for v in ([0, 1], [5], [[1, 2]]))
    pages, q, kv, tab = zeros(8, 2, 16, 128), zeros(1, 4, 128), zeros(1, 2, 128), zeros(64, 64, dtype=torch.float32)
    ws = zeros(512, dtype=torch.uint8)
    return [lambda: k.paged_attention(q, cu, lens, table, pages, pages, q, 0.1, 1, workspace=ws),
            lambda: k.packed_attention(q, kv, kv, cu, q, 0.1, 1, workspace=ws),
            lambda: k.paged_kv_read(cu, table, pages, pages, kv, kv),
            lambda: k.paged_qkv(zeros(1, 8 * 128), cu, lens, table, pages, pages, q, tab, tab)]


def test_tensors_of_a_device_that_is_not_current_are_refused(shim, monkeypatch):
    """The library launches on the current device, where another device's pointers mean nothing."""
    for current in (0, 1):
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current)
        shim.lib.calls.clear()
        for call in paged_calls(shim, current):
            call()
        assert len(shim.lib.calls) == 4
        for call in paged_calls(shim, 1 - current):
            with pytest.raises(RuntimeError, match="current"):
                call()
        assert len(shim.lib.calls) == 4


def test_a_capture_never_takes_the_streams_own_workspace(shim, monkeypatch):
    """Not even where an earlier call on the stream has made it: its replays may run beside calls that use it."""
    capturing = False
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: capturing)
    monkeypatch.setattr(shim, "attention_workspace", lambda device: gpu(torch.zeros(512, dtype=torch.uint8)))
    q, kv, pages = bf16(1, 4, 128), bf16(1, 2, 128), bf16(8, 2, 16, 128)
    attend = [lambda **kw: shim.paged_attention(q, ints([0, 1]), ints([5]), ints([[1, 2]]), pages, pages, q, 0.1, 1, **kw),
              lambda **kw: shim.packed_attention(q, kv, kv, ints([0, 1]), q, 0.1, 1, **kw)]
    for call in attend:
        call()
    capturing = True
    for call in attend:
        with pytest.raises(RuntimeError, match="before the capture"):
            call()
        call(workspace=gpu(torch.zeros(512, dtype=torch.uint8)))
    assert len(shim.lib.calls) == 4


OVERLAPS = [dict(row=0, head=128), dict(row=4096, head=0), dict(row=64, head=4096), dict(row=128, head=128), dict(row=4096, head=64),
            dict(row=512, head=128), dict(row=128, head=256), dict(row=384, head=256)]


@pytest.mark.parametrize("bad", OVERLAPS, ids=str)
def test_outputs_whose_rows_overlap_are_refused(bad):
    """An expanded output, or one whose rows and heads run into each other: what it would hold depends on the order of
    the stores. (8 rows of 8 heads; every call is refused before a launch.)"""
    import os
    import kernels
    if not os.path.exists(kernels.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    lib, (row, head) = kernels.load_library(), bad.values()
    cache = (256, 256, 0, 0, 256, 256, 256, 2, 8, 10, 16, 4, 4, 0)
    att = kernels._ATTENTION_ARGS.pack(*cache, 256, 256, 256, 256, 256, 8, 8, 8, 1024, 128, 1024, 128, row, head, 1 << 40, 0.1)
    for f, args in ((lib.qk_paged_attention, att), (lib.qk_packed_attention, att),
                    (lib.qk_paged_kv_read, kernels._READ_ARGS.pack(*cache, 0, 256, 256, 8, row, head))):
        assert f(args, 0) == 1 and b"overlap" in lib.qk_last_error()


def test_recovery_resets_every_scratch(linear):
    """Counters that a timed-out wait left mid-count: of the GEMV's and the linears' scratch, and of those that larger calls
    replaced and a graph may still run on."""
    k, call = linear
    tensors = []
    for units in (4, 8):
        tensors.append(k.scratch(torch.device("cpu"), 64, units)[1])
    call(4)
    tensors.append(k._scratch[("gemm", 0)])
    call(128)
    tensors.append(k._scratch[("gemm", 0)])
    k._scratch[("ragged", 0, 0)] = torch.zeros(64, dtype=torch.uint8)
    tensors.append(k._scratch[("ragged", 0, 0)])
    for t in tensors:
        t.fill_(1)
    k.reset_scratch()
    assert not any(t.any() for t in tensors)

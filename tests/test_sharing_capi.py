"""The host side of the operators for sequences that share pages, without a GPU: bad arguments are refused with a message
before anything is launched, and the shim refuses tensors of the wrong kind."""
import os

import pytest
import torch


@pytest.fixture(scope="module")
def k():
    import kernels
    if not os.path.exists(kernels.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return kernels


M = 1 << 20   # addresses far enough apart
PLAN = dict(refs=1 * M, lens=2 * M, fresh=3 * M, table=4 * M, groups=5 * M, refs_out=6 * M, table_out=7 * M, cu=8 * M, seq_lens=9 * M,
            slots=10 * M, positions=11 * M, shared=12 * M, info=13 * M, batch=3, width=4, stride=4, out_stride=4, pages=10, page=16, rows=9,
            n_groups=1)
FORK = dict(refs=1 * M, lens=2 * M, parents=3 * M, table=4 * M, refs_out=6 * M, table_out=7 * M, lens_out=8 * M, info=9 * M, k=10 * M,
            v=11 * M, ks=0, vs=0, batch=3, rows=2, width=4, stride=4, out_stride=4, layers=2, pages=10, n_kv=8, page=16, fp8=0)
BEAM = dict(logits=1 * M, scores=2 * M, cu=3 * M, out_scores=4 * M, out_parents=5 * M, out_tokens=6 * M, workspace=7 * M, rows=4, batch=1,
            vocab=100, k=8, row_stride=100, fp32=0, workspace_bytes=1 << 40)
SHARED = dict(k_pages=256, v_pages=256, k_scale=0, v_scale=0, cu=256, lens=256, table=256, batch=2, n_kv=8, pages=10, page=16, width=4,
              stride=4, fp8=0, q=256, k=0, v=0, out=256, workspace=256, rows=3, n_q=32, max_q=1, q_row=4096, q_head=128, kv_row=0, kv_head=0,
              o_row=4096, o_head=128, workspace_bytes=1 << 40, scale=0.1, groups=256, shared=256, n_groups=1)


@pytest.mark.parametrize("bad", [
    dict(refs=0), dict(lens=0), dict(fresh=0), dict(table=0), dict(refs_out=0), dict(table_out=0), dict(cu=0), dict(seq_lens=0),
    dict(groups=0), dict(shared=0), dict(n_groups=-1), dict(n_groups=1 << 20), dict(batch=-1), dict(batch=16385), dict(width=0),
    dict(stride=3), dict(out_stride=0), dict(pages=0), dict(page=24), dict(page=8), dict(pages=1 << 28), dict(rows=-2), dict(rows=-1),
    dict(rows=1 << 40), dict(table_out=4 * M + 4), dict(table_out=4 * M, out_stride=5), dict(refs_out=M + 4), dict(seq_lens=2 * M),
    dict(seq_lens=3 * M + 8), dict(width=1 << 28, stride=1 << 28, out_stride=1 << 28)], ids=str)
def test_paged_plan_refuses(k, bad):
    lib, a = k.load_library(), {**PLAN, **bad}
    assert lib.qk_paged_plan(k._PLAN_ARGS.pack(*a.values()), 0) == 1 and lib.qk_last_error()


@pytest.mark.parametrize("bad", [
    dict(refs=0), dict(lens=0), dict(parents=0), dict(table=0), dict(refs_out=0), dict(table_out=0), dict(lens_out=0), dict(k=0),
    dict(v=0), dict(fp8=1), dict(batch=16385), dict(rows=16385), dict(rows=-1), dict(width=0), dict(stride=3), dict(out_stride=0),
    dict(layers=0), dict(layers=1 << 20), dict(n_kv=0), dict(pages=0), dict(pages=1 << 25), dict(page=48), dict(k=10 * M + 8),
    dict(table_out=4 * M), dict(lens_out=2 * M), dict(lens_out=3 * M + 4), dict(refs_out=M + 8)], ids=str)
def test_paged_fork_refuses(k, bad):
    lib, a = k.load_library(), {**FORK, **bad}
    assert lib.qk_paged_fork(k._FORK_ARGS.pack(*a.values()), 0) == 1 and lib.qk_last_error()


@pytest.mark.parametrize("bad", [
    dict(logits=0), dict(scores=0), dict(cu=0), dict(out_scores=0), dict(out_parents=0), dict(out_tokens=0), dict(workspace=0),
    dict(rows=-1), dict(rows=1 << 20), dict(batch=-1), dict(batch=16385), dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(k=0), dict(k=65),
    dict(row_stride=-1), dict(logits=M + 1), dict(logits=M + 2, fp32=1), dict(workspace_bytes=100), dict(workspace=7 * M + 16)], ids=str)
def test_beam_select_refuses(k, bad):
    lib, a = k.load_library(), {**BEAM, **bad}
    assert lib.qk_beam_select(k._BEAM_ARGS.pack(*a.values()), 0) == 1 and lib.qk_last_error()


@pytest.mark.parametrize("bad", [
    dict(groups=0), dict(shared=0), dict(n_groups=-1), dict(n_groups=1 << 20), dict(q=0), dict(out=0), dict(workspace=0), dict(k_pages=0),
    dict(lens=0), dict(page=24), dict(n_q=33), dict(n_q=8 * 33), dict(rows=-1), dict(max_q=0), dict(scale=0.0), dict(q_row=4100),
    dict(o_head=4), dict(workspace_bytes=8), dict(workspace=272), dict(fp8=1)], ids=str)
def test_shared_attention_refuses(k, bad):
    lib, a = k.load_library(), {**SHARED, **bad}
    assert lib.qk_shared_attention(k._SHARED_ARGS.pack(*a.values()), 0) == 1 and lib.qk_last_error()


def test_null_structs_are_refused(k):
    lib = k.load_library()
    for f in (lib.qk_paged_plan, lib.qk_paged_fork, lib.qk_beam_select, lib.qk_shared_attention):
        assert f(None, 0) == 1 and b"null" in lib.qk_last_error()


def test_workspace_sizes(k):
    lib = k.load_library()
    sizes = [lib.qk_beam_workspace_bytes(r, v, n) for r, v, n in ((0, 1, 1), (4, 32003, 8), (4, 151936, 8), (4, 151936, 64), (128, 151936, 64))]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for bad in ((-1, 100, 8), (1 << 20, 100, 8), (1, 0, 8), (1, 2 << 20, 8), (1, 100, 0), (1, 100, 65)):
        assert lib.qk_beam_workspace_bytes(*bad) == -1
    assert 0 < lib.qk_shared_attention_workspace_bytes(1, 8) <= lib.qk_shared_attention_workspace_bytes(512, 32)
    for bad in ((-1, 8), (1 << 40, 8), (1, 0), (1, 1 << 20)):
        assert lib.qk_shared_attention_workspace_bytes(*bad) == -1


def test_shim_refuses_host_tensors(k):
    o = k.DecodeOps(k.load_library())
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)   # noqa: E731
    pages = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA device"):
        o.paged_plan(i(4), i(2), i(2), i(2, 3), i(3), i(2), 16)
    with pytest.raises(RuntimeError, match="CUDA device"):
        o.paged_fork(i(4), i(2), i(2), i(2, 3), i(2, 3), i(2), pages, pages)
    with pytest.raises(RuntimeError, match="CUDA device"):
        o.beam_select(torch.zeros(2, 9), torch.zeros(2), i(2), torch.zeros(1, 4), i(1, 4), i(1, 4))
    x = torch.zeros(2, 32, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA device"):
        o.shared_attention(x, i(3), i(2), i(2, 2), i(2), i(1), pages, pages, x, 0.1, 1)

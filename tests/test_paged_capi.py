"""The paged-serving entry points' host side, without a GPU: bad arguments are refused with a message before anything
is launched, the shim refuses tensors off the GPU, and the rotary tables are the formulas'."""
import math
import os

import pytest
import torch

import model as M


@pytest.fixture(scope="module")
def k():
    import kernels
    if not os.path.exists(kernels.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return kernels


CACHE = dict(k_pages=256, v_pages=256, k_scale=0, v_scale=0, cu=256, lens=256, table=256, batch=2, n_kv=8, pages=10, page=16,
             width=4, stride=4, fp8=0)
QKV = dict(qkv=256, q_out=256, k_out=0, q_norm=0, k_norm=0, cos=256, sin=256, rows=3, n_q=32, qkv_stride=6144, q_stride=4096,
           k_stride=0, max_pos=64, half=64, interleaved=0, eps=1e-6)
READ = dict(starts=0, k_out=256, v_out=256, rows=3, row=1024, head=128)
ATT = dict(q=256, k=256, v=256, out=256, workspace=256, rows=3, n_q=32, max_q=1, q_row=4096, q_head=128, kv_row=1024,
           kv_head=128, o_row=4096, o_head=128, workspace_bytes=1 << 40, scale=0.1)
BAD_CACHE = [dict(k_pages=0), dict(v_pages=0), dict(cu=0), dict(table=0), dict(fp8=1), dict(page=24), dict(page=8), dict(page=256),
             dict(pages=0), dict(n_kv=0), dict(batch=-1), dict(pages=1 << 30), dict(width=0), dict(stride=3), dict(k_pages=264),
             dict(width=1 << 28, stride=1 << 28), dict(n_kv=1 << 40), dict(batch=1 << 33)]


@pytest.mark.parametrize("bad", BAD_CACHE + [
    dict(qkv=0), dict(q_out=0), dict(cos=0), dict(lens=0), dict(q_norm=256), dict(rows=-1), dict(n_q=0), dict(half=4), dict(half=72),
    dict(half=12), dict(max_pos=0), dict(qkv_stride=6000), dict(q_stride=100), dict(k_out=256, k_stride=8), dict(qkv_stride=6148),
    dict(q_out=264), dict(sin=260)], ids=str)
def test_paged_qkv_refuses(k, bad):
    lib, a = k.load_library(), {**CACHE, **QKV, **bad}
    assert lib.qk_paged_qkv(k._QKV_ARGS.pack(*a.values()), 0) == 1 and lib.qk_last_error()


@pytest.mark.parametrize("bad", BAD_CACHE + [dict(k_out=0), dict(v_out=264), dict(rows=-1), dict(row=64), dict(head=64), dict(row=1028),
                                             dict(head=132)], ids=str)
def test_paged_kv_read_refuses(k, bad):
    lib, a = k.load_library(), {**CACHE, **READ, **bad}
    assert lib.qk_paged_kv_read(k._READ_ARGS.pack(*a.values()), 0) == 1 and lib.qk_last_error()


BAD_ATT = [dict(q=0), dict(out=0), dict(workspace=0), dict(rows=-1), dict(rows=1 << 40), dict(n_q=0), dict(n_q=33), dict(n_q=8 * 33),
           dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(max_q=0), dict(q=264), dict(q_row=4100),
           dict(o_head=4), dict(o_row=-8), dict(workspace_bytes=8), dict(workspace=272)]


@pytest.mark.parametrize("bad", BAD_CACHE + BAD_ATT + [dict(lens=0)], ids=str)
def test_paged_attention_refuses(k, bad):
    lib, a = k.load_library(), {**CACHE, **ATT, **bad}
    assert lib.qk_paged_attention(k._ATTENTION_ARGS.pack(*a.values()), 0) == 1 and lib.qk_last_error()


@pytest.mark.parametrize("bad", BAD_ATT + [dict(k=0), dict(v=0), dict(cu=0), dict(batch=-1), dict(n_kv=0), dict(k=264), dict(kv_row=1028),
                                           dict(kv_head=-8)], ids=str)
def test_packed_attention_refuses(k, bad):
    lib, a = k.load_library(), {**CACHE, **ATT, **bad}
    assert lib.qk_packed_attention(k._ATTENTION_ARGS.pack(*a.values()), 0) == 1 and lib.qk_last_error()


def test_null_structs_are_refused(k):
    lib = k.load_library()
    for f in (lib.qk_paged_qkv, lib.qk_paged_kv_read, lib.qk_paged_attention, lib.qk_packed_attention):
        assert f(None, 0) == 1 and b"null" in lib.qk_last_error()


def test_shim_refuses_host_tensors(k):
    o = k.DecodeOps(k.load_library())
    x = torch.zeros(2, 48, 128, dtype=torch.bfloat16)
    pages, cu, table = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16), torch.tensor([0, 2], dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device"):
        o.paged_attention(x[:, :32], cu, cu[1:], table, pages, pages, x[:, :32], 0.1, 2)
    with pytest.raises(RuntimeError, match="CUDA device"):
        o.packed_attention(x[:, :32], x[:, 32:40], x[:, 40:], cu, x[:, :32], 0.1, 2)


@pytest.mark.parametrize("rot", [16, 64, 96, 128])
def test_rope_angles(rot):
    cos, sin = M.rope_angles(300, rot, 1e6, "cpu")
    assert cos.shape == sin.shape == (300, rot // 2) and cos.dtype == torch.float32
    for p, i in ((0, 0), (1, 0), (299, 0), (299, rot // 2 - 1), (123, rot // 4)):
        a = p * 1e6 ** (-2 * i / rot)
        assert abs(cos[p, i].item() - math.cos(a)) < 1e-6 and abs(sin[p, i].item() - math.sin(a)) < 1e-6
    lin, _ = M.rope_angles(300, rot, 1e6, "cpu", {"type": "linear", "factor": 2.0})
    assert torch.equal(lin[::2], cos[:150])
    f, n = 4.0, 100
    y, ys = M.rope_angles(300, rot, 1e6, "cpu", {"type": "yarn", "factor": f, "original_max_position": n})
    mul = 0.1 * math.log(f) + 1
    for p, i in ((1, 0), (299, rot // 2 - 1), (77, rot // 8), (200, 2)):
        w = 1e6 ** (-2 * i / rot)
        keep = min(1.0, max(0.0, (n * w / (2 * math.pi) - 1) / 31))
        a = p * (w * keep + w / f * (1 - keep))
        assert abs(y[p, i].item() - mul * math.cos(a)) < 2e-6 and abs(ys[p, i].item() - mul * math.sin(a)) < 2e-6
    for bad in (dict(type="other", factor=2.0), dict(type="linear", factor=0.5), dict(type="yarn", factor=math.nan)):
        with pytest.raises(ValueError):
            M.rope_angles(8, rot, 1e6, "cpu", bad)
    for r in (8, 24, 144):
        with pytest.raises(ValueError):
            M.rope_angles(8, r, 1e6, "cpu")

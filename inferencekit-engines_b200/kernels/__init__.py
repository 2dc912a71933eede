"""Loads the B200 decode kernels (C ABI, libqwen3_b200.so) and exposes them under the reference's op names.

Drop-in for the reference's `kernels.ops()` (qwen3-8b-fp8_rtx-5090/kernels/__init__.py:11-24), whose pybind11
module exports fp8_gemv, attention, lm_head_argmax, embed, finalize, set_pdl and set_timeline
(kernels/decode.cu:822-830). The methods below take the same positional arguments in the same order and
launch on torch's current CUDA stream without a host sync, so `Engine.decode_step` can be captured into a
CUDA graph exactly as before. There is no fallback: if the library is missing or the device is not an
sm_100 GPU, `ops()` raises.

Differences a caller must know:
  * FP8 weights must be in `model.pack_fp8` layout (the B200 kernels' tile order). `pack_fp8` returns a
    `PackedFP8` tensor (`PackedFP8Pairs` for gate|up); `fp8_gemv` and the FP8 `lm_head_argmax` raise
    RuntimeError for any other tensor, e.g. weights in the reference's `tile_fp8` layout (convert those
    with `model.pack_reference_tiled`). `depth` maps to ring stages per warp, `warps` to warps per CTA,
    `pre` to ring stages issued before waiting on the previous kernel. `kmajor` must be 0 or 1 and `trig`
    must be -1 or a K block in [0, K/128), as in the reference; neither changes anything here (the layout
    is fixed by the tag, and every kernel lets its successor launch right after its own wait).
  * Scales may be 128x128 blocks [N/128, K/128] or per output channel [N]; the layout is read off the
    tensor's shape.
  * `lm_head_argmax` also takes an FP8 head: pass `w_scale=` (fp32 [V]) with packed fp8 weights.
  * The split-K scratch of the GEMV is owned by this object (allocated on first use per device, before any
    graph capture when the engine warms up eagerly).
"""
from __future__ import annotations

import ctypes
import os
import struct

import torch

_here = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_here, "libqwen3_b200.so")

GEMV_QKV, GEMV_O, GEMV_GATE_UP, GEMV_DOWN = 0, 1, 2, 3
GEMV_PARTIAL, GEMV_QKV_RESADD, GEMV_GATE_UP_RESADD = 5, 6, 7
SCALE_BLOCK128, SCALE_CHANNEL = 0, 1

_VP, _I, _F, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong
_SIGS = {
    "qk_version": ([], _I),
    "qk_last_error": ([], ctypes.c_char_p),
    "qk_set_pdl": ([_I], _I),
    "qk_set_timeline": ([_VP, _I], _I),
    "qk_get_device_error": ([ctypes.POINTER(_I), _VP], _I),
    "qk_wait_probe": ([_I, _VP, ctypes.c_ulonglong, _VP, _VP], _I),
    "qk_fp8_gemv": ([_I, _VP, _VP, _I, _VP, _VP, _VP, _VP, _VP, _I, _I, _F, _VP, _VP, _I, _I, _I, _I, _I, _VP], _I),
    "qk_attention": ([_VP] * 12 + [_I, _I, _I, _I, _I, _I, _F, _F, _I, _VP], _I),
    "qk_lm_head_argmax": ([_VP, _VP, _I, _VP, _VP, _VP, _VP, _I, _I, _F, _VP, _VP, _I, _VP], _I),
    "qk_embed": ([_VP, _VP, _VP, _I, _I, _VP], _I),
    "qk_decode_step": ([_VP, _I, _VP, _VP, ctypes.c_longlong, _VP, _VP, _VP, _VP, _I, _VP, _VP, _VP, _VP, _VP, _I,
                        _VP, _VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_longlong, _VP, _I, _VP, _VP, _VP, _VP, _I, _I,
                        _F, _I, _VP, _VP], _I),
    "qk_decode_step_tp": ([_VP, _I, _VP, _VP, ctypes.c_longlong, _VP, _VP, _VP, _VP, _I, _VP, _VP, _VP, _VP, _VP,
                           _I, _VP, _VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_longlong, _VP, _I, _VP, _VP, _VP, _VP,
                           _I, _I, _F, _VP, _VP, _I, _VP, _VP], _I),
    "qk_tp_area_bytes": ([], ctypes.c_longlong),
    "qk_tp_area_alloc": ([ctypes.POINTER(_VP), _VP], _I),
    "qk_tp_area_open": ([_VP, ctypes.POINTER(_VP)], _I),
    "qk_tp_area_close": ([_VP], _I),
    "qk_tp_area_free": ([_VP], _I),
    "qk_tp_area_reset": ([_VP, _VP], _I),
    "qk_residual_add": ([_VP, _VP, _I, _VP], _I),
    "qk_argmax_key_flip": ([_VP, _I, _VP], _I),
    "qk_decode_step_part_floats": ([_I], ctypes.c_longlong),
    "qk_decode_step_counters": ([_I], _I),
    "qk_fp8_gemv_noalloc": ([_I, _VP, _VP, _I, _VP, _VP, _VP, _VP, _VP, _I, _I, _F, _VP], _I),
    "qk_finalize": ([_VP, _VP, _VP, _VP, _I, _I, _VP], _I),
    "qk_fp8_gemm_rows_scratch_bytes": ([_I, _I, _I], ctypes.c_longlong),
    "qk_fp8_gemm_rows": ([_VP, _VP, _I, _I, _VP, _VP, _I, _I, _F, _VP, _VP, ctypes.c_longlong, _VP], _I),
    "qk_fp8_gemm_tiles": ([_VP, _VP, _I, _I, _VP, _VP, _I, _I, _F, _VP, _VP, ctypes.c_longlong, _VP], _I),
    "qk_attention_fp8kv": ([_VP] * 13 + [_I, _I, _I, _I, _I, _I, _F, _F, _VP], _I),
    "qk_embed_rows": ([_VP, _I, _VP, _I, _VP, _VP], _I),
    "qk_prefill_qkv": ([_VP, _I, _I, _I, _I, _VP, _VP, _VP, _VP, _F, _VP, _VP, _I, _VP, _VP], _I),
    "qk_prefill_attention": ([_VP, _I, _I, _I, _I, _VP, _VP, _I, _F, _VP, _VP], _I),
    "qk_add_rows": ([_VP, _VP, ctypes.c_longlong, _VP], _I),
    "qk_swiglu_rows": ([_VP, _I, _I, _VP, _VP], _I),
    "qk_argmax_rows": ([_VP, _I, _I, _VP, _VP], _I),
    "qk_paged_qkv": ([_VP, _VP], _I),
    "qk_paged_kv_read": ([_VP, _VP], _I),
    "qk_ragged_attention_workspace_bytes": ([], _L),
    "qk_paged_attention": ([_VP, _VP], _I),
    "qk_packed_attention": ([_VP, _VP], _I),
    "qk_paged_plan": ([_VP, _VP], _I),
    "qk_paged_fork": ([_VP, _VP], _I),
    "qk_beam_workspace_bytes": ([_L, _L, _L], _L),
    "qk_beam_select": ([_VP, _VP], _I),
    "qk_shared_attention_workspace_bytes": ([_L, _L], _L),
    "qk_shared_attention": ([_VP, _VP], _I),
}


class PackedFP8(torch.Tensor):
    """uint8 weights in the `model.pack_fp8` layout (16-row units of 2 KiB tiles). The type survives
    `.to()`, `.cuda()`, views and slicing, so the ops can tell packed weights from any other fp8/uint8
    tensor of the same size."""


class PackedTiles(torch.Tensor):
    """fp8 [N, K] weights in the `model.pack_fp8_tiles` layout: 128 x 128 tiles, each in the 128-byte-swizzle
    image the tcgen05 linear's MMAs read, tile-major. Keeps its type through `.to()` and views."""


class PackedFP8Pairs(PackedFP8):
    """gate|up weights packed as 16 gate rows + the matching 16 up rows per unit (`pack_fp8(w, pairs=True)`)."""


def check_packed(w, pairs: bool, what: str):
    """Raise RuntimeError unless `w` is a pack_fp8 tensor of the right kind (gate|up pairs or plain)."""
    if not isinstance(w, PackedFP8) or isinstance(w, PackedFP8Pairs) != pairs:
        want = "pack_fp8(w, pairs=True)" if pairs else "pack_fp8(w)"
        got = type(w).__name__ if isinstance(w, PackedFP8) else f"an untagged {getattr(w, 'dtype', type(w))} tensor"
        raise RuntimeError(f"{what}: weights must be in the model.{want} layout, got {got} (weights in the "
                           "reference's tile_fp8 layout convert with model.pack_reference_tiled)")


def load_library(path: str = LIB_PATH) -> ctypes.CDLL:
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is missing: build it with `make -C {os.path.dirname(_here)}` "
                           "(or __graft_entry__.build())")
    lib = ctypes.CDLL(path)
    for name, (args, res) in _SIGS.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    return lib


class QkTpComm(ctypes.Structure):
    """qk_tp_comm_t"""
    _fields_ = [("tp", ctypes.c_int), ("rank", ctypes.c_int), ("areas", ctypes.c_void_p)]


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _launch_stream(what: str, dev: int) -> int:
    """The stream for a call on tensors of GPU `dev`, which has to be the current one: the library launches there; as an
    integer (no stream object, and the bindings behind torch.cuda's functions: the paged calls' host time is their launch)."""
    current = torch._C._cuda_getDevice()
    if current != dev:
        raise RuntimeError(f"{what}: the tensors are on GPU {dev}, the current device is {current}")
    return torch._C._cuda_getCurrentRawStream(dev)


_E4M3 = (torch.float8_e4m3fn, torch.uint8)
_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
# qk_paged_qkv_t, qk_paged_kv_read_t and qk_ragged_attention_t (the first 14 fields of each: qk_paged_cache_t)
_QKV_ARGS, _READ_ARGS, _ATTENTION_ARGS = (struct.Struct(f) for f in ("7Q7q7Q8qd", "7Q7q3Q3q", "7Q7q5Q10qd"))
# qk_paged_plan_t, qk_paged_fork_t, qk_beam_select_t and qk_shared_attention_t
_PLAN_ARGS, _FORK_ARGS, _BEAM_ARGS, _SHARED_ARGS = (struct.Struct(f) for f in ("13Q8q", "12Q10q", "7Q7q", "7Q7q5Q10qd2Qq"))


class DecodeOps:
    """The reference's op set over the C ABI (see module docstring)."""

    TL_SLOT_WORDS = 2048     # u64 words per launch in a timeline buffer (256 CTAs x 8 stamps)

    def __init__(self, lib: ctypes.CDLL):
        self.lib = lib
        self._scratch = {}
        self._outgrown = []          # scratch that larger calls replaced: a captured graph may still run on it
        self.timeline_names = None   # launch names in timeline-slot order while a timeline is set

    # ---- helpers ------------------------------------------------------------------------------------------
    def _check(self, status: int, what: str):
        if status != 0:
            raise RuntimeError(f"{what}: {self.lib.qk_last_error().decode()}")

    def scratch(self, device: torch.device, part_floats: int, units: int):
        """Split-K scratch for the GEMV on `device` (grown, never shrunk; counters start at zero)."""
        key = device.index if device.index is not None else torch.cuda.current_device()
        part, counters = self._scratch.get(key, (None, None))
        if part is None or part.numel() < part_floats or counters.numel() < units:
            n_part = max(part_floats, 0 if part is None else part.numel())
            n_cnt = max(units, 0 if counters is None else counters.numel())
            if part is not None:
                self._outgrown.append((part, counters))
            part = torch.empty(n_part, dtype=torch.float32, device=device)
            counters = torch.zeros(n_cnt, dtype=torch.int32, device=device)
            self._scratch[key] = (part, counters)
        return part, counters

    def reset_scratch(self):
        """Zero the counters of every scratch and workspace of this object's, after a failed launch and with none in flight."""
        for s in [*self._scratch.values(), *self._outgrown]:
            (s[1] if isinstance(s, tuple) else s).zero_()   # the GEMV's (block dots, unit counters); a whole buffer

    def device_error(self) -> int:
        """Read and clear the device error word (bounded waits that gave up, bad state)."""
        v = ctypes.c_int(0)
        self._check(self.lib.qk_get_device_error(ctypes.byref(v), _stream()), "qk_get_device_error")
        return v.value

    # ---- the reference's ops -----------------------------------------------------------------------------
    def set_pdl(self, on: bool):
        self._check(self.lib.qk_set_pdl(int(bool(on))), "set_pdl")

    def set_timeline(self, buf=None):
        """buf: zeroed int64 CUDA tensor of n_slots * 2048 words, or None to disable. Launch i after this
        call stamps slot i (layout in include/qwen3_b200.h); `timeline_names[i]` names it."""
        n = 0 if buf is None else buf.numel() // self.TL_SLOT_WORDS
        self._check(self.lib.qk_set_timeline(_p(buf), n), "set_timeline")
        self.timeline_names = None if buf is None else []

    def _tl(self, name):
        if self.timeline_names is not None:
            self.timeline_names.append(name)

    def fp8_gemv(self, kind, w, ws, x, norm_w, out, N, eps, depth=0, warps=0, pre=-1, trig=-1, kmajor=1,
                 resadd=None, resid_out=None, stage_tiles=0, ctas_per_sm=0):
        N = int(N)
        check_packed(w, int(kind) in (GEMV_GATE_UP, GEMV_GATE_UP_RESADD), "fp8_gemv")
        K = w.numel() // N
        if int(kmajor) not in (0, 1):
            raise RuntimeError(f"fp8_gemv: kmajor must be 0 or 1, got {kmajor}")
        if int(trig) != -1 and not 0 <= int(trig) < K // 128:
            raise RuntimeError(f"fp8_gemv: trig must be -1 or a K block in [0, {K // 128}), got {trig}")
        scale_mode = SCALE_CHANNEL if ws.dim() == 1 else SCALE_BLOCK128
        part, counters = self.scratch(w.device, N * K // 128, N // 8)
        st = self.lib.qk_fp8_gemv(int(kind), _p(w), _p(ws), scale_mode, _p(x), _p(norm_w), _p(resadd),
                                  _p(resid_out), _p(out), N, K, float(eps), _p(part), _p(counters),
                                  int(warps), int(depth), int(stage_tiles), int(pre), int(ctas_per_sm), _stream())
        self._check(st, "fp8_gemv")
        self._tl(f"gemv{int(kind)}")

    def attention(self, qkv, q_norm_w, k_norm_w, cos_tab, sin_tab, state, k_cache, v_cache, o_part, ml_part,
                  counters, out, scale, eps, late_trigger=0, chunk=64, batch=None, state_stride=2):
        """k_cache/v_cache: one layer, [n_kv, max_seq, 128] (batch 1, as the reference) or
        [batch, n_kv, max_seq, 128]."""
        if k_cache.dim() == 3:
            b, n_kv, max_seq = 1, k_cache.shape[0], k_cache.shape[1]
        else:
            b, n_kv, max_seq = k_cache.shape[0], k_cache.shape[1], k_cache.shape[2]
        if batch is not None:
            b = batch
        max_splits = o_part.shape[-2]
        qkv_stride = qkv.shape[-1] if qkv.dim() > 1 else qkv.numel()
        st = self.lib.qk_attention(_p(qkv), _p(q_norm_w), _p(k_norm_w), _p(cos_tab), _p(sin_tab), _p(state),
                                   _p(k_cache), _p(v_cache), _p(o_part), _p(ml_part), _p(counters), _p(out),
                                   b, n_kv, max_seq, max_splits, qkv_stride, int(state_stride), float(scale),
                                   float(eps), int(chunk), _stream())
        self._check(st, "attention")
        self._tl("attention")

    def attention_fp8kv(self, qkv, q_norm_w, k_norm_w, cos_tab, sin_tab, state, k_cache, k_scale, v_cache, v_scale,
                        o_part, ml_part, out, scale, eps, batch=None, state_stride=2):
        """Decode attention over an FP8 KV cache (e4m3 rows + one fp32 scale per row), 64-key splits.
        k_cache/v_cache: one layer, uint8 or float8_e4m3fn [n_kv, max_seq, 128] (batch 1) or
        [batch, n_kv, max_seq, 128]; k_scale/v_scale: fp32 [n_kv, max_seq] or [batch, n_kv, max_seq]."""
        if k_cache.dim() == 3:
            b, n_kv, max_seq = 1, k_cache.shape[0], k_cache.shape[1]
        else:
            b, n_kv, max_seq = k_cache.shape[0], k_cache.shape[1], k_cache.shape[2]
        if batch is not None:
            b = batch
        if k_cache.element_size() != 1 or v_cache.element_size() != 1 or k_scale.dtype != torch.float32:
            raise RuntimeError("attention_fp8kv: caches must be 1-byte e4m3 rows, scales fp32")
        max_splits = o_part.shape[-2]
        qkv_stride = qkv.shape[-1] if qkv.dim() > 1 else qkv.numel()
        st = self.lib.qk_attention_fp8kv(_p(qkv), _p(q_norm_w), _p(k_norm_w), _p(cos_tab), _p(sin_tab), _p(state),
                                         _p(k_cache), _p(k_scale), _p(v_cache), _p(v_scale), _p(o_part), _p(ml_part),
                                         _p(out), b, n_kv, max_seq, max_splits, qkv_stride, int(state_stride),
                                         float(scale), float(eps), _stream())
        self._check(st, "attention_fp8kv")

    def lm_head_argmax(self, w, x, norm_w, logits, best, eps, ctas=0, w_scale=None, row_offset=0):
        V = logits.numel()
        fp8 = w_scale is not None
        part = counters = None
        if fp8:
            check_packed(w, False, "lm_head_argmax")
            part, counters = self.scratch(w.device, V * 4096 // 128, V // 8)
        elif w.dtype != torch.bfloat16 or isinstance(w, PackedFP8):
            raise RuntimeError("lm_head_argmax: a bf16 [V, 4096] head, or packed fp8 weights with w_scale=")
        st = self.lib.qk_lm_head_argmax(_p(w), _p(w_scale), int(fp8), _p(x), _p(norm_w), _p(logits), _p(best), V,
                                        int(row_offset), float(eps), _p(part), _p(counters), int(ctas), _stream())
        self._check(st, "lm_head_argmax")
        self._tl("lm_head")

    def decode_step(self, layer_table, n_layers, k_cache, v_cache, embed, final_norm, w_head, s_head, cos_tab,
                    sin_tab, token, state, out_tokens, best, resid, qkv, attn, h, logits, part, counters, o_part,
                    ml_part, attn_counters, sync, max_seq, eps, scale_mode, timeline=None):
        """The fused decode step (qk_decode_step): one launch per token. layer_table: int64 CUDA tensor
        [n_layers, 12] of device pointers in qk_layer_t order; k_cache/v_cache: bf16 [n_layers, 1, 8, max_seq, 128]
        (a layer stride of any multiple of 16 bytes); timeline: optional int64 CUDA tensor of
        #SMs * (5*n_layers + 1) * 24 words (layout in include/qwen3_b200.h)."""
        if k_cache.stride() != v_cache.stride() or k_cache.shape[-2] != max_seq or k_cache.shape[-1] != 128:
            raise ValueError("k_cache/v_cache must be [layers, 1, 8, max_seq, 128] with equal strides")
        if s_head is not None:
            check_packed(w_head, False, "decode_step")
        elif w_head.dtype != torch.bfloat16:
            raise RuntimeError("decode_step: without s_head the head must be bf16 [vocab, 4096]")
        stride = k_cache.stride(0) * k_cache.element_size()
        st = self.lib.qk_decode_step(_p(layer_table), int(n_layers), _p(k_cache), _p(v_cache), stride, _p(embed),
                                     _p(final_norm), _p(w_head),
                                     _p(s_head), embed.shape[0], _p(cos_tab), _p(sin_tab), _p(token), _p(state),
                                     _p(out_tokens), out_tokens.numel(), _p(best), _p(resid), _p(qkv), _p(attn), _p(h),
                                     _p(logits), _p(part), part.numel(), _p(counters), counters.numel(), _p(o_part),
                                     _p(ml_part), _p(attn_counters), _p(sync), int(max_seq), o_part.shape[-2],
                                     float(eps), int(scale_mode), _p(timeline), _stream())
        self._check(st, "decode_step")

    def decode_step_tp(self, layer_table, n_layers, k_cache, v_cache, embed, final_norm, w_head, s_head, cos_tab,
                       sin_tab, token, state, out_tokens, best, resid, qkv, attn, h, logits, part, counters, o_part,
                       ml_part, attn_counters, sync, max_seq, eps, resid_alt, vocab_offset, comm, timeline=None):
        """The fused tensor-parallel step of one rank (qk_decode_step_tp); comm: a `TPComm` (areas exchanged)."""
        stride = k_cache.stride(0) * k_cache.element_size()
        st = self.lib.qk_decode_step_tp(_p(layer_table), int(n_layers), _p(k_cache), _p(v_cache), stride, _p(embed),
                                        _p(final_norm), _p(w_head), _p(s_head), logits.numel(), _p(cos_tab),
                                        _p(sin_tab), _p(token), _p(state), _p(out_tokens), out_tokens.numel(),
                                        _p(best), _p(resid), _p(qkv), _p(attn), _p(h), _p(logits), _p(part),
                                        part.numel(), _p(counters), counters.numel(), _p(o_part), _p(ml_part),
                                        _p(attn_counters), _p(sync), int(max_seq), o_part.shape[-2], float(eps),
                                        _p(timeline), _p(resid_alt), int(vocab_offset), ctypes.byref(comm),
                                        _stream())
        self._check(st, "decode_step_tp")

    def tp_area_alloc(self):
        """A zeroed TP area on the current device and its 64-byte CUDA IPC handle (bytes)."""
        area = ctypes.c_void_p()
        handle = ctypes.create_string_buffer(64)
        self._check(self.lib.qk_tp_area_alloc(ctypes.byref(area), handle), "tp_area_alloc")
        return area.value, handle.raw

    def tp_area_open(self, handle: bytes):
        peer = ctypes.c_void_p()
        buf = ctypes.create_string_buffer(handle, 64)
        self._check(self.lib.qk_tp_area_open(buf, ctypes.byref(peer)), "tp_area_open")
        return peer.value

    def tp_area_close(self, peer):
        self._check(self.lib.qk_tp_area_close(ctypes.c_void_p(peer)), "tp_area_close")

    def tp_area_free(self, area):
        self._check(self.lib.qk_tp_area_free(ctypes.c_void_p(area)), "tp_area_free")

    def tp_area_reset(self, area):
        """Zero this rank's own TP area on the current stream (recovery after a failed step)."""
        self._check(self.lib.qk_tp_area_reset(ctypes.c_void_p(area), _stream()), "tp_area_reset")

    def residual_add(self, resid, sum_f32):
        """resid = bf16(resid + bf16(sum)) (after the all-reduce of a row-parallel partial)."""
        self._check(self.lib.qk_residual_add(_p(resid), _p(sum_f32), resid.numel(), _stream()), "residual_add")

    def argmax_key_flip(self, keys):
        """Unsigned <-> signed order of packed argmax keys (int64 tensor), in place."""
        self._check(self.lib.qk_argmax_key_flip(_p(keys), keys.numel(), _stream()), "argmax_key_flip")

    def embed(self, token, table, resid):
        b = token.numel()
        self._check(self.lib.qk_embed(_p(token), _p(table), _p(resid), table.shape[0], b, _stream()), "embed")

    def gemm_scratch(self, device, rows: int, shapes) -> torch.Tensor:
        """A scratch for fp8_gemm_rows calls of up to `rows` rows and weights of any of these (N, K) shapes (zeroed once;
        every call leaves it ready for the next). Calls that may run at the same time need one each."""
        need = [self.lib.qk_fp8_gemm_rows_scratch_bytes(rows, N, K) for N, K in shapes]
        if not need or min(need) < 0:
            raise RuntimeError(f"gemm_scratch: unsupported rows={rows} or shapes {list(shapes)}")
        return torch.zeros(max(need), dtype=torch.uint8, device=device)

    def fp8_gemm_rows(self, x, w, w_scale, out, norm_w=None, eps=1e-6, scratch=None):
        """Batched FP8 linear on the tcgen05 tensor cores: out[m] = bf16 W8A8 linear of x[m] (optionally
        RMS-normalised with norm_w first), for M = 1..128 rows (K <= 12288 above 64). x bf16 [M, K]; w fp8 [N, K],
        either a plain row-major matrix (read through TMA boxes) or a `PackedTiles` tensor from
        `model.pack_fp8_tiles` (read as contiguous tiles; not the GEMV's pack_fp8 layout); w_scale fp32 [N] or
        [N/128, K/128]; out bf16 [M, N]. scratch: from gemm_scratch; by default this object's own, one per device, which
        every caller without one shares."""
        tiles = isinstance(w, PackedTiles)
        if (isinstance(w, PackedFP8) or w.dtype != torch.float8_e4m3fn or w.dim() != 2 or not w.is_contiguous()):
            raise RuntimeError("fp8_gemm_rows: w must be a row-major float8_e4m3fn [N, K] matrix or "
                               "model.pack_fp8_tiles(w) (not pack_fp8)")
        M, K = x.shape
        N = w.shape[0]
        nbytes = self.lib.qk_fp8_gemm_rows_scratch_bytes(M, N, K)
        if nbytes < 0:
            raise RuntimeError(f"fp8_gemm_rows: unsupported shape M={M} N={N} K={K} (M 1..128; N, K multiples of "
                               "128; K at most 16384, or 12288 above 64 rows)")
        sc = scratch
        if sc is None:
            key = ("gemm", x.device.index if x.device.index is not None else torch.cuda.current_device())
            sc = self._scratch.get(key)
            if sc is None or sc.numel() < nbytes:
                if sc is not None:
                    self._outgrown.append(sc)
                sc = self._scratch[key] = torch.zeros(nbytes, dtype=torch.uint8, device=x.device)
        elif sc.dtype != torch.uint8 or sc.device != x.device or not sc.is_contiguous() or sc.numel() < nbytes:
            raise RuntimeError(f"fp8_gemm_rows: scratch must come from gemm_scratch() for these rows, on x's device ({nbytes} bytes)")
        scale_mode = SCALE_CHANNEL if w_scale.dim() == 1 else SCALE_BLOCK128
        fn = self.lib.qk_fp8_gemm_tiles if tiles else self.lib.qk_fp8_gemm_rows
        st = fn(_p(x), _p(norm_w), M, K, _p(w), _p(w_scale), scale_mode, N, float(eps), _p(out), _p(sc), sc.numel(),
                _stream())
        self._check(st, "fp8_gemm_rows")

    def embed_rows(self, tokens, table, out):
        """out[m] = table[tokens[m]] for the chunk's int32 tokens [M]; out bf16 [M, H]."""
        M = tokens.numel()
        self._check(self.lib.qk_embed_rows(_p(tokens), M, _p(table), table.shape[0], _p(out), _stream()),
                    "embed_rows")

    def prefill_qkv(self, qkv, p0, q_norm, k_norm, cos, sin, eps, k_cache, v_cache, q_out):
        """Per-head RMSNorm + RoPE of the chunk's q and k rows (positions p0 .. p0+M-1), K and V appended to
        one layer's cache [n_kv, max_seq, 128]; q_out bf16 [M, n_q, 128]."""
        M = qkv.shape[0]
        n_kv, max_seq = k_cache.shape[0], k_cache.shape[1]
        n_q = q_out.shape[1]
        st = self.lib.qk_prefill_qkv(_p(qkv), M, int(p0), n_q, n_kv, _p(q_norm), _p(k_norm), _p(cos), _p(sin),
                                     float(eps), _p(k_cache), _p(v_cache), max_seq, _p(q_out), _stream())
        self._check(st, "prefill_qkv")

    def prefill_attention(self, q, p0, k_cache, v_cache, scale, out):
        """Causal GQA attention of the chunk's queries q [M, n_q, 128] over cache rows 0 .. p0+m; out bf16
        [M, n_q * 128] (or [M, n_q, 128])."""
        M, n_q = q.shape[0], q.shape[1]
        n_kv, max_seq = k_cache.shape[0], k_cache.shape[1]
        st = self.lib.qk_prefill_attention(_p(q), M, int(p0), n_q, n_kv, _p(k_cache), _p(v_cache), max_seq,
                                           float(scale), _p(out), _stream())
        self._check(st, "prefill_attention")

    def add_rows(self, resid, y):
        """resid = bf16(resid + y), elementwise."""
        self._check(self.lib.qk_add_rows(_p(resid), _p(y), resid.numel(), _stream()), "add_rows")

    def swiglu_rows(self, gu, h):
        """h[m] = bf16(bf16(silu(gate)) * up) for gu = [gate | up] rows [M, 2I]; h [M, I]."""
        M, I = h.shape
        self._check(self.lib.qk_swiglu_rows(_p(gu), M, I, _p(h), _stream()), "swiglu_rows")

    def argmax_rows(self, logits, best):
        """best[r] = packed argmax key of bf16 logits row r ([rows, V]; ties to the lowest index)."""
        rows, V = logits.shape
        self._check(self.lib.qk_argmax_rows(_p(logits), rows, V, _p(best), _stream()), "argmax_rows")

    # ---- serving from a paged KV cache ---------------------------------------------------------------------
    # A ragged batch: sequence b owns rows cu[b] .. cu[b+1]-1 (int32 [B+1]) and ends, with them, at length seq_lens[b]
    # (int32 [B]); its position p lies in slot p % page_size of page block_table[b, p // page_size] (int32 [B, width], the
    # rows any distance of at least `width` apart, or one row for all: an expanded table).
    # k_pages/v_pages: bf16 [pages, n_kv, page_size, 128], or e4m3 (uint8 or float8_e4m3fn) with fp32 row scales
    # k_scale/v_scale [pages, n_kv, page_size]; page_size 16, 32, 64 or 128. Lengths and tables live on the device
    # (the calls can be captured); a position or page outside them sets the device error word and is not written.
    # The arguments go to the library as one packed struct: a ctypes call with 30 arguments costs more host time
    # than the launch.
    @staticmethod
    def _paged(what, k_pages, v_pages, k_scale, v_scale, cu, lens, block_table):
        """Check the cache and the batch (lens None: none wanted); returns (B, n_kv, device index, the fields of
        qk_paged_cache_t)."""
        dev = k_pages.get_device()
        shape, dt = k_pages.shape, k_pages.dtype
        if len(shape) != 4 or shape != v_pages.shape or not (k_pages.is_contiguous() and v_pages.is_contiguous()):
            raise RuntimeError(f"{what}: k_pages and v_pages must be contiguous [pages, n_kv, page_size, 128]")
        pages, n_kv, page, hd = shape
        if hd != 128 or v_pages.dtype is not dt or (dt is not _BF16 and dt not in _E4M3):
            raise RuntimeError(f"{what}: pages must be bf16, or e4m3 bytes (uint8 or float8_e4m3fn), 128 values per row")
        ks = vs = fp8 = 0
        if dt is not _BF16:
            for s in (k_scale, v_scale):
                if s is None or s.dtype is not _F32 or s.shape != shape[:3] or not s.is_contiguous() or s.get_device() != dev:
                    raise RuntimeError(f"{what}: an e4m3 cache needs contiguous fp32 k_scale and v_scale [pages, n_kv, page_size]")
            ks, vs, fp8 = k_scale.data_ptr(), v_scale.data_ptr(), 1
        elif k_scale is not None or v_scale is not None:
            raise RuntimeError(f"{what}: a bf16 cache has no row scales")
        if cu.dtype is not _I32 or block_table.dtype is not _I32 or block_table.dim() != 2 or cu.dim() != 1 or not cu.is_contiguous():
            raise RuntimeError(f"{what}: cu must be int32 [B+1] and block_table int32 [B, width]")
        B, width = block_table.shape
        stride, inner = block_table.stride()
        if inner != 1 and width > 1:
            raise RuntimeError(f"{what}: block_table rows must be contiguous")
        if cu.numel() != B + 1:
            raise RuntimeError(f"{what}: cu has {cu.numel()} entries for {B} sequences (B + 1 wanted)")
        if dev < 0 or v_pages.get_device() != dev or cu.get_device() != dev or block_table.get_device() != dev:
            raise RuntimeError(f"{what}: every tensor must be on the same CUDA device")
        lens_ptr = 0
        if lens is not None:
            if lens.dtype is not _I32 or lens.dim() != 1 or lens.numel() != B or lens.get_device() != dev or not lens.is_contiguous():
                raise RuntimeError(f"{what}: seq_lens must be int32 [{B}] on the cache's device")
            lens_ptr = lens.data_ptr()
        return B, n_kv, dev, (k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, cu.data_ptr(), lens_ptr, block_table.data_ptr(),
                              B, n_kv, pages, page, width, stride if B > 1 else width, fp8)

    @staticmethod
    def _heads(what, name, t, dev):
        """(rows, heads, row stride, head stride) of a bf16 [rows, heads, 128] or [rows, heads * 128] tensor."""
        shape, strides = t.shape, t.stride()
        if t.dtype is _BF16 and t.get_device() == dev and strides[-1] == 1:
            if len(shape) == 3 and shape[2] == 128:
                return shape[0], shape[1], strides[0], strides[1]
            if len(shape) == 2 and shape[1] % 128 == 0:
                return shape[0], shape[1] // 128, strides[0], 128
        raise RuntimeError(f"{what}: {name} must be bf16 [rows, heads, 128] or [rows, heads * 128] on the call's device, the "
                           "last dimension contiguous")

    def attention_workspace(self, device) -> torch.Tensor:
        """A workspace for paged_attention and packed_attention on `device` (zeroed once; every call leaves it
        ready for the next). Calls that may run at the same time, on two streams, need one each."""
        return torch.zeros(self.lib.qk_ragged_attention_workspace_bytes(), dtype=torch.uint8, device=device)

    def _workspace(self, what, ws, dev, stream, maker="attention_workspace", nbytes=0):
        if ws is None:   # one per device and stream, kept; never a graph's, whose replays may run beside the stream's calls
            if stream and torch._C._cuda_isCurrentStreamCapturing():   # (stream 0 cannot be captured)
                raise RuntimeError(f"{what}: pass workspace={maker}(device), made before the capture")
            key = ("ragged" if maker == "attention_workspace" else maker, dev, stream)
            ws = self._scratch.get(key)
            if ws is None or ws.numel() < nbytes:
                # (no graph runs on an outgrown one, and the stream's calls are done with it before its memory is given out again: dropped,
                # and replaced by half as much again, so that slowly growing calls replace few)
                dest, grown = torch.device("cuda", dev), 0 if ws is None else ws.numel() * 3 // 2
                ws = self._scratch[key] = torch.zeros(max(nbytes, grown), dtype=torch.uint8, device=dest) if nbytes else self.attention_workspace(dest)
        elif ws.dtype is not torch.uint8 or ws.get_device() != dev or not ws.is_contiguous():
            raise RuntimeError(f"{what}: workspace must come from {maker}() on the call's device")
        return ws

    def paged_qkv(self, qkv, cu, seq_lens, block_table, k_pages, v_pages, q_out, cos, sin, q_norm=None, k_norm=None,
                  eps=1e-6, interleaved=False, k_scale=None, v_scale=None, k_out=None):
        """The qkv projection's rows [T, (n_q + 2 n_kv) * 128] (bf16, any row stride): per-head RMSNorm with q_norm/k_norm
        (bf16 [128], both or neither), rotary positions, q to q_out ([T, n_q, 128]), K and V rows into their
        sequences' pages (quantised per row for an e4m3 cache). cos/sin: fp32 [max_pos, r / 2] (`model.rope_angles`);
        the first r dims of a head turn, in pairs (i, i + r/2) or, interleaved, (2i, 2i + 1). k_out [T, n_kv, 128]
        also takes the keys before quantisation (for `packed_attention` over the same rows). fp32 inside, one
        rounding. Rows past cu[B] are left alone."""
        B, n_kv, dev, cache = self._paged("paged_qkv", k_pages, v_pages, k_scale, v_scale, cu, seq_lens, block_table)
        T, n_q, q_row, q_head = self._heads("paged_qkv", "q_out", q_out, dev)
        w = (n_q + 2 * n_kv) * 128
        if qkv.dtype != torch.bfloat16 or qkv.shape != (T, w) or qkv.stride(1) != 1 or qkv.get_device() != dev:
            raise RuntimeError(f"paged_qkv: qkv must be bf16 [{T}, {w}], the last dimension contiguous")
        if q_head != 128:
            raise RuntimeError("paged_qkv: the heads of a q_out row must be contiguous")
        k_row = k_ptr = qn = kn = 0
        if k_out is not None:
            kT, heads, k_row, k_head = self._heads("paged_qkv", "k_out", k_out, dev)
            if (kT, heads, k_head) != (T, n_kv, 128):
                raise RuntimeError(f"paged_qkv: k_out must be [{T}, {n_kv}, 128], the heads of a row contiguous")
            k_ptr = k_out.data_ptr()
        tab = cos.shape
        if cos.dtype != torch.float32 or len(tab) != 2 or tab != sin.shape or sin.dtype != torch.float32 \
                or not (cos.is_contiguous() and sin.is_contiguous()) or cos.get_device() != dev or sin.get_device() != dev:
            raise RuntimeError("paged_qkv: cos and sin must be contiguous fp32 [max_pos, rotary dims / 2] tables")
        if q_norm is not None or k_norm is not None:
            for t in (q_norm, k_norm):
                if t is None or t.dtype != torch.bfloat16 or t.shape != (128,) or t.get_device() != dev or t.stride(0) != 1:
                    raise RuntimeError("paged_qkv: q_norm and k_norm must be bf16 [128], both or neither")
            qn, kn = q_norm.data_ptr(), k_norm.data_ptr()
        if T == 0 or B == 0:
            return
        st = self.lib.qk_paged_qkv(_QKV_ARGS.pack(*cache, qkv.data_ptr(), q_out.data_ptr(), k_ptr, qn, kn, cos.data_ptr(),
                                                  sin.data_ptr(), T, n_q, qkv.stride(0), q_row, k_row, tab[0], tab[1],
                                                  bool(interleaved), eps), _launch_stream("paged_qkv", dev))
        if st:
            self._check(st, "paged_qkv")

    def paged_kv_read(self, cu, block_table, k_pages, v_pages, k_out, v_out, k_scale=None, v_scale=None, starts=None):
        """Positions starts[b] .. (0 without starts, int32 [B]) of each sequence out of the pages: row cu[b] + i of
        k_out and v_out (bf16 [T, n_kv, 128], equal strides, any row and head stride: a contiguous cache's
        [n_kv, max_seq, 128] transposed will do) is position starts[b] + i, dequantised."""
        B, n_kv, dev, cache = self._paged("paged_kv_read", k_pages, v_pages, k_scale, v_scale, cu, None, block_table)
        rows = self._heads("paged_kv_read", "k_out", k_out, dev)
        if rows[1] != n_kv or self._heads("paged_kv_read", "v_out", v_out, dev) != rows:
            raise RuntimeError(f"paged_kv_read: k_out and v_out must be [T, {n_kv}, 128] with equal strides")
        first = 0
        if starts is not None:
            if starts.dtype != torch.int32 or starts.shape != (B,) or starts.get_device() != dev or not starts.is_contiguous():
                raise RuntimeError(f"paged_kv_read: starts must be int32 [{B}] on the cache's device")
            first = starts.data_ptr()
        if rows[0] == 0 or B == 0:
            return
        st = self.lib.qk_paged_kv_read(_READ_ARGS.pack(*cache, first, k_out.data_ptr(), v_out.data_ptr(), rows[0], rows[2],
                                                       rows[3]), _launch_stream("paged_kv_read", dev))
        if st:
            self._check(st, "paged_kv_read")

    def paged_attention(self, q, cu, seq_lens, block_table, k_pages, v_pages, out, scale, max_q, k_scale=None,
                        v_scale=None, workspace=None):
        """Causal attention of each sequence's new tokens over its paged cache, their own rows included (`paged_qkv`
        first): row cu[b] + i sees positions 0 .. seq_lens[b] - n_b + i of sequence b; a row that sees none gives zeros.
        q and out: bf16 [T, n_q, 128] (or [T, n_q * 128]), 1 to 32 query heads per KV head; max_q: at least the most
        new tokens of a sequence (1 for a decode step). Rows past cu[B] are left alone."""
        B, n_kv, dev, cache = self._paged("paged_attention", k_pages, v_pages, k_scale, v_scale, cu, seq_lens, block_table)
        T, n_q, q_row, q_head = self._heads("paged_attention", "q", q, dev)
        oT, on, o_row, o_head = self._heads("paged_attention", "out", out, dev)
        if oT != T or on != n_q:
            raise RuntimeError(f"paged_attention: out must have q's shape, [{T}, {n_q}, 128]")
        if T == 0 or B == 0:
            return
        stream = _launch_stream("paged_attention", dev)
        ws = self._workspace("paged_attention", workspace, dev, stream)
        st = self.lib.qk_paged_attention(_ATTENTION_ARGS.pack(*cache, q.data_ptr(), 0, 0, out.data_ptr(), ws.data_ptr(), T, n_q,
                                                              max_q, q_row, q_head, 0, 0, o_row, o_head, ws.numel(), scale), stream)
        if st:
            self._check(st, "paged_attention")

    def packed_attention(self, q, k, v, cu, out, scale, max_q, workspace=None):
        """Causal attention of whole prompts packed without padding: prompt b is rows cu[b] .. cu[b+1]-1 (int32 [B+1]) of
        q [T, n_q, 128], k and v [T, n_kv, 128] (bf16, any 16-byte-aligned row and head strides, k's equal to v's:
        views of one qkv projection will do) and out; max_q: at least the longest prompt."""
        dev = q.get_device()
        T, n_q, q_row, q_head = self._heads("packed_attention", "q", q, dev)
        kv = self._heads("packed_attention", "k", k, dev)
        oT, on, o_row, o_head = self._heads("packed_attention", "out", out, dev)
        if kv[0] != T or self._heads("packed_attention", "v", v, dev) != kv or oT != T or on != n_q:
            raise RuntimeError("packed_attention: q, k, v and out must have the same rows, k and v equal shapes and strides, "
                               "out q's shape")
        if dev < 0 or cu.dtype != torch.int32 or cu.dim() != 1 or len(cu) < 1 or not cu.is_contiguous() or cu.get_device() != dev:
            raise RuntimeError("packed_attention: cu must be int32 [B+1] on q's CUDA device")
        B = len(cu) - 1
        if T == 0 or B == 0:
            return
        stream = _launch_stream("packed_attention", dev)
        ws = self._workspace("packed_attention", workspace, dev, stream)
        st = self.lib.qk_packed_attention(
            _ATTENTION_ARGS.pack(0, 0, 0, 0, cu.data_ptr(), 0, 0, B, kv[1], 0, 0, 0, 0, 0, q.data_ptr(), k.data_ptr(),
                                 v.data_ptr(), out.data_ptr(), ws.data_ptr(), T, n_q, max_q, q_row, q_head, kv[2], kv[3], o_row,
                                 o_head, ws.numel(), scale), stream)
        if st:
            self._check(st, "packed_attention")

    # ---- sequences that share pages ------------------------------------------------------------------------
    # refs (int32 [pages]) counts the sequences that hold a page, 0 for a free one; a sequence of length n holds the first
    # ceil(n / page_size) entries of its block-table row. Free pages are taken lowest first, in the order of the sequences.
    # With too few of them a call takes nothing and sets the device error word (8).
    @staticmethod
    def _ints(what, name, t, shape, dev):
        """The address of a contiguous int32 tensor of `shape` (None: any one-dimensional) on GPU dev; 0 for None."""
        if t is None:
            return 0
        if t.dtype is _I32 and t.get_device() == dev and (t.shape == shape or (shape is None and t.dim() == 1)) and t.is_contiguous():
            return t.data_ptr()
        raise RuntimeError(f"{what}: {name} must be contiguous int32 {list(shape) if shape else '[n]'} on the call's CUDA device")

    @staticmethod
    def _table(what, name, t, rows, width, dev):
        """(address, row stride) of an int32 [rows, width] block table on GPU dev (width None: any)."""
        if t.dtype is not _I32 or t.dim() != 2 or t.shape[0] != rows or t.get_device() != dev or (width is not None and t.shape[1] != width) \
                or (t.stride(1) != 1 and t.shape[1] > 1):
            raise RuntimeError(f"{what}: {name} must be int32 [{rows}, {'width' if width is None else width}] on the call's CUDA device, "
                               "rows contiguous")
        return t.data_ptr(), t.stride(0)

    def paged_plan(self, refs, lens, new, block_table, cu, seq_lens, page_size, refs_out=None, table_out=None, slots=None,
                   positions=None, groups=None, shared=None, info=None):
        """The pass in which new[b] tokens enter sequence b, which has lens[b] positions in the cache (int32 [B]): writes cu [B+1]
        and seq_lens [B] (what the paged calls take), free pages into the new entries of block_table, their refs 1. slots and
        positions (int32 [T]): of every token row, page * page_size + slot in the page, and the position. groups (int32
        [G+1], group g is the sequences groups[g] .. groups[g+1]-1) and shared (int32 [G]): how many leading positions a group's
        sequences have in the same pages (for `shared_attention`). info (int32 [2]): pages missing (0: done), free pages left.
        All or nothing: where pages are missing, or slots are too few for the rows, cu is 0 and seq_lens is lens.
        refs_out and table_out: where the new state goes (default: in place)."""
        what, dev = "paged_plan", refs.get_device()
        if dev < 0:
            raise RuntimeError("paged_plan: every tensor must be on the same CUDA device")
        refs_ptr, lens_ptr = self._ints(what, "refs", refs, None, dev), self._ints(what, "lens", lens, None, dev)
        B = lens.shape[0]
        table_ptr, stride = self._table(what, "block_table", block_table, B, None, dev)
        width = block_table.shape[1]
        out_ptr, out_stride = (table_ptr, stride) if table_out is None else self._table(what, "table_out", table_out, B, width, dev)
        if (groups is None) != (shared is None):
            raise RuntimeError("paged_plan: groups and shared go together")
        G = 0 if groups is None else len(groups) - 1
        if G < 0:
            raise RuntimeError("paged_plan: groups must have at least one entry")
        T = -1 if slots is None and positions is None else len(positions if slots is None else slots)
        st = self.lib.qk_paged_plan(
            _PLAN_ARGS.pack(refs_ptr, lens_ptr, self._ints(what, "new", new, (B,), dev), table_ptr,
                            self._ints(what, "groups", groups, None, dev),
                            refs_ptr if refs_out is None else self._ints(what, "refs_out", refs_out, tuple(refs.shape), dev), out_ptr,
                            self._ints(what, "cu", cu, (B + 1,), dev), self._ints(what, "seq_lens", seq_lens, (B,), dev),
                            self._ints(what, "slots", slots, (T,), dev), self._ints(what, "positions", positions, (T,), dev),
                            self._ints(what, "shared", shared, (G,), dev), self._ints(what, "info", info, (2,), dev),
                            B, width, stride, out_stride, refs.shape[0], page_size, T, G), _launch_stream(what, dev))
        if st:
            self._check(st, what)

    def paged_fork(self, refs, lens, parents, block_table, table_out, lens_out, k_pages, v_pages, k_scale=None, v_scale=None,
                   refs_out=None, info=None):
        """The sequences in a new order: row i of table_out [N, width] and lens_out [N] (not the inputs) continues row parents[i]
        (int32 [N]; -1: an empty row) of block_table [B, width] and lens [B]. Whole pages are shared by count; a partly filled last
        page stays with the first new row that ends in it, unless a sequence outside the call or a longer new row holds it too; the
        others get a free page and a copy of the filled rows. Pools: [pages, n_kv,
        page_size, 128] or [layers, pages, n_kv, page_size, 128] (bf16, or e4m3 with scales of the leading dimensions), whose
        pages are copied in every layer. One row into many spreads a prompt over its beams, parents of -1 end sequences. refs_out:
        where the counts go (default: in place). info (int32 [2]): pages missing (0: done; else refs is as it was and the new rows are
        empty), free pages left."""
        what, dev, shape, dt = "paged_fork", refs.get_device(), k_pages.shape, k_pages.dtype
        if dev < 0 or k_pages.get_device() != dev or v_pages.get_device() != dev:
            raise RuntimeError("paged_fork: every tensor must be on the same CUDA device")
        if len(shape) not in (4, 5) or shape != v_pages.shape or not (k_pages.is_contiguous() and v_pages.is_contiguous()) or shape[-1] != 128 \
                or v_pages.dtype is not dt or (dt is not _BF16 and dt not in _E4M3):
            raise RuntimeError("paged_fork: k_pages and v_pages must be contiguous [pages, n_kv, page_size, 128] or [layers, ...] pools, bf16 "
                               "or e4m3 bytes")
        ks = vs = fp8 = 0
        if dt is not _BF16:
            for s in (k_scale, v_scale):
                if s is None or s.dtype is not _F32 or s.shape != shape[:-1] or not s.is_contiguous() or s.get_device() != dev:
                    raise RuntimeError("paged_fork: an e4m3 cache needs contiguous fp32 k_scale and v_scale, the pools' leading dimensions")
            ks, vs, fp8 = k_scale.data_ptr(), v_scale.data_ptr(), 1
        elif k_scale is not None or v_scale is not None:
            raise RuntimeError("paged_fork: a bf16 cache has no row scales")
        pages, n_kv, page = shape[-4:-1]
        refs_ptr, lens_ptr = self._ints(what, "refs", refs, (pages,), dev), self._ints(what, "lens", lens, None, dev)
        parents_ptr = self._ints(what, "parents", parents, None, dev)
        B, N = lens.shape[0], parents.shape[0]
        table_ptr, stride = self._table(what, "block_table", block_table, B, None, dev)
        width = block_table.shape[1]
        out_ptr, out_stride = self._table(what, "table_out", table_out, N, width, dev)
        st = self.lib.qk_paged_fork(
            _FORK_ARGS.pack(refs_ptr, lens_ptr, parents_ptr, table_ptr,
                            refs_ptr if refs_out is None else self._ints(what, "refs_out", refs_out, (pages,), dev), out_ptr,
                            self._ints(what, "lens_out", lens_out, (N,), dev), self._ints(what, "info", info, (2,), dev),
                            k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, B, N, width, stride, out_stride,
                            shape[0] if len(shape) == 5 else 1, pages, n_kv, page, fp8), _launch_stream(what, dev))
        if st:
            self._check(st, what)

    def beam_workspace(self, device, rows: int, vocab: int, k: int) -> torch.Tensor:
        """A workspace for beam_select calls of up to these sizes (zeroed once). Calls that may run at the same time need one each."""
        nbytes = self.lib.qk_beam_workspace_bytes(rows, vocab, k)
        if nbytes < 0:
            raise RuntimeError(f"beam_workspace: unsupported rows={rows} vocab={vocab} k={k} (vocab at most 1048576, k at most 64)")
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)

    def beam_select(self, logits, scores, cu, out_scores, out_parents, out_tokens, workspace=None):
        """The k best continuations of each request: its beams are rows cu[b] .. cu[b+1]-1 (int32 [B+1], at most 128 a request) of
        logits [R, V] (bf16 or fp32, any row stride) with their scores so far (fp32 [R]). out_scores (fp32), out_parents (the
        row) and out_tokens (int32), all [B, k] with k <= 64: the largest scores[r] + log_softmax(logits[r])[v], in order,
        equal ones by row, then logit and token; -inf, -1, -1 where fewer have a score above -inf. A logit of -inf excludes a token, a score of
        -inf a beam. A NaN or +inf among a row's logits (or as its score) sets the device error word (2) and excludes the row."""
        what, dev = "beam_select", logits.get_device()
        if dev < 0 or logits.dim() != 2 or logits.dtype not in (_BF16, _F32) or (logits.stride(1) != 1 and logits.shape[1] > 1):
            raise RuntimeError("beam_select: logits must be bf16 or fp32 [rows, vocab] on a CUDA device, rows contiguous")
        R, V = logits.shape
        if scores.dtype is not _F32 or tuple(scores.shape) != (R,) or scores.get_device() != dev or not scores.is_contiguous():
            raise RuntimeError(f"beam_select: scores must be fp32 [{R}] on the logits' device")
        cu_ptr = self._ints(what, "cu", cu, None, dev)
        B = len(cu) - 1
        if B < 0 or out_scores.dim() != 2 or out_scores.dtype is not _F32 or out_scores.shape[0] != B or out_scores.get_device() != dev \
                or not out_scores.is_contiguous():
            raise RuntimeError("beam_select: out_scores must be contiguous fp32 [requests, k] on the logits' device, cu [requests + 1]")
        k = out_scores.shape[1]
        nbytes = self.lib.qk_beam_workspace_bytes(R, V, k)
        if nbytes < 0:
            raise RuntimeError(f"beam_select: unsupported rows={R} vocab={V} k={k} (vocab at most 1048576, k 1 to 64)")
        stream = _launch_stream(what, dev)
        ws = self._workspace(what, workspace, dev, stream, "beam_workspace", nbytes)
        st = self.lib.qk_beam_select(
            _BEAM_ARGS.pack(logits.data_ptr(), scores.data_ptr(), cu_ptr, out_scores.data_ptr(),
                            self._ints(what, "out_parents", out_parents, (B, k), dev), self._ints(what, "out_tokens", out_tokens, (B, k), dev),
                            ws.data_ptr(), R, B, V, k, logits.stride(0), logits.dtype is _F32, ws.numel()), stream)
        if st:
            self._check(st, what)

    def shared_workspace(self, device, rows: int, n_q: int) -> torch.Tensor:
        """A workspace for shared_attention calls of up to `rows` token rows and n_q query heads (zeroed once; every call leaves it
        ready for the next). Calls that may run at the same time need one each."""
        nbytes = self.lib.qk_shared_attention_workspace_bytes(rows, n_q)
        if nbytes < 0:
            raise RuntimeError(f"shared_workspace: unsupported rows={rows} n_q={n_q}")
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)

    def shared_attention(self, q, cu, seq_lens, block_table, groups, shared, k_pages, v_pages, out, scale, max_q, k_scale=None,
                         v_scale=None, workspace=None):
        """`paged_attention` over sequences that share their first positions: group g, the sequences groups[g] .. groups[g+1]-1
        (int32 [G+1]), has its first shared[g] positions (int32 [G]; `paged_plan` finds them) in the same pages, or in pages of equal
        contents, all of them before its new tokens. They are read once for the whole group, through its first sequence's table.
        Sequences in no group are on their own."""
        what = "shared_attention"
        B, n_kv, dev, cache = self._paged(what, k_pages, v_pages, k_scale, v_scale, cu, seq_lens, block_table)
        T, n_q, q_row, q_head = self._heads(what, "q", q, dev)
        oT, on, o_row, o_head = self._heads(what, "out", out, dev)
        if oT != T or on != n_q:
            raise RuntimeError(f"shared_attention: out must have q's shape, [{T}, {n_q}, 128]")
        groups_ptr = self._ints(what, "groups", groups, None, dev)
        G = len(groups) - 1
        if G < 0:
            raise RuntimeError("shared_attention: groups must have at least one entry")
        shared_ptr = self._ints(what, "shared", shared, (G,), dev)
        nbytes = self.lib.qk_shared_attention_workspace_bytes(T, n_q)
        if nbytes < 0:
            raise RuntimeError(f"shared_attention: unsupported rows={T} n_q={n_q}")
        if T == 0 or B == 0:
            return
        stream = _launch_stream(what, dev)
        ws = self._workspace(what, workspace, dev, stream, "shared_workspace", nbytes)
        st = self.lib.qk_shared_attention(_SHARED_ARGS.pack(*cache, q.data_ptr(), 0, 0, out.data_ptr(), ws.data_ptr(), T, n_q, max_q, q_row,
                                                            q_head, 0, 0, o_row, o_head, ws.numel(), scale, groups_ptr, shared_ptr, G), stream)
        if st:
            self._check(st, what)

    def finalize(self, best, token, out_tokens, state):
        b = token.numel()
        out_len = out_tokens.shape[-1]
        self._check(self.lib.qk_finalize(_p(best), _p(token), _p(out_tokens), _p(state), out_len, b, _stream()),
                    "finalize")


_ops = None


def ops() -> DecodeOps:
    """The decode ops (loads libqwen3_b200.so once). Raises if the library or an sm_100 GPU is missing."""
    global _ops
    if _ops is None:
        lib = load_library()
        if not torch.cuda.is_available():
            raise RuntimeError("the B200 decode kernels need a CUDA device")
        major, minor = torch.cuda.get_device_capability()
        if (major, minor) != (10, 0):
            raise RuntimeError(f"libqwen3_b200.so is built for sm_100a; this device is sm_{major}{minor}")
        _ops = DecodeOps(lib)
    return _ops

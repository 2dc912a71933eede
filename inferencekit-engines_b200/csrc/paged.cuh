// The paged KV cache: rows written from a qkv projection (per-head RMSNorm, rotary positions, optional e4m3
// quantisation) and read back.
//
// A call describes a ragged batch: sequence b owns token rows cu[b] .. cu[b+1]-1 and ends, with them, at length
// seq_lens[b], so row cu[b] + i sits at position seq_lens[b] - (cu[b+1] - cu[b]) + i. Position p of sequence b lies
// in slot p % page_size of page block_table[b][p / page_size]. A page holds [n_kv][page_size][128] values: the rows
// of one head are one contiguous block, which a single copy moves. bf16 pages hold the rows; e4m3 pages hold
// q = e4m3(x / s) with one fp32 scale s = max|x| / 448 per row in [n_pages][n_kv][page_size] (the format of the
// contiguous FP8 cache, attention_fp8kv.cuh).
#pragma once
#include "common.cuh"

namespace qk {

struct PagedCache {
  uint8_t* k;           // [n_pages][n_kv][page_size][128] bf16 or e4m3
  uint8_t* v;
  float* ks;            // [n_pages][n_kv][page_size], e4m3 only
  float* vs;
  const int* table;     // [B] rows of table_width entries, table_stride apart
  const int* cu;        // [B + 1]
  const int* seq_lens;  // [B]
  int B, n_kv, n_pages, page_shift, table_width, table_stride;
};

// The sequence that owns token row t: the number of cu[1 .. B] that are <= t (B where t is past the last row).
// All 32 lanes take part; 32 probes a round, so one load for B <= 32 and two up to 1024.
__device__ __forceinline__ int seq_of_row(const int* cu, int B, int t, int lane) {
  int lo = 0, n = B;                       // the answer lies in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32, i = (lane + 1) * step;
    const bool le = i <= n && __ldg(cu + lo + i) <= t;
    const int k = __popc(__ballot_sync(0xffffffffu, le));   // probes 1 .. k hold: the answer is >= lo + k * step
    lo += k * step;
    n = min(n - k * step, step - 1);
  }
  return lo;
}

// 8 floats -> 8 e4m3 bytes x / s, round to nearest even (a zero scale gives zeros). IEEE division: bf16 rows over
// their own maximum land on rounding ties often enough to see which way a last-bit difference goes.
__device__ __forceinline__ uint2 quant8(const float (&x)[8], float s) {
  uint32_t h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = s != 0.f ? __fdiv_rn(x[2 * j], s) : 0.f, b = s != 0.f ? __fdiv_rn(x[2 * j + 1], s) : 0.f;
    h[j] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 pack_bf16x8(const float (&x)[8]) {
  return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
__device__ __forceinline__ void unpack_bf16x8(const uint4 r, float (&x)[8]) {
  x[0] = bf16lo(r.x), x[1] = bf16hi(r.x), x[2] = bf16lo(r.y), x[3] = bf16hi(r.y);
  x[4] = bf16lo(r.z), x[5] = bf16hi(r.z), x[6] = bf16lo(r.w), x[7] = bf16hi(r.w);
}
// Sum and maximum over the 16 lanes that hold one head's row; the maximum keeps a NaN.
__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float half_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

struct PagedQkvParams {
  PagedCache c;
  const bf16* qkv;      // [T] rows of (n_q + 2 n_kv) * 128 values, qkv_stride apart
  bf16* q_out;          // [T][n_q][128], rows q_stride apart
  bf16* k_out;          // [T][n_kv][128], rows k_stride apart, or null
  const bf16* q_norm;   // [128] or null
  const bf16* k_norm;
  const float* cos;     // [max_pos][half]
  const float* sin;
  long long qkv_stride, q_stride, k_stride;
  int T, n_q, max_pos, half, interleaved;
  float eps;
};

// A half-warp (16 lanes, 8 dims each) handles one head of one row: everything it needs is in its own registers and
// a row is one 256-byte load. Heads 0 .. n_q-1 are queries, then n_kv keys, then n_kv values. All arithmetic in
// fp32, one rounding at the store (bf16, or e4m3 after the division by the row's scale).
template <bool FP8>
__global__ void __launch_bounds__(256) paged_qkv_kernel(const __grid_constant__ PagedQkvParams p) {
  const int lane = threadIdx.x & 31, sub = lane & 15;
  const int H = p.n_q + 2 * p.c.n_kv, pairs = (H + 1) / 2;
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = w / pairs, h = 2 * (w - t * pairs) + (lane >> 4);
  if (t >= p.T) return;
  grid_dep_wait();
  grid_dep_launch();
  const int b = seq_of_row(p.c.cu, p.c.B, t, lane);
  if (b >= p.c.B) return;                     // a padding row past the last sequence
  const bool on = h < H;
  float x[8];
  unpack_bf16x8(on ? ldg_stream(p.qkv + t * p.qkv_stride + h * HEAD_DIM + sub * 8) : make_uint4(0, 0, 0, 0), x);
  const int pos = __ldg(p.c.seq_lens + b) - (__ldg(p.c.cu + b + 1) - t);
  const int page_at = pos >> p.c.page_shift;
  int page = -1;
  if (pos >= 0 && pos < p.max_pos && page_at < p.c.table_width)
    page = __ldg(p.c.table + (size_t)b * p.c.table_stride + page_at);
  if (page < 0 || page >= p.c.n_pages) {      // outside the table or the pool: nothing to write to
    if (lane == 0) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    return;
  }
  const bool is_q = h < p.n_q, is_v = h >= p.n_q + p.c.n_kv;
  const bf16* nw = is_q ? p.q_norm : p.k_norm;
  if (p.q_norm) {                             // both norms, or neither
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
    const float rstd = rsqrtf(half_sum(ss) * (1.f / HEAD_DIM) + p.eps);
    if (!is_v) {
      float wt[8];
      unpack_bf16x8(*reinterpret_cast<const uint4*>(nw + sub * 8), wt);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * rstd * wt[j];
    }
  }
  const int half = p.half, d0 = sub * 8;
  const float* cos = p.cos + (size_t)pos * half;
  const float* sin = p.sin + (size_t)pos * half;
  if (p.interleaved) {                        // pairs (2i, 2i+1): both in this lane, angle i = d / 2
    if (!is_v && d0 < 2 * half) {
      const float4 c4 = *reinterpret_cast<const float4*>(cos + d0 / 2), s4 = *reinterpret_cast<const float4*>(sin + d0 / 2);
      const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = x[2 * j], q = x[2 * j + 1];
        x[2 * j] = a * cc[j] - q * sn[j];
        x[2 * j + 1] = q * cc[j] + a * sn[j];
      }
    }
  } else {                                    // pairs (i, i + half): the partner is half / 8 lanes away
    const int off = half / 8, first = sub < off;
    const int from = (lane & 16) | ((first ? sub + off : sub - off) & 15);
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = __shfl_sync(0xffffffffu, x[j], from);
    if (!is_v && d0 < 2 * half) {
      const int a0 = first ? d0 : d0 - half;
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 c4 = *reinterpret_cast<const float4*>(cos + a0 + j), s4 = *reinterpret_cast<const float4*>(sin + a0 + j);
        const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j + i] = x[j + i] * cc[i] + (first ? -y[j + i] : y[j + i]) * sn[i];
      }
    }
  }
  float s = 0.f;
  if (FP8) {
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = max_nan(a, fabsf(x[j]));
    s = __fdiv_rn(half_max(a), 448.f);
  }
  if (!on) return;
  const uint4 rb = pack_bf16x8(x);
  if (is_q) {
    *reinterpret_cast<uint4*>(p.q_out + t * p.q_stride + h * HEAD_DIM + d0) = rb;
    return;
  }
  const int g = is_v ? h - p.n_q - p.c.n_kv : h - p.n_q;
  if (p.k_out && !is_v) *reinterpret_cast<uint4*>(p.k_out + t * p.k_stride + g * HEAD_DIM + d0) = rb;
  const int slot = pos & ((1 << p.c.page_shift) - 1);
  const size_t row = (((size_t)page * p.c.n_kv + g) << p.c.page_shift) + slot;
  uint8_t* pool = is_v ? p.c.v : p.c.k;
  if (FP8) {
    *reinterpret_cast<uint2*>(pool + row * HEAD_DIM + d0) = quant8(x, s);
    if (sub == 0) (is_v ? p.c.vs : p.c.ks)[row] = s;
  } else {
    *reinterpret_cast<uint4*>(pool + (row * HEAD_DIM + d0) * 2) = rb;
  }
}

struct PagedReadParams {
  PagedCache c;
  const int* starts;    // first position of each sequence, or null for 0
  bf16* k_out;          // row t, head g at k_out + t * row_stride + g * head_stride
  bf16* v_out;
  long long row_stride, head_stride;
  int T;
};

// Rows back out of the pages: output row cu[b] + i is position starts[b] + i of sequence b, dequantised in fp32 and
// rounded to bf16 once. A half-warp handles one head's K and V row.
template <bool FP8>
__global__ void __launch_bounds__(256) paged_kv_read_kernel(const __grid_constant__ PagedReadParams p) {
  const int lane = threadIdx.x & 31, sub = lane & 15;
  const int n_kv = p.c.n_kv, pairs = (n_kv + 1) / 2;
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = w / pairs, g = 2 * (w - t * pairs) + (lane >> 4);
  if (t >= p.T) return;
  grid_dep_wait();
  grid_dep_launch();
  const int b = seq_of_row(p.c.cu, p.c.B, t, lane);
  if (b >= p.c.B) return;
  const int pos = (p.starts ? __ldg(p.starts + b) : 0) + t - __ldg(p.c.cu + b), page_at = pos >> p.c.page_shift;
  int page = -1;
  if (pos >= 0 && page_at < p.c.table_width) page = __ldg(p.c.table + (size_t)b * p.c.table_stride + page_at);
  if (page < 0 || page >= p.c.n_pages) {
    if (lane == 0) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    return;
  }
  if (g >= n_kv) return;
  const size_t row = (((size_t)page * n_kv + g) << p.c.page_shift) + (pos & ((1 << p.c.page_shift) - 1));
  const size_t at = t * p.row_stride + g * p.head_stride + sub * 8;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint8_t* pool = which ? p.c.v : p.c.k;
    uint4 r;
    if (FP8) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(pool + row * HEAD_DIM + sub * 8));
      const float s = __ldg((which ? p.c.vs : p.c.ks) + row);
      const uint32_t h[4] = {e4m3x2_to_f16x2(q.x), e4m3x2_to_f16x2(q.x >> 16), e4m3x2_to_f16x2(q.y), e4m3x2_to_f16x2(q.y >> 16)};
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        x[2 * j] = f.x * s;
        x[2 * j + 1] = f.y * s;
      }
      r = pack_bf16x8(x);
    } else {
      r = ldg_stream(pool + (row * HEAD_DIM + sub * 8) * 2);
    }
    *reinterpret_cast<uint4*>((which ? p.v_out : p.k_out) + at) = r;
  }
}

}  // namespace qk

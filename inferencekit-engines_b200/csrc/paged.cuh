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
#include <type_traits>

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
__device__ __forceinline__ void pairs_of(const uint4 r, uint64_t (&x)[4]) {
  x[0] = (uint64_t)(r.x & 0xFFFF0000u) << 32 | r.x << 16, x[1] = (uint64_t)(r.y & 0xFFFF0000u) << 32 | r.y << 16;
  x[2] = (uint64_t)(r.z & 0xFFFF0000u) << 32 | r.z << 16, x[3] = (uint64_t)(r.w & 0xFFFF0000u) << 32 | r.w << 16;
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

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two fp32 values in a register pair, for the packed instructions (half the issue slots)
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float f32x2_lo(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float f32x2_hi(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 8 floats (as packed pairs) of a row whose largest magnitude is amax, s = amax / 448 -> 8 e4m3 bytes: the fp32 quotients
// x / s, rounded to nearest even (a zero row gives zeros). bf16 rows lie on ties of e4m3 often, so the quotient has to be the
// rounded one: x * (448 / amax) is off by an ulp here and there, and a correction by its remainder x - q s, which an fma
// gives without rounding the product, makes it right (Markstein, IBM J. Res. Dev. 34, 1990), for two packed fmas a pair.
// Rows whose remainders could fall below fp32's range, and those with an infinity or NaN, are divided.
__device__ __forceinline__ uint2 quant8(const uint64_t (&x)[4], float amax, float s) {
  uint32_t h[4];
  const bool plain = amax >= 1e-20f && amax < INFINITY;
  const float r = plain ? __fdiv_rn(448.f, amax) : 0.f;   // 1 / s to an ulp or two, beside s and not behind it
  const uint64_t inv = f32x2(r, r), neg = f32x2(-s, -s);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint64_t q = mul2(x[j], inv);
    q = fma2(fma2(q, neg, x[j]), inv, q);
    float a = f32x2_lo(q), b = f32x2_hi(q);
    if (!plain) a = s != 0.f ? __fdiv_rn(f32x2_lo(x[j]), s) : 0.f, b = s != 0.f ? __fdiv_rn(f32x2_hi(x[j]), s) : 0.f;
    h[j] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
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
  int T, n_q, max_pos, half, span;
  float eps;
};

// A warp takes `span` pairs of heads of one row, a half-warp (16 lanes, 8 dims each) per head: finding the row's sequence,
// position and page is a chain of four dependent loads, and its angles and the norm's weights are the same for every
// head, so they are fetched once for the span. All arithmetic in fp32, one rounding at the store (bf16, or e4m3 after the
// division by the row's scale).
// With w the norm's weights and (c, s) a pair's angle, the rotated value of dim j is rstd * (x_j A_j + x_j' B_j), j' its
// partner, A_j = w_j c and B_j = +-w_j' s, both computed once per warp: two products and a multiplication per value.
// Pairs of heads: ceil(n_q / 2) of queries, then ceil(n_kv / 2) of keys and as many of values; a pair has one kind.
// Bound by issue slots, not bytes, when written head by head with its own angles (160 us for 16,384 rows of 32 + 16
// heads into e4m3 pages, 2.4 TB/s); 80 us in a graph, 4.7 TB/s so.
enum { ROW_Q, ROW_K, ROW_V };
template <bool FP8, bool INTER>
__global__ void __launch_bounds__(256, 4) paged_qkv_kernel(const __grid_constant__ PagedQkvParams p) {
  const int lane = threadIdx.x & 31, sub = lane & 15, d0 = sub * 8, side = lane >> 4;
  const int n_kv = p.c.n_kv, n_q = p.n_q, q_pairs = (n_q + 1) / 2, kv_pairs = (n_kv + 1) / 2;
  const int pairs = q_pairs + 2 * kv_pairs, parts = (pairs + p.span - 1) / p.span;
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = w / parts, first = (w - t * parts) * p.span, last = min(pairs, first + p.span);
  if (t >= p.T) return;
  grid_dep_wait();
  grid_dep_launch();
  const int b = seq_of_row(p.c.cu, p.c.B, t, lane);
  if (b >= p.c.B) return;                     // a padding row past the last sequence
  const int pos = __ldg(p.c.seq_lens + b) - (__ldg(p.c.cu + b + 1) - t);
  const int page_at = pos >> p.c.page_shift;
  int page = -1;
  if (pos >= 0 && pos < p.max_pos && page_at < p.c.table_width)
    page = __ldg(p.c.table + (size_t)b * p.c.table_stride + page_at);
  if (page < 0 || page >= p.c.n_pages) {      // outside the table or the pool: nothing to write to
    if (lane == 0) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    return;
  }
  // Interleaved: pairs (2i, 2i+1), both in this lane, angle i = d / 2 (four of them). Otherwise pairs (i, i + half): the
  // partner is half / 8 lanes away, and its sine counts negative for the lower one.
  const int half = p.half, off = half / 8;
  const bool lower = sub < off, turns = d0 < 2 * half;
  const int partner = INTER || !turns ? sub : lower ? sub + off : sub - off;
  uint64_t A[4], B[4];
  auto weights = [&](const bf16* nw) {
    float wt[8], wp[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) wt[j] = wp[j] = 1.f;
    if (nw) {
      unpack_bf16x8(*reinterpret_cast<const uint4*>(nw + d0), wt);
      unpack_bf16x8(*reinterpret_cast<const uint4*>(nw + partner * 8), wp);
    }
    if (!turns) {
#pragma unroll
      for (int j = 0; j < 4; ++j) A[j] = f32x2(wt[2 * j], wt[2 * j + 1]), B[j] = 0;
      return;
    }
    const size_t a0 = (size_t)pos * half + (INTER ? d0 / 2 : lower ? d0 : d0 - half);
    float cs[8], sn[8];
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      if (INTER && j) break;
      const float4 c4 = *reinterpret_cast<const float4*>(p.cos + a0 + j), s4 = *reinterpret_cast<const float4*>(p.sin + a0 + j);
      cs[j] = c4.x, cs[j + 1] = c4.y, cs[j + 2] = c4.z, cs[j + 3] = c4.w;
      sn[j] = s4.x, sn[j + 1] = s4.y, sn[j + 2] = s4.z, sn[j + 3] = s4.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (INTER) {
        A[j] = f32x2(wt[2 * j] * cs[j], wt[2 * j + 1] * cs[j]);
        B[j] = f32x2(-wt[2 * j + 1] * sn[j], wt[2 * j] * sn[j]);
      } else {
        const float sign = lower ? -1.f : 1.f;
        A[j] = f32x2(wt[2 * j] * cs[2 * j], wt[2 * j + 1] * cs[2 * j + 1]);
        B[j] = f32x2(sign * wp[2 * j] * sn[2 * j], sign * wp[2 * j + 1] * sn[2 * j + 1]);
      }
    }
  };
  const int slot = pos & ((1 << p.c.page_shift) - 1);
  const size_t row0 = (((size_t)page * n_kv) << p.c.page_shift) + slot;
  // pairs [from, to) of one kind, whose heads begin at src and end at n
  auto rows = [&](auto kind, int from, int to, int n, const bf16* src) {
    constexpr int KIND = decltype(kind)::value, AHEAD = 2;
    auto load = [&](int pair) {
      const int h = 2 * pair + side;
      return pair < to && h < n ? ldg_stream(src + h * HEAD_DIM) : make_uint4(0, 0, 0, 0);
    };
    uint4 next[AHEAD];                        // two pairs' rows are on their way while two are computed
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) next[i] = load(from + i);
    for (int pair = from; pair < to; pair += AHEAD) {
      uint4 in[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) in[i] = next[i];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) next[i] = load(pair + AHEAD + i);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (pair + i >= to) break;
        const int h = 2 * (pair + i) + side;
        const bool on = h < n;
        uint64_t x2[4];                       // the packed instructions halve the issue slots, which bound this
        pairs_of(in[i], x2);
        if (KIND != ROW_V) {                  // norm and rotation
          uint4 o = in[i];
          if (!INTER) {
            const int lane_of = (lane & 16) | partner;
            o.x = __shfl_sync(0xffffffffu, o.x, lane_of), o.y = __shfl_sync(0xffffffffu, o.y, lane_of);
            o.z = __shfl_sync(0xffffffffu, o.z, lane_of), o.w = __shfl_sync(0xffffffffu, o.w, lane_of);
          } else {                            // neighbours change places
            o.x = __byte_perm(o.x, 0, 0x1032), o.y = __byte_perm(o.y, 0, 0x1032);
            o.z = __byte_perm(o.z, 0, 0x1032), o.w = __byte_perm(o.w, 0, 0x1032);
          }
          float rstd = 1.f;
          if (p.q_norm) {
            uint64_t ss = mul2(x2[0], x2[0]);
#pragma unroll
            for (int j = 1; j < 4; ++j) ss = fma2(x2[j], x2[j], ss);
            rstd = rsqrtf(half_sum(f32x2_lo(ss) + f32x2_hi(ss)) * (1.f / HEAD_DIM) + p.eps);
          }
          const uint64_t r2 = f32x2(rstd, rstd);
          uint64_t y2[4];
          pairs_of(o, y2);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x2[j] = mul2(x2[j], A[j]);
            if (turns) x2[j] = fma2(y2[j], B[j], x2[j]);   // (not as 0 * y where nothing turns: y may be infinite)
            x2[j] = mul2(x2[j], r2);
          }
        }
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[2 * j] = f32x2_lo(x2[j]), x[2 * j + 1] = f32x2_hi(x2[j]);
        if (KIND == ROW_Q) {
          if (on) *reinterpret_cast<uint4*>(p.q_out + t * p.q_stride + h * HEAD_DIM + d0) = pack_bf16x8(x);
          continue;
        }
        if (KIND == ROW_K && p.k_out && on) *reinterpret_cast<uint4*>(p.k_out + t * p.k_stride + h * HEAD_DIM + d0) = pack_bf16x8(x);
        const size_t row = row0 + ((size_t)h << p.c.page_shift);
        uint8_t* pool = KIND == ROW_K ? p.c.k : p.c.v;
        if (FP8) {
          float a = 0.f;
#pragma unroll
          for (int j = 0; j < 8; j += 2) a = max3_nan(a, fabsf(x[j]), fabsf(x[j + 1]));
          a = half_max(a);
          const float s = __fdiv_rn(a, 448.f);
          const uint2 q = quant8(x2, a, s);
          if (on) *reinterpret_cast<uint2*>(pool + row * HEAD_DIM + d0) = q;
          if (on && sub == 0) (KIND == ROW_K ? p.c.ks : p.c.vs)[row] = s;
        } else if (on) {
          *reinterpret_cast<uint4*>(pool + (row * HEAD_DIM + d0) * 2) = KIND == ROW_K ? pack_bf16x8(x) : in[i];
        }
      }
    }
  };
  const bf16* src = p.qkv + t * p.qkv_stride + d0;
  const int k0 = q_pairs, v0 = q_pairs + kv_pairs;
  if (first < k0) {
    weights(p.q_norm);
    rows(std::integral_constant<int, ROW_Q>{}, first, min(last, k0), n_q, src);
  }
  if (first < v0 && last > k0) {
    weights(p.k_norm);
    rows(std::integral_constant<int, ROW_K>{}, max(first, k0) - k0, min(last, v0) - k0, n_kv, src + n_q * HEAD_DIM);
  }
  if (last > v0) rows(std::integral_constant<int, ROW_V>{}, max(first, v0) - v0, last - v0, n_kv, src + (n_q + n_kv) * HEAD_DIM);
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
// rounded to bf16 once. A warp takes all 2 n_kv rows (K, then V) of one position, 16 bytes a lane: two bf16 rows or four
// e4m3 rows at a time, two such loads in flight, 48 warps an SM: 134 us in a graph for 131,000 positions of 8 heads out of
// e4m3 pages (6.1 TB/s). Four loads a lane take 160 us (registers), one 144 (too little in flight), 64 warps 154 (too few
// registers), 40 warps 137.
template <bool FP8>
__global__ void __launch_bounds__(256, 6) paged_kv_read_kernel(const __grid_constant__ PagedReadParams p) {
  constexpr int LANES = FP8 ? 8 : 16, ROWS = 32 / LANES, AHEAD = 2;
  const int lane = threadIdx.x & 31, sub = lane % LANES;
  const int n_kv = p.c.n_kv;
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
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
  const size_t row0 = (((size_t)page * n_kv) << p.c.page_shift) + (pos & ((1 << p.c.page_shift) - 1));
  const int first = lane / LANES;
  for (int i0 = 0; i0 < 2 * n_kv; i0 += ROWS * AHEAD) {
    uint4 q[AHEAD];
    float s[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = i0 + a * ROWS + first, g = i < n_kv ? i : i - n_kv;
      const size_t row = row0 + ((size_t)g << p.c.page_shift);
      if (i < 2 * n_kv) {
        q[a] = ldg_stream((i < n_kv ? p.c.k : p.c.v) + (row * (FP8 ? 8 : 16) + sub) * 16);
        if (FP8) s[a] = __ldg((i < n_kv ? p.c.ks : p.c.vs) + row);
      }
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = i0 + a * ROWS + first, g = i < n_kv ? i : i - n_kv;
      if (i >= 2 * n_kv) continue;
      uint4* dst = reinterpret_cast<uint4*>((i < n_kv ? p.k_out : p.v_out) + t * p.row_stride + g * p.head_stride) + sub * (FP8 ? 2 : 1);
      if (FP8) {
        const uint32_t words[4] = {q[a].x, q[a].y, q[a].z, q[a].w};
        uint32_t y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t h = e4m3x2_to_f16x2(words[j >> 1] >> (16 * (j & 1)));
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
          y[j] = pack_bf16(f.x * s[a], f.y * s[a]);
        }
        dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
        dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
      } else {
        *dst = q[a];
      }
    }
  }
}

}  // namespace qk

// Causal attention of ragged batches: new tokens over a paged cache (bf16 or e4m3 rows), or whole packed prompts.
//
//   out[t][h] = sum over j <= pos(t) of softmax_j(scale * q[t][h] . K[g][j]) V[g][j],   g = h / (n_q / n_kv)
//
// One pass over the keys with a running maximum m and sum l in fp32; a row that sees no key gives zeros.
#pragma once
#include "attention_tc.cuh"

namespace qk {

// A warp per (row, query head): 32 keys a step, a key per lane for the scores, then 4 dims per lane for P.V.
template <int SRC>
__global__ void __launch_bounds__(256) ragged_attention_kernel(const __grid_constant__ RaggedParams p) {
  __shared__ float qs[8][HEAD_DIM];
  const int lane = threadIdx.x & 31, wib = threadIdx.x >> 5;
  const long long w = (long long)blockIdx.x * 8 + wib;
  const int t = (int)(w / p.n_q), h = (int)(w - (long long)t * p.n_q), g = h / p.group;
  if (t >= p.T) return;
  const int b = seq_of_row(p.c.cu, p.c.B, t, lane);
  if (b >= p.c.B) return;
  const int r0 = __ldg(p.c.cu + b), n = __ldg(p.c.cu + b + 1) - r0;
  const int len = SRC == SRC_PACKED ? n : __ldg(p.c.seq_lens + b), keys = max(0, len - n + (t - r0) + 1);
  const uint2 qr = *reinterpret_cast<const uint2*>(p.q + t * p.q_row + h * p.q_head + lane * 4);
  qs[wib][lane * 4] = bf16lo(qr.x), qs[wib][lane * 4 + 1] = bf16hi(qr.x);
  qs[wib][lane * 4 + 2] = bf16lo(qr.y), qs[wib][lane * 4 + 3] = bf16hi(qr.y);
  __syncwarp();
  auto row_of = [&](int j) -> size_t {
    if (SRC == SRC_PACKED) return (size_t)(r0 + j);
    const int at = j >> p.c.page_shift;
    int page = at < p.c.table_width ? __ldg(p.c.table + (size_t)b * p.c.table_stride + at) : -1;
    if (page < 0 || page >= p.c.n_pages) {
      atomicOr(&g_dev_error, DEVERR_BAD_STATE);
      page = 0;
    }
    return (((size_t)page * p.c.n_kv + g) << p.c.page_shift) + (j & ((1 << p.c.page_shift) - 1));
  };
  auto load4 = [&](const uint8_t* pool, const float* sc, const bf16* rows, size_t row, int d, float (&x)[4]) {
    if (SRC == SRC_PAGED_FP8) {
      const uint32_t q = __ldg(reinterpret_cast<const uint32_t*>(pool + row * HEAD_DIM + d));
      const float s = __ldg(sc + row);
      const uint32_t a = e4m3x2_to_f16x2(q), c = e4m3x2_to_f16x2(q >> 16);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a)), e = __half22float2(*reinterpret_cast<const __half2*>(&c));
      x[0] = f.x * s, x[1] = f.y * s, x[2] = e.x * s, x[3] = e.y * s;
    } else {
      const uint2 r = SRC == SRC_PAGED ? __ldg(reinterpret_cast<const uint2*>(pool + (row * HEAD_DIM + d) * 2))
                                       : __ldg(reinterpret_cast<const uint2*>(rows + row * p.kv_row + g * p.kv_head + d));
      x[0] = bf16lo(r.x), x[1] = bf16hi(r.x), x[2] = bf16lo(r.y), x[3] = bf16hi(r.y);
    }
  };
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < keys; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    size_t row = 0;
    if (j < keys) {
      row = row_of(j);
      s = 0.f;
      for (int d = 0; d < HEAD_DIM; d += 4) {
        float x[4];
        load4(p.c.k, p.c.ks, p.k, row, d, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fmaf(qs[wib][d + e], x[e], s);
      }
      s *= p.scale;
    }
    const float mn = fmaxf(m, warp_max(s)), base = mn == -INFINITY ? 0.f : mn;
    const float pj = expf(s - base), f = expf(m - base);
    l = l * f + warp_sum(pj);
    m = mn;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= f;
    for (int i = 0; i < min(32, keys - j0); ++i) {
      const float pi = __shfl_sync(0xffffffffu, pj, i);
      const size_t ri = __shfl_sync(0xffffffffu, (unsigned long long)row, i);
      float x[4];
      load4(p.c.v, p.c.vs, p.v, ri, lane * 4, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(pi, x[e], o[e]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  *reinterpret_cast<uint2*>(p.out + t * p.out_row + h * p.out_head + lane * 4) =
      make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
}

}  // namespace qk

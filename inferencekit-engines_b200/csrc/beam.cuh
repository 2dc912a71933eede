// Beam search's selection: for each request the best k of  s(r, v) = score_r + x_rv - logsumexp_v'(x_rv')  over its beams r
// and the vocabulary v, ties to the lowest (r, v).
//
// Bound by the logits' bytes, which are read once.
//  * A CTA holds a chunk of a row in registers (8 16-byte vectors a thread: 16,384 bf16 or 8,192 fp32 values a CTA of 256): one
//    trip through memory for the maximum, the sum of exponentials and the chunk's own k best values.
//  * The order inside a row is the order of its logits, which needs no logsumexp: a chunk leaves (max, sum) and its k best keys,
//    value and ~index, in order. The CTA that completes a request's count merges the chunks' lists: row sums and scores in 64
//    bits there, so that two beams' candidates are ordered by more than fp32 shows.
//  * exp in fp32, a thread's 64 terms under its own maximum; a row's sum is off by some 2^-22 of itself.
#pragma once
#include "paged.cuh"

namespace qk {

constexpr int BEAM_THREADS = 256, BEAM_WARPS = BEAM_THREADS / 32;
constexpr int BEAM_VECTORS = 8;            // 16-byte vectors of a row that a thread holds
constexpr int BEAM_MAX_K = 64;
constexpr int BEAM_MAX_ROWS = 128;         // beams of a request
constexpr int BEAM_MAX_VOCAB = 1 << 20;
template <typename T>
constexpr int beam_chunk() { return BEAM_THREADS * BEAM_VECTORS * 16 / (int)sizeof(T); }   // values
// Chunks of a row: it may begin anywhere in a 16-byte vector.
__host__ __device__ constexpr int beam_chunks(int V, int size) {
  const int per = 16 / size;
  return ((V + per - 1 + per - 1) / per + BEAM_THREADS * BEAM_VECTORS - 1) / (BEAM_THREADS * BEAM_VECTORS);
}
constexpr int BEAM_MAX_LISTS = BEAM_MAX_ROWS * beam_chunks(BEAM_MAX_VOCAB, 4);

struct BeamParams {
  const void* logits;   // row r at r * row_stride
  const float* scores;  // [R]
  const int* cu;        // [B + 1]
  float* out_scores;    // [B][K]
  int* out_parents;
  int* out_tokens;
  float2* ml;           // [R][chunks] maximum, sum under it
  unsigned long long* keys;   // [R][chunks][K]
  int* counters;        // [B], zero between launches
  long long row_stride;
  int B, R, V, K, chunks, granules;   // granules: 16-byte vectors of a chunk
};

// A value's place in the order: larger values first, then lower indices; 0 is less than every one of them.
__device__ __forceinline__ unsigned long long beam_key(float x, int v) { return argmax_key(x + 0.f, v); }   // (-0 is 0)
__device__ __forceinline__ float beam_value(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int beam_index(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }

struct BeamBest {            // a candidate of the merge: its score, then its flat place in the request (row * V + token)
  double s;
  unsigned at;
  int list;
};
__device__ __forceinline__ bool beam_better(double a, unsigned ia, double b, unsigned ib) { return a > b || (a == b && ia < ib); }

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS) beam_select_kernel(const __grid_constant__ BeamParams p) {
  constexpr int PER = 16 / sizeof(T), N = BEAM_VECTORS * PER;   // values of a vector; of a thread
  __shared__ unsigned long long red[BEAM_WARPS];
  __shared__ float red_m[BEAM_WARPS], red_l[BEAM_WARPS];
  __shared__ int s_b, s_last;
  __shared__ double lse[BEAM_MAX_ROWS];
  __shared__ BeamBest red_c[BEAM_WARPS];
  __shared__ uint8_t head[BEAM_MAX_LISTS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
  grid_dep_wait();
  grid_dep_launch();
  // ---- the rows' requests: all or nothing, so that every CTA comes to the same count ------------------------------------------
  if (tid == 0) s_b = -1;
  __syncthreads();
  bool bad = false;
  for (int b = tid; b < p.B; b += BEAM_THREADS) {
    const int lo = __ldg(p.cu + b), hi = __ldg(p.cu + b + 1);
    bad |= lo < 0 || hi < lo || hi > p.R || hi - lo > BEAM_MAX_ROWS;
    if (lo <= row && row < hi) s_b = b;
    if (lo == hi && b == (int)blockIdx.x)   // (the grid has a CTA for each request) without beams
      for (int i = 0; i < p.K; ++i) {
        const size_t at = (size_t)b * p.K + i;
        p.out_scores[at] = -INFINITY, p.out_parents[at] = p.out_tokens[at] = -1;
      }
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    return;
  }
  const int b = s_b;
  if (b < 0 || row >= p.R) return;

  // ---- the chunk ----------------------------------------------------------------------------------------------------------------
  const float score = __ldg(p.scores + row);
  const uintptr_t base = reinterpret_cast<uintptr_t>(p.logits) + (size_t)row * p.row_stride * sizeof(T);
  const int lead = (int)(base & 15) / (int)sizeof(T);       // values of the first vector before the row
  const uint4* vec = reinterpret_cast<const uint4*>(base & ~(uintptr_t)15);
  const T* x0 = reinterpret_cast<const T*>(base);
  const int g0 = chunk * p.granules;
  alignas(16) T x[N];
  auto index = [&](int i) { return (g0 + (i / PER) * BEAM_THREADS + tid) * PER - lead + i % PER; };
#pragma unroll
  for (int i = 0; i < BEAM_VECTORS; ++i) {
    const int in_chunk = i * BEAM_THREADS + tid, first = index(i * PER);
    uint4 w;
    if (score != -INFINITY && in_chunk < p.granules && first >= 0 && first + PER <= p.V) {
      w = ldg_stream(vec + g0 + in_chunk);
      *reinterpret_cast<uint4*>(x + i * PER) = w;
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const bool in = score != -INFINITY && in_chunk < p.granules && first + j >= 0 && first + j < p.V;
        x[i * PER + j] = in ? x0[first + j] : (T)-INFINITY;
      }
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, (float)x[i]);
  const float under = m == -INFINITY ? 0.f : m;
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) l += exp2f(((float)x[i] - under) * 1.4426950408889634f);
  // the k best, one a round: the thread that gave it looks for its next
  auto next_best = [&](unsigned long long below) {
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = (float)x[i];
      const unsigned long long key = v > -INFINITY ? beam_key(v, index(i)) : 0;   // (a NaN is none)
      if (key < below && key > best) best = key;
    }
    return best;
  };
  unsigned long long mine = next_best(~0ull);
  unsigned long long* keys = p.keys + ((size_t)row * p.chunks + chunk) * p.K;
  for (int k = 0; k < p.K; ++k) {
    unsigned long long best = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) red[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BEAM_WARPS; ++w) best = max(best, red[w]);
    if (tid == 0) keys[k] = best;
    if (best && best == mine) mine = next_best(mine);
    __syncthreads();
  }
  // (max, sum) of the chunk
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), ol = __shfl_xor_sync(0xffffffffu, l, o), to = fmaxf(m, om);
    const float z = to == -INFINITY ? 0.f : to;
    l = l * exp2f((m - z) * 1.4426950408889634f) + ol * exp2f((om - z) * 1.4426950408889634f);
    m = to;
  }
  if (lane == 0) red_m[warp] = m, red_l[warp] = l;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < BEAM_WARPS; ++w) {
      const float to = fmaxf(m, red_m[w]), z = to == -INFINITY ? 0.f : to;
      l = l * exp2f((m - z) * 1.4426950408889634f) + red_l[w] * exp2f((red_m[w] - z) * 1.4426950408889634f);
      m = to;
    }
    p.ml[(size_t)row * p.chunks + chunk] = make_float2(m, l);
  }
  __syncthreads();
  const int r0 = __ldg(p.cu + b), rows = __ldg(p.cu + b + 1) - r0;
  if (tid == 0) {
    __threadfence();
    const int before = atomicAdd(p.counters + b, 1);
    s_last = before == rows * p.chunks - 1;
    if (s_last) p.counters[b] = 0;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;

  // ---- the request is complete: its lists, merged -------------------------------------------------------------------------------
  for (int r = warp; r < rows; r += BEAM_WARPS) {
    const float2* ml = p.ml + (size_t)(r0 + r) * p.chunks;
    float M = -INFINITY;
    for (int c = lane; c < p.chunks; c += 32) M = fmaxf(M, __ldcg(&ml[c].x));
    M = warp_max(M);
    double L = 0.;
    for (int c = lane; c < p.chunks; c += 32) {
      const float2 v = __ldcg(ml + c);
      if (v.x != -INFINITY) L += (double)v.y * exp((double)v.x - (double)M);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    const float s = __ldg(p.scores + r0 + r);
    const bool none = s == -INFINITY || (L == 0. && M == -INFINITY), wrong = !none && !(fabsf(s) < INFINITY && L > 0. && L < 1e300);
    if (lane == 0) {
      if (wrong) atomicOr(&g_dev_error, DEVERR_BAD_STATE);   // a NaN or +infinity among its logits, or as its score
      lse[r] = none || wrong ? INFINITY : (double)M + log(L);
    }
  }
  const int lists = rows * p.chunks;
  for (int i = tid; i < lists; i += BEAM_THREADS) head[i] = 0;
  __syncthreads();
  auto pick = [&]() {                       // the best head of this thread's lists
    BeamBest best = {-INFINITY, 0xffffffffu, -1};
    for (int i = tid; i < lists; i += BEAM_THREADS) {
      const int r = i / p.chunks;
      if (head[i] >= p.K || lse[r] == INFINITY) continue;
      const unsigned long long key = __ldcg(p.keys + ((size_t)r0 * p.chunks + i) * p.K + head[i]);
      if (!key) continue;
      const double s = (double)__ldg(p.scores + r0 + r) + ((double)beam_value(key) - lse[r]);
      const unsigned at = (unsigned)r * (unsigned)p.V + (unsigned)beam_index(key);
      if (best.list < 0 || beam_better(s, at, best.s, best.at)) best = {s, at, i};
    }
    return best;
  };
  BeamBest own = pick();
  for (int k = 0; k < p.K; ++k) {
    BeamBest best = own;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double s = __shfl_xor_sync(0xffffffffu, best.s, o);
      const unsigned at = __shfl_xor_sync(0xffffffffu, best.at, o);
      const int list = __shfl_xor_sync(0xffffffffu, best.list, o);
      if (list >= 0 && (best.list < 0 || beam_better(s, at, best.s, best.at))) best = {s, at, list};
    }
    if (lane == 0) red_c[warp] = best;
    __syncthreads();
    best = red_c[0];
    for (int w = 1; w < BEAM_WARPS; ++w) {
      const BeamBest o = red_c[w];
      if (o.list >= 0 && (best.list < 0 || beam_better(o.s, o.at, best.s, best.at))) best = o;
    }
    if (tid == 0) {
      const size_t at = (size_t)b * p.K + k;
      const bool any = best.list >= 0;
      p.out_scores[at] = any ? (float)best.s : -INFINITY;
      p.out_parents[at] = any ? r0 + (int)(best.at / (unsigned)p.V) : -1;
      p.out_tokens[at] = any ? (int)(best.at % (unsigned)p.V) : -1;
    }
    if (best.list >= 0 && best.list == own.list) {
      ++head[best.list];
      own = pick();
    }
    __syncthreads();
  }
}

}  // namespace qk

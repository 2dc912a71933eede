// Beam search's selection: for each request the best k of  s(r, v) = score_r + x_rv - logsumexp_v'(x_rv')  over its beams r
// and the vocabulary v, ties to the lowest (r, v).
//
// Bound by the logits' bytes, which are read once.
//  * A CTA holds a chunk of a row in registers (8 16-byte vectors a thread: 16,384 bf16 or 8,192 fp32 values a CTA of 256): one
//    trip through memory for the maximum, the sum of exponentials and the chunk's own k best values.
//  * The order inside a row is the order of its logits, which needs no logsumexp: a chunk leaves (max, sum) and its k best keys,
//    value and ~index, in order. The CTA that completes a request's count merges the chunks' lists: row sums and scores in 64
//    bits there, so that two beams' candidates are ordered by more than fp32 shows.
//  * k best of many, twice: the k-th largest of some of them (the largest value of each thread or group of threads) is a lower
//    bound of the k-th largest of all, which few more than k reach; those are ranked by counting. Where too many reach it (ties,
//    sorted rows), k rounds of a maximum take their place.
//  * exp in fp32, a thread's 64 terms under its own maximum; a row's sum is off by some 2^-22 of itself.
#pragma once
#include "attention_few.cuh"   // LOG2E

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
  int list;                 // where it is from; -1: none
};
__device__ __forceinline__ bool beam_better(double a, unsigned ia, double b, unsigned ib) { return a > b || (a == b && ia < ib); }

constexpr int BEAM_CAP = 512;              // candidates that are ranked by counting

// exp2 of x - m, both already in units of log2 e
__device__ __forceinline__ float beam_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <typename T>
__device__ __forceinline__ float beam_value_of(uint32_t w, int j) {   // value j (0 or 1; fp32: 0) of a word
  return sizeof(T) == 4 ? __uint_as_float(w) : j ? bf16hi(w) : bf16lo(w);
}

struct BeamSmem {
  union {
    unsigned long long keys[BEAM_CAP];     // a chunk's candidates
    struct {                               // the merge's
      double score[BEAM_CAP];
      unsigned at[BEAM_CAP];
    } c;
  };
  float top[BEAM_THREADS];                 // the groups' largest
  unsigned short lists[BEAM_CAP];          // the merge: lists that can hold one of the k best
  unsigned long long red[BEAM_WARPS];
  float red_m[BEAM_WARPS], red_l[BEAM_WARPS];
  double lse[BEAM_MAX_ROWS];
  BeamBest red_c[BEAM_WARPS];
  uint8_t head[BEAM_MAX_LISTS];
  float border;
  int b, r0, rows, last, count, n_lists;
};

// sm.border: the k-th largest of the first n of sm.top (a multiple of 4, at most the threads), -inf where there are fewer. Two barriers.
__device__ __forceinline__ void beam_border(BeamSmem& sm, int n, int k) {
  const int tid = threadIdx.x;
  if (tid == 0) sm.border = -INFINITY;
  __syncthreads();
  if (tid < n) {
    const float v = sm.top[tid];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < n; i += 4) {
      const float4 o = *reinterpret_cast<const float4*>(&sm.top[i]);
      rank += (o.x > v || (o.x == v && i < tid)) + (o.y > v || (o.y == v && i + 1 < tid)) + (o.z > v || (o.z == v && i + 2 < tid)) +
              (o.w > v || (o.w == v && i + 3 < tid));
    }
    if (rank == k - 1) sm.border = v;
  }
  __syncthreads();
}

// The merge of a request's lists, by the CTA that completed it.
__device__ __forceinline__ void beam_merge(const BeamParams& p, BeamSmem& sm, int b, int r0, int rows) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sm.count = sm.n_lists = 0;
  for (int r = warp; r < rows; r += BEAM_WARPS) {
    const float2* ml = p.ml + (size_t)(r0 + r) * p.chunks;
    const float s = __ldg(p.scores + r0 + r);
    float M = -INFINITY;
    double L = 0.;
    for (int c0 = 0; c0 < p.chunks; c0 += 32) {
      const float2 v = c0 + lane < p.chunks ? __ldcg(ml + c0 + lane) : make_float2(-INFINITY, 0.f);
      const float to = fmaxf(M, warp_max(v.x)), z = to == -INFINITY ? 0.f : to;
      L = L * beam_ex2((M - z) * LOG2E) + (double)v.y * beam_ex2((v.x - z) * LOG2E);
      M = to;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    const bool none = s == -INFINITY || (L == 0. && M == -INFINITY), wrong = !none && !(fabsf(s) < INFINITY && L > 0. && L < 1e300);
    if (lane == 0) {
      if (wrong) atomicOr(&g_dev_error, DEVERR_BAD_STATE);   // a NaN or +infinity among its logits, or as its score
      sm.lse[r] = none || wrong ? INFINITY : (double)M + log(L);
    }
  }
  __syncthreads();
  const int lists = rows * p.chunks;
  auto key_of = [&](int list, int i) { return __ldcg(p.keys + ((size_t)r0 * p.chunks + list) * p.K + i); };
  auto score_of = [&](int list, unsigned long long key) {   // -inf: none
    const int r = list / p.chunks;
    return key && sm.lse[r] != INFINITY ? (double)__ldg(p.scores + r0 + r) + ((double)beam_value(key) - sm.lse[r]) : -INFINITY;
  };
  auto place_of = [&](int list, unsigned long long key) { return (unsigned)(list / p.chunks) * (unsigned)p.V + (unsigned)beam_index(key); };
  // (scores rounded down to fp32 for the borders: what reaches a border of theirs is a lower bound too)
  // ---- which lists: with many, those whose first candidate is among the k best firsts (or equal to the last of them) --------------
  const bool few = lists * p.K <= BEAM_CAP * 8 || lists <= p.K;
  if (!few) {
    float top = -INFINITY;
    for (int i = tid; i < lists; i += BEAM_THREADS) top = fmaxf(top, __double2float_rd(score_of(i, key_of(i, 0))));
    sm.top[tid] = top;
    beam_border(sm, BEAM_THREADS, p.K);
    for (int i = tid; i < lists; i += BEAM_THREADS) {
      const float s = __double2float_rd(score_of(i, key_of(i, 0)));
      if (s < sm.border || s == -INFINITY) continue;
      const int at = atomicAdd(&sm.n_lists, 1);
      if (at < BEAM_CAP) sm.lists[at] = (unsigned short)i;
    }
    __syncthreads();
  }
  const int n_lists = few ? lists : sm.n_lists;
  if (n_lists <= BEAM_CAP) {
    // ---- their candidates, by depth, so that a list's go to different threads ------------------------------------------------------
    auto each = [&](auto f) {
#pragma unroll 4
      for (int c = tid; c < n_lists * p.K; c += BEAM_THREADS) {
        const int i = c / n_lists, list = few ? c - i * n_lists : sm.lists[c - i * n_lists];
        f(list, key_of(list, i));
      }
    };
    float top = -INFINITY;
    each([&](int list, unsigned long long key) { top = fmaxf(top, __double2float_rd(score_of(list, key))); });
    sm.top[tid] = top;
    beam_border(sm, BEAM_THREADS, p.K);
    each([&](int list, unsigned long long key) {
      const double s = score_of(list, key);
      if (s == -INFINITY || __double2float_rd(s) < sm.border) return;
      const int at = atomicAdd(&sm.count, 1);
      if (at < BEAM_CAP) sm.c.score[at] = s, sm.c.at[at] = place_of(list, key);
    });
  } else if (tid == 0) {
    sm.count = BEAM_CAP + 1;
  }
  __syncthreads();
  const size_t out = (size_t)b * p.K;
  auto write = [&](int k, bool any, double s, unsigned at) {
    p.out_scores[out + k] = any ? (float)s : -INFINITY;
    p.out_parents[out + k] = any ? r0 + (int)(at / (unsigned)p.V) : -1;
    p.out_tokens[out + k] = any ? (int)(at % (unsigned)p.V) : -1;
  };
  const int n = sm.count;
  if (n <= BEAM_CAP) {
    for (int i = tid; i < n; i += BEAM_THREADS) {
      const double s = sm.c.score[i];
      const unsigned at = sm.c.at[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += beam_better(sm.c.score[j], sm.c.at[j], s, at);
      if (rank < p.K) write(rank, true, s, at);
    }
    for (int k = n + tid; k < p.K; k += BEAM_THREADS) write(k, false, 0., 0u);
    return;
  }
  // many equal ones: a round each, among the heads of the lists
  for (int i = tid; i < lists; i += BEAM_THREADS) sm.head[i] = 0;
  auto pick = [&]() {                       // (a thread's own lists)
    BeamBest best = {-INFINITY, 0xffffffffu, -1};
    for (int i = tid; i < lists; i += BEAM_THREADS) {
      if (sm.head[i] >= p.K) continue;
      const unsigned long long key = key_of(i, sm.head[i]);
      const BeamBest c = {score_of(i, key), place_of(i, key), i};
      if (c.s > -INFINITY && (best.list < 0 || beam_better(c.s, c.at, best.s, best.at))) best = c;
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
    if (lane == 0) sm.red_c[warp] = best;
    __syncthreads();
    best = sm.red_c[0];
    for (int w = 1; w < BEAM_WARPS; ++w) {
      const BeamBest o = sm.red_c[w];
      if (o.list >= 0 && (best.list < 0 || beam_better(o.s, o.at, best.s, best.at))) best = o;
    }
    if (tid == 0) write(k, best.list >= 0, best.s, best.at);
    if (best.list >= 0 && best.list == own.list) {
      ++sm.head[best.list];
      own = pick();
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 4) beam_select_kernel(const __grid_constant__ BeamParams p) {
  constexpr int PER = 16 / sizeof(T), PW = 4 / sizeof(T), WORDS = BEAM_VECTORS * 4;   // values of a vector and a word; words of a thread
  __shared__ BeamSmem sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
  grid_dep_wait();
  grid_dep_launch();
  // ---- the chunk: on its way before anything else is looked at ------------------------------------------------------------------
  const uintptr_t base = reinterpret_cast<uintptr_t>(p.logits) + (size_t)row * p.row_stride * sizeof(T);
  const int lead = (int)(base & 15) / (int)sizeof(T);       // values of the first vector before the row
  const uint4* vec = reinterpret_cast<const uint4*>(base & ~(uintptr_t)15);
  const int g0 = chunk * p.granules;
  constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;   // -inf
  const float beam = row < p.R ? __ldg(p.scores + row) : 0.f;
  uint32_t x[WORDS];
  auto index = [&](int word) { return (g0 + (word / 4) * BEAM_THREADS + tid) * PER - lead + (word % 4) * PW; };   // of its first value
#pragma unroll
  for (int i = 0; i < BEAM_VECTORS; ++i) {
    const int at = i * BEAM_THREADS + tid, first = index(4 * i);
    uint4 w = make_uint4(NONE, NONE, NONE, NONE);
    if (row < p.R && at < p.granules && first < p.V && first > -PER) {
      if (first >= 0 && first + PER <= p.V) {
        w = ldg_stream(vec + g0 + at);
      } else {                              // a row's first and last vector: its own values only
        uint64_t half[2] = {(uint64_t)NONE << 32 | NONE, (uint64_t)NONE << 32 | NONE};
        const T* src = reinterpret_cast<const T*>(base);
#pragma unroll 1
        for (int j = max(0, -first); j < min(PER, p.V - first); ++j) {
          const uint32_t v = sizeof(T) == 4 ? __float_as_uint((float)src[first + j]) : (uint32_t)__bfloat16_as_ushort((bf16)src[first + j]);
          const int bit = j * (int)sizeof(T) * 8;
          const uint64_t mask = (sizeof(T) == 4 ? 0xffffffffull : 0xffffull) << (bit & 63);
          if (bit < 64) half[0] = (half[0] & ~mask) | (uint64_t)v << (bit & 63);
          else half[1] = (half[1] & ~mask) | (uint64_t)v << (bit & 63);
        }
        w = make_uint4((uint32_t)half[0], (uint32_t)(half[0] >> 32), (uint32_t)half[1], (uint32_t)(half[1] >> 32));
      }
    }
    x[4 * i] = w.x, x[4 * i + 1] = w.y, x[4 * i + 2] = w.z, x[4 * i + 3] = w.w;
  }
  // ---- the rows' requests: all or nothing, so that every CTA comes to the same count ------------------------------------------
  if (tid == 0) sm.b = -1, sm.count = 0;
  __syncthreads();
  bool bad = false;
  for (int b = tid; b < p.B; b += BEAM_THREADS) {
    const int lo = __ldg(p.cu + b), hi = __ldg(p.cu + b + 1);
    bad |= lo < 0 || hi < lo || hi > p.R || hi - lo > BEAM_MAX_ROWS;
    if (lo <= row && row < hi) sm.b = b, sm.r0 = lo, sm.rows = hi - lo;
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
  const int b = sm.b, r0 = sm.r0, rows = sm.rows;
  if (b < 0 || row >= p.R) return;
  if (beam == -INFINITY) {   // a beam that is none: whatever its logits are
#pragma unroll
    for (int i = 0; i < WORDS; ++i) x[i] = NONE;
  }

  // ---- maximum, sum ---------------------------------------------------------------------------------------------------------------
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < WORDS; ++i)
#pragma unroll
    for (int j = 0; j < PW; ++j) m = fmaxf(m, beam_value_of<T>(x[i], j));
  const float under = m == -INFINITY ? 0.f : -m * LOG2E;
  float l = 0.f, l1 = 0.f;
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    l += beam_ex2(fmaf(beam_value_of<T>(x[i], 0), LOG2E, under));
    if (PW == 2) l1 += beam_ex2(fmaf(beam_value_of<T>(x[i], 1), LOG2E, under));
  }
  l += l1;
  // ---- the k best ---------------------------------------------------------------------------------------------------------------
  const int share = p.K > 16 ? 2 : 4;       // threads of a group
  float top = m;
  for (int o = 1; o < share; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (tid % share == 0) sm.top[tid / share] = top;
  float M = warp_max(m);                    // the warp's sum under its maximum
  l = warp_sum(M == -INFINITY ? 0.f : l * beam_ex2((m - M) * LOG2E));
  if (lane == 0) sm.red_m[warp] = M, sm.red_l[warp] = l;
  beam_border(sm, BEAM_THREADS / share, p.K);
  if (warp == BEAM_WARPS - 1) {             // (max, sum) of the chunk
    const float wm = lane < BEAM_WARPS ? sm.red_m[lane] : -INFINITY;
    M = warp_max(wm);
    l = warp_sum(wm == -INFINITY ? 0.f : sm.red_l[lane] * beam_ex2((wm - M) * LOG2E));
    if (lane == 0) p.ml[(size_t)row * p.chunks + chunk] = make_float2(M, l);
  }
  const float border = sm.border;
  if (m >= border && m > -INFINITY) {
    uint32_t hits = 0;                      // words with a value that reaches the border
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const float v0 = beam_value_of<T>(x[i], 0), v1 = PW == 2 ? beam_value_of<T>(x[i], 1) : v0;
      hits |= (fmaxf(v0, v1) >= border ? 1u : 0u) << i;
    }
    const T* src = reinterpret_cast<const T*>(base);   // (few, and read again: registers have no index)
    while (hits) {
      const int i = __ffs(hits) - 1;
      hits &= hits - 1;
      const int first = index(i);
#pragma unroll
      for (int j = 0; j < PW; ++j) {
        const float v = first + j >= 0 && first + j < p.V ? (float)src[first + j] : -INFINITY;
        if (v >= border && v > -INFINITY) {
          const int at = atomicAdd(&sm.count, 1);
          if (at < BEAM_CAP) sm.keys[at] = beam_key(v, first + j);
        }
      }
    }
  }
  __syncthreads();
  unsigned long long* keys = p.keys + ((size_t)row * p.chunks + chunk) * p.K;
  const int n = sm.count;
  if (n <= BEAM_CAP) {
    for (int i = tid; i < n; i += BEAM_THREADS) {
      const unsigned long long key = sm.keys[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sm.keys[j] > key;
      if (rank < p.K) keys[rank] = key;
    }
    for (int k = n + tid; k < p.K; k += BEAM_THREADS) keys[k] = 0;
  } else {                                  // one a round: the thread that gave it looks for its next
    const T* src = reinterpret_cast<const T*>(base);   // (read again: registers have no index)
    auto next_best = [&](unsigned long long below) {
      unsigned long long best = 0;
#pragma unroll 1
      for (int i = 0; i < BEAM_VECTORS; ++i) {
        const int at = index(4 * i);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const bool in = i * BEAM_THREADS + tid < p.granules && at + j >= 0 && at + j < p.V;
          const float v = in ? (float)src[at + j] : -INFINITY;
          const unsigned long long key = v > -INFINITY ? beam_key(v, at + j) : 0;   // (a NaN is none)
          if (key < below && key > best) best = key;
        }
      }
      return best;
    };
    unsigned long long mine = ~0ull;
    bool stale = true;
    for (int k = 0; k < p.K; ++k) {
      if (stale) mine = next_best(mine);
      unsigned long long best = mine;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
      if (lane == 0) sm.red[warp] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < BEAM_WARPS; ++w) best = max(best, sm.red[w]);
      if (tid == 0) keys[k] = best;
      stale = best && best == mine;
      __syncthreads();
    }
  }
  __syncthreads();
  if (tid == 0) {                           // releases the CTA's stores (ordered before by the barrier), acquires the others'
    int before;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.counters + b) : "memory");
    sm.last = before == rows * p.chunks - 1;
    if (sm.last) p.counters[b] = 0;
  }
  __syncthreads();
  if (sm.last) beam_merge(p, sm, b, r0, rows);
}

}  // namespace qk

// Beam search's selection: for each request the best k of  s(r, v) = score_r + x_rv - logsumexp_v'(x_rv')  over its beams r
// and the vocabulary v; of equal scores the lowest r first, in a row the largest logit, then the lowest v.
//
// The logits' bytes are read once, and their exponentials (16 a cycle and SM) take 70 % of the time that bf16 logits need to arrive. What
// bounds the kernels is neither: in a chunk the chain of dependent instructions from vector to vector (18 % of the copy rate for 128 rows of
// 151,936), in the merge its own short steps.
//  * beam_chunk_kernel: the order inside a row is the order of its logits, which needs no logsumexp. The rows' chunks are dealt in
//    equal contiguous ranges to two CTAs an SM. A chunk (16,384 bf16 or 8,192 fp32 values) comes by a bulk copy into a ring of
//    three, so that up to 192 KB an SM are on their way. A CTA leaves, for its part of a row, (max, sum of exponentials) and the
//    k best keys, value and ~index, in order. (Vectors in registers, unrolled: no faster, and twice the code.)
//  * k best of many: the k-th largest of some of them (the largest of each group of threads, in a part's first chunk) is a lower
//    bound of the k-th largest of all. What reaches it is collected, chunk after chunk, and ranked by counting at the end. Chunks
//    in which too many reach it (ties, rising rows) take k rounds of a maximum instead.
//  * beam_merge_kernel: a CTA per request makes its rows' logsumexps and merges their parts' lists, in the same way. Row sums and
//    scores are in 64 bits there, so that two beams' candidates are ordered by more than fp32 shows.
//  * exp in fp32, a thread's terms under its own maximum; a row's sum is off by some 2^-22 of itself.
#pragma once
#include "attention_few.cuh"   // LOG2E, ex2

namespace qk {

constexpr int BEAM_THREADS = 256, BEAM_WARPS = BEAM_THREADS / 32;
constexpr int BEAM_VECTORS = 8;            // 16-byte vectors of a chunk that a thread takes
constexpr int BEAM_MAX_K = 64;
constexpr int BEAM_MAX_ROWS = 128;         // beams of a request
constexpr int BEAM_MAX_VOCAB = 1 << 20;
constexpr int BEAM_CAP = 1024;             // candidates that are ranked by counting

// 16-byte vectors of a row, which may begin anywhere in one.
__host__ __device__ constexpr int beam_granules(int V, int size) { return (V + 2 * (16 / size) - 2) / (16 / size); }
__host__ __device__ constexpr int beam_min_chunks(int V, int size) {
  return (beam_granules(V, size) + BEAM_THREADS * BEAM_VECTORS - 1) / (BEAM_THREADS * BEAM_VECTORS);
}
constexpr int BEAM_MAX_CHUNKS = beam_min_chunks(BEAM_MAX_VOCAB, 4);
constexpr int BEAM_MAX_LISTS = BEAM_MAX_ROWS * BEAM_MAX_CHUNKS;

// CTAs for `all` chunks on `sms` SMs: two an SM, and no more than that (all + 1) CTAs and chunks multiply within 32 bits. (The most
// chunks, 65,536 rows of 129, leave 508.)
inline int beam_grid(long long all, int sms) {
  return (int)std::max(1ll, std::min(std::min(all, 2ll * sms), 0xffffffffll / (all + 1)));
}

struct BeamParams {
  const void* logits;   // row r at r * row_stride
  const float* scores;  // [R]
  const int* cu;        // [B + 1]
  float* out_scores;    // [B][K]
  int* out_parents;
  int* out_tokens;
  float2* ml;           // [R][chunks], at a part's first chunk: maximum, sum under it
  unsigned long long* keys;   // [R][chunks][K], likewise, 0 behind the last
  long long row_stride;
  int B, R, V, K, chunks, granules, grid;   // granules: 16-byte vectors of a chunk; grid: of the chunks' kernel
};
// CTA c has the chunks from beam_first(c) to beam_first(c + 1). (32 bits hold the products: beam_grid.)
__device__ __forceinline__ int beam_first(const BeamParams& p, int c) { return (int)((unsigned)c * (unsigned)(p.R * p.chunks) / (unsigned)p.grid); }
__device__ __forceinline__ int beam_owner(const BeamParams& p, int u) {
  return (int)(((unsigned)(u + 1) * (unsigned)p.grid - 1) / (unsigned)(p.R * p.chunks));
}

template <typename T>
__device__ __forceinline__ float beam_value_of(uint32_t w, int j) {   // value j (0 or 1; fp32: 0) of a word
  return sizeof(T) == 4 ? __uint_as_float(w) : j ? bf16hi(w) : bf16lo(w);
}
// A value's place in the order: larger values first, then lower indices; 0 is less than every one of them.
__device__ __forceinline__ unsigned long long beam_key(float x, int v) { return argmax_key(x + 0.f, v); }   // (-0 is 0)
__device__ __forceinline__ float beam_value(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int beam_index(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }

// The k-th largest of the groups' largest values `top` (-inf where there are fewer): 64 groups of threads, or 128 for k > 16 (some
// -groups ln(1 - k / groups) values reach it, of many that lie anywhere: 18 for k = 16, 89 for k = 64). All threads; two barriers.
struct BeamBorder {
  float top[128], border;
};
__device__ __forceinline__ float beam_border(BeamBorder& sm, float top, int k) {
  const int tid = threadIdx.x, share = k > 16 ? 2 : 4, n = BEAM_THREADS / share;
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  if (share == 4) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if (tid % share == 0) sm.top[tid / share] = top;
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
  return sm.border;
}

constexpr int BEAM_STAGES = 3, BEAM_CHECK = 4;   // chunks in the ring; chunks between looks at the number of candidates
struct BeamChunkSmem {
  uint4 ring[BEAM_STAGES][BEAM_THREADS * BEAM_VECTORS];
  unsigned long long cand[BEAM_CAP];       // keys
  uint32_t hit[BEAM_CAP];                  // vectors with a value that reaches the border: vector of the row, top bit: of the first chunk
  BeamBorder border;
  unsigned long long red[BEAM_WARPS];
  float red_m[BEAM_WARPS], red_l[BEAM_WARPS];
  uint64_t full[BEAM_STAGES], empty[BEAM_STAGES];
  int count, hits;
};

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 2) beam_chunk_kernel(const __grid_constant__ BeamParams p) {
  constexpr int PER = 16 / sizeof(T), PW = 4 / sizeof(T);   // values of a vector and a word
  constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;   // -inf
  extern __shared__ __align__(128) uint8_t beam_smem[];
  BeamChunkSmem& sm = *reinterpret_cast<BeamChunkSmem*>(beam_smem);
  auto &cand = sm.cand;
  int &count = sm.count, &hits = sm.hits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < BEAM_STAGES; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], BEAM_WARPS);
    }
    fence_mbar_init();
  }
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();
  const int u0 = beam_first(p, blockIdx.x), u1 = beam_first(p, blockIdx.x + 1);

  // chunk u: its row's address, the values of that row's first vector that lie before it, its first vector, and those of its
  // vectors (from .. to - 1 of the row) that lie whole within the tensor, which are copied
  struct Chunk {
    uintptr_t base;
    int lead, g0, from, to;
  };
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p.logits), hi = lo + ((size_t)(p.R - 1) * p.row_stride + p.V) * sizeof(T);
  auto chunk_of = [&](int u) {
    const int row = u / p.chunks;
    Chunk c;
    c.base = lo + (size_t)row * p.row_stride * sizeof(T);
    c.lead = (int)(c.base & 15) / (int)sizeof(T);
    c.g0 = (u - row * p.chunks) * p.granules;
    const uintptr_t v0 = c.base & ~(uintptr_t)15;
    const int all = (c.lead + p.V + PER - 1) / PER;
    c.from = c.g0 == 0 && v0 < lo ? 1 : c.g0;
    c.to = min(c.g0 + p.granules, all);
    if (c.to == all && v0 + (size_t)all * 16 > hi) --c.to;
    return c;
  };
  auto copy = [&](int u) {                  // thread 0
    const Chunk c = chunk_of(u);
    const int st = (u - u0) % BEAM_STAGES, n = max(0, c.to - c.from);
    mbar_arrive_expect_tx(&sm.full[st], (uint32_t)n * 16);
    if (n) bulk_g2s(&sm.ring[st][c.from - c.g0], reinterpret_cast<const void*>((c.base & ~(uintptr_t)15) + (size_t)c.from * 16), (uint32_t)n * 16, &sm.full[st]);
  };
  // vector v of a row at its edge: its own values only
  auto gather = [&](uintptr_t base, int first) {
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
    return make_uint4((uint32_t)half[0], (uint32_t)(half[0] >> 32), (uint32_t)half[1], (uint32_t)(half[1] >> 32));
  };
  // this thread's vector i of the chunk; what is not the row's is -inf
  auto take = [&](const Chunk& c, int st, int i) {
    const int at = i * BEAM_THREADS + tid, first = (c.g0 + at) * PER - c.lead;
    uint4 w = make_uint4(NONE, NONE, NONE, NONE);
    if (at < p.granules && first < p.V && first > -PER) w = first >= 0 && first + PER <= p.V ? sm.ring[st][at] : gather(c.base, first);
    return w;
  };
  auto largest = [&](const uint4& w) {      // (a NaN is none, but for a vector of them)
    if (sizeof(T) == 4) return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
    const __nv_bfloat162 mx = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(mx), __high2float(mx));
  };
  // cand[0 .. n): the k best of them to the front, in order (0 where there are fewer)
  auto rank_all = [&](int n) {
    unsigned long long key[BEAM_CAP / BEAM_THREADS];
    int rank[BEAM_CAP / BEAM_THREADS];
#pragma unroll
    for (int i = 0; i < BEAM_CAP / BEAM_THREADS; ++i) {
      const int at = i * BEAM_THREADS + tid;
      key[i] = at < n ? cand[at] : 0;
      rank[i] = 0;
    }
    for (int i = 0; i * BEAM_THREADS < n; ++i) {
      int above = 0;
      const unsigned long long own = i * BEAM_THREADS + tid < n ? cand[i * BEAM_THREADS + tid] : ~0ull;
#pragma unroll 4
      for (int j = 0; j < n; ++j) above += cand[j] > own;
#pragma unroll
      for (int k = 0; k < BEAM_CAP / BEAM_THREADS; ++k)
        if (k == i) rank[k] = above;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BEAM_CAP / BEAM_THREADS; ++i)
      if (key[i] && rank[i] < p.K) cand[rank[i]] = key[i];
    for (int k = n + tid; k < p.K; k += BEAM_THREADS) cand[k] = 0;
    __syncthreads();
  };
  if (tid == 0)
    for (int u = u0; u < min(u1, u0 + BEAM_STAGES); ++u) copy(u);
  int first_u = u0;                         // the part's first chunk
  float m = -INFINITY, border = -INFINITY;
  float sum = 0.f;
  int kept = 0, since = 0, looked = u0;     // candidates at the last look; chunks since; the next one
  bool ok = true;
  for (int u = u0; u < u1; ++u) {
    const Chunk c = chunk_of(u);
    const bool ends = u + 1 == u1 || (u + 1) % p.chunks == 0;
    const int st = (u - u0) % BEAM_STAGES, turn = (u - u0) / BEAM_STAGES;
    const bool begins = u == first_u;
    ok = __all_sync(0xffffffffu, ok && mbar_wait_small(&sm.full[st], (uint32_t)(turn & 1)));
    auto push = [&](int i) {
      const int at = atomicAdd(&hits, 1);
      if (at < BEAM_CAP) sm.hit[at] = (uint32_t)(c.g0 + i * BEAM_THREADS + tid) | (begins ? 1u << 31 : 0);
    };
    // ---- maximum, sum, what reaches the border (equal values of later chunks have higher indices than k that are kept already) -------
    float top = -INFINITY;
#pragma unroll 2
    for (int i = 0; i < BEAM_VECTORS; ++i) {
      const uint4 w = take(c, st, i);
      const float vm = largest(w), mn = fmaxf(m, vm), z = mn == -INFINITY ? 0.f : mn;   // (x - z first: its product's rounding goes by it)
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = ex2((beam_value_of<T>(words[j], 0) - z) * LOG2E);
        if (PW == 2) e[j] += ex2((beam_value_of<T>(words[j], 1) - z) * LOG2E);
      }
      sum = sum * ex2((m - z) * LOG2E) + ((e[0] + e[1]) + (e[2] + e[3]));
      m = mn;
      top = fmaxf(top, vm);
      if (!begins && vm > border) push(i);
    }
    if (begins) {
      if (tid == 0) count = hits = 0;
      kept = 0;
      border = beam_border(sm.border, top, p.K);
      if (top >= border && top > -INFINITY)
#pragma unroll 1
        for (int i = 0; i < BEAM_VECTORS; ++i) {
          const float vm = largest(take(c, st, i));
          if (vm >= border && vm > -INFINITY) push(i);
        }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.empty[st]);
    if (tid == 0 && u + BEAM_STAGES < u1 && ok) {
      ok = mbar_wait_small(&sm.empty[st], (uint32_t)(turn & 1));
      if (ok) copy(u + BEAM_STAGES);
    }
    if (!ends && ++since < BEAM_CHECK) continue;
    since = 0;
    __syncthreads();
    const int vectors = hits;
    if (!ends) {                            // (a warp that goes on adds to them: not before all have read)
      __syncthreads();
      if (vectors <= BEAM_CAP / 2) continue;
    }
    // ---- the vectors' values that reach the border, the k best of them and of those before -----------------------------------------
    for (int i = tid; i < min(vectors, BEAM_CAP); i += BEAM_THREADS) {
      const int first = (int)(sm.hit[i] & 0x7fffffffu) * PER - c.lead;
      const bool in_first = sm.hit[i] >> 31;
      const uint4 w = first >= 0 && first + PER <= p.V ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(c.base) + first) : gather(c.base, first);
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
      uint32_t reach = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float v = beam_value_of<T>(words[j / PW], j % PW);
        reach |= ((in_first ? v >= border && v > -INFINITY : v > border) ? 1u : 0u) << j;
      }
      while (reach) {
        const int j = __ffs(reach) - 1, at = atomicAdd(&count, 1);
        reach &= reach - 1;
        if (at < BEAM_CAP) cand[at] = beam_key((float)reinterpret_cast<const T*>(c.base)[first + j], first + j);
      }
    }
    __syncthreads();
    int n = vectors > BEAM_CAP ? BEAM_CAP + 1 : count;
    if (n > BEAM_CAP) {
      // one a round: the thread that gave it looks for its next, among those kept at the last look and the values since
      const T* src = reinterpret_cast<const T*>(c.base);
      const int row_u = u / p.chunks * p.chunks, v0 = max(0, (max(first_u, looked) - row_u) * p.granules * PER - c.lead);
      const int v1 = min(p.V, (u + 1 - row_u) * p.granules * PER - c.lead);
      auto next_best = [&](unsigned long long below) {
        unsigned long long best = 0;
        for (int i = tid; i < kept; i += BEAM_THREADS)
          if (cand[i] < below && cand[i] > best) best = cand[i];
#pragma unroll 8
        for (int i = v0 + tid; i < v1; i += BEAM_THREADS) {
          const float v = (float)src[i];
          const unsigned long long key = v > -INFINITY ? beam_key(v, i) : 0;   // (a NaN is none)
          if (key < below && key > best) best = key;
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
        if (tid == 0) cand[BEAM_CAP - BEAM_MAX_K + k] = best;   // (those kept are in front)
        stale = best && best == mine;
        __syncthreads();
      }
      if (tid < p.K) cand[tid] = cand[BEAM_CAP - BEAM_MAX_K + tid];
      __syncthreads();
    } else {
      rank_all(n);
    }
    kept = min(n, p.K);                     // the k best are in front
    if (kept == p.K) border = fmaxf(border, beam_value(cand[p.K - 1]));
    if (tid == 0) count = kept, hits = 0;
    looked = u + 1;
    if (ends) {
      const float M = warp_max(m);          // the warp's sum under its maximum
      float l = warp_sum(M == -INFINITY ? sum : sum * ex2((m - M) * LOG2E));   // (a NaN stays)
      if (lane == 0) sm.red_m[warp] = M, sm.red_l[warp] = l;
      unsigned long long* keys = p.keys + (size_t)first_u * p.K;
      if (tid < p.K) keys[tid] = cand[tid];
      __syncthreads();
      if (warp == 0) {
        const float wm = lane < BEAM_WARPS ? sm.red_m[lane] : -INFINITY, wl = lane < BEAM_WARPS ? sm.red_l[lane] : 0.f, top_m = warp_max(wm);
        l = warp_sum(top_m == -INFINITY ? wl : wl * ex2((wm - top_m) * LOG2E));
        if (lane == 0) p.ml[first_u] = make_float2(top_m, l);
      }
      first_u = u + 1;
      m = -INFINITY;
      sum = 0.f;
    }
    __syncthreads();                        // the next chunk's candidates come behind, or in the place of these
  }
  if (!ok && lane == 0) atomicOr(&g_dev_error, DEVERR_MBAR_TIMEOUT);
  if (__syncthreads_or(!ok) && tid == 0)    // a wait gave up: the copies in flight land before the shared memory goes away
    for (int u = max(u0, u1 - BEAM_STAGES); u < u1; ++u)
      mbar_wait_small(&sm.full[(u - u0) % BEAM_STAGES], (uint32_t)((u - u0) / BEAM_STAGES & 1), 1000000ull);
}

constexpr int BEAM_MAX_USED = 256;         // lists that are merged side by side

// What orders candidates whose scores are equal in 64 bits, the larger first: the lower row of the request, in it the larger logit (which
// a score far larger may have swallowed), then the lower token. 7, 32 and 20 bits.
__device__ __forceinline__ unsigned long long beam_place(int row, unsigned long long key) {
  return (unsigned long long)(BEAM_MAX_ROWS - 1 - row) << 52 | key >> 32 << 20 | (BEAM_MAX_VOCAB - 1 - beam_index(key));
}
static_assert(BEAM_MAX_ROWS <= 1 << 7 && BEAM_MAX_VOCAB <= 1 << 20, "a candidate's place has 59 bits");

struct BeamBest {            // a candidate of the merge: its score, then its place
  double s;
  unsigned long long at;
  int list;                 // where it is from; -1: none
};
__device__ __forceinline__ bool beam_better(double a, unsigned long long ia, double b, unsigned long long ib) { return a > b || (a == b && ia > ib); }

struct BeamMergeSmem {
  double cand_s[BEAM_CAP];
  unsigned long long cand_at[BEAM_CAP];
  BeamBorder border;
  // A logit x of row r scores (x - max[r]) + off[r], off = score - log of the sum under the maximum; -inf: the row has nothing. (The
  // difference first: a row of the type's lowest values has its maximum there too, beside which the rest would be lost.)
  double off[BEAM_MAX_ROWS];
  float max[BEAM_MAX_ROWS];
  float2 ml[BEAM_MAX_USED];
  BeamBest red[BEAM_WARPS];
  int list_at[BEAM_MAX_ROWS + 4];          // lists of the rows before
  int chunk[BEAM_MAX_USED];                // of the lists that can hold one of the k best: the first chunk, the row
  uint8_t row[BEAM_MAX_USED];
  uint8_t head[BEAM_MAX_LISTS];
  int count, n_of, reach;
};
// The lists of a request, in the order of their rows, become one.
__global__ void __launch_bounds__(BEAM_THREADS) beam_merge_kernel(const __grid_constant__ BeamParams p) {
  extern __shared__ __align__(16) uint8_t beam_smem[];
  BeamMergeSmem& sm = *reinterpret_cast<BeamMergeSmem*>(beam_smem);
  float* value = reinterpret_cast<float*>(beam_smem + sizeof(BeamMergeSmem));   // [lists][K]: the candidates' logits, -inf: none
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x;
  if (tid == 0) sm.count = sm.n_of = sm.reach = 0;
  if (p.R * p.chunks == 0) grid_dep_wait();   // (else the chunks' kernel waited for what precedes it before it let this one start)
  const int r0 = __ldg(p.cu + b);
  int rows = __ldg(p.cu + b + 1) - r0;
  if (r0 < 0 || rows < 0 || rows > BEAM_MAX_ROWS || r0 > p.R - rows) {
    if (tid == 0) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    rows = 0;
  }
  const size_t out = (size_t)b * p.K;
  auto write = [&](int k, bool any, double s, unsigned long long at) {
    p.out_scores[out + k] = any ? (float)s : -INFINITY;
    p.out_parents[out + k] = any ? r0 + BEAM_MAX_ROWS - 1 - (int)(at >> 52) : -1;
    p.out_tokens[out + k] = any ? BEAM_MAX_VOCAB - 1 - (int)(at & (BEAM_MAX_VOCAB - 1)) : -1;
  };
  // ---- the rows' parts: row r's lists are list_at[r] .. list_at[r + 1] - 1, one for each CTA that had chunks of it -------------------
  if (warp == 0) {
    int before = 0;
    for (int r = 0; r < rows; r += 32) {
      const int u = (r0 + r + lane) * p.chunks, n = r + lane < rows ? beam_owner(p, u + p.chunks - 1) - beam_owner(p, u) + 1 : 0;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (r + lane < rows) sm.list_at[r + lane] = before + incl - n;
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) sm.list_at[rows] = before;
  }
  const float score = tid < rows ? __ldg(p.scores + r0 + tid) : -INFINITY;   // of row tid
  __syncthreads();
  const int lists = sm.list_at[rows];
  auto row_of = [&](int list) {
    int lo = 0, hi = rows;                  // list_at[lo] <= list
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (sm.list_at[mid] <= list) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  auto chunk_of = [&](int r, int list) {    // the first chunk of a list of row r
    const int u = (r0 + r) * p.chunks, i = list - sm.list_at[r];
    return i == 0 ? u : beam_first(p, beam_owner(p, u) + i);
  };
  const bool few = lists <= BEAM_MAX_USED;
  if (few && tid < lists) {
    const int r = row_of(tid);
    sm.row[tid] = (uint8_t)r;
    sm.chunk[tid] = chunk_of(r, tid);
  }
  __syncthreads();
  grid_dep_wait();                          // the chunks' lists are there
  grid_dep_launch();
  auto key_at = [&](int chunk, int i) { return __ldcg(p.keys + (size_t)chunk * p.K + i); };
  // ---- the lists' values on their way, the rows' sums ------------------------------------------------------------------------------
  auto fetch = [&](int n) {
    const float per_k = 1.f / p.K;
#pragma unroll 1
    for (int c0 = tid; c0 < n * p.K; c0 += 8 * BEAM_THREADS) {
      unsigned long long key[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = min(c0 + j * BEAM_THREADS, n * p.K - 1), at = (int)(((float)c + 0.5f) * per_k);   // c / K (c < 2^14, K <= 64)
        key[j] = key_at(sm.chunk[at], c - at * p.K);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j * BEAM_THREADS < n * p.K) value[c0 + j * BEAM_THREADS] = key[j] ? beam_value(key[j]) : -INFINITY;
    }
  };
  if (few) {
    if (tid < lists) sm.ml[tid] = __ldcg(p.ml + sm.chunk[tid]);
    fetch(lists);
  }
  __syncthreads();
  if (tid < rows) {
    float M = -INFINITY;
    double L = 0.;
    for (int i = sm.list_at[tid]; i < sm.list_at[tid + 1]; ++i) {
      const float2 v = few ? sm.ml[i] : __ldcg(p.ml + chunk_of(tid, i));
      const float to = fmaxf(M, v.x), z = to == -INFINITY ? 0.f : to;
      L = L * ex2((M - z) * LOG2E) + (double)v.y * (v.x == z ? 1.f : ex2((v.x - z) * LOG2E));
      M = to;
    }
    const bool none = score == -INFINITY || (L == 0. && M == -INFINITY), wrong = !none && !(fabsf(score) < INFINITY && L > 0. && L < 1e300);
    if (wrong) atomicOr(&g_dev_error, DEVERR_BAD_STATE);   // a NaN or +infinity among its logits, or as its score
    const double off = none || wrong ? -INFINITY : (double)score - log(L);
    sm.off[tid] = off;
    sm.max[tid] = none || wrong ? 0.f : M;
    if (off != -INFINITY) atomicMax(&sm.reach, __float_as_int(fabsf((float)off)));
  }
  __syncthreads();
  // Borders are found among fp32 scores, each within 2^-23 of |score| + |off| of the 64-bit one; what may be among the k best reaches
  // the border less twice that.
  auto lowered = [&](float border) { return border == -INFINITY ? border : border - 0x1p-21f * (fabsf(border) + __int_as_float(sm.reach)); };
  // ---- which lists: with many, those whose first candidate can be among the k best firsts -----------------------------------------
  if (!few) {
    auto first = [&](int list, int& r, int& chunk) {
      r = row_of(list);
      chunk = chunk_of(r, list);
      const unsigned long long key = key_at(chunk, 0);
      return key ? (beam_value(key) - sm.max[r]) + (float)sm.off[r] : -INFINITY;
    };
    int r, chunk;
    float top = -INFINITY;
    for (int i = tid; i < lists; i += BEAM_THREADS) top = fmaxf(top, first(i, r, chunk));
    const float border = lowered(beam_border(sm.border, top, p.K));
    for (int i = tid; i < lists; i += BEAM_THREADS) {
      const float s = first(i, r, chunk);
      if (!(s >= border && s > -INFINITY)) continue;
      const int at = atomicAdd(&sm.n_of, 1);
      if (at < BEAM_MAX_USED) sm.row[at] = (uint8_t)r, sm.chunk[at] = chunk;
    }
    __syncthreads();
    if (sm.n_of <= BEAM_MAX_USED) fetch(sm.n_of);
    __syncthreads();
  }
  const int n_lists = few ? lists : sm.n_of;
  if (n_lists <= BEAM_MAX_USED) {
    // ---- their candidates: a warp a list, its first one another lane's in each ------------------------------------------------------
    auto each = [&](auto f) {
      for (int at = warp; at < n_lists; at += BEAM_WARPS) {
        const float off = (float)sm.off[sm.row[at]], max = sm.max[sm.row[at]];
        for (int i = (lane - 5 * (at / BEAM_WARPS)) & 31; i < p.K; i += 32) f(at, i, (value[at * p.K + i] - max) + off);
      }
    };
    float top = -INFINITY;
    each([&](int, int, float s) { top = fmaxf(top, s); });
    const float border = lowered(beam_border(sm.border, top, p.K));
    each([&](int at, int i, float s) {
      if (!(s >= border && s > -INFINITY)) return;   // (nor what an infinite logit makes NaN)
      const int to = atomicAdd(&sm.count, 1);
      if (to >= BEAM_CAP) return;
      const int r = sm.row[at];
      const unsigned long long key = key_at(sm.chunk[at], i);
      sm.cand_s[to] = ((double)beam_value(key) - (double)sm.max[r]) + sm.off[r];
      sm.cand_at[to] = beam_place(r, key);
    });
  } else if (tid == 0) {
    sm.count = BEAM_CAP + 1;
  }
  __syncthreads();
  const int n = sm.count;
  if (n <= BEAM_CAP) {
    for (int i = tid; i < n; i += BEAM_THREADS) {
      const double s = sm.cand_s[i];
      const unsigned long long at = sm.cand_at[i];
      int rank = 0, equal = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const double o = sm.cand_s[j];
        rank += o > s;
        equal += o == s;
      }
      if (equal > 1)                        // (rare: the places' loads beside the scores' took 2 us of 34 for 64 of 8,000)
        for (int j = 0; j < n; ++j) rank += sm.cand_s[j] == s && sm.cand_at[j] > at;
      if (rank < p.K) write(rank, true, s, at);
    }
    for (int k = n + tid; k < p.K; k += BEAM_THREADS) write(k, false, 0., 0ull);
    return;
  }
  // many equal ones: a round each, among the heads of the lists
  for (int i = tid; i < lists; i += BEAM_THREADS) sm.head[i] = 0;
  auto pick = [&]() {                       // (a thread's own lists)
    BeamBest best = {-INFINITY, 0, -1};
    for (int i = tid; i < lists; i += BEAM_THREADS) {
      if (sm.head[i] >= p.K) continue;
      const int r = row_of(i);
      const unsigned long long key = key_at(chunk_of(r, i), sm.head[i]);
      const BeamBest c = {key ? ((double)beam_value(key) - (double)sm.max[r]) + sm.off[r] : -INFINITY, beam_place(r, key), i};
      if ((float)c.s > -INFINITY && (best.list < 0 || beam_better(c.s, c.at, best.s, best.at))) best = c;
    }
    return best;
  };
  BeamBest own = pick();
  for (int k = 0; k < p.K; ++k) {
    BeamBest best = own;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double s = __shfl_xor_sync(0xffffffffu, best.s, o);
      const unsigned long long at = __shfl_xor_sync(0xffffffffu, best.at, o);
      const int list = __shfl_xor_sync(0xffffffffu, best.list, o);
      if (list >= 0 && (best.list < 0 || beam_better(s, at, best.s, best.at))) best = {s, at, list};
    }
    if (lane == 0) sm.red[warp] = best;
    __syncthreads();
    best = sm.red[0];
    for (int w = 1; w < BEAM_WARPS; ++w) {
      const BeamBest o = sm.red[w];
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

}  // namespace qk

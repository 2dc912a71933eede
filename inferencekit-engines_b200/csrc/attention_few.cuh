// Paged attention for few query rows: the decode step's one token, or a handful (speculated tokens), per sequence.
//
//   out[t][h] = sum over j <= pos(t) of softmax_j(scale * q[t][h] . K[g][j]) V[g][j]
//
// Bound by the cache bytes: up to 16 query rows (tokens x heads of a KV head) meet each K and V row once, so the only
// aim is to keep HBM busy.
//  * Work: the (sequence, KV head, key tile) triples, tile-major, are dealt in equal contiguous ranges to one CTA
//    per SM, whatever the lengths are: a 32k context beside short ones leaves no SM idle. A unit (sequence, head)
//    split between CTAs leaves fp32 partials (o, m, l); the CTA that completes the unit's count adds them in CTA
//    order (the same bits every run).
//  * A producer warp keeps a ring of 128 KB of tiles in flight: TMA boxes of one page's rows each, 128-byte
//    swizzle, so every shared-memory read below is free of bank conflicts.
//  * Consumer warps take KW keys of a tile each and keep a running softmax and output registers of their own, so nothing
//    waits on a neighbour until the piece ends. Products are warp-level MMAs with the keys as M: S^T = K Q^T and
//    O^T = V^T P^T (m16n8k16), 8 query rows a tile of N, so a decode step's 4 heads fill half of it, where rows as M would
//    fill a quarter, with twice the MMAs and accumulators. P^T turns from one's result into the other's operand with a
//    movmatrix. A tcgen05 tile of 128 rows would hold 4 in use and pass every score through TMEM.
//  * bf16 cache: bf16 MMAs, P in two parts, its rounding to bf16 and what that leaves: 16 bits of P, more than the output
//    shows, as in the contiguous cache's attention, whose P is fp32. 1 % more time (16 sequences at up to 32k).
//  * e4m3 cache: the bytes become f16 exactly; q is scaled to f16 range by a power of two per row; the K scale multiplies
//    the score in fp32; P times the V scale is rounded to f16 (11 bits: an eighth of the output's own rounding),
//    brought to at most 2^15 by a running power of two per row, so that what falls below f16's smallest value is below 2^-39
//    of the row's largest weight times V scale, whatever the scales are. The conversions (4 issue cycles for two values)
//    are what bounds this path beside HBM.
#pragma once
#include "gemm_tc.cuh"     // tma_load_2d
#include "paged.cuh"

namespace qk {

constexpr int FEW_RING = 131072;      // bytes of K and V in the ring
constexpr int FEW_MIN_TILES = 1;      // a CTA's least share (one sequence of 13 tiles and 8 heads: 9.0 us in a graph; 10.7 with 2, 11.7 with 4)
constexpr float LOG2E = 1.4426950408889634f;

struct RaggedParams {
  PagedCache c;         // pages, table, cu, seq_lens; packed prompts use cu alone
  const bf16* q;        // row t, head h at q + t * q_row + h * q_head
  const bf16* k;        // packed keys: row t, head g at k + t * kv_row + g * kv_head (null for a paged cache)
  const bf16* v;
  bf16* out;
  long long q_row, q_head, kv_row, kv_head, out_row, out_head;
  int T, n_q, group;
  float scale;
};

struct FewParams {
  CUtensorMap tm_k, tm_v;   // the pools as [n_pages * n_kv * page_size] rows: box {128 bytes, min(page_size, keys of a tile) rows}
  RaggedParams r;
  float* part;              // [grid][2][rows][128]
  float* ml;                // [grid][2][rows][2]
  int* counters;            // [grid], zero between launches
  int strict;               // 1: no other kernel takes the sequences with more rows
};

// A sequence's part in the few-row kernel: its token rows and keys (rows 0: not this kernel's).
struct FewSeq {
  int row0, n, len;
};
template <int ROWS>
__device__ __forceinline__ FewSeq few_seq(const RaggedParams& r, int b, int strict) {
  FewSeq s;
  s.row0 = __ldg(r.c.cu + b);
  s.n = __ldg(r.c.cu + b + 1) - s.row0;
  s.len = __ldg(r.c.seq_lens + b);
  const long long cap = (long long)r.c.table_width << r.c.page_shift;
  if (s.len > cap) {
    atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    s.len = (int)cap;
  }
  const bool bad = s.row0 < 0 || s.n < 0 || s.n > r.T - s.row0, more = !bad && s.n * r.group > ROWS;
  if (bad || (more && strict)) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
  if (bad || more) s.n = 0;
  return s;
}
// Tiles of one of its heads; a sequence without a key still has rows to set to zero.
template <int KEYS>
__device__ __forceinline__ int few_tiles(const FewSeq& s) {
  return s.n > 0 ? max(1, (s.len + KEYS - 1) / KEYS) : 0;
}

// NT: 8-row tiles of query rows (1 or 2).
template <bool FP8, int NT>
struct FewShape {
  static constexpr int ROWS = 8 * NT;
  static constexpr int KEYS = FP8 ? 128 : 64;            // keys of a tile: 16 KB of K (and of V) either way; e4m3 tiles
                                                         // of 64 keys cost the loading warp its pace (102 us against 88)
  static constexpr int CW = 8;                           // consumer warps
  static constexpr int KW = FP8 || NT == 1 ? 32 : 16;    // keys of a tile that a warp takes (bf16, 16 rows: 16 leaves no spills)
  static constexpr int GROUPS = CW * KW / KEYS;      // groups of warps, a tile each in turn
  static constexpr int TILE = KEYS * HEAD_DIM * (FP8 ? 1 : 2);
  // Stages: a multiple of GROUPS, so that tile i and stage i % S belong to the same group: a group meets every phase of
  // its stages' barriers, and a wait by parity cannot mistake one phase for the one two before it.
  static constexpr int S = FEW_RING / (2 * TILE) / GROUPS * GROUPS;
  static_assert(S >= GROUPS && S > 0, "every group needs a stage");
  // 16 rows need more registers than nine warps can have (168 each: three of them share a scheduler's); with three idle
  // warps beside the loading one the three warpgroups have 384 x 168, which become 256 x 208 and 128 x 88 (16 sequences
  // of 4 tokens at 16k, e4m3: 114 us; 135 without). 8 rows fit.
  static constexpr bool SPLIT = NT == 2;
  static constexpr int THREADS = CW * 32 + (SPLIT ? 128 : 32);
  static constexpr int CONSUMER = 208, PRODUCER = 88;
  static_assert(256 * CONSUMER + 128 * PRODUCER <= 384 * 168, "setmaxnreg would wait for ever");
};
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <bool FP8, int NT>
struct FewSmem {
  using Sh = FewShape<FP8, NT>;
  uint8_t k[Sh::S][Sh::TILE], v[Sh::S][Sh::TILE];
  float sum[Sh::CW][Sh::ROWS][HEAD_DIM + 4];   // the warps' outputs on their way to one
  float ks[FP8 ? Sh::S : 1][Sh::KEYS], vs[FP8 ? Sh::S : 1][Sh::KEYS];
  float wm[Sh::CW][Sh::ROWS], wl[Sh::CW][Sh::ROWS];
  uint64_t full[Sh::S], empty[Sh::S];
  int last;
};

// mbar_wait in fewer instructions, for kernels with many waits in unrolled code (instructions that are not in the cache cost
// a short call most): the clock and the error word are looked at every 256 polls, the limits are the same.
__device__ __forceinline__ bool mbar_wait_small(uint64_t* bar, uint32_t parity, unsigned long long limit_ns = WAIT_LIMIT_NS) {
  unsigned long long t0 = 0;
#pragma unroll 1
  for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i) {
    if (i & 255) continue;
    const unsigned long long now = globaltimer();
    if (t0 == 0) t0 = now;
    if (wait_failed()) return false;
    if (now - t0 > limit_ns) {
      atomicOr(&g_dev_error, DEVERR_MBAR_TIMEOUT);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {   // an 8 x 8 tile of 16-bit values across the warp
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ int add_acq_rel(int* p, int v) {
  int r;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(r) : "l"(p), "r"(v) : "memory");
  return r;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}
template <bool FP8>
__device__ __forceinline__ void few_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (FP8) hmma16816(d, a[0], a[1], a[2], a[3], b0, b1);
  else mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^e of the smallest power of two above |x| (0 for x = 0), as its exponent
__device__ __forceinline__ int exponent_above(float x) {
  const int e = (int)((__float_as_uint(x) >> 23) & 0xff);
  return e == 0 ? -126 : e - 126;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }

__device__ __forceinline__ void few_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }
// The CTA whose range holds tile u, for ranges [c * W / G, (c + 1) * W / G).
__device__ __forceinline__ int owner_of(long long u, long long W, int G) { return (int)(((u + 1) * G - 1) / W); }

template <bool FP8, int NT>
__global__ void __launch_bounds__(FewShape<FP8, NT>::THREADS, 1) few_attention_kernel(const __grid_constant__ FewParams p) {
  using Sh = FewShape<FP8, NT>;
  using Smem = FewSmem<FP8, NT>;
  constexpr int ROWS = Sh::ROWS, CW = Sh::CW, KW = Sh::KW, GROUPS = Sh::GROUPS, S = Sh::S, TILE = Sh::TILE;
  constexpr int KEYS = Sh::KEYS, KT = KW / 16;   // 16-key tiles of M that a warp takes
  extern __shared__ __align__(1024) uint8_t few_smem[];
  Smem& sm = *reinterpret_cast<Smem*>(few_smem);
  const RaggedParams& r = p.r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c = blockIdx.x, n_kv = r.c.n_kv;
  if (tid == 0) {
    prefetch_map(&p.tm_k);
    prefetch_map(&p.tm_v);
    for (int s = 0; s < S; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], KEYS / KW);
    }
    fence_mbar_init();
  }
  grid_dep_wait();
  grid_dep_launch();

  // ---- this CTA's range of tiles: the total, then the sequence its first tile lies in; every warp for itself -----------
  const int per = (r.c.B + 31) / 32;
  long long mine = 0;
  FewSeq s = {0, 0, 0};
  for (int i = lane * per; i < min(r.c.B, (lane + 1) * per); ++i) {
    s = few_seq<ROWS>(r, i, p.strict);
    mine += (long long)few_tiles<KEYS>(s) * n_kv;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  const long long W = __shfl_sync(0xffffffffu, incl, 31);
  const int G = (int)min((long long)gridDim.x, max(1ll, W / FEW_MIN_TILES));   // every CTA below G has a tile
  if (c >= G || W == 0) return;             // (CTA-uniform) nothing to do
  const long long u0 = c * W / G, u1 = (c + 1) * W / G;
  const int owner = __ffs(__ballot_sync(0xffffffffu, incl > u0)) - 1;
  long long start = __shfl_sync(0xffffffffu, incl - mine, owner);
  int b = owner * per;
  if (per == 1) {
    s = {__shfl_sync(0xffffffffu, s.row0, owner), __shfl_sync(0xffffffffu, s.n, owner), __shfl_sync(0xffffffffu, s.len, owner)};
  } else {
    for (;; ++b) {
      s = few_seq<ROWS>(r, b, 0);
      const long long tiles = (long long)few_tiles<KEYS>(s) * n_kv;
      if (u0 < start + tiles) break;
      start += tiles;
    }
  }
  __syncthreads();                          // the barriers are initialised

  // Every warp walks the same pieces: b, its tiles per head, the head, the tiles [t0, t1) of the head.
  int n = few_tiles<KEYS>(s);
  int g = (int)((u0 - start) / n), t0 = (int)((u0 - start) - (long long)g * n);
  const uint32_t bytes_row = FP8 ? HEAD_DIM : 2 * HEAD_DIM;

  if (warp >= CW) {   // ---- producer ----
    if constexpr (Sh::SPLIT) regs_dec<Sh::PRODUCER>();
    if (warp > CW) return;
    const int RB = min(1 << r.c.page_shift, KEYS), boxes = KEYS / RB;
    int it = 0;
    bool ok = true;
    for (long long u = u0; u < u1 && ok;) {
      const int t1 = (int)min((long long)n, t0 + (u1 - u));
      // page numbers of 32 / boxes tiles a load, the next ones on their way: one load a tile would take as long as the
      // tile's whole share of HBM's time
      const int batch = 32 / boxes;
      auto pages_of = [&](int t) {          // lane: box lane % boxes of tile t + lane / boxes; -1 where it holds no key
        const int tile = t + lane / boxes, j = tile * KEYS + (lane % boxes) * RB;
        if (tile >= t1 || j >= s.len) return -1;
        int pg = __ldg(r.c.table + (size_t)b * r.c.table_stride + (j >> r.c.page_shift));
        if (pg < 0 || pg >= r.c.n_pages) {
          atomicOr(&g_dev_error, DEVERR_BAD_STATE);
          pg = 0;
        }
        return pg;
      };
      int cur = pages_of(t0), next = pages_of(t0 + batch), in = 0;
      for (int t = t0; t < t1; ++t, ++it, ++in) {
        const int st = it % S;
        if (in == batch) {
          cur = next;
          next = pages_of(t + batch);
          in = 0;
        }
        const int of_box = __shfl_sync(0xffffffffu, cur, in * boxes + lane % boxes), page = lane < boxes ? of_box : -1;
        if (it >= S) ok = __all_sync(0xffffffffu, mbar_wait_small(&sm.empty[st], (uint32_t)((it / S - 1) & 1)));
        if (!ok) break;
        const int nb = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_arrive_expect_tx(&sm.full[st], (uint32_t)(nb * RB) * (2 * bytes_row + (FP8 ? 8 : 0)));
        __syncwarp();
        if (page >= 0) {
          const int row = ((page * n_kv + g) << r.c.page_shift) + ((t * KEYS + lane * RB) & ((1 << r.c.page_shift) - 1));
          uint8_t *kd = sm.k[st] + lane * RB * 128, *vd = sm.v[st] + lane * RB * 128;
          tma_load_2d(kd, &p.tm_k, 0, row, &sm.full[st]);
          if (!FP8) tma_load_2d(kd + TILE / 2, &p.tm_k, 64, row, &sm.full[st]);
          if (FP8) bulk_g2s(&sm.ks[FP8 ? st : 0][lane * RB], r.c.ks + row, RB * 4, &sm.full[st]);
          tma_load_2d(vd, &p.tm_v, 0, row, &sm.full[st]);
          if (!FP8) tma_load_2d(vd + TILE / 2, &p.tm_v, 64, row, &sm.full[st]);
          if (FP8) bulk_g2s(&sm.vs[FP8 ? st : 0][lane * RB], r.c.vs + row, RB * 4, &sm.full[st]);
        }
      }
      u += t1 - t0;
      t0 = 0;
      if (u < u1 && ++g == n_kv) {
        g = 0;
        do s = few_seq<ROWS>(r, ++b, 0);
        while (few_tiles<KEYS>(s) == 0);
        n = few_tiles<KEYS>(s);
      }
    }
    if (ok)   // the last stages' copies are waited for by the consumers
      return;
    // a wait gave up: let the copies in flight land before the CTA's shared memory goes away
    for (int i = max(0, it - S); i < it; ++i) mbar_wait_small(&sm.full[i % S], (uint32_t)((i / S) & 1), 1000000ull);
    return;
  }

  // ---- consumers ----
  if constexpr (Sh::SPLIT) regs_inc<Sh::CONSUMER>();
  const int grp = warp / (KEYS / KW), part = warp % (KEYS / KW), lg = lane >> 2, lt = lane & 3;
  const float sl2 = r.scale * LOG2E;
  bool ok = true;
  int it = 0;
  for (long long u = u0; u < u1;) {
    const int t1 = (int)min((long long)n, t0 + (u1 - u));
    const int rows = s.n * r.group;
    // the query rows as B fragments: thread (lg, lt) holds row lg of each tile; the dims of its MMA k slots are the ones
    // its 16-byte K chunks below hold
    uint32_t qf[NT][8][2];
    float qs[NT][2];                        // of rows 2 lt, 2 lt + 1: scale * log2 e, fp8: times the power of two that undoes q's
    int lim[NT][2];                         // the last key each of them sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 8 + lg;
      uint4 x[4] = {};
      if (row < rows) {
        const bf16* src = r.q + (long long)(s.row0 + row / r.group) * r.q_row + (long long)(g * r.group + row % r.group) * r.q_head;
#pragma unroll
        for (int i = 0; i < 4; ++i)         // bf16: chunks 2 lt, 2 lt + 1 of each 64-dim half; e4m3: dims 32 lt .. + 31
          x[i] = *reinterpret_cast<const uint4*>(src + (FP8 ? 32 * lt + 8 * i : 64 * (i >> 1) + 16 * lt + 8 * (i & 1)));
      }
      float own = sl2;
      if (FP8) {
        float f[4][8], mx = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          unpack_bf16x8(x[i], f[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(f[i][e]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e2 = min(max(exponent_above(mx), -110), 110);
        const float up = pow2(8 - e2);      // the row's largest value lands in [2^7, 2^8)
        own = sl2 * pow2(e2 - 8);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = make_uint4(pack_f16(f[i][0] * up, f[i][1] * up), pack_f16(f[i][2] * up, f[i][3] * up),
                            pack_f16(f[i][4] * up, f[i][5] * up), pack_f16(f[i][6] * up, f[i][7] * up));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qf[nt][2 * i][0] = x[i].x, qf[nt][2 * i][1] = x[i].y;
        qf[nt][2 * i + 1][0] = x[i].z, qf[nt][2 * i + 1][1] = x[i].w;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qs[nt][e] = __shfl_sync(0xffffffffu, own, (2 * lt + e) * 4);
        lim[nt][e] = min(s.len - 1, s.len - s.n + (nt * 8 + 2 * lt + e) / r.group);
      }
    }
    float o[8][NT][4], m[NT][2], l[NT][2];
    // fp8: the largest weight times V scale of each row so far, under the running maximum; P times the V scale is taken over
    // the power of two above it
    float big[NT][2];
    auto unit = [](float x) { return max(exponent_above(x), -100); };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
      big[nt][0] = big[nt][1] = 0.f;
    }
    for (int t = t0; t < t1; ++t, ++it) {
      if (GROUPS > 1 && it % GROUPS != grp) continue;
      const int st = it % S, j0 = t * KEYS + part * KW;
      ok = __all_sync(0xffffffffu, ok && mbar_wait_small(&sm.full[st], (uint32_t)((it / S) & 1)));
      if (ok && j0 < s.len) {
        const uint32_t kb = smem_u32(sm.k[st]) + (part * KW) * 128, vb = smem_u32(sm.v[st]) + (part * KW) * 128;
        if (j0 + KW > s.len) {              // the sequence ends inside: what lies behind it must not reach P.V, as 0 x NaN
          for (int i = lane; i < (j0 + KW - s.len) * (FP8 ? 8 : 16); i += 32) {
            const int row = (s.len - j0) + i / (FP8 ? 8 : 16), ch = i % (FP8 ? 8 : 16);
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vb + (ch >> 3) * (TILE / 2) + row * 128 + (ch & 7) * 16), "r"(0) : "memory");
          }
          fence_proxy_async_smem();         // the ring's next copy into these rows comes after
          __syncwarp();
        }
        // scores of KT tiles of 16 keys: thread (lg, lt) has keys lg and lg + 8 of query rows 2 lt and 2 lt + 1
        float sc[KT][NT][4];
#pragma unroll
        for (int j = 0; j < KT; ++j) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[j][nt][0] = sc[j][nt][1] = sc[j][nt][2] = sc[j][nt][3] = 0.f;
          const uint32_t ra = kb + (16 * j + lg) * 128;   // row & 7 == lg, of row + 8 too
#pragma unroll
          for (int i = 0; i < (FP8 ? 2 : 4); ++i) {
            const uint32_t at = ra + (FP8 ? 0 : (i >> 1) * (TILE / 2)) + ((2 * lt + (i & 1)) ^ lg) * 16;
            const uint4 w = lds128_at(at), z = lds128_at(at + 8 * 128);
            if (FP8) {
              const uint32_t ww[4] = {w.x, w.y, w.z, w.w}, zz[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t af[4] = {e4m3x2_to_f16x2(ww[e]), e4m3x2_to_f16x2(zz[e]), e4m3x2_to_f16x2(ww[e] >> 16), e4m3x2_to_f16x2(zz[e] >> 16)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) few_mma<FP8>(sc[j][nt], af, qf[nt][4 * i + e][0], qf[nt][4 * i + e][1]);
              }
            } else {
              const uint32_t a0[4] = {w.x, z.x, w.y, z.y}, a1[4] = {w.z, z.z, w.w, z.w};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                few_mma<FP8>(sc[j][nt], a0, qf[nt][2 * i][0], qf[nt][2 * i][1]);
                few_mma<FP8>(sc[j][nt], a1, qf[nt][2 * i + 1][0], qf[nt][2 * i + 1][1]);
              }
            }
          }
        }
        float kscale[KT][2], vscale[KT][2];
        if (FP8) {
#pragma unroll
          for (int j = 0; j < KT; ++j)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const int key = part * KW + 16 * j + 8 * hh + lg;
              kscale[j][hh] = sm.ks[st][key];
              vscale[j][hh] = t * KEYS + key < s.len ? sm.vs[st][key] : 0.f;
            }
        }
        const bool edge = j0 + KW - 1 > s.len - s.n;    // some row does not see some of the keys
        uint32_t pf[KT][NT][2], pl[FP8 ? 1 : KT][NT][2];   // bf16: and what rounding P to it leaves
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = m[nt][e];
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                float& x = sc[j][nt][2 * hh + e];
                x *= FP8 ? qs[nt][e] * kscale[j][hh] : qs[nt][e];
                if (edge && j0 + 16 * j + 8 * hh + lg > lim[nt][e]) x = -INFINITY;
                mx = fmaxf(mx, x);
              }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float base = mx == -INFINITY ? 0.f : mx;
            f[e] = ex2(m[nt][e] - base);
            m[nt][e] = mx;
            float add = 0.f;
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                float& x = sc[j][nt][2 * hh + e];
                x = ex2(x - base);
                add += x;
                if (FP8) x *= vscale[j][hh];
              }
            l[nt][e] = l[nt][e] * f[e] + add;
            if (FP8) {                      // into f16's range, each row by what its own sum is made of
              float top = 0.f;
#pragma unroll
              for (int j = 0; j < KT; ++j) top = fmaxf(top, fmaxf(sc[j][nt][e], sc[j][nt][2 + e]));
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              const int before = unit(big[nt][e]);
              big[nt][e] = fmaxf(big[nt][e] * f[e], top);
              const int now = unit(big[nt][e]);
              f[e] *= pow2(before - now);   // (the exponent falls only as far as f does)
              const float dn = pow2(-now) * 32768.f;
#pragma unroll
              for (int j = 0; j < KT; ++j) sc[j][nt][e] *= dn, sc[j][nt][2 + e] *= dn;
            }
          }
          if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i][nt][0] *= f[0], o[i][nt][1] *= f[1], o[i][nt][2] *= f[0], o[i][nt][3] *= f[1];
          }
#pragma unroll
          for (int j = 0; j < KT; ++j)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const float a = sc[j][nt][2 * hh], e = sc[j][nt][2 * hh + 1];
              const uint32_t p2 = FP8 ? pack_f16(a, e) : pack_bf16(a, e);
              pf[j][nt][hh] = transpose8x8(p2);
              if (!FP8) pl[FP8 ? 0 : j][nt][hh] = transpose8x8(pack_bf16(a - bf16lo(p2), e - bf16hi(p2)));
            }
        }
        // O^T: 8 tiles of 16 dims
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          if (FP8) {                        // row lg of tile i is dim 16 lg + 2 i, row lg + 8 the next: a thread's chunk lg holds all its dims
            uint4 w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = 8 * (k >> 1) + 2 * lt + (k & 1);
              w[k] = lds128_at(vb + (16 * j + row) * 128 + ((lg ^ (row & 7)) * 16));
            }
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              uint32_t a[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) a[k] = q4 == 0 ? w[k].x : q4 == 1 ? w[k].y : q4 == 2 ? w[k].z : w[k].w;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t lo = __byte_perm(a[0], a[1], i ? 0x7362 : 0x5140), hi = __byte_perm(a[2], a[3], i ? 0x7362 : 0x5140);
                const uint32_t af[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2(hi >> 16)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) few_mma<FP8>(o[2 * q4 + i][nt], af, pf[j][nt][0], pf[j][nt][1]);
              }
            }
          } else {                          // row lg of tile i is dim 16 i + lg
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int row = (lane & 7) + 8 * (lane >> 4), ch = (2 * i + ((lane >> 3) & 1)) & 7;
              uint32_t af[4];
              ldmatrix4_trans(af, vb + (i >> 2) * (TILE / 2) + (16 * j + row) * 128 + ((ch ^ (row & 7)) * 16));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                few_mma<FP8>(o[i][nt], af, pf[j][nt][0], pf[j][nt][1]);
                few_mma<FP8>(o[i][nt], af, pl[FP8 ? 0 : j][nt][0], pl[FP8 ? 0 : j][nt][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[st]);
    }

    // ---- the warps' sums become one, then the output or a partial --------------------------------------------------
    const long long unit0 = u - t0;         // the unit's first tile
    const bool whole = t1 - t0 == n;
    const int cf = owner_of(unit0, W, G), cl = owner_of(unit0 + n - 1, W, G);
    const int slot = u == u0 ? 0 : 1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
        if (lg == 0) sm.wm[warp][nt * 8 + 2 * lt + e] = m[nt][e], sm.wl[warp][nt * 8 + 2 * lt + e] = l[nt][e];
      }
    few_sync(CW * 32);
    float f[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < CW; ++w) M = fmaxf(M, sm.wm[w][nt * 8 + 2 * lt + e]);
        f[nt][e] = M == -INFINITY ? 1.f : ex2(m[nt][e] - M);
        if (FP8) f[nt][e] *= pow2(unit(big[nt][e])) * (1.f / 32768.f);
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = FP8 ? 16 * lg + 2 * i + (e >> 1) : 16 * i + 8 * (e >> 1) + lg;
          sm.sum[warp][nt * 8 + 2 * lt + (e & 1)][d] = o[i][nt][e] * f[nt][e & 1];
        }
    few_sync(CW * 32);
    // thread: 8 dims of a row (16 threads a row)
    for (int i = tid; i < rows * 16; i += CW * 32) {
      const int row = i >> 4, d0 = (i & 15) * 8;
      float x[8] = {};
#pragma unroll
      for (int w = 0; w < CW; ++w) {
        const float4 a = *reinterpret_cast<const float4*>(&sm.sum[w][row][d0]), e = *reinterpret_cast<const float4*>(&sm.sum[w][row][d0 + 4]);
        x[0] += a.x, x[1] += a.y, x[2] += a.z, x[3] += a.w, x[4] += e.x, x[5] += e.y, x[6] += e.z, x[7] += e.w;
      }
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < CW; ++w) M = fmaxf(M, sm.wm[w][row]);
#pragma unroll
      for (int w = 0; w < CW; ++w) L += M == -INFINITY ? sm.wl[w][row] : sm.wl[w][row] * ex2(sm.wm[w][row] - M);
      if (whole) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= inv;
        *reinterpret_cast<uint4*>(r.out + (long long)(s.row0 + row / r.group) * r.out_row +
                                  (long long)(g * r.group + row % r.group) * r.out_head + d0) = pack_bf16x8(x);
      } else {
        const size_t at = (size_t)(c * 2 + slot) * ROWS + row;
        *reinterpret_cast<float4*>(p.part + at * HEAD_DIM + d0) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p.part + at * HEAD_DIM + d0 + 4) = make_float4(x[4], x[5], x[6], x[7]);
        if (d0 == 0) *reinterpret_cast<float2*>(p.ml + at * 2) = make_float2(M, L);
      }
    }
    few_sync(CW * 32);                      // sum, wm and wl are free again
    if (!whole) {
      if (tid == 0) {                       // releases the CTA's stores (ordered before by few_sync), acquires the others'
        const int before = add_acq_rel(p.counters + cf, 1);
        sm.last = before == cl - cf;
        if (sm.last) p.counters[cf] = 0;
      }
      few_sync(CW * 32);
      if (sm.last) {                        // every piece is there: add them, Q threads a row and 8 dims, in a fixed order
        const int T = CW * 32, items = rows * 16, Q = max(1, min(CW, T / items));
        for (int i = tid; i < items * Q; i += T) {
          const int q = i / items, row = i / 16 % rows, d0 = (i & 15) * 8;
          auto at_of = [&](int cc) {        // the unit is CTA cc's first one, unless it begins inside the first owner's range
            return (size_t)(cc * 2 + (cc == cf && cc * W / G != unit0 ? 1 : 0)) * ROWS + row;
          };
          float M = -INFINITY, L = 0.f, x[8] = {};
#pragma unroll 4
          for (int cc = cf + q; cc <= cl; cc += Q) {
            const size_t at = at_of(cc);
            const float2 mlv = __ldcg(reinterpret_cast<const float2*>(p.ml + at * 2));
            const float4 a = __ldcg(reinterpret_cast<const float4*>(p.part + at * HEAD_DIM + d0));
            const float4 e = __ldcg(reinterpret_cast<const float4*>(p.part + at * HEAD_DIM + d0 + 4));
            const float mn = fmaxf(M, mlv.x), f0 = M == -INFINITY ? 1.f : ex2(M - mn), f = mlv.x == -INFINITY ? 1.f : ex2(mlv.x - mn);
            M = mn;
            L = L * f0 + mlv.y * f;
            x[0] = x[0] * f0 + a.x * f, x[1] = x[1] * f0 + a.y * f, x[2] = x[2] * f0 + a.z * f, x[3] = x[3] * f0 + a.w * f;
            x[4] = x[4] * f0 + e.x * f, x[5] = x[5] * f0 + e.y * f, x[6] = x[6] * f0 + e.z * f, x[7] = x[7] * f0 + e.w * f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) sm.sum[q][row][d0 + e] = x[e];
          if (d0 == 0) sm.wm[q][row] = M, sm.wl[q][row] = L;
        }
        few_sync(T);
        for (int i = tid; i < items; i += T) {
          const int row = i / 16, d0 = (i & 15) * 8;
          float M = -INFINITY, L = 0.f, x[8] = {};
          for (int q = 0; q < Q; ++q) M = fmaxf(M, sm.wm[q][row]);
          for (int q = 0; q < Q; ++q) {
            const float f = sm.wm[q][row] == -INFINITY ? 1.f : ex2(sm.wm[q][row] - M);
            L += sm.wl[q][row] * f;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] += sm.sum[q][row][d0 + e] * f;
          }
          const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= inv;
          *reinterpret_cast<uint4*>(r.out + (long long)(s.row0 + row / r.group) * r.out_row +
                                    (long long)(g * r.group + row % r.group) * r.out_head + d0) = pack_bf16x8(x);
        }
        few_sync(T);
      }
    }
    u += t1 - t0;
    t0 = 0;
    if (u < u1 && ++g == n_kv) {
      g = 0;
      do s = few_seq<ROWS>(r, ++b, 0);
      while (few_tiles<KEYS>(s) == 0);
      n = few_tiles<KEYS>(s);
    }
  }
  if (!ok && lane == 0) atomicOr(&g_dev_error, DEVERR_MBAR_TIMEOUT);
}

}  // namespace qk

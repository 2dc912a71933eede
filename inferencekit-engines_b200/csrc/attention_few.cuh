// Paged attention for few query rows: the decode step's one token, or a handful (speculated tokens), per sequence.
//
//   out[t][h] = sum over j <= pos(t) of softmax_j(scale * q[t][h] . K[g][j]) V[g][j]
//
// Bound by the cache bytes: up to 32 query rows (tokens x heads of a KV head) meet each K and V row once, so the only
// aim is to keep HBM busy.
//  * Work: the (sequence, KV head, 64-key tile) triples, tile-major, are dealt in equal contiguous ranges to one CTA
//    per SM, whatever the lengths are: a 32k context beside short ones leaves no SM idle. A unit (sequence, head)
//    split between CTAs leaves fp32 partials (o, m, l); the CTA that completes the unit's count adds them in CTA
//    order (the same bits every run).
//  * A producer warp keeps a ring of 192 KB of tiles in flight: TMA boxes of one page's rows each, 128-byte
//    swizzle, so every shared-memory read below is free of bank conflicts.
//  * Eight consumer warps (four for 17 to 32 rows): 16 keys of a tile each, and each its own running softmax and
//    output registers, so nothing waits on a neighbour until the piece ends. Scores and P.V are warp-level MMAs
//    (m16n8k16) with the query rows as M: the tensor work is some 5 % of what these units do, while a 128-row
//    tcgen05 tile would hold 4 rows in use and pass every score through TMEM.
//  * bf16 cache: bf16 MMAs, P rounded to bf16. e4m3 cache: the bytes become f16 exactly; q is scaled to f16 range by
//    a power of two per row; the K scale multiplies the score in fp32; P times the V scale is brought into f16 range
//    by a running power of two, 2^15 at most, so what falls below f16's smallest value is below 2^-39 of the row's
//    largest weight.
#pragma once
#include "gemm_tc.cuh"     // tma_load_2d
#include "paged.cuh"

namespace qk {

constexpr int FEW_KEYS = 64;          // keys of a tile
constexpr int FEW_RING = 196608;      // bytes of K and V in the ring
constexpr int FEW_MIN_TILES = 1;      // a CTA's least share
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
  CUtensorMap tm_k, tm_v;   // the pools as [n_pages * n_kv * page_size] rows: box {128 bytes, min(page_size, 64) rows}
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
__device__ __forceinline__ int few_tiles(const FewSeq& s) {
  return s.n > 0 ? max(1, (s.len + FEW_KEYS - 1) / FEW_KEYS) : 0;
}

template <bool FP8>
struct FewSmem {
  static constexpr int TILE = FEW_KEYS * HEAD_DIM * (FP8 ? 1 : 2);
  static constexpr int S = FEW_RING / (2 * TILE);
  // Even, so that tile i and stage i % S belong to the same group of warps (i & 1): a group meets every phase of its
  // stages' barriers, and a wait by parity cannot mistake one phase for the one two before it.
  static_assert(S % 2 == 0, "a stage must stay with one group of consumer warps");
  uint8_t k[S][TILE], v[S][TILE];
  float sum[2][16][HEAD_DIM + 4];       // the warps' outputs on their way to one
  float ks[FP8 ? S : 1][FEW_KEYS], vs[FP8 ? S : 1][FEW_KEYS];
  float wm[8][16], wl[8][16];
  uint64_t full[S], empty[S];
  long long chunk[288], total, start_prefix;
  int start_b, last;
};

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

// MT: 16-row M tiles (1 or 2).
__device__ __forceinline__ void few_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }
// The CTA whose range holds tile u, for ranges [c * W / G, (c + 1) * W / G).
__device__ __forceinline__ int owner_of(long long u, long long W, int G) { return (int)(((u + 1) * G - 1) / W); }

template <bool FP8, int MT>
__global__ void __launch_bounds__(MT == 1 ? 288 : 160, 1) few_attention_kernel(const __grid_constant__ FewParams p) {
  constexpr int ROWS = 16 * MT, CW = MT == 1 ? 8 : 4, GROUPS = CW / 4, THREADS = CW * 32 + 32;
  using Smem = FewSmem<FP8>;
  constexpr int S = Smem::S, TILE = Smem::TILE;
  extern __shared__ __align__(1024) uint8_t few_smem[];
  Smem& sm = *reinterpret_cast<Smem*>(few_smem);
  const RaggedParams& r = p.r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c = blockIdx.x, n_kv = r.c.n_kv;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 4);
    }
    fence_mbar_init();
  }
  grid_dep_wait();
  grid_dep_launch();

  // ---- this CTA's range of tiles: the total, then the sequence its first tile lies in -----------------------------
  const int per = (r.c.B + THREADS - 1) / THREADS;
  long long mine = 0;
  for (int b = tid * per; b < min(r.c.B, (tid + 1) * per); ++b) mine += (long long)few_tiles(few_seq<ROWS>(r, b, p.strict)) * n_kv;
  sm.chunk[tid] = mine;
  __syncthreads();
  if (warp == 0) {                          // inclusive sums over the threads' chunks
    long long at = 0;
    for (int i = 0; i < THREADS; i += 32) {
      long long v = sm.chunk[i + lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      sm.chunk[i + lane] = at + v;
      at += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) sm.total = at;
  }
  __syncthreads();
  const long long W = sm.total;
  const int G = (int)min((long long)gridDim.x, max(1ll, W / FEW_MIN_TILES));   // every CTA below G has a tile
  const long long u0 = c * W / G, u1 = (c + 1) * W / G;
  if (c >= G || W == 0) return;             // (CTA-uniform) nothing to do
  if (sm.chunk[tid] - mine <= u0 && u0 < sm.chunk[tid]) {   // exactly one thread
    long long at = sm.chunk[tid] - mine;
    int b = tid * per;
    for (;; ++b) {
      const long long n = (long long)few_tiles(few_seq<ROWS>(r, b, 0)) * n_kv;
      if (u0 < at + n) break;
      at += n;
    }
    sm.start_b = b;
    sm.start_prefix = at;
  }
  __syncthreads();

  // Every warp walks the same pieces: b, its tiles per head, the head, the tiles [t0, t1) of the head.
  int b = sm.start_b;
  FewSeq s = few_seq<ROWS>(r, b, 0);
  int n = few_tiles(s);
  int g = (int)((u0 - sm.start_prefix) / n), t0 = (int)((u0 - sm.start_prefix) - (long long)g * n);
  const uint32_t bytes_row = FP8 ? HEAD_DIM : 2 * HEAD_DIM;

  if (warp == CW) {   // ---- producer ----
    const int RB = min(1 << r.c.page_shift, FEW_KEYS), boxes = FEW_KEYS / RB;
    int it = 0;
    bool ok = true;
    for (long long u = u0; u < u1 && ok;) {
      const int t1 = (int)min((long long)n, t0 + (u1 - u));
      auto page_of = [&](int t) {           // this lane's box of tile t: its page, -1 where it holds no key
        const int j = t * FEW_KEYS + lane * RB;
        if (lane >= boxes || j >= s.len) return -1;
        int pg = __ldg(r.c.table + (size_t)b * r.c.table_stride + (j >> r.c.page_shift));
        if (pg < 0 || pg >= r.c.n_pages) {
          atomicOr(&g_dev_error, DEVERR_BAD_STATE);
          pg = 0;
        }
        return pg;
      };
      int next = page_of(t0);
      for (int t = t0; t < t1; ++t, ++it) {
        const int st = it % S, page = next;
        if (t + 1 < t1) next = page_of(t + 1);
        if (it >= S) ok = __all_sync(0xffffffffu, mbar_wait(&sm.empty[st], (uint32_t)((it / S - 1) & 1)));
        if (!ok) break;
        const int nb = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_arrive_expect_tx(&sm.full[st], (uint32_t)(nb * RB) * (2 * bytes_row + (FP8 ? 8 : 0)));
        __syncwarp();
        if (page >= 0) {
          const int row = ((page * n_kv + g) << r.c.page_shift) + ((t * FEW_KEYS + lane * RB) & ((1 << r.c.page_shift) - 1));
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
        while (few_tiles(s) == 0);
        n = few_tiles(s);
      }
    }
    if (ok)   // the last stages' copies are waited for by the consumers
      return;
    // a wait gave up: let the copies in flight land before the CTA's shared memory goes away
    for (int i = max(0, it - S); i < it; ++i) mbar_wait(&sm.full[i % S], (uint32_t)((i / S) & 1), 1000000ull);
    return;
  }

  // ---- consumers ----
  const int grp = warp / 4, quarter = warp & 3, lg = lane >> 2, lt = lane & 3;   // keys 16 * quarter .. + 15 of a tile
  const float sl2 = r.scale * LOG2E;
  bool ok = true;
  int it = 0;
  for (long long u = u0; u < u1;) {
    const int t1 = (int)min((long long)n, t0 + (u1 - u));
    const int rows = s.n * r.group;
    // the query rows as A fragments: thread (lg, lt) holds rows lg and lg + 8; the dims of its MMA k slots are the ones
    // its 16-byte K chunks below hold
    uint32_t qf[MT][8][4];
    float qs[MT][2];                        // fp8: the power of two that undoes the row's scaling, times scale * log2 e
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = mt * 16 + hh * 8 + lg;
        uint4 x[4] = {};
        if (row < rows) {
          const bf16* src = r.q + (long long)(s.row0 + row / r.group) * r.q_row + (long long)(g * r.group + row % r.group) * r.q_head;
#pragma unroll
          for (int i = 0; i < 4; ++i)       // bf16: chunks 2 lt, 2 lt + 1 of each 64-dim half; e4m3: dims 32 lt .. + 31
            x[i] = *reinterpret_cast<const uint4*>(src + (FP8 ? 32 * lt + 8 * i : 64 * (i >> 1) + 16 * lt + 8 * (i & 1)));
        }
        qs[mt][hh] = sl2;
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
          const float up = pow2(8 - e2);    // the row's largest value lands in [2^7, 2^8)
          qs[mt][hh] = sl2 * pow2(e2 - 8);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[i] = make_uint4(pack_f16(f[i][0] * up, f[i][1] * up), pack_f16(f[i][2] * up, f[i][3] * up),
                              pack_f16(f[i][4] * up, f[i][5] * up), pack_f16(f[i][6] * up, f[i][7] * up));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qf[mt][2 * i][hh] = x[i].x, qf[mt][2 * i][2 + hh] = x[i].y;
          qf[mt][2 * i + 1][hh] = x[i].z, qf[mt][2 * i + 1][2 + hh] = x[i].w;
        }
      }
    int lim[MT][2];                         // the last key each row sees
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) lim[mt][hh] = min(s.len - 1, s.len - s.n + (mt * 16 + hh * 8 + lg) / r.group);
    float o[MT][16][4], m[MT][2], l[MT][2];
    int ev = -100;                          // fp8: P is multiplied by the V scale over 2^ev
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f;
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.f;
    }
    for (int t = t0; t < t1; ++t, ++it) {
      if (GROUPS == 2 && (it & 1) != grp) continue;
      const int st = it % S, j0 = t * FEW_KEYS + quarter * 16;
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&sm.full[st], (uint32_t)((it / S) & 1)));
      if (ok && j0 < s.len) {
        const uint32_t kb = smem_u32(sm.k[st]) + (quarter * 16) * 128, vb = smem_u32(sm.v[st]) + (quarter * 16) * 128;
        if (j0 + 16 > s.len) {              // the sequence ends inside: what lies behind it must not reach P.V, as 0 x NaN
          for (int i = lane; i < (j0 + 16 - s.len) * (FP8 ? 8 : 16); i += 32) {
            const int row = (s.len - j0) + i / (FP8 ? 8 : 16), ch = i % (FP8 ? 8 : 16);
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vb + (ch >> 3) * (TILE / 2) + row * 128 + (ch & 7) * 16), "r"(0) : "memory");
          }
          fence_proxy_async_smem();         // the ring's next copy into these rows comes after
          __syncwarp();
        }
        // scores: two 8-key tiles
        float sc[MT][2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) sc[mt][j][0] = sc[mt][j][1] = sc[mt][j][2] = sc[mt][j][3] = 0.f;
          const uint32_t ra = kb + (8 * j + lg) * 128;   // row & 7 == lg
#pragma unroll
          for (int i = 0; i < (FP8 ? 2 : 4); ++i) {
            const int ch = (2 * lt + (i & 1)) ^ lg;
            const uint4 w = lds128_at(ra + (FP8 ? 0 : (i >> 1) * (TILE / 2)) + ch * 16);
            if (FP8) {
              const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t b0 = e4m3x2_to_f16x2(ww[e]), b1 = e4m3x2_to_f16x2(ww[e] >> 16);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) few_mma<FP8>(sc[mt][j], qf[mt][4 * i + e], b0, b1);
              }
            } else {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                few_mma<FP8>(sc[mt][j], qf[mt][2 * i], w.x, w.y);
                few_mma<FP8>(sc[mt][j], qf[mt][2 * i + 1], w.z, w.w);
              }
            }
          }
        }
        float kscale[2][2], vscale[2][2];
        if (FP8) {
          float vmax = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = quarter * 16 + 8 * j + 2 * lt + e;
              kscale[j][e] = sm.ks[st][key];
              vscale[j][e] = t * FEW_KEYS + key < s.len ? sm.vs[st][key] : 0.f;
              vmax = fmaxf(vmax, vscale[j][e]);
            }
          vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 1));
          vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
          const int e2 = exponent_above(vmax);   // the same in every lane
          if (e2 > ev) {
            const float f = pow2(ev - e2);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[mt][i][0] *= f, o[mt][i][1] *= f, o[mt][i][2] *= f, o[mt][i][3] *= f;
            ev = e2;
          }
          const float dn = pow2(-ev);
#pragma unroll
          for (int j = 0; j < 2; ++j) vscale[j][0] *= dn * 32768.f, vscale[j][1] *= dn * 32768.f;
        }
        const bool edge = j0 + 15 > s.len - s.n;        // some row does not see some of the 16 keys
        uint32_t pf[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float f[2];
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float raw = sc[mt][j][2 * hh + e] * qs[mt][hh];
                x[2 * j + e] = FP8 ? raw * kscale[j][e] : raw;
                if (edge && j0 + 8 * j + 2 * lt + e > lim[mt][hh]) x[2 * j + e] = -INFINITY;
              }
            float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m[mt][hh], mx), base = mn == -INFINITY ? 0.f : mn;
            f[hh] = ex2(m[mt][hh] - base);
            m[mt][hh] = mn;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = ex2(x[e] - base);
            l[mt][hh] = l[mt][hh] * f[hh] + ((x[0] + x[1]) + (x[2] + x[3]));
#pragma unroll
            for (int j = 0; j < 2; ++j)
              pf[mt][2 * j + hh] = FP8 ? pack_f16(x[2 * j] * vscale[j][0], x[2 * j + 1] * vscale[j][1]) : pack_bf16(x[2 * j], x[2 * j + 1]);
          }
          if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[mt][i][0] *= f[0], o[mt][i][1] *= f[0], o[mt][i][2] *= f[1], o[mt][i][3] *= f[1];
          }
        }
        // P.V: 16 tiles of 8 output columns
        if (FP8) {                          // column n of tile i is dim 16 n + i: a thread's chunk lg holds all its tiles
          uint4 w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = 8 * (j >> 1) + 2 * lt + (j & 1);
            w[j] = lds128_at(vb + row * 128 + ((lg ^ (row & 7)) * 16));
          }
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const uint32_t a[4] = {q4 == 0 ? w[0].x : q4 == 1 ? w[0].y : q4 == 2 ? w[0].z : w[0].w,
                                   q4 == 0 ? w[1].x : q4 == 1 ? w[1].y : q4 == 2 ? w[1].z : w[1].w,
                                   q4 == 0 ? w[2].x : q4 == 1 ? w[2].y : q4 == 2 ? w[2].z : w[2].w,
                                   q4 == 0 ? w[3].x : q4 == 1 ? w[3].y : q4 == 2 ? w[3].z : w[3].w};
            const uint32_t lo0 = __byte_perm(a[0], a[1], 0x5140), hi0 = __byte_perm(a[0], a[1], 0x7362);
            const uint32_t lo1 = __byte_perm(a[2], a[3], 0x5140), hi1 = __byte_perm(a[2], a[3], 0x7362);
            const uint32_t b0[4] = {e4m3x2_to_f16x2(lo0), e4m3x2_to_f16x2(lo0 >> 16), e4m3x2_to_f16x2(hi0), e4m3x2_to_f16x2(hi0 >> 16)};
            const uint32_t b1[4] = {e4m3x2_to_f16x2(lo1), e4m3x2_to_f16x2(lo1 >> 16), e4m3x2_to_f16x2(hi1), e4m3x2_to_f16x2(hi1 >> 16)};
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) few_mma<FP8>(o[mt][4 * q4 + e], pf[mt], b0[e], b1[e]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const int row = lane & 15, ch = (i + (lane >> 4)) & 7;
            uint32_t w[4];
            ldmatrix4_trans(w, vb + (i >> 3) * (TILE / 2) + row * 128 + ((ch ^ (row & 7)) * 16));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              few_mma<FP8>(o[mt][i], pf[mt], w[0], w[1]);
              few_mma<FP8>(o[mt][i + 1], pf[mt], w[2], w[3]);
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
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        l[mt][hh] += __shfl_xor_sync(0xffffffffu, l[mt][hh], 1);
        l[mt][hh] += __shfl_xor_sync(0xffffffffu, l[mt][hh], 2);
        if (lt == 0) sm.wm[warp][hh * 8 + lg] = m[mt][hh], sm.wl[warp][hh * 8 + lg] = l[mt][hh];
      }
      few_sync(CW * 32);
      float f[2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < CW; ++w) M = fmaxf(M, sm.wm[w][hh * 8 + lg]);
        f[hh] = M == -INFINITY ? 1.f : ex2(m[mt][hh] - M);
        if (FP8) f[hh] *= pow2(ev) * (1.f / 32768.f);
      }
      auto put = [&](float (&dst)[16][HEAD_DIM + 4], bool add) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = FP8 ? 16 * (2 * lt + (e & 1)) + i : 8 * i + 2 * lt + (e & 1);
            float& x = dst[(e >> 1) * 8 + lg][d];
            const float y = o[mt][i][e] * f[e >> 1];
            x = add ? x + y : y;
          }
      };
#pragma unroll
      for (int w = CW - 2; w >= 0; w -= 2) {  // two warps at a time
        if ((warp & ~1) == w) put(sm.sum[warp & 1], w != CW - 2);
        few_sync(CW * 32);
      }
      // thread: 8 dims of a row (16 threads a row)
      for (int i = tid; i < 16 * 16; i += CW * 32) {
        const int rr = i >> 4, d0 = (i & 15) * 8, row = mt * 16 + rr;
        if (row >= rows) continue;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = sm.sum[0][rr][d0 + e] + sm.sum[1][rr][d0 + e];
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < CW; ++w) M = fmaxf(M, sm.wm[w][rr]);
#pragma unroll
        for (int w = 0; w < CW; ++w) L += M == -INFINITY ? sm.wl[w][rr] : sm.wl[w][rr] * ex2(sm.wm[w][rr] - M);
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
      few_sync(CW * 32);                    // sum, wm and wl are free again
    }
    if (!whole) {
      __threadfence();
      few_sync(CW * 32);
      if (tid == 0) {
        const int before = atomicAdd(p.counters + cf, 1);
        sm.last = before == cl - cf;
        if (sm.last) {
          __threadfence();
          p.counters[cf] = 0;
        }
      }
      few_sync(CW * 32);
      if (sm.last) {                        // every piece is there: add them in CTA order
        for (int i = tid; i < rows * 16; i += CW * 32) {
          const int row = i >> 4, d0 = (i & 15) * 8;
          float M = -INFINITY, L = 0.f, x[8] = {};
          auto at_of = [&](int cc) {        // the unit is CTA cc's first one, unless it begins inside the first owner's range
            return (size_t)(cc * 2 + (cc == cf && cc * W / G != unit0 ? 1 : 0)) * ROWS + row;
          };
          for (int cc = cf; cc <= cl; ++cc) M = fmaxf(M, __ldcg(p.ml + at_of(cc) * 2));
          for (int cc = cf; cc <= cl; ++cc) {
            const size_t at = at_of(cc);
            const float2 mlv = __ldcg(reinterpret_cast<const float2*>(p.ml + at * 2));
            const float4 a = __ldcg(reinterpret_cast<const float4*>(p.part + at * HEAD_DIM + d0));
            const float4 e = __ldcg(reinterpret_cast<const float4*>(p.part + at * HEAD_DIM + d0 + 4));
            const float f = M == -INFINITY ? 1.f : ex2(mlv.x - M);
            L += mlv.y * f;
            x[0] += a.x * f, x[1] += a.y * f, x[2] += a.z * f, x[3] += a.w * f;
            x[4] += e.x * f, x[5] += e.y * f, x[6] += e.z * f, x[7] += e.w * f;
          }
          const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= inv;
          *reinterpret_cast<uint4*>(r.out + (long long)(s.row0 + row / r.group) * r.out_row +
                                    (long long)(g * r.group + row % r.group) * r.out_head + d0) = pack_bf16x8(x);
        }
      }
    }
    u += t1 - t0;
    t0 = 0;
    if (u < u1 && ++g == n_kv) {
      g = 0;
      do s = few_seq<ROWS>(r, ++b, 0);
      while (few_tiles(s) == 0);
      n = few_tiles(s);
    }
  }
  if (!ok && lane == 0) atomicOr(&g_dev_error, DEVERR_MBAR_TIMEOUT);
}

}  // namespace qk

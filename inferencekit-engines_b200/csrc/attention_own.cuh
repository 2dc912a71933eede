// Attention of sequences that share their first positions (shared_attention): what is not the tensor-core kernel's.
//
//   out[t][h] = (sum over the prefix's keys + sum over the sequence's own keys of w_j V_j) / (the same sums of w_j),
//   w_j = exp2(scale log2 e q . K_j - m), each part under its own maximum m
//
// Three launches, each of which starts as the one before it leaves the SMs:
//  * the sequences' own keys. They are few and short beside the prefix, and what costs is each unit's chain of latencies (lengths,
//    pages, rows of q, the first tile, the sums' way out). So a warp is a CTA of its own here, with a ring of its own: six on an SM
//    hide each other's chains. (64 sequences of up to 500 keys and 8 KV heads: 22 us; the few-row kernel, whose eight warps take
//    each unit together, 40 out of a cold cache.)
//    Prefixes of groups with few query rows are sequences like these, in blocks of 16 rows.
//  * the prefixes of larger groups (attention_tc.cuh): a group's rows, as one sequence's, over the keys they share, read once;
//  * prefix_merge_kernel: a row's sums over its own keys and its prefix, in pieces where CTAs or warps shared them out, become the output.
#pragma once
#include "attention_few.cuh"

namespace qk {

// Sums (o under a maximum m in log2 units, and l) of row t, head h at t * n_q + h: over its own keys where one warp or CTA took them
// all, and over its prefix, in 1, 2 or 4 parts, where one CTA did. In blocks, so that where a row's are goes by its number alone: calls
// of any shape, on any part of a workspace, find info as the last one left it.
constexpr int SHARED_BLOCK = 1024;
struct SharedRows {
  float own_o[SHARED_BLOCK][HEAD_DIM], o[SHARED_BLOCK][4][HEAD_DIM];
  float2 own_ml[SHARED_BLOCK], ml[SHARED_BLOCK][4];
  int own_info[SHARED_BLOCK], info[SHARED_BLOCK];   // what the kernels left (OWN_*, PREFIX_*), zero between launches
};
struct SharedParams {
  const int* groups;        // [G + 1]: group g is the sequences groups[g] .. groups[g + 1] - 1
  const int* shared;        // [G]: positions that they have in common
  int G;
  SharedRows* rows;
  __device__ __forceinline__ float* own_o(int at) const { return rows[(unsigned)at / SHARED_BLOCK].own_o[(unsigned)at % SHARED_BLOCK]; }
  __device__ __forceinline__ float* o(int at, int part) const { return rows[(unsigned)at / SHARED_BLOCK].o[(unsigned)at % SHARED_BLOCK][part]; }
  __device__ __forceinline__ float2* own_ml(int at) const { return &rows[(unsigned)at / SHARED_BLOCK].own_ml[(unsigned)at % SHARED_BLOCK]; }
  __device__ __forceinline__ float2* ml(int at, int part) const { return &rows[(unsigned)at / SHARED_BLOCK].ml[(unsigned)at % SHARED_BLOCK][part]; }
  __device__ __forceinline__ int* own_info(int at) const { return &rows[(unsigned)at / SHARED_BLOCK].own_info[(unsigned)at % SHARED_BLOCK]; }
  __device__ __forceinline__ int* info(int at) const { return &rows[(unsigned)at / SHARED_BLOCK].info[(unsigned)at % SHARED_BLOCK]; }
  float* part;              // the prefixes' pieces, as in the tensor-core kernel, with maxima in log2 units
  float* part_ml;
  float* own_part;          // own keys' pieces: [warp][2][16 rows][128]
  float2* own_part_ml;      // [warp][2][16 rows]
};
// info: the CTAs first .. last that have pieces (bits 0-7 and 8-15; the first one's second piece, the others' first), the row of a
// tile pair that has the row's first part (16-23), parts as a power of two (24-25), and one of these. 0: nothing.
constexpr int PREFIX_WHOLE = 1 << 26, PREFIX_PIECES = 1 << 27, PREFIX_WARPS = 1 << 28;   // the last: the rest is as in own_info
// own_info: the warps first .. last that have pieces (0-9 and 10-19), the row of the block (20-23), whether the first one's is its
// second piece (24), and one of these. 0: the output is written.
constexpr int OWN_SUMS = 1 << 25, OWN_PIECES = 1 << 26;
constexpr int SHARED_TILE = 128;      // a prefix is cut to whole key tiles: what is left of it is read with a sequence's own keys
constexpr int SHARED_MIN_KEYS = 256;  // shorter ones too
// The tensor cores' launch pays where it saves so many reads of a key (for one KV head) in all: it and the merge of its sums take some
// 10 us, and a shared page that is read again comes out of the L2 cache. Measured, shared against not: 16 sequences behind
// 2,048 keys (246,000 reads) 25 us against 27; 64 behind 512 (258,000) 33 against 32; 8 groups of 8 behind 512 (229,000) 31
// against 33, behind 1,024 38 against 47; e4m3 pages alike. (So near the border it is wrong by 1 or 2 us either way: the number of reads
// does not say it all.)
constexpr long long SHARED_MIN_READS = 240000;
// A prefix that the warps take is read once for every 16 rows (the second time out of the L2 cache): those of one block of rows, and of
// up to four where that is few reads in all. Measured, warps against tensor cores: 8 sequences behind 4,096 keys (65,000 reads) 25 us against
// 33, 16 (131,000) 27 against 31, 8 groups of 8 (524,000) 71 against 59, 8 of 4 (one block) 48 against 55.
constexpr long long OWN_PREFIX_READS = 200000;
struct SharedGroup {
  int first, end, keys;               // its sequences; the keys that are read once
  int row0, n;                        // their rows
  bool warps;                         // whether the prefix is the warps'
};
// `large`: whether prefixes that are not the warps' are shared at all.
__device__ __forceinline__ SharedGroup shared_group(const SharedParams& x, const RaggedParams& r, int g, bool large) {
  const PagedCache& c = r.c;
  SharedGroup s = {__ldg(x.groups + g), __ldg(x.groups + g + 1), __ldg(x.shared + g), 0, 0, false};
  bool bad = s.first < 0 || s.end < s.first || s.end > c.B || s.keys < 0 || s.keys > (long long)c.table_width << c.page_shift;
  s.keys = bad || s.end - s.first < 2 || s.keys < SHARED_MIN_KEYS ? 0 : s.keys / SHARED_TILE * SHARED_TILE;
  if (s.keys) {
    s.row0 = __ldg(c.cu + s.first);
    s.n = __ldg(c.cu + s.end) - s.row0;
    if (s.row0 < 0 || s.n < 0 || s.n > r.T - s.row0) bad = true, s.keys = s.n = 0;
    const int blocks = (s.n * r.group + 15) / 16;
    s.warps = blocks <= 1 || (blocks <= 4 && (long long)blocks * s.keys * c.n_kv * x.G <= OWN_PREFIX_READS);
    if (!s.warps && !large) s.keys = 0;
  }
  if (bad) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
  return s;
}
// Reads that a large prefix saves: a sequence's own keys are read once for each 16 of its rows.
__device__ __forceinline__ long long saved_reads(const SharedGroup& s, const RaggedParams& r) {
  return s.keys && !s.warps ? (long long)(max(s.end - s.first, s.n * r.group / 16) - 1) * s.keys * r.c.n_kv : 0;
}
// Whether what the large prefixes save is worth their launch; a whole warp.
__device__ __forceinline__ bool large_prefixes(const SharedParams& x, const RaggedParams& r, int lane) {
  long long reads = 0;
  for (int g = lane; g < x.G; g += 32) reads += saved_reads(shared_group(x, r, g, true), r);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) reads += __shfl_xor_sync(0xffffffffu, reads, o);
  return reads >= SHARED_MIN_READS;
}
// The keys of sequence b that its group's prefix has.
__device__ __forceinline__ int shared_keys(const SharedParams& x, const RaggedParams& r, int b, bool large) {
  int lo = 0, hi = x.G;                // the group: the last one that begins at or before b
  if (hi == 0) return 0;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (__ldg(x.groups + mid) <= b) lo = mid;
    else hi = mid;
  }
  const SharedGroup s = shared_group(x, r, lo, large);
  return s.first <= b && b < s.end ? s.keys : 0;
}

constexpr int OWN_WARPS = 6, OWN_MAX_GRID = 160 * OWN_WARPS;   // warps on an SM, and of a launch over a sequence's own keys

struct MergeParams {
  SharedParams x;
  bf16* out;
  long long out_row, out_head;
  int n_q, rows;            // T * n_q
};
// Four warps for two rows, whose 16-byte columns lie beside each other in a piece, so that every 32-byte sector is used; each
// warp takes every fourth part, up to 24 of them on their way at once.
__global__ void __launch_bounds__(256) prefix_merge_kernel(const __grid_constant__ MergeParams p) {
  __shared__ float4 sum[8][2][32];
  __shared__ float2 sum_ml[8][32];
  const SharedParams& x = p.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quarter = warp & 3;
  const int at = (blockIdx.x * 2 + (warp >> 2)) * 2 + (lane & 1), q0 = lane >> 1;
  grid_dep_wait();
  grid_dep_launch();
  const int info = at < p.rows ? __ldcg(x.info(at)) : 0, own = at < p.rows ? __ldcg(x.own_info(at)) : 0;
  if (__syncthreads_or(info | own) == 0) return;
  const bool whole = info & PREFIX_WHOLE && !(info & PREFIX_WARPS);
  const int split = info >> 24 & 3, first = min(info & 255, 159), last = min(info >> 8 & 255, 159), row = info >> 16 & 255;
  // what warps left: the own keys' sums, or pieces; a prefix's likewise
  struct Warps {
    int first, parts, code;
  };
  auto warps_of = [&](int code) {
    Warps w = {min(code & 1023, OWN_MAX_GRID - 1), 0, code};
    w.parts = code & OWN_SUMS ? 1 : code & OWN_PIECES ? max(0, min(code >> 10 & 1023, OWN_MAX_GRID - 1) - w.first + 1) : 0;
    return w;
  };
  const bool prefix_by_warps = info & PREFIX_WARPS;
  const Warps w_own = warps_of(own), w_pre = warps_of(prefix_by_warps ? info & (PREFIX_WARPS - 1) : 0);
  const int by_warp = w_own.parts + w_pre.parts;
  const int parts = by_warp + (info == 0 || prefix_by_warps ? 0 : (whole ? 1 : last - first + 1) << split);
  float M = -INFINITY, L = 0.f;
  float4 o[2] = {};
  auto add = [&](float2 v, float4 a, float4 b) {
    if (v.y == 0.f) return;                 // nothing of it counts
    const float mn = fmaxf(M, v.x), f0 = M == -INFINITY ? 0.f : ex2(M - mn), f = ex2(v.x - mn);
    M = mn;
    L = L * f0 + v.y * f;
    o[0].x = o[0].x * f0 + a.x * f, o[0].y = o[0].y * f0 + a.y * f, o[0].z = o[0].z * f0 + a.z * f, o[0].w = o[0].w * f0 + a.w * f;
    o[1].x = o[1].x * f0 + b.x * f, o[1].y = o[1].y * f0 + b.y * f, o[1].z = o[1].z * f0 + b.z * f, o[1].w = o[1].w * f0 + b.w * f;
  };
  constexpr int BATCH = 6;                  // parts of a warp that are on their way at once
#pragma unroll 1
  for (int i0 = quarter; i0 < parts; i0 += 4 * BATCH) {
    float2 v[BATCH];
    float4 a[BATCH], b[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int i = i0 + 4 * j;
      v[j] = make_float2(-INFINITY, 0.f);
      if (i >= parts) continue;
      const float2* ml;
      const float* src;
      int step = 64;                        // to the second 64 dims
      if (i < by_warp) {
        const bool pre = i >= w_own.parts;
        const Warps& w = pre ? w_pre : w_own;
        const int k = pre ? i - w_own.parts : i;
        const size_t at_row = (size_t)((w.first + k) * 2 + (k == 0 ? w.code >> 24 & 1 : 0)) * 16 + (w.code >> 20 & 15);
        const bool sums = w.code & OWN_SUMS;
        ml = !sums ? x.own_part_ml + at_row : pre ? x.ml(at, 0) : x.own_ml(at);
        src = (!sums ? x.own_part + at_row * HEAD_DIM : pre ? x.o(at, 0) : x.own_o(at)) + 4 * q0;
      } else {
        const int k = i - by_warp, part = k & ((1 << split) - 1), c = first + (k >> split), r = (row & 127) + part * (128 >> split);
        const size_t slot = ((size_t)(c * 2 + (c == first ? 1 : 0)) * 2 + (row >> 7)) * 128;
        ml = whole ? x.ml(at, part) : reinterpret_cast<const float2*>(x.part_ml) + slot + (r & 127);
        src = whole ? x.o(at, part) + 4 * q0 : x.part + slot * 128 + (size_t)q0 * 512 + (r & 127) * 4;
        if (!whole) step = 16 * 512;
      }
      v[j] = __ldcg(ml);
      a[j] = __ldcg(reinterpret_cast<const float4*>(src));
      b[j] = __ldcg(reinterpret_cast<const float4*>(src + step));
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
      if (i0 + 4 * j < parts) add(v[j], a[j], b[j]);
  }
  if (quarter) {
    sum[warp][0][lane] = o[0], sum[warp][1][lane] = o[1];
    sum_ml[warp][lane] = make_float2(M, L);
  }
  __syncthreads();
  if (quarter || (info | own) == 0) return;
  if (q0 == 0) *x.info(at) = *x.own_info(at) = 0;
  if (own == 0) return;                     // a sequence with more rows than max_q says: nobody took its own keys
#pragma unroll
  for (int k = 1; k < 4; ++k) add(sum_ml[warp + k][lane], sum[warp + k][0][lane], sum[warp + k][1][lane]);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int t = at / p.n_q;
  uint2* dst = reinterpret_cast<uint2*>(p.out + t * p.out_row + (long long)(at - t * p.n_q) * p.out_head);
  dst[q0] = make_uint2(pack_bf16(o[0].x * inv, o[0].y * inv), pack_bf16(o[0].z * inv, o[0].w * inv));
  dst[q0 + 16] = make_uint2(pack_bf16(o[1].x * inv, o[1].y * inv), pack_bf16(o[1].z * inv, o[1].w * inv));
}

// A sequence's part here: up to OWN_MAX_ROWS query rows per KV head, in blocks of 8 or 16.
constexpr int OWN_MAX_ROWS = 64;
constexpr int OWN_MIN_TILES = 1;           // a warp's least share
constexpr int OWN_UNIT_COST = 2;           // what a unit costs beside its tiles (rows of q, the sums' way out), in tiles
template <bool FP8, int NT>
struct OwnShape {
  static constexpr int ROWS = 8 * NT, KEYS = 32;
  static constexpr int TILE = KEYS * HEAD_DIM * (FP8 ? 1 : 2);   // bytes of K (and of V)
  static constexpr int S = FP8 ? 4 : 2;    // 32 KB
};
// Up to so many sequences, and groups, are looked up once, side by side, and kept in shared memory: a warp would else come to
// its first tile by a chain of some ten loads from memory.
constexpr int OWN_KEPT = 128, OWN_KEPT_GROUPS = 32;

template <bool FP8, int NT>
struct OwnSmem {
  using Sh = OwnShape<FP8, NT>;
  uint8_t k[Sh::S][Sh::TILE], v[Sh::S][Sh::TILE];
  float ks[FP8 ? Sh::S : 1][Sh::KEYS], vs[FP8 ? Sh::S : 1][Sh::KEYS];
  uint64_t full[Sh::S];
  int4 seq[OWN_KEPT];        // OwnSeq
  int4 group[OWN_KEPT_GROUPS], prefix[OWN_KEPT_GROUPS];   // its sequences and keys; OwnSeq
};

struct OwnParams {
  CUtensorMap tm_k, tm_v;   // as the few-row kernel's, boxes of at most 32 rows
  RaggedParams r;
  SharedParams x;
  int strict;               // 1: no other kernel takes the sequences with more rows
};

struct OwnSeq {
  int row0, n, len, start;  // token rows (n 0: not this kernel's), own keys, keys of the prefix before them (-1 - table row: a prefix)
};
// Of sequence b, with row0 = cu[b], end = cu[b + 1], len and its group's keys
__device__ __forceinline__ OwnSeq own_seq(const OwnParams& p, int row0, int end, int len, int keys) {
  const RaggedParams& r = p.r;
  OwnSeq s = {row0, end - row0, len, 0};
  const long long cap = (long long)r.c.table_width << r.c.page_shift;
  bool wrong = s.len > cap;
  if (wrong) s.len = (int)cap;
  const bool bad = s.row0 < 0 || s.n < 0 || s.n > r.T - s.row0, more = !bad && (long long)s.n * r.group > OWN_MAX_ROWS;
  wrong |= bad || (more && p.strict);
  if (bad || more) s.n = 0;
  if (s.n) {
    s.start = keys;
    s.len -= s.start;
    wrong |= s.start && s.len < s.n;        // a new token among the prefix's
  }
  if (wrong) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
  return s;
}
__device__ __forceinline__ OwnSeq own_seq(const OwnParams& p, int b, bool large) {
  return own_seq(p, __ldg(p.r.c.cu + b), __ldg(p.r.c.cu + b + 1), __ldg(p.r.c.seq_lens + b), shared_keys(p.x, p.r, b, large));
}
// A group's prefix as a sequence: every row sees all of its keys.
__device__ __forceinline__ OwnSeq own_prefix(const SharedGroup& g) {
  return {g.row0, g.keys && g.warps ? g.n : 0, g.keys, -1 - g.first};
}
// The walk over a warp's range of tiles: sequences, their blocks of rows, KV heads, tiles of 32 keys.
template <int ROWS, int KEYS>
struct OwnWalk {
  const OwnParams& p;
  const int4 *kept, *kept_prefix;           // sequences and prefixes in shared memory, or null
  bool large;                               // large_prefixes
  OwnSeq s;
  int b, block, g, t, n, blocks;            // t: the next tile of the unit's n
  __device__ __forceinline__ OwnWalk(const OwnParams& p_, const int4* kept_, const int4* prefix_, bool large_, int b_)
      : p(p_), kept(kept_), kept_prefix(prefix_), large(large_), b(b_), block(0), g(0), t(0) { seq(); }
  __device__ __forceinline__ void seq() {
    const int g = b - p.r.c.B;              // the prefixes come behind the sequences
    if (kept) {
      const int4 v = g < 0 ? kept[b] : kept_prefix[g];
      s = {v.x, v.y, v.z, v.w};
    } else {
      s = g < 0 ? own_seq(p, b, large) : own_prefix(shared_group(p.x, p.r, g, large));
    }
    blocks = (s.n * p.r.group + ROWS - 1) / ROWS;
    n = max(1, (s.len + KEYS - 1) / KEYS);   // (a sequence without a key still has rows to be written)
  }
  __device__ __forceinline__ long long cost() const { return (long long)blocks * p.r.c.n_kv * (n + OWN_UNIT_COST); }
  __device__ __forceinline__ void next_unit() {   // (there is one)
    t = 0;
    if (++g < p.r.c.n_kv) return;
    g = 0;
    if (++block < blocks) return;
    block = 0;
    do {
      ++b;
      seq();
    } while (blocks == 0);
  }
};

template <bool FP8, int NT>
__global__ void __launch_bounds__(32) own_attention_kernel(const __grid_constant__ OwnParams p) {
  using Sh = OwnShape<FP8, NT>;
  constexpr int ROWS = Sh::ROWS, KEYS = Sh::KEYS, TILE = Sh::TILE, S = Sh::S;
  using Walk = OwnWalk<ROWS, KEYS>;
  extern __shared__ __align__(1024) uint8_t own_smem[];
  OwnSmem<FP8, NT>& sm = *reinterpret_cast<OwnSmem<FP8, NT>*>(own_smem);
  const RaggedParams& r = p.r;
  const int lane = threadIdx.x, lg = lane >> 2, lt = lane & 3, c = blockIdx.x;
  if (lane == 0) {
    prefetch_map(&p.tm_k);
    prefetch_map(&p.tm_v);
    for (int i = 0; i < S; ++i) mbar_init(&sm.full[i], 1);
    fence_mbar_init();
  }
  grid_dep_wait();
  grid_dep_launch();
  // ---- this warp's range: the total, then the sequence its first tile lies in -------------------------------------------------
  const int seqs = r.c.B + p.x.G, per = (seqs + 31) / 32;
  const int4* kept = r.c.B <= OWN_KEPT && p.x.G <= OWN_KEPT_GROUPS ? sm.seq : nullptr;
  bool large = false;
  if (kept) {
    int row0[OWN_KEPT / 32], end[OWN_KEPT / 32], len[OWN_KEPT / 32];
#pragma unroll
    for (int i = 0; i < OWN_KEPT / 32; ++i) {
      const int b = 32 * i + lane;
      row0[i] = end[i] = len[i] = 0;
      if (b < r.c.B) row0[i] = __ldg(r.c.cu + b), end[i] = __ldg(r.c.cu + b + 1), len[i] = __ldg(r.c.seq_lens + b);
    }
    SharedGroup g = {0, 0, 0, 0, 0, false};
    if (lane < p.x.G) g = shared_group(p.x, r, lane, true);
    long long reads = saved_reads(g, r);    // (as large_prefixes)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) reads += __shfl_xor_sync(0xffffffffu, reads, o);
    large = reads >= SHARED_MIN_READS;
    if (!g.warps && !large) g.keys = 0;
    if (lane < p.x.G) {
      const OwnSeq s = own_prefix(g);
      sm.group[lane] = make_int4(g.first, g.end, g.keys, 0);
      sm.prefix[lane] = make_int4(s.row0, s.n, s.len, s.start);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < OWN_KEPT / 32; ++i) {
      const int b = 32 * i + lane;
      if (b >= r.c.B) break;
      int lo = 0, hi = p.x.G;               // (as shared_keys)
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sm.group[mid].x <= b) lo = mid;
        else hi = mid;
      }
      const int4 g = sm.group[lo];
      const OwnSeq s = own_seq(p, row0[i], end[i], len[i], g.x <= b && b < g.y ? g.z : 0);
      sm.seq[b] = make_int4(s.row0, s.n, s.len, s.start);
    }
    __syncwarp();
  }
  if (!kept) large = large_prefixes(p.x, r, lane);
  long long mine = 0;
  for (int i = lane * per; i < min(seqs, (lane + 1) * per); ++i) mine += Walk(p, kept, sm.prefix, large, i).cost();
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  const long long W = __shfl_sync(0xffffffffu, incl, 31);
  const int G = (int)min((long long)gridDim.x, max(1ll, W / OWN_MIN_TILES));
  if (c >= G || W == 0) return;
  const long long u0 = c * W / G, u1 = (c + 1) * W / G;
  const int owner = __ffs(__ballot_sync(0xffffffffu, incl > u0)) - 1;
  long long start = __shfl_sync(0xffffffffu, incl - mine, owner);
  Walk at(p, kept, sm.prefix, large, owner * per);
  while (u0 >= start + at.cost()) {
    start += at.cost();
    ++at.b;
    at.seq();
  }
  long long unit0;                          // where the unit begins: its cost, then its tiles
  {
    const long long unit = (u0 - start) / (at.n + OWN_UNIT_COST);
    unit0 = start + unit * (at.n + OWN_UNIT_COST);
    at.t = max(0, (int)(u0 - unit0) - OWN_UNIT_COST);
    at.block = (int)(unit / r.c.n_kv);
    at.g = (int)(unit - (long long)at.block * r.c.n_kv);
  }
  __syncwarp();

  // ---- loads: S tiles ahead of the products, page numbers 32 boxes at a time ---------------------------------------------------
  Walk ld = at;
  const int RB = min(1 << r.c.page_shift, KEYS), boxes = KEYS / RB, batch = 32 / boxes;
  long long next = unit0 + OWN_UNIT_COST + at.t;   // where the next tile to load is
  int loaded = 0;
  int pages = -1, in = batch;               // this lane's box of tile (first of the batch) + lane / boxes; the place in the batch
  auto load = [&]() {                       // the next tile of the range
    const int st = loaded % S;
    if (in == batch) {
      const int j = (ld.t + lane / boxes) * KEYS + (lane % boxes) * RB;
      pages = -1;
      if (j < ld.s.len) {
        const int start = ld.s.start;
        pages = __ldg(r.c.table + (size_t)(start < 0 ? -1 - start : ld.b) * r.c.table_stride + ((j + max(start, 0)) >> r.c.page_shift));
        if (pages < 0 || pages >= r.c.n_pages) {
          atomicOr(&g_dev_error, DEVERR_BAD_STATE);
          pages = 0;
        }
      }
      in = 0;
    }
    const int of_box = __shfl_sync(0xffffffffu, pages, in * boxes + lane % boxes), page = lane < boxes ? of_box : -1;
    const int nb = __popc(__ballot_sync(0xffffffffu, page >= 0));
    if (lane == 0) mbar_arrive_expect_tx(&sm.full[st], (uint32_t)(nb * RB) * (FP8 ? 2 * HEAD_DIM + 8 : 4 * HEAD_DIM));
    __syncwarp();
    if (page >= 0) {
      const int row = ((page * r.c.n_kv + ld.g) << r.c.page_shift) + ((ld.t * KEYS + lane * RB) & ((1 << r.c.page_shift) - 1));
      uint8_t *kd = sm.k[st] + lane * RB * 128, *vd = sm.v[st] + lane * RB * 128;
      tma_load_2d(kd, &p.tm_k, 0, row, &sm.full[st]);
      if (!FP8) tma_load_2d(kd + TILE / 2, &p.tm_k, 64, row, &sm.full[st]);
      if (FP8) bulk_g2s(&sm.ks[FP8 ? st : 0][lane * RB], r.c.ks + row, RB * 4, &sm.full[st]);
      tma_load_2d(vd, &p.tm_v, 0, row, &sm.full[st]);
      if (!FP8) tma_load_2d(vd + TILE / 2, &p.tm_v, 64, row, &sm.full[st]);
      if (FP8) bulk_g2s(&sm.vs[FP8 ? st : 0][lane * RB], r.c.vs + row, RB * 4, &sm.full[st]);
    }
    ++loaded;
    ++in;
    ++next;
    if (++ld.t == ld.n) {
      next += OWN_UNIT_COST;
      if (next < u1) ld.next_unit();
      in = batch;
    }
  };
  for (int i = 0; i < S && next < u1; ++i) load();

  FewRows<FP8, NT, KEYS / 16> w;
  bool ok = true;
  for (int it = 0;;) {
    const int n = at.n, t0 = at.t, t1 = (int)min((long long)n, u1 - unit0 - OWN_UNIT_COST), from = at.block * ROWS;
    if (t1 <= t0) break;                    // (the range ends before the unit's first tile)
    const OwnSeq s = at.s;
    const bool prefix = s.start < 0;
    const int after = prefix ? 1 : s.n;     // tokens that do not see all of the keys, and the last one
    const int rows = min(ROWS, s.n * r.group - from), first = s.len - after + by_group(from, r.group);
    w.begin(r, s.row0, after, s.len, from, rows, at.g, lane);
    for (int t = t0; t < t1; ++t, ++it) {
      const int st = it % S;
      ok = __all_sync(0xffffffffu, ok && mbar_wait_small(&sm.full[st], (uint32_t)((it / S) & 1)));
      if (!ok) break;
      if (t * KEYS < s.len)
        w.step(smem_u32(sm.k[st]), smem_u32(sm.v[st]), TILE / 2, sm.ks[FP8 ? st : 0], sm.vs[FP8 ? st : 0], t * KEYS, s.len, first, lane);
      __syncwarp();
      if (next < u1) load();
    }
    if (!ok) break;
    w.finish();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) w.o[i][nt][e] *= w.unscale(nt, e & 1);
    const bool whole = t1 - t0 == n;
    if (!whole || s.start) {                // sums, for the merge with other pieces' and the prefix's, or the own keys'
      const long long tile0 = unit0 + OWN_UNIT_COST;
      const int cf = owner_of(tile0, W, G), cl = owner_of(tile0 + n - 1, W, G);
      const int code = whole ? OWN_SUMS : OWN_PIECES | (cf * W / G < unit0 ? 1 << 24 : 0) | cl << 10 | cf;
      const size_t slot = (size_t)(c * 2 + (u0 < unit0 ? 1 : 0)) * 16;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = nt * 8 + 2 * lt + e;
          if (row >= rows) continue;
          const int sum_at = (s.row0 + by_group(from + row, r.group)) * r.n_q + at.g * r.group + from + row - by_group(from + row, r.group) * r.group;
          if (lg == 0) {
            *(!whole ? p.x.own_part_ml + slot + row : prefix ? p.x.ml(sum_at, 0) : p.x.own_ml(sum_at)) = make_float2(w.m[nt][e], w.l[nt][e]);
            if (t0 == 0) *(prefix ? p.x.info(sum_at) : p.x.own_info(sum_at)) = code | row << 20 | (prefix ? PREFIX_WARPS : 0);
          }
          float* dst = !whole ? p.x.own_part + (slot + row) * HEAD_DIM : prefix ? p.x.o(sum_at, 0) : p.x.own_o(sum_at);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            if (FP8) {                      // 16 dims in a row
              *reinterpret_cast<float4*>(dst + w.dim(i, 0, lg)) = make_float4(w.o[i][nt][e], w.o[i][nt][2 + e], w.o[i + 1][nt][e], w.o[i + 1][nt][2 + e]);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) dst[w.dim(i + (k >> 1), 2 * (k & 1), lg)] = w.o[i + (k >> 1)][nt][2 * (k & 1) + e];
            }
          }
        }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float inv = w.l[nt][e] == 0.f ? 0.f : 1.f / w.l[nt][e];
#pragma unroll
          for (int i = 0; i < 8; ++i) w.o[i][nt][e] *= inv, w.o[i][nt][2 + e] *= inv;
        }
        auto row_of = [&](int row) {
          const int tok = by_group(from + row, r.group);
          return r.out + (long long)(s.row0 + tok) * r.out_row + (long long)(at.g * r.group + from + row - tok * r.group) * r.out_head;
        };
        if (FP8) {                          // 16 dims of rows 2 lt and 2 lt + 1
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = nt * 8 + 2 * lt + e;
            if (row >= rows) continue;
            uint4* dst = reinterpret_cast<uint4*>(row_of(row) + 16 * lg);
#pragma unroll
            for (int h = 0; h < 2; ++h)
              dst[h] = make_uint4(pack_bf16(w.o[4 * h][nt][e], w.o[4 * h][nt][2 + e]), pack_bf16(w.o[4 * h + 1][nt][e], w.o[4 * h + 1][nt][2 + e]),
                                  pack_bf16(w.o[4 * h + 2][nt][e], w.o[4 * h + 2][nt][2 + e]), pack_bf16(w.o[4 * h + 3][nt][e], w.o[4 * h + 3][nt][2 + e]));
          }
        } else {                            // 8 x 8 tiles of (dim, row), turned: two dims of row lg a thread
          const int row = nt * 8 + lg;
          bf16* dst = row_of(min(row, rows - 1)) + 2 * lt;
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t y = transpose8x8(pack_bf16(w.o[i][nt][2 * h], w.o[i][nt][2 * h + 1]));
              if (row < rows) *reinterpret_cast<uint32_t*>(dst + 16 * i + 8 * h) = y;
            }
        }
      }
    }
    unit0 += n + OWN_UNIT_COST;
    if (unit0 + OWN_UNIT_COST >= u1) break;
    at.next_unit();
  }
  if (!ok) {                                // a wait gave up: the copies in flight land before the shared memory goes away
    if (lane == 0) atomicOr(&g_dev_error, DEVERR_MBAR_TIMEOUT);
    for (int i = max(0, loaded - S); i < loaded; ++i) mbar_wait_small(&sm.full[i % S], (uint32_t)((i / S) & 1), 1000000ull);
  }
}

}  // namespace qk

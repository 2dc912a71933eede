// Causal attention on the 5th-generation tensor cores: whole packed prompts, and chunks of new tokens over a paged cache.
//
//   out[t][h] = sum over j <= pos(t) of softmax_j(scale * q[t][h] . K[g][j]) V[g][j],   g = h / (n_q / n_kv)
//
// Bound by the tensor cores: 2 x 128 x 128 x 128 multiply-adds per (128 query rows, 128 keys), and beside them 128 x 128
// exponentials, whose unit is as long at it as the two products are at the matrix units.
//  * The query rows of a KV head are its tokens times its heads, token-major: a tile of 128 rows is 128 / group tokens,
//    so grouped heads share every K and V tile that is loaded. A CTA (one per SM) works on two such tiles at a time,
//    whose softmax warps take turns with the matrix unit.
//  * One pass over the keys in tiles of 128. S = Q K^T (operands in shared memory, accumulator in TMEM); a softmax
//    thread owns one row: it reads its 128 scores with tcgen05.ld, keeps the running maximum m and sum l, writes
//    P = exp2(S - m), but for a constant, as bf16 over S in TMEM; O += P V reads P from TMEM and V from shared memory
//    (dims contiguous: the MN-major operand). P is rounded to bf16, the type of V's tile, which costs an output about as
//    much as its own rounding (2.2e-3 together, of its norm, against 1.5e-3); P in two parts would be half as many products
//    again, of what bounds this. l sums the fp32 values.
//  * O stays in TMEM. Its rows are multiplied by exp2(m_old - m_new) only when a maximum grew by more than 2^32 in
//    weight: until then the old m serves. P, l and O have fp32's exponents, so a P of 2^16 is as exact as one of 1; the
//    rescale becomes rare, and a tile's exponentials need not wait for its maximum. (A limit of 2^8 costs nothing where scores
//    deviate by 1 or 2, but 40 % where they deviate by 4: 630 us for one prompt of 8,192 tokens.) P is exp2(S - m - 16), so
//    that it stays below 2^16 under a stale maximum; the sums pass fp32's range where V's values times the keys that count
//    are above 2^112, and lose bits where V's values are below 2^-110.
//  * Warps: 0-3 and 4-7 the softmax of the two tiles, 8 the loads (TMA, 128-byte swizzle, a ring of five 32 KB K and V
//    tiles), 9 issues the MMAs from one thread (10 clears V rows past a sequence's end, 11 fills the warpgroup, which
//    gives registers to the softmax): Q0 K0, Q1 K0, then per key tile P0 V, Q0 K', P1 V, Q1 K', with P in two parts, the
//    first multiplied while the second is computed. While one tile's softmax runs, the matrix unit has the other's two
//    products to do.
//  * Measured (one prompt of 8,192 tokens, 32 heads on 8): 437 to 445 us in bursts of four calls, 1,235 to
//    1,258 TFLOP/s; some 505 us under the 1,000 W cap. A period of a pair of tiles is 3,150 cycles, the matrix unit's share
//    2,130: the chain of one tile's softmax (2,060), its last P V and next S (800) is longer than half of it. Slower were:
//    exponentials partly on the FMA pipe, halves of S loaded apart, an issuing warp per tile, P in halves (452 us),
//    128-byte transposed output stores.
//  * Work: (sequence, KV head, tile pair, key tile) in that order, dealt in equal contiguous ranges to the CTAs: causal
//    rows and ragged lengths balance by themselves, and a few rows over a long context spread over every SM. A boundary
//    nearer than TCA_MIN_PIECE tiles to the end of a unit moves there. Units cut by one leave fp32 partials (O, m, l) per
//    piece; the CTA that completes the unit's count adds them in order.
//  * An e4m3 cache: the loads bring raw tiles, and six more warps write them as bf16 tiles in the image the MMAs read: the
//    e4m3 values, exactly. The softmax multiplies each score by its key's K scale and each P by its V scale (packed
//    multiplications and broadcast loads); P times the V scale is what is rounded to bf16. Folding the scales into the tiles,
//    rounded to bf16, was a fifth faster and half as far off again (3.4e-3 against 2.3e-3; fp32 sums rounded once: 1.7e-3).
#pragma once
#include "attention_own.cuh"

namespace qk {

constexpr int TCA_KEYS = 128;             // keys of a tile
constexpr int TCA_TILE = TCA_KEYS * HEAD_DIM * 2;   // 32 KB: two 64-dim halves of 128 rows x 128 B
constexpr int TCA_MIN_PIECE = 4;          // tiles
constexpr int TCA_UNIT_COST = 2;          // what a unit costs beside its key tiles (Q load, first scores, output), in tiles
constexpr int TCA_FIRST = 6;              // 16-key steps of P handed over first, of 8 (one prompt of 8,192 tokens, in a burst: 444 us; 452 with 4, 464 with 2)
constexpr float TCA_LAZY = 32.f;          // log2 of the growth that a stale maximum may hide
constexpr float TCA_SHIFT = 16.f;         // P's largest value under a fresh maximum is 2^-16, under a stale one 2^16

enum { SRC_PACKED = 0, SRC_PAGED = 1, SRC_PAGED_FP8 = 2 };
// What the kernel's sequences are: whole ones; the groups of shared_attention, whose rows all see all of the prefix and whose
// sums it leaves to the next launches; or what follows a sequence's prefix, whose sums are added.
enum { TC_WHOLE = 0, TC_PREFIX = 1, TC_OWN = 2 };

struct TcAttnParams {
  CUtensorMap tm_q;         // {128 dims, n_q heads, T rows}: box {64, group, 128 / group}
  CUtensorMap tm_k, tm_v;   // packed: {128 dims, n_kv, T}, box {64, 1, 128}; paged: the pool's rows, box {64, min(page, 128)}
  RaggedParams r;
  float* part;              // [grid][2][2 tiles][32 column quads][128 rows][4]
  float* ml;                // [grid][2][2 tiles][128 rows][2]
  int* counters;            // [grid], zero between launches
  int min_rows;             // sequences with fewer query rows per KV head are another kernel's
  int after;                // launched behind another kernel of the same call, which it need not wait for at its start
  int seqs;                 // sequences, or groups
  SharedParams x;           // (prefixes: part and ml are its)
};

struct TcSeq {
  int row0, n, len;         // token rows, keys (n 0: nothing to do here)
  int table, start;         // the row of the block table; keys before these that a shared prefix has
};
template <int SRC, int MODE>
__device__ __forceinline__ TcSeq tc_seq(const TcAttnParams& p, int b, bool large) {   // large: large_prefixes
  const RaggedParams& r = p.r;
  TcSeq s;
  s.table = b;
  s.start = 0;
  if (MODE == TC_PREFIX) {
    const SharedGroup g = shared_group(p.x, r, b, large);
    s.table = g.first;
    s.row0 = g.row0;
    s.n = g.keys && !g.warps ? g.n : 0;
    s.len = g.keys;
    return s;
  }
  s.row0 = __ldg(r.c.cu + b);
  s.n = __ldg(r.c.cu + b + 1) - s.row0;
  s.len = s.n;
  if (SRC != SRC_PACKED) {
    s.len = __ldg(r.c.seq_lens + b);
    const int cap = r.c.table_width << r.c.page_shift;
    if (s.len > cap) {
      atomicOr(&g_dev_error, DEVERR_BAD_STATE);
      s.len = cap;
    }
    s.len = max(s.len, 0);
  }
  const bool bad = s.row0 < 0 || s.n < 0 || s.n > r.T - s.row0;
  if (bad) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
  if (bad || s.n * r.group < p.min_rows) s.n = 0;
  if (MODE == TC_OWN && s.n) {
    s.start = shared_keys(p.x, r, b, large);
    s.len -= s.start;
    if (s.start && s.len < s.n) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    s.len = max(s.len, 0);
  }
  return s;
}
// sum over i < n of floor((a i + b) / 128), a and b not negative (Euclid's scheme: the lattice points under a line)
__host__ __device__ __forceinline__ long long floor_sum(unsigned n, unsigned a, unsigned b) {
  long long sum = 0;
  unsigned m = TCA_KEYS;
#pragma unroll 1
  while (n) {
    const unsigned qa = a / m, qb = b / m;
    sum += (long long)n * (n - 1) / 2 * qa + (long long)n * qb;
    a -= qa * m;
    b -= qb * m;
    const unsigned long long y = (unsigned long long)a * n + b;
    if (y < m) break;
    if (y >> 32) {                          // (64-bit divisions are several times slower)
      n = (unsigned)(y / m);
      b = (unsigned)(y % m);
    } else {
      n = (unsigned)y / m;
      b = (unsigned)y - n * m;
    }
    const unsigned t = m;
    m = a;
    a = t;
  }
  return sum;
}
__device__ __forceinline__ long long div_short(long long a, long long b) {   // both positive
  return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}
// The cost of a sequence's tile pairs: pair i covers tokens [i step, (i + 1) step) and the keys its last token sees, so
// many tiles (one where it sees none: there still are rows to set to zero), and TCA_UNIT_COST.
// FLAT: every token sees all keys.
template <bool FLAT>
struct TcPairs {
  int n, step, a, len;      // pairs; tokens of a pair; keys before the first token; keys
  __host__ __device__ __forceinline__ TcPairs(const TcSeq& s, int step_) : n((s.n + step_ - 1) / step_), step(step_), a(s.len - s.n), len(s.len) {}
  __host__ __device__ __forceinline__ int tiles(int i) const {
    const int x = FLAT || i == n - 1 ? len : a + (i + 1) * step;
    return max(1, (x + TCA_KEYS - 1) / TCA_KEYS);
  }
  __host__ __device__ __forceinline__ int cost(int i) const { return tiles(i) + TCA_UNIT_COST; }
  __host__ __device__ __forceinline__ long long before(int i) const {   // cost of the pairs 0 .. i - 1
    if (FLAT) return (long long)i * cost(0);
    const int q = min(i, n - 1), z = a < 0 ? min(q, -a / step) : 0;
    if (i <= 0) return 0;
    return z + floor_sum(q - z, step, a + (z + 1) * step + TCA_KEYS - 1) + (i == n ? tiles(n - 1) : 0) + (long long)i * TCA_UNIT_COST;
  }
};

struct TcPlace {              // where a range begins
  int b, g, pair, t;
  long long u;
};
template <int SRC, int MODE>
struct TcAttnSmem {
  // K and V tiles of the ring; e4m3 tiles on their way to bf16 (prefixes are bound by what is on its way from memory)
  static constexpr int S = SRC != SRC_PAGED_FP8 ? 5 : MODE == TC_PREFIX ? 3 : 4;
  static constexpr int RAW = SRC != SRC_PAGED_FP8 ? 0 : MODE == TC_PREFIX ? 4 : 2;
  uint8_t q[2][TCA_TILE];
  uint8_t kv[S][TCA_TILE];
  uint8_t raw[RAW ? RAW : 1][RAW ? TCA_KEYS * HEAD_DIM : 16];
  // scale * log2 e times the K scales of a key tile, and the V scales, for the softmax. Three tiles of K's: tile j + 3 is
  // converted into the stage of tile j + 1, which is free once both query tiles' scores of j + 1 are done, behind their
  // P V of j. Two of V's: tile j + 2 goes into the stage of tile j, free after its P V.
  float k_scale[RAW ? 3 : 1][RAW ? TCA_KEYS : 4], v_scale[RAW ? 2 : 1][RAW ? TCA_KEYS : 4];
  long long total;
  TcPlace at[2];
  uint64_t q_full, q_empty, full[S], empty[S], raw_full[RAW ? RAW : 1], raw_empty[RAW ? RAW : 1];
  uint64_t s_full[2], p_full[2][2], o_full[2], v_clean[S];   // per tile (P in two halves); per stage
  uint32_t tmem;
  int last;
  bool large;
};

__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// D fp32, A and B bf16, M = N = 128; b_mn: B is stored with N contiguous
__host__ __device__ constexpr uint32_t tca_idesc(bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
}
// V [128 keys][128 dims]: 64-dim halves TCA_TILE / 2 apart, groups of 8 keys 1024 bytes apart
__device__ __forceinline__ uint64_t tca_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((TCA_TILE / 2) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tca_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum), "r"(0)
      : "memory");
}
__device__ __forceinline__ void tca_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum), "r"(0)
      : "memory");
}
// 32 consecutive 32-bit columns of this warp's 32 TMEM lanes, one lane a thread
__device__ __forceinline__ void tca_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tca_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
      "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
      "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),
      "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tca_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                 "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(taddr));
}
__device__ __forceinline__ void tca_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
               "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
               : "memory");
}
template <int N>
__device__ __forceinline__ void tca_st(uint32_t taddr, const uint32_t* v) {   // N columns, 16, 32 or 48
  if (N >= 32) tca_st32(taddr, v);
  if (N & 16) tca_st16(taddr + (N & 32), v + (N & 32));
}
__device__ __forceinline__ void tca_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// P of 2 N scores: p = exp2(s * scale + base), bf16 pairs to out (which may be the scores' first half), sums to sum. The
// packed instructions halve the issue slots beside the exponential unit, which is what bounds this.
// With F32 it stays as fp32 in the scores' place (out unused), for tca_pack.
template <int N, bool F32>
__device__ __forceinline__ void tca_exp(uint32_t* s, uint32_t* out, uint64_t scale, uint64_t base, uint64_t (&sum)[2]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint64_t x = fma2(f32x2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale, base);
    x = f32x2(ex2(f32x2_lo(x)), ex2(f32x2_hi(x)));
    sum[i & 1] = add2(sum[i & 1], x);
    if (F32) s[2 * i] = (uint32_t)x, s[2 * i + 1] = (uint32_t)(x >> 32);
    else out[i] = pack_bf16(f32x2_lo(x), f32x2_hi(x));
  }
}
// P times the keys' V scales (l is without them), to bf16 pairs.
template <int N>
__device__ __forceinline__ void tca_pack(const uint32_t* s, uint32_t* out, const float* vs) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float4 v4 = *reinterpret_cast<const float4*>(vs + 2 * i);
    const uint64_t a = mul2(f32x2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), f32x2(v4.x, v4.y));
    const uint64_t b = mul2(f32x2(__uint_as_float(s[2 * i + 2]), __uint_as_float(s[2 * i + 3])), f32x2(v4.z, v4.w));
    out[i] = pack_bf16(f32x2_lo(a), f32x2_hi(a));
    out[i + 1] = pack_bf16(f32x2_lo(b), f32x2_hi(b));
  }
}

// Nothing that uses these values moves before this point (a tcgen05.ld's registers are its own until the wait after it).
__device__ __forceinline__ void tca_tie32(uint32_t* v) {
  asm volatile("" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
               "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]),
               "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
               "+r"(v[30]), "+r"(v[31]));
}
// One lane of a converged warp, the same one every time. The compiler knows it for a single lane (which `lane == 0` does
// not tell it), so the MMAs' descriptors go straight to the uniform registers that they are taken from.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// Rows FIRST to LAST - 1 of a tile of e4m3 rows to bf16 ones in the image the MMAs read, exactly; 8 threads a row, ROWS rows at a
// time, from `tail` on zeros.
// 8 bytes and 8 again: two swizzled 16-byte chunks of a row. Three rows' loads go before their stores: one at a time, each load's
// latency and each conversion's in turn, a tile took 2,500 cycles of six warps.
template <int ROWS, int FIRST, int LAST>
__device__ __forceinline__ void tca_convert(uint32_t src, uint32_t dst, int th, int tail) {
  const int ch = th & 7, half = ch >> 2;    // this thread's 16 dims
#pragma unroll
  for (int k0 = 0; FIRST + k0 * ROWS < LAST; k0 += 3) {
    uint2 q[3][2];
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) {         // the second half's lanes begin with their other chunk: no bank conflict
        const int row = FIRST + (k0 + k) * ROWS + (th >> 3);
        if (FIRST + (k0 + k) * ROWS < LAST && row < LAST)
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(q[k][j].x), "=r"(q[k][j].y) : "r"(src + row * HEAD_DIM + ch * 16 + (j ^ half) * 8));
      }
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = FIRST + (k0 + k) * ROWS + (th >> 3);
        if (FIRST + (k0 + k) * ROWS >= LAST || row >= LAST) break;
        uint32_t y[4];
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) {
          const uint32_t h = e4m3x2_to_f16x2((i2 < 2 ? q[k][j].x : q[k][j].y) >> (16 * (i2 & 1)));
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
          y[i2] = pack_bf16(f.x, f.y);
        }
        if (row >= tail) y[0] = y[1] = y[2] = y[3] = 0;
        const int c16 = ((ch & 3) * 2 + (j ^ half)) ^ (row & 7);
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + half * (TCA_TILE / 2) + row * 128 + c16 * 16), "r"(y[0]), "r"(y[1]),
                     "r"(y[2]), "r"(y[3])
                     : "memory");
      }
  }
}

// A prefix with few rows: a tile's four warps of 32 rows hold them 2 or 4 times (`parts`), each part for its own half or quarter of
// every key tile. What a tile costs then is the chain from its scores to its product with V, and a thread's 128 exponentials
// are the longest part of that: 128 / parts remain (and zeros for the other parts' keys).
__device__ __forceinline__ int prefix_parts(int n, int tpq) { return n <= tpq ? 4 : n <= 2 * tpq ? 2 : 1; }

// A CTA's walk over its pieces; every role walks the same one.
template <int SRC, int MODE>
struct TcWalk {
  const TcAttnParams& p;
  int b, g, pair, t0, step;
  bool large;
  TcSeq s;
  TcPairs<MODE == TC_PREFIX> pr;
  long long u, u1;
  int n, t1;                // the unit's key tiles; the piece is [t0, t1)
  __device__ __forceinline__ TcWalk(const TcAttnParams& p_, const TcAttnSmem<SRC, MODE>& sm, int step_)
      : p(p_), b(sm.at[0].b), g(sm.at[0].g), pair(sm.at[0].pair), t0(max(0, sm.at[0].t - TCA_UNIT_COST)), step(step_), large(sm.large), s(tc_seq<SRC, MODE>(p_, sm.at[0].b, sm.large)), pr(s, step_),
        u(sm.at[0].u), u1(sm.at[1].u) {
    piece();
  }
  __device__ __forceinline__ int cost() const { return t0 ? 0 : TCA_UNIT_COST; }   // a unit's own falls to its first piece
  __device__ __forceinline__ void piece() {
    n = pr.tiles(pair);
    t1 = (int)min((long long)n, t0 + (u1 - u) - cost());
  }
  __device__ __forceinline__ bool more() const { return u < u1; }
  __device__ __forceinline__ void next() {
    u += t1 - t0 + cost();
    t0 = 0;
    if (u >= u1) return;
    if (++pair == pr.n) {
      pair = 0;
      if (++g == p.r.c.n_kv) {
        g = 0;
        do s = tc_seq<SRC, MODE>(p, ++b, large);
        while (s.n == 0);
        pr = TcPairs<MODE == TC_PREFIX>(s, step);
      }
    }
    piece();
  }
  // of tile x of the pair: its first token, whether it has any, and its key tiles in this piece
  __device__ __forceinline__ int tok0(int x) const { return pair * step + x * (step / 2); }
  __device__ __forceinline__ bool two() const { return tok0(1) < s.n; }
  __device__ __forceinline__ int end(int x) const {
    if (tok0(x) >= s.n) return t0;
    const int keys = MODE == TC_PREFIX ? s.len : min(s.len, s.len - s.n + min(tok0(x) + step / 2, s.n));
    return max(t0, min(t1, max(1, (keys + TCA_KEYS - 1) / TCA_KEYS)));
  }
};

// Threads, and their registers: 384 x 168 at launch become 256 x 208 + 128 x 88; with four warps more (they, 10 and 11 turn
// e4m3 tiles into bf16 ones), 512 x 128 become 256 x 200 + 256 x 56.
template <int SRC>
struct TcShape {
  static constexpr int THREADS = SRC == SRC_PAGED_FP8 ? 512 : 384;
  static constexpr int SOFTMAX = SRC == SRC_PAGED_FP8 ? 200 : 208, OTHER = SRC == SRC_PAGED_FP8 ? 56 : 88;
  static_assert(256 * SOFTMAX + (THREADS - 256) * OTHER <= THREADS * (SRC == SRC_PAGED_FP8 ? 128 : 168), "setmaxnreg would wait for ever");
};
template <int SRC, int MODE>
__global__ void __launch_bounds__(TcShape<SRC>::THREADS, 1) tc_attention_kernel(const __grid_constant__ TcAttnParams p) {
  extern __shared__ __align__(1024) uint8_t tca_smem[];
  using Smem = TcAttnSmem<SRC, MODE>;
  using Pairs = TcPairs<MODE == TC_PREFIX>;
  using Walk = TcWalk<SRC, MODE>;
  Smem& sm = *reinterpret_cast<Smem*>(tca_smem);
  constexpr int TCA_STAGES = Smem::S, RAW = Smem::RAW ? Smem::RAW : 1;
  constexpr bool FP8 = SRC == SRC_PAGED_FP8;
  const RaggedParams& r = p.r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x, n_kv = r.c.n_kv;
  const int tpq = 32 / r.group;           // prefixes: tokens of a warp's 32 rows
  const int step = MODE == TC_PREFIX ? 8 * tpq : 2 * (128 / r.group);   // tokens of a tile pair
  if (tid == 0) {
    prefetch_map(&p.tm_q);
    if (!FP8) prefetch_map(&p.tm_k), prefetch_map(&p.tm_v);
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int i = 0; i < TCA_STAGES; ++i) {
      mbar_init(&sm.full[i], !FP8 ? 1 : MODE == TC_PREFIX ? 10 : 6);   // the copies; the converting warps
      mbar_init(&sm.empty[i], FP8 ? 1 : 2);   // the MMAs; they and the V cleaner
      mbar_init(&sm.v_clean[i], 1);
    }
    for (int i = 0; i < RAW; ++i) {
      mbar_init(&sm.raw_full[i], 1);
      mbar_init(&sm.raw_empty[i], MODE == TC_PREFIX ? 10 : 6);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sm.s_full[x], 1);
      mbar_init(&sm.p_full[x][0], 4);
      mbar_init(&sm.p_full[x][1], 4);
      mbar_init(&sm.o_full[x], 1);
    }
    fence_mbar_init();
  }
  // Behind the few-row kernel: that one let this one start after its own wait, so what came before both is complete, and
  // the two share neither rows nor scratch. CTAs take the SMs as the other's leave them; this kernel waits for the other
  // at its end, so that whatever follows it follows both.
  if (!p.after) grid_dep_wait();
  grid_dep_launch();

  // ---- this CTA's range of key tiles: sums over the sequences, 32 chunks of them; warp 0 finds where it begins, warp 1
  // where the next one does ---------------------------------------------------------------------------------------------
  if (warp < 2) {
    const bool large = MODE != TC_WHOLE && large_prefixes(p.x, r, lane);
    const int per = (p.seqs + 31) / 32;
    long long mine = 0, tot = 0;
    TcSeq s = {0, 0, 0, 0, 0};
    for (int b = lane * per; b < min(p.seqs, (lane + 1) * per); ++b) {
      s = tc_seq<SRC, MODE>(p, b, large);
      const Pairs pr(s, step);
      tot = pr.n ? pr.before(pr.n) : 0;
      mine += tot * n_kv;
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const long long W = __shfl_sync(0xffffffffu, incl, 31);
    const int G = (int)min((long long)gridDim.x, max(1ll, W / TCA_MIN_PIECE));
    const long long u = div_short(min(c + warp, G) * W, G);
    int b = p.seqs, g = 0, pair = 0, t = 0;
    long long at = W;
    if (u < W) {
      const int first = __ffs(__ballot_sync(0xffffffffu, incl > u)) - 1;
      at = __shfl_sync(0xffffffffu, incl - mine, first);
      b = first * per;
      if (per == 1) {                       // the lane's sequence is the one
        s = {__shfl_sync(0xffffffffu, s.row0, first), __shfl_sync(0xffffffffu, s.n, first), __shfl_sync(0xffffffffu, s.len, first), 0, 0};
        tot = __shfl_sync(0xffffffffu, tot, first);
      } else {
        for (;; ++b) {
          s = tc_seq<SRC, MODE>(p, b, large);
          const Pairs pr(s, step);
          tot = pr.n ? pr.before(pr.n) : 0;
          if (u < at + tot * n_kv) break;
          at += tot * n_kv;
        }
      }
      const Pairs pr(s, step);
      g = (int)div_short(u - at, tot);
      at += g * tot;
      int lo = 0, hi = pr.n;                // the pair: before(lo) <= u - at < before(hi)
#pragma unroll 1
      while (hi - lo > 1) {
        const int d = (hi - lo + 31) / 32, i = lo + (lane + 1) * d;
        const bool le = i < hi && pr.before(i) <= u - at;
        const int k = __popc(__ballot_sync(0xffffffffu, le));
        lo += k * d;
        hi = min(hi, lo + d);
      }
      pair = lo;
      at += pr.before(pair);
      t = (int)(u - at);                    // into the unit's cost: TCA_UNIT_COST, then its tiles
      const int n = pr.cost(pair);
      if (t < TCA_UNIT_COST + TCA_MIN_PIECE) t = 0;
      else if (n - t < TCA_MIN_PIECE) {     // the range begins with the next unit
        at += n;
        t = 0;
        if (++pair == pr.n) {
          pair = 0;
          if (++g == n_kv) {
            g = 0;
            do ++b;
            while (b < p.seqs && tc_seq<SRC, MODE>(p, b, large).n == 0);
          }
        }
      }
    }
    if (lane == 0) {
      sm.at[warp] = {b, g, pair, t, at + t};   // u and t count cost: key tile t - TCA_UNIT_COST
      sm.total = W;
      sm.large = large;
    }
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const long long W = sm.total;
  const bool work = sm.at[0].u < sm.at[1].u;
  // TMEM columns: S (and P) of the tiles at 0 and 128, O at 256 and 384

  // the register split stands inside the roles' branches: after a join the compiler would have to take the smaller share
  if (warp >= 8) {
    regs_dec<TcShape<SRC>::OTHER>();
    if (work && warp == 8) {   // ---- loads ----
      Walk w(p, sm, step);
      const int RB = SRC == SRC_PACKED ? TCA_KEYS : min(1 << r.c.page_shift, TCA_KEYS);
      const uint32_t q_bytes = (uint32_t)(step / 2) * r.group * HEAD_DIM * 2;
      int it = 0;
      bool ok = true;
      for (int unit = 0; w.more() && ok; w.next(), ++unit) {
        if (unit) ok = __all_sync(0xffffffffu, mbar_wait_small(&sm.q_empty, (uint32_t)((unit - 1) & 1)));
        if (!ok) break;
        const bool two = w.two();
        if (lane == 0) {
          mbar_arrive_expect_tx(&sm.q_full, two ? 2 * q_bytes : q_bytes);
          for (int x = 0; x < (two ? 2 : 1); ++x)
            for (int h = 0; h < 2; ++h) {
              if (MODE == TC_PREFIX) {
                const int per = 4 / prefix_parts(w.s.n, tpq);   // a part's quarters
                for (int k = 0; k < 4; ++k)
                  tma_load_3d(sm.q[x] + h * (TCA_TILE / 2) + k * 32 * 128, &p.tm_q, 64 * h, w.g * r.group, w.s.row0 + w.tok0(x) + k % per * tpq, &sm.q_full);
              } else {
                tma_load_3d(sm.q[x] + h * (TCA_TILE / 2), &p.tm_q, 64 * h, w.g * r.group, w.s.row0 + w.tok0(x), &sm.q_full);
              }
            }
        }
        auto page_of = [&](int t) {           // this lane's box of tile t: its page, -1 where it holds no key
          const int j = t * TCA_KEYS + lane * RB;
          if (lane * RB >= TCA_KEYS || j >= w.s.len) return -1;
          int pg = __ldg(r.c.table + (size_t)(MODE == TC_PREFIX ? w.s.table : w.b) * r.c.table_stride + ((MODE == TC_OWN ? j + w.s.start : j) >> r.c.page_shift));
          if (pg < 0 || pg >= r.c.n_pages) {
            atomicOr(&g_dev_error, DEVERR_BAD_STATE);
            pg = 0;
          }
          return pg;
        };
        int next = SRC == SRC_PACKED ? 0 : page_of(w.t0);
        for (int t = w.t0; t < w.t1 && ok; ++t) {
          const int page = next;
          if (SRC != SRC_PACKED && t + 1 < w.t1) next = page_of(t + 1);
          for (int v = 0; v < 2; ++v, ++it) {   // K, then V
            constexpr int N = FP8 ? RAW : TCA_STAGES;
            const int st = it % N;
            uint64_t* full = FP8 ? &sm.raw_full[st] : &sm.full[st];
            if (it >= N) ok = __all_sync(0xffffffffu, mbar_wait_small(FP8 ? &sm.raw_empty[st] : &sm.empty[st], (uint32_t)((it / N - 1) & 1)));
            if (!ok) break;
            const CUtensorMap* tm = v ? &p.tm_v : &p.tm_k;
            if (SRC == SRC_PACKED) {
              if (lane == 0) {
                mbar_arrive_expect_tx(full, TCA_TILE);
                for (int h = 0; h < 2; ++h) tma_load_3d(sm.kv[st] + h * (TCA_TILE / 2), tm, 64 * h, w.g, w.s.row0 + t * TCA_KEYS, full);
              }
            } else {
              const int nb = __popc(__ballot_sync(0xffffffffu, page >= 0));
              if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(nb * RB) * (FP8 ? HEAD_DIM : 2 * HEAD_DIM));
              __syncwarp();
              if (page >= 0) {
                const int row = ((page * n_kv + w.g) << r.c.page_shift) + ((t * TCA_KEYS + lane * RB) & ((1 << r.c.page_shift) - 1));
                if (FP8) {                    // a page's rows of a head are contiguous
                  bulk_g2s(sm.raw[FP8 ? st : 0] + lane * RB * HEAD_DIM, (v ? r.c.v : r.c.k) + (size_t)row * HEAD_DIM, RB * HEAD_DIM, full);
                } else {
                  for (int h = 0; h < 2; ++h) tma_load_2d(sm.kv[st] + h * (TCA_TILE / 2) + lane * RB * 128, tm, 64 * h, row, full);
                }
              }
            }
          }
        }
      }
      if (!ok)   // a wait gave up: let the copies in flight land before the shared memory goes away
        for (int n = FP8 ? RAW : TCA_STAGES, i = max(0, it - n); i < it; ++i)
          mbar_wait_small(FP8 ? &sm.raw_full[i % n] : &sm.full[i % n], (uint32_t)((i / n) & 1), 1000000ull);
    } else if (work && warp == 9) {   // ---- MMA issue: one thread, nothing between the products but its waits ----
      if (elect_one()) {
        constexpr uint32_t id_s = tca_idesc(false), id_o = tca_idesc(true);
        Walk w(p, sm, step);
        uint32_t st = 0, par = 0, np[2] = {0, 0}, clean = 0;   // st, par: the next tile's stage, its `full` parity; clean: v_clean's
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          ok = ok && mbar_wait_small(bar, parity);
          tc_fence_after();
        };
        auto take = [&]() {                   // the next K or V tile of the ring
          wait(&sm.full[st], par);
          const uint32_t at = st;
          if (++st == TCA_STAGES) st = 0, par ^= 1;
          return at;
        };
        auto scores = [&](int x, uint32_t at) {   // S = Q K^T
          const uint64_t qd = tc_desc_sw128(smem_u32(sm.q[x])), kd = tc_desc_sw128(smem_u32(sm.kv[at]));
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t off = ((k >> 2) * (TCA_TILE / 2) + (k & 3) * 32) >> 4;
            tca_mma_ss(tmem + 128 * x, qd + off, kd + off, id_s, k > 0);
          }
          tc_commit(&sm.s_full[x]);
        };
        for (int unit = 0; w.more() && ok; w.next(), ++unit) {
          const int e[2] = {w.end(0), w.end(1)};
          wait(&sm.q_full, (uint32_t)(unit & 1));
          uint32_t ks = take();
          if (!ok) break;
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (w.t0 < e[x]) scores(x, ks);
          tc_commit(&sm.empty[ks]);
          if (w.t1 - w.t0 == 1) tc_commit(&sm.q_empty);
          for (int t = w.t0; t < w.t1; ++t) {
            const uint32_t vs = take();
            const bool more = t + 1 < w.t1;
            if (!FP8 && w.s.len - t * TCA_KEYS < TCA_KEYS) {
              wait(&sm.v_clean[vs], clean >> vs & 1);
              clean ^= 1u << vs;
            }
            if (more) ks = take();
            if (!ok) break;
            const uint64_t vd = tca_desc_mn(smem_u32(sm.kv[vs]));
#pragma unroll                              // (the arrays stay in registers)
            for (int x = 0; x < 2; ++x) {
              if (t < e[x]) {
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                  wait(&sm.p_full[x][hh], np[x] & 1);
                  if (!ok) break;
#pragma unroll
                  for (int k = hh ? TCA_FIRST : 0; k < (hh ? 8 : TCA_FIRST); ++k)
                    tca_mma_ts(tmem + 256 + 128 * x, tmem + 128 * x + 8 * k, vd + k * (2048 >> 4), id_o, k > 0 || t > w.t0);
                }
                if (t + 1 == e[x]) tc_commit(&sm.o_full[x]);
                ++np[x];
              }
              if (t + 1 < e[x] && ok) scores(x, ks);
            }
            if (!ok) break;
            tc_commit(&sm.empty[vs]);
            if (more) tc_commit(&sm.empty[ks]);
            if (t + 2 == w.t1) tc_commit(&sm.q_empty);
          }
        }
      }
      __syncwarp();
    } else if (!FP8 && work && warp == 10) {   // ---- V rows past a sequence's end: another's, or nothing; 0 x NaN must not reach O ----
      Walk w(p, sm, step);
      uint32_t st = 0, par = 0;
      bool ok = true;
      for (; w.more() && ok; w.next())
        for (int i = 2 * w.t0; i < 2 * w.t1 && ok; ++i) {   // every tile of the ring in turn, K and V
          ok = __all_sync(0xffffffffu, mbar_wait_small(&sm.full[st], par));
          const int tail = w.s.len - (i >> 1) * TCA_KEYS;
          if ((i & 1) && tail < TCA_KEYS) {
            const uint32_t va = smem_u32(sm.kv[st]);
            for (int k = max(tail, 0) * 16 + lane; k < TCA_KEYS * 16; k += 32)
              asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(va + ((k >> 3) & 1) * (TCA_TILE / 2) + (k >> 4) * 128 + (k & 7) * 16), "r"(0) : "memory");
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.v_clean[st]);
          }
          if (lane == 0) mbar_arrive(&sm.empty[st]);
          if (++st == TCA_STAGES) st = 0, par ^= 1;
        }
    } else if (FP8 && work) {   // ---- warps 10 to 15: e4m3 tiles to bf16 ones (exact), and their rows' scales ----
      Walk w(p, sm, step);
      const int th = tid - 320;
      // the scales of key th of tile t: fetched a tile ahead, and the number of the page that they are in two
      auto page_of = [&](int t) {
        const int j = t * TCA_KEYS + th;
        return th < TCA_KEYS && t < w.t1 && j < w.s.len
                   ? __ldg(r.c.table + (size_t)(MODE == TC_PREFIX ? w.s.table : w.b) * r.c.table_stride + ((MODE == TC_OWN ? j + w.s.start : j) >> r.c.page_shift))
                   : -1;
      };
      auto scales_of = [&](int t, int pg) {
        const int j = t * TCA_KEYS + th;
        float2 y = make_float2(0.f, 0.f);
        if (th < TCA_KEYS && t < w.t1 && j < w.s.len) {
          if (pg < 0 || pg >= r.c.n_pages) pg = 0;   // (the loads say so)
          const int at = ((pg * n_kv + w.g) << r.c.page_shift) + (j & ((1 << r.c.page_shift) - 1));
          y = make_float2(__ldg(r.c.ks + at) * (r.scale * LOG2E), __ldg(r.c.vs + at));
        }
        return y;
      };
      uint32_t it = 0;
      bool ok = true;
      for (; w.more() && ok; w.next()) {
        int page = page_of(w.t0 + 1);
        float2 scales = scales_of(w.t0, page_of(w.t0)), ahead = make_float2(0.f, 0.f);
        for (int i = 2 * w.t0; i < 2 * w.t1 && ok; ++i, ++it) {   // K and V in turn
          const uint32_t rs = it % RAW, st = it % TCA_STAGES;
          const bool is_v = i & 1;
          if (!is_v) {
            ahead = scales_of((i >> 1) + 1, page);
            page = page_of((i >> 1) + 2);
          }
          ok = mbar_wait_small(&sm.raw_full[rs], (it / RAW) & 1);
          if (it >= TCA_STAGES) ok = ok && mbar_wait_small(&sm.empty[st], (it / TCA_STAGES - 1) & 1);
          ok = __all_sync(0xffffffffu, ok);
          const int tail = w.s.len - (i >> 1) * TCA_KEYS;   // rows from here on were not loaded, or are not the sequence's
          const uint32_t src = smem_u32(sm.raw[FP8 ? rs : 0]), dst = smem_u32(sm.kv[st]);
          if (th < TCA_KEYS) {
            if (is_v) sm.v_scale[FP8 ? (it >> 1) & 1 : 0][FP8 ? th : 0] = scales.y;
            else sm.k_scale[FP8 ? (it >> 1) % 3 : 0][FP8 ? th : 0] = scales.x;
          }
          if (is_v) scales = ahead;
          const bool ten = MODE == TC_PREFIX && !w.two();   // with tile 1's softmax warps, which have no rows
          if (ten) tca_convert<24, 80, TCA_KEYS>(src, dst, th, TCA_KEYS);
          else tca_convert<24, 0, TCA_KEYS>(src, dst, th, tail);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {                    // (a prefix's barriers wait for ten warps)
            const uint32_t n = MODE == TC_PREFIX && !ten && warp == 10 ? 5 : 1;
            mbar_arrive_n(&sm.full[st], n);
            mbar_arrive_n(&sm.raw_empty[rs], n);
          }
        }
      }
    }
  } else {
    regs_inc<TcShape<SRC>::SOFTMAX>();
    if (work) {   // ---- softmax: thread = one row of tile x ----
      const int x = warp >> 2, row = tid & 127;
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + lanes + 128 * x, to = tmem + lanes + 256 + 128 * x;
      const float sl2 = FP8 ? 1.f : r.scale * LOG2E;   // (an e4m3 cache: already in the keys' scales)
      Walk w(p, sm, step);
      int ns = 0, no = 0, kt = 0;             // kt: key tiles of the pieces before
      bool ok = true;
      for (; w.more(); w.next()) {
        const int parts = MODE == TC_PREFIX ? prefix_parts(w.s.n, tpq) : 1, per = 4 / parts;
        const int own = MODE == TC_PREFIX ? lane / r.group : row / r.group, hq = MODE == TC_PREFIX ? lane % r.group : row % r.group;
        const int e = w.end(x), tok = w.tok0(x) + own + (MODE == TC_PREFIX ? (warp & 3) % per * tpq : 0), pos = MODE == TC_PREFIX ? w.s.len - 1 : w.s.len - w.s.n + tok;
        const bool valid = (MODE == TC_PREFIX ? own < tpq : row < (step / 2) * r.group) && tok < w.s.n;
        const int first = MODE == TC_PREFIX ? w.s.len - 1 : w.s.len - w.s.n + w.tok0(x);   // the last key that the tile's first row sees
        float m = -INFINITY, l = 0.f, base = 0.f;   // base = -m * sl2 - TCA_SHIFT
        // No rows in tile 1 (a prefix in parts, or a last pair of few rows): its warps do most of the tiles' conversion. That also
        // keeps them in step with the ring, whose phases they know by parity only: none of them passes a piece without its tiles.
        if (FP8 && MODE == TC_PREFIX && x == 1 && !w.two()) {
          for (uint32_t it = 2 * kt; it < (uint32_t)(2 * (kt + w.t1 - w.t0)); ++it) {
            const uint32_t rs = it % RAW, st = it % TCA_STAGES;
            ok = ok && mbar_wait_small(&sm.raw_full[rs], (it / RAW) & 1);
            if (it >= TCA_STAGES) ok = ok && mbar_wait_small(&sm.empty[st], (it / TCA_STAGES - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tca_convert<16, 0, 80>(smem_u32(sm.raw[FP8 ? rs : 0]), smem_u32(sm.kv[st]), row, TCA_KEYS);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&sm.full[st]);
              mbar_arrive(&sm.raw_empty[rs]);
            }
          }
        } else if (MODE == TC_PREFIX && parts > 1) {
          auto tiles = [&](auto n_parts) {
            constexpr int N = 128 / decltype(n_parts)::value;   // keys of a tile that are this part's: from k0 on
            const int part = (warp & 3) / per, k0 = part * N;
            for (int t = w.t0; t < e; ++t) {
              ok = __all_sync(0xffffffffu, ok && mbar_wait_small(&sm.s_full[x], (uint32_t)(ns++ & 1)));
              tc_fence_after();
              uint32_t v[N];
#pragma unroll
              for (int i = 0; i < N; i += 32) tca_ld32(ts + k0 + i, v + i);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < N; i += 32) tca_tie32(v + i);
              if (FP8) {
                const float* ks = sm.k_scale[FP8 ? (kt + t - w.t0) % 3 : 0] + (FP8 ? k0 : 0);
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * ks[FP8 ? i : 0]);
              }
              float mx[2] = {m, m};
#pragma unroll
              for (int i = 0; i < N; i += 2) mx[(i >> 1) & 1] = max3_nan(mx[(i >> 1) & 1], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
              const float mn = max_nan(mx[0], mx[1]);
              const bool grow = valid && !((mn - m) * sl2 <= TCA_LAZY);
              if (__any_sync(0xffffffffu, grow)) {
                float f = 1.f;
                if (grow) {
                  f = m == -INFINITY ? 0.f : ex2((m - mn) * sl2);
                  m = mn;
                  l *= f;
                  base = m == -INFINITY ? 0.f : m == INFINITY ? __int_as_float(0x7fffffff) : -m * sl2 - TCA_SHIFT;
                }
                if (t > w.t0) {               // the products before this tile's scores are done: O is whole
#pragma unroll 1
                  for (int i = 0; i < 8; ++i) {
                    uint32_t o[16];
                    tca_ld16(to + 16 * i, o);
                    tc_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                    tca_st16(to + 16 * i, o);
                  }
                }
              }
              uint64_t sum[2] = {0, 0};
              tca_exp<N / 2, FP8>(v, v, f32x2(sl2, sl2), f32x2(base, base), sum);
              if (FP8) {                      // V's tile, and with it the scales, is there (its stage waits for this P)
                const uint32_t i = 2 * (kt + t - w.t0) + 1;
                ok = __all_sync(0xffffffffu, ok && mbar_wait_small(&sm.full[i % TCA_STAGES], (i / TCA_STAGES) & 1));
                tca_pack<N / 2>(v, v, sm.v_scale[FP8 ? (kt + t - w.t0) & 1 : 0] + (FP8 ? k0 : 0));
              }
              uint32_t none[N / 2];
#pragma unroll
              for (int i = 0; i < N / 2; ++i) none[i] = 0;
#pragma unroll
              for (int k = 0; k < 128 / N; ++k) {
                if (k == part) tca_st<N / 2>(ts + k * (N / 2), v);
                else tca_st<N / 2>(ts + k * (N / 2), none);
              }
              tca_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive(&sm.p_full[x][0]);
                mbar_arrive(&sm.p_full[x][1]);
              }
              l += (f32x2_lo(sum[0]) + f32x2_hi(sum[0])) + (f32x2_lo(sum[1]) + f32x2_hi(sum[1]));
            }
          };
          if (parts == 4) tiles(std::integral_constant<int, 4>{});
          else tiles(std::integral_constant<int, 2>{});
        } else
        for (int t = w.t0; t < e; ++t) {
          ok = __all_sync(0xffffffffu, ok && mbar_wait_small(&sm.s_full[x], (uint32_t)(ns++ & 1)));
          tc_fence_after();
          uint32_t v[128];
          const int lim = t * TCA_KEYS + TCA_KEYS - 1 > first ? min(pos, w.s.len - 1) - t * TCA_KEYS : TCA_KEYS;
          const bool edge = t * TCA_KEYS + TCA_KEYS - 1 > first;
          auto load_s = [&](int from, int to_) {
#pragma unroll
            for (int i = from; i < to_; ++i) tca_ld32(ts + 32 * i, v + 32 * i);
            tc_wait_ld();
#pragma unroll
            for (int i = from; i < to_; ++i) tca_tie32(v + 32 * i);
            if (FP8) {                        // the K scales, exactly
              const float* ks = sm.k_scale[FP8 ? (kt + t - w.t0) % 3 : 0];
#pragma unroll
              for (int i = 32 * from; i < 32 * to_; i += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(ks + (FP8 ? i : 0));
                const uint64_t a = mul2(f32x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), f32x2(k4.x, k4.y));
                const uint64_t b = mul2(f32x2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), f32x2(k4.z, k4.w));
                v[i] = (uint32_t)a, v[i + 1] = (uint32_t)(a >> 32), v[i + 2] = (uint32_t)b, v[i + 3] = (uint32_t)(b >> 32);
              }
            }
            if (edge) {
#pragma unroll
              for (int i = 32 * from; i < 32 * to_; ++i)
                if (i > lim) v[i] = 0xff800000u;   // -inf
            }
          };
          load_s(0, 4);
          float mx[4] = {m, m, m, m};
#pragma unroll
          for (int i = 0; i < 128; i += 2) mx[(i >> 1) & 3] = max3_nan(mx[(i >> 1) & 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
          const float mn = max_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3]);
          const uint64_t scale2 = f32x2(sl2, sl2);
          // The first half's exponentials are computed under the old maximum while the new one is found. It stands unless
          // some row has none yet (all of them in the piece's first tile), or one that grew by more than TCA_LAZY, or a NaN.
          uint64_t sum[2] = {0, 0};
          const bool early = t > w.t0;
          if (early) tca_exp<8 * TCA_FIRST, FP8>(v, v, scale2, f32x2(base, base), sum);
          const bool grow = valid && !((mn - m) * sl2 <= TCA_LAZY);
          if (__any_sync(0xffffffffu, grow)) {   // (each row by its own scores: neighbours, and rows that are none, change nothing)
            float f = 1.f;
            if (grow) {
              f = m == -INFINITY ? 0.f : ex2((m - mn) * sl2);
              m = mn;
              l *= f;
              // an infinite maximum makes the row NaN, as inf - inf does
              base = m == -INFINITY ? 0.f : m == INFINITY ? __int_as_float(0x7fffffff) : -m * sl2 - TCA_SHIFT;
            }
            if (early) {                      // the products before this tile's scores are done: O is whole
#pragma unroll 1
              for (int i = 0; i < 8; ++i) {
                uint32_t o[16];
                tca_ld16(to + 16 * i, o);
                tc_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                tca_st16(to + 16 * i, o);
              }
            }
            if (early) load_s(0, (TCA_FIRST + 1) / 2);
            sum[0] = sum[1] = 0;
            tca_exp<8 * TCA_FIRST, FP8>(v, v, scale2, f32x2(base, base), sum);
          }
          auto hand_over = [&](int hh) {
            tca_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.p_full[x][hh]);
          };
          const float* vs = sm.v_scale[FP8 ? (kt + t - w.t0) & 1 : 0];
          if (FP8) {                          // V's tile, and with it the scales, is there (its stage waits for this P)
            const uint32_t i = 2 * (kt + t - w.t0) + 1;
            ok = __all_sync(0xffffffffu, ok && mbar_wait_small(&sm.full[i % TCA_STAGES], (i / TCA_STAGES) & 1));
            tca_pack<8 * TCA_FIRST>(v, v, vs);
          }
          tca_st<8 * TCA_FIRST>(ts, v);
          hand_over(0);
          tca_exp<64 - 8 * TCA_FIRST, FP8>(v + 16 * TCA_FIRST, v + 8 * TCA_FIRST, scale2, f32x2(base, base), sum);
          if (FP8) tca_pack<64 - 8 * TCA_FIRST>(v + 16 * TCA_FIRST, v + 8 * TCA_FIRST, vs + (FP8 ? 16 * TCA_FIRST : 0));
          tca_st<64 - 8 * TCA_FIRST>(ts + 8 * TCA_FIRST, v + 8 * TCA_FIRST);
          hand_over(1);
          l += (f32x2_lo(sum[0]) + f32x2_hi(sum[0])) + (f32x2_lo(sum[1]) + f32x2_hi(sum[1]));
        }

        kt += w.t1 - w.t0;
        // ---- the piece's end: the output rows, or a partial --------------------------------------------------------
        const bool any = e > w.t0;
        if (any) {
          ok = __all_sync(0xffffffffu, ok && mbar_wait_small(&sm.o_full[x], (uint32_t)(no++ & 1)));
          tc_fence_after();
        }
        bf16* dst = r.out + (long long)(w.s.row0 + tok) * r.out_row + (long long)(w.g * r.group + hq) * r.out_head;
        auto store = [&](const float* o, float inv, int col) {   // 32 columns
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = o[k + i] * inv;
            *reinterpret_cast<uint4*>(dst + col + k) = pack_bf16x8(y);
          }
        };
        // sums for prefix_merge_kernel: of the own keys, or of a prefix that no other CTA has keys of, in parts
        const int row_at = (w.s.row0 + tok) * r.n_q + w.g * r.group + hq, part = MODE == TC_PREFIX ? (warp & 3) / per : 0;
        const int split = parts == 4 ? 2 : parts - 1;
        const float m2 = m == -INFINITY ? m : m * sl2 + TCA_SHIFT;
        if ((MODE == TC_PREFIX || (MODE == TC_OWN && w.s.start)) && w.t0 == 0 && w.t1 == w.n) {
          if (any) {
            float* sums = MODE == TC_PREFIX ? p.x.o(row_at, part) : p.x.own_o(row_at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t o[32];
              tca_ld32(to + 32 * i, o);
              tc_wait_ld();
              tca_tie32(o);
              if (valid) {
#pragma unroll
                for (int k = 0; k < 32; k += 4) *reinterpret_cast<uint4*>(sums + 32 * i + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
              }
              __syncwarp();
            }
            if (valid) {
              *(MODE == TC_PREFIX ? p.x.ml(row_at, part) : p.x.own_ml(row_at)) = make_float2(m2, l);
              if (MODE == TC_OWN) *p.x.own_info(row_at) = OWN_SUMS;
              else if (part == 0) *p.x.info(row_at) = PREFIX_WHOLE | split << 24;
            }
            __syncwarp();
          }
          continue;
        }
        if (w.t0 == 0 && w.t1 == w.n) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          if (any) {
            uint32_t o[128];
#pragma unroll
            for (int i = 0; i < 4; ++i) tca_ld32(to + 32 * i, o + 32 * i);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 4; ++i) tca_tie32(o + 32 * i);
            if (valid) {
#pragma unroll
              for (int i = 0; i < 4; ++i) store(reinterpret_cast<const float*>(o + 32 * i), inv, 32 * i);
            }
            __syncwarp();
          }
          continue;
        }
        // boundaries inside the unit: c_lo .. c_hi; its first piece is CTA c_lo - 1's last (slot 1), piece i > 0 is CTA
        // c_lo + i - 1's first (slot 0)
        const long long a0 = w.u - w.t0 - (w.t0 ? TCA_UNIT_COST : 0);
        const int G = (int)min((long long)gridDim.x, max(1ll, W / TCA_MIN_PIECE));
        const int c_lo = (int)div_short((a0 + TCA_UNIT_COST + TCA_MIN_PIECE) * G + W - 1, W);
        const int c_hi = (int)div_short((a0 + TCA_UNIT_COST + w.n - TCA_MIN_PIECE + 1) * G + W - 1, W) - 1;
        const size_t slot = ((size_t)(c * 2 + (w.t0 == 0 ? 1 : 0)) * 2 + x) * 128;
        *reinterpret_cast<float2*>(p.ml + (slot + row) * 2) = make_float2(MODE == TC_PREFIX ? m2 : m, l);
        if (any) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t o[32];
            tca_ld32(to + 32 * i, o);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<uint4*>(p.part + slot * 128 + (size_t)(8 * i + k / 4) * 512 + row * 4) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
        }
        if (MODE == TC_PREFIX) {              // (the merge adds the pieces)
          if (valid && w.t0 == 0 && part == 0) *p.x.info(row_at) = PREFIX_PIECES | (c_lo - 1) | c_hi << 8 | (x * 128 + row) << 16 | split << 24;
          __syncwarp();
          continue;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (tid == 0) {                       // releases the CTA's stores (ordered before by the barrier), acquires the others'
          const int before = add_acq_rel(p.counters + c_lo - 1, 1);
          sm.last = before == c_hi - c_lo + 1;
          if (sm.last) p.counters[c_lo - 1] = 0;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const bool last = sm.last;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (last && valid) {
          auto slot_of = [&](int cc) { return ((size_t)(cc * 2 + (cc == c_lo - 1 ? 1 : 0)) * 2 + x) * 128; };
          float M = -INFINITY;
#pragma unroll 4
          for (int cc = c_lo - 1; cc <= c_hi; ++cc) M = fmaxf(M, __ldcg(p.ml + (slot_of(cc) + row) * 2));
#pragma unroll 1
          for (int col = 0; col < 128; col += 64) {   // 16 loads in flight a piece
            float o[64] = {}, L = 0.f;
            for (int cc = c_lo - 1; cc <= c_hi; ++cc) {
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.ml + (slot_of(cc) + row) * 2));
              float4 q[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) q[k] = __ldcg(reinterpret_cast<const float4*>(p.part + slot_of(cc) * 128 + (size_t)(col / 4 + k) * 512 + row * 4));
              if (ml.y == 0.f) continue;      // no key of the piece was visible (and its O may not have been written)
              const float f = M == -INFINITY ? 1.f : ex2((ml.x - M) * sl2);
              L += ml.y * f;
#pragma unroll
              for (int k = 0; k < 16; ++k)
                o[4 * k] += q[k].x * f, o[4 * k + 1] += q[k].y * f, o[4 * k + 2] += q[k].z * f, o[4 * k + 3] += q[k].w * f;
            }
            if (MODE == TC_OWN && w.s.start) {
#pragma unroll
              for (int k = 0; k < 64; k += 4) *reinterpret_cast<float4*>(p.x.own_o(row_at) + col + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
              if (col == 0) *p.x.own_ml(row_at) = make_float2(M == -INFINITY ? M : M * sl2 + TCA_SHIFT, L), *p.x.own_info(row_at) = OWN_SUMS;
              continue;
            }
            const float inv = L == 0.f ? 0.f : 1.f / L;
            store(o, inv, col);
            store(o + 32, inv, col + 32);
          }
        }
        __syncwarp();
      }
      if (!ok && lane == 0) atomicOr(&g_dev_error, DEVERR_MBAR_TIMEOUT);
    }
  }
  if (p.after) grid_dep_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace qk

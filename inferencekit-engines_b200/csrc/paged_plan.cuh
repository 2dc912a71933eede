// The bookkeeping of a paged cache whose sequences share pages, on the device: free pages into the block tables of a pass,
// and the reordering of sequences that fork.
//
// refs[p] counts the sequences that hold page p; 0 is a free page. A sequence of length n holds the first ceil(n / page_size)
// entries of its block table. Both kernels give out the lowest free pages, in the order of the sequences, so what they leave
// depends on their inputs alone.
//
//   plan: need_b = ceil((len_b + new_b) / P) - ceil(len_b / P), all of them or none; cu = prefix sums of new; slot of every
//         new row; per group of sequences the leading positions that lie in the same pages
//   fork: row i continues row parents[i]: refs of the old rows' pages fall, those of the new rows' rise; a partly filled last page
//         goes to the first row that ends in it, the others get a page of their own and a copy of the filled rows
//
// Both are chains of short dependent steps (prefix sums over sequences, over pages, then tables, then slots), bound by the
// latency of each, so each is one launch: a CTA, or a cluster of eight for large batches and pools, which share out the
// pages, the table rows and the slots and meet at a barrier between the steps (700 sequences, 43,000 rows, 46,000 pages: 25 us; 92 with one
// CTA). Prefix sums over sequences are every CTA's own.
#pragma once
#include "paged.cuh"

namespace qk {

constexpr int PLAN_THREADS = 1024, PLAN_WARPS = PLAN_THREADS / 32;
constexpr int PLAN_MAX_BATCH = 16384;      // sequences of a call: their prefix sums lie in shared memory

struct PlanParams {
  const int* refs;      // [pages]
  int* refs_out;        // may be refs
  const int* table;     // [B] rows of width entries
  int* table_out;       // may be table
  const int* lens;      // [B] positions in the cache
  const int* fresh;     // [B] tokens that enter
  int* cu;              // [B + 1]
  int* seq_lens;        // [B]
  int* slots;           // [T], or null
  int* positions;       // [T], or null
  const int* groups;    // [G + 1]
  int* shared;          // [G]
  int* info;            // [2], or null: pages missing, free pages left
  long long table_stride, out_stride;
  int B, width, pages, page_shift, T, G;
};

// The warps' sums; the arrays over sequences (and pages) lie behind them.
struct PlanSmem {
  long long need[PLAN_WARPS], rows[PLAN_WARPS];
  int free[PLAN_WARPS], copies[PLAN_WARPS], cta_free, pad[3];
};

// The CTAs of a launch are one cluster (or a single one).
__device__ __forceinline__ void plan_sync() {
  if (gridDim.x == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The int that CTA `rank` of the cluster has at the place of `p`.
__device__ __forceinline__ int plan_remote(const int* p, int rank) {
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ long long warp_scan(long long v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Free pages, counted and dealt out by warps: warp w of n takes pages [w * per, (w + 1) * per), 128 at a time, four a lane, the
// next ones on their way.
struct FreePages {
  int first, last;
  __device__ __forceinline__ FreePages(int pages, int w, int n) {
    const int per = ((pages + n - 1) / n + 127) / 128 * 128;
    first = (int)min((long long)pages, (long long)w * per);
    last = (int)min((long long)pages, (long long)(w + 1) * per);
  }
  // f(page, refs of it, whether it is free, free pages of the range before it): for every page of the range, whose refs are get(page).
  // Returns the free ones.
  template <typename G, typename F>
  __device__ __forceinline__ int each(G get, int lane, F f) const {
    int before = 0, next[4];
    auto load = [&](int p0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = p0 + 32 * k + lane;
        next[k] = p < last ? get(p) : 1;
      }
    };
    load(first);
    for (int p0 = first; p0 < last; p0 += 128) {
      int v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = next[k];
      load(p0 + 128);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned free = __ballot_sync(0xffffffffu, v[k] == 0);
        const int p = p0 + 32 * k + lane;
        if (p < last) f(p, v[k], v[k] == 0, before + __popc(free & ((1u << lane) - 1)));
        before += __popc(free);
      }
    }
    return before;
  }
};

// The sequence that takes the page of rank r: the last one whose exclusive sum is <= r, of those that take any.
__device__ __forceinline__ int taker_of(const int* sums, int n, int r) {
  int lo = 0, hi = n;                       // sums[lo] <= r
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (sums[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS, 1) paged_plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ __align__(16) uint8_t plan_smem[];
  PlanSmem& sm = *reinterpret_cast<PlanSmem*>(plan_smem);
  int* need_at = reinterpret_cast<int*>(&sm + 1);   // [B] pages of the sequences before
  int* new_at = need_at + p.B;              // [B + 1] rows of the sequences before
  auto &w_need = sm.need, &w_new = sm.rows;
  auto &w_free = sm.free;
  int& cta_free = sm.cta_free;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x, ctas = gridDim.x;
  const int all_warps = PLAN_WARPS * ctas, my_warp = cta * PLAN_WARPS + warp;
  const int P = 1 << p.page_shift;
  grid_dep_wait();
  grid_dep_launch();
  auto pages_of = [&](int n) { return (int)(((long long)n + P - 1) >> p.page_shift); };
  // ---- lengths: prefix sums over the sequences, in chunks of a thread's contiguous ones ------------------------------------
  auto rows_of = [&](int b, int& len) {     // the rows that enter; a sequence with a bad length sits out
    len = __ldg(p.lens + b);
    const int n = __ldg(p.fresh + b);
    const bool bad = len < 0 || n < 0 || (long long)len + n > ((long long)p.width << p.page_shift);
    if (bad) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    return bad ? 0 : n;
  };
  const int per = (p.B + PLAN_THREADS - 1) / PLAN_THREADS;
  long long need = 0, rows = 0;
  for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) {
    int len;
    const int n = rows_of(b, len);
    need += n ? pages_of(len + n) - pages_of(len) : 0;
    rows += n;
  }
  const long long need_in = warp_scan(need, lane), rows_in = warp_scan(rows, lane);
  if (lane == 31) w_need[warp] = need_in, w_new[warp] = rows_in;
  const FreePages range(p.pages, my_warp, all_warps);
  auto refs_of = [&](int page) { return __ldcg(p.refs + page); };
  const int free_here = range.each(refs_of, lane, [](int, int, bool, int) {});
  if (lane == 0) w_free[warp] = free_here;
  __syncthreads();
  if (ctas > 1 && warp == 0) {
    const int v = __reduce_add_sync(0xffffffffu, w_free[lane]);
    if (lane == 0) cta_free = v;
  }
  if (ctas > 1) plan_sync();
  long long need_before = 0, rows_before = 0, all_need = 0, all_rows = 0;
  int free_before = 0, all_free = 0;
  for (int w = 0; w < PLAN_WARPS; ++w) {
    if (w < warp) need_before += w_need[w], rows_before += w_new[w], free_before += w_free[w];
    all_need += w_need[w], all_rows += w_new[w], all_free += w_free[w];
  }
  if (ctas > 1) {
    all_free = 0;
    for (int c = 0; c < ctas; ++c) {
      const int v = plan_remote(&cta_free, c);
      if (c < cta) free_before += v;
      all_free += v;
    }
  }
  const bool too_many = all_rows > 0x7fffffff || (p.T >= 0 && all_rows > p.T);   // (T -1: no row is written)
  const bool fits = all_need <= all_free && !too_many;
  if (tid == 0) new_at[p.B] = fits ? (int)all_rows : 0;
  if (tid == 0 && cta == 0) {
    if (too_many) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    if (all_need > all_free) atomicOr(&g_dev_error, DEVERR_NO_PAGES);
    if (p.info) {
      p.info[0] = (int)max(0ll, all_need - all_free);
      p.info[1] = all_free - (fits ? (int)all_need : 0);
    }
    p.cu[p.B] = fits ? (int)all_rows : 0;
  }
  need_before += need_in - need, rows_before += rows_in - rows;
  for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) {
    int len;
    const int n = fits ? rows_of(b, len) : (len = __ldg(p.lens + b), 0);
    need_at[b] = (int)need_before;
    new_at[b] = fits ? (int)rows_before : 0;
    if (cta == 0) p.cu[b] = new_at[b], p.seq_lens[b] = len + n;
    need_before += n ? pages_of(len + n) - pages_of(len) : 0;
    rows_before += n;
  }
  __syncthreads();

  // ---- pages: those of rank below the sum go to the sequences ----------------------------------------------------------------
  const int take = fits ? (int)all_need : 0;
  if (p.refs_out != p.refs || (free_before < take && free_here))
    range.each(refs_of, lane, [&](int page, int refs, bool free, int before) {
      const int rank = free_before + before;
      const bool taken = free && rank < take;
      if (taken) {
        const int b = taker_of(need_at, p.B, rank);
        p.table_out[b * p.out_stride + pages_of(__ldg(p.lens + b)) + rank - need_at[b]] = page;
      }
      if (taken || p.refs_out != p.refs) p.refs_out[page] = taken ? 1 : refs;
    });
  if (p.table_out != p.table)               // the entries that were there
    for (int b = my_warp; b < p.B; b += all_warps) {
      const int len = __ldg(p.lens + b), n = new_at[b + 1] - new_at[b];
      const int have = n ? pages_of(len) : p.width, want = n ? pages_of(len + n) : p.width;
      for (int j = lane; j < p.width; j += 32)
        if (j < have || j >= want) p.table_out[b * p.out_stride + j] = __ldg(p.table + b * p.table_stride + j);
    }
  plan_sync();

  // ---- rows: a warp per sequence ---------------------------------------------------------------------------------------------
  if (p.slots || p.positions)
    for (int b = my_warp; b < p.B; b += all_warps) {
      const int len = __ldg(p.lens + b), r0 = new_at[b], n = new_at[b + 1] - r0;
      for (int i = lane; i < n; i += 32) {
        const int pos = len + i;
        if (p.positions) p.positions[r0 + i] = pos;
        if (!p.slots) continue;
        const int page = __ldcg(p.table_out + b * p.out_stride + (pos >> p.page_shift));   // (another CTA may have written it)
        const bool bad = page < 0 || page >= p.pages;   // an old entry that names no page
        if (bad) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
        p.slots[r0 + i] = bad ? -1 : (page << p.page_shift) + (pos & (P - 1));
      }
    }
  // ---- groups: leading entries that all members have in the same page, at most what all of them have ---------------------------
  for (int g = my_warp; g < p.G; g += all_warps) {
    const int b0 = __ldg(p.groups + g), b1 = __ldg(p.groups + g + 1);
    int n = 0;
    if (b0 < 0 || b1 < b0 || b1 > p.B) {
      if (lane == 0) atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    } else if (b1 > b0) {
      n = 0x7fffffff;
      for (int b = b0 + lane; b < b1; b += 32) n = min(n, __ldg(p.lens + b));
      n = max(0, __reduce_min_sync(0xffffffffu, n));
      n = (int)min((long long)n, (long long)p.width << p.page_shift);
      const int entries = pages_of(n);
      for (int j0 = 0; j0 < entries; j0 += 32) {
        const int j = j0 + lane;
        bool same = true;
        if (j < entries) {
          const int page = p.table[b0 * p.table_stride + j];
          same = page >= 0;
#pragma unroll 8
          for (int b = b0 + 1; b < b1; ++b) same &= p.table[b * p.table_stride + j] == page;
        }
        const unsigned other = __ballot_sync(0xffffffffu, !same);
        if (other) {
          n = min(n, (j0 + __ffs(other) - 1) << p.page_shift);
          break;
        }
      }
    }
    if (lane == 0) p.shared[g] = n;
  }
}

struct ForkParams {
  const int* refs;
  int* refs_out;        // may be refs
  const int* table;     // [B] rows
  const int* lens;      // [B]
  const int* parents;   // [N], -1: an empty row
  int* table_out;       // [N] rows
  int* lens_out;        // [N]
  int* info;            // [2], or null
  uint8_t* k;           // [layers][pages][n_kv][page_size] rows
  uint8_t* v;
  float* ks;            // [layers][pages][n_kv][page_size], or null
  float* vs;
  long long table_stride, out_stride;
  int B, N, width, pages, page_shift, layers, n_kv, row_bytes, parts;
};

// The tables and counts of a fork. Row i copies where copied(i): its parent's last page is partly filled and an earlier new row ends in
// it too, or something else holds it: a new row that goes past it, or a sequence outside the call.
__global__ void __launch_bounds__(PLAN_THREADS, 1) paged_fork_kernel(const __grid_constant__ ForkParams p) {
  extern __shared__ __align__(16) uint8_t plan_smem[];
  PlanSmem& sm = *reinterpret_cast<PlanSmem*>(plan_smem);
  int* copy_at = reinterpret_cast<int*>(&sm + 1);   // [N] copies of the rows before
  auto refs_of = [&](int page) { return __ldcg(p.refs_out + page); };
  auto &w_copies = sm.copies, &w_free = sm.free;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = 1 << p.page_shift;
  grid_dep_wait();
  grid_dep_launch();
  const int cap = (int)min((long long)p.width << p.page_shift, 0x7fffffffll);
  auto length = [&](int b) {                // of an old row; a bad one is empty
    const int len = __ldg(p.lens + b);
    if (len >= 0 && len <= cap) return len;
    atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    return 0;
  };
  auto pages_of = [&](int n) { return (int)(((long long)n + P - 1) >> p.page_shift); };
  auto parent = [&](int i) {                // -1: empty
    const int b = __ldg(p.parents + i);
    if (b >= -1 && b < p.B) return b;
    atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    return -1;
  };
  auto old_page = [&](int b, int j) {       // -1: not one of the pool's
    const int page = __ldg(p.table + b * p.table_stride + j);
    if (page >= 0 && page < p.pages) return page;
    atomicOr(&g_dev_error, DEVERR_BAD_STATE);
    return -1;
  };
  auto open_page = [&](int i) {             // the partly filled page that row i's parent ends in; -1: none
    const int b = parent(i), n = b < 0 ? 0 : length(b);
    return n & (P - 1) ? old_page(b, n >> p.page_shift) : -1;
  };
  auto count = [&](int b, int entries, int by) {   // a warp: the first entries of an old row
    for (int j = lane; j < entries; j += 32) {
      const int page = old_page(b, j);
      if (page >= 0) atomicAdd(p.refs_out + page, by);
    }
  };
  if (p.refs_out != p.refs) {
#pragma unroll 4
    for (int i = tid; i < p.pages; i += PLAN_THREADS) p.refs_out[i] = __ldcg(p.refs + i);
    __syncthreads();
  }
  // ---- the old rows' pages, and the new rows' but for those partly filled ----------------------------------------------------------
  for (int b = warp; b < p.B; b += PLAN_WARPS) count(b, pages_of(length(b)), -1);
  for (int i = warp; i < p.N; i += PLAN_WARPS) {
    const int b = parent(i);
    if (b >= 0) count(b, length(b) >> p.page_shift, 1);
  }
  __syncthreads();
  // ---- a partly filled page that nothing else holds is the first row's that ends in it: i - N, the least, in the place of its count -----
  const int per = (p.N + PLAN_THREADS - 1) / PLAN_THREADS, i0 = tid * per, i1 = min(p.N, i0 + per);
  for (int i = i0; i < i1; ++i) {
    const int page = open_page(i);
    if (page >= 0 && refs_of(page) <= 0) atomicMin(p.refs_out + page, i - p.N);
  }
  __syncthreads();
  // ---- which rows copy, and the sums of that -----------------------------------------------------------------------------------
  int mine = 0;
  for (int i = i0; i < i1; ++i) {
    const int page = open_page(i);
    copy_at[i] = page >= 0 && refs_of(page) != i - p.N;   // (a flag for now)
    mine += copy_at[i];
  }
  const int incl = (int)warp_scan(mine, lane);
  if (lane == 31) w_copies[warp] = incl;
  __syncthreads();
  int before = incl - mine, wanted = 0;
  for (int w = 0; w < PLAN_WARPS; ++w) {
    if (w < warp) before += w_copies[w];
    wanted += w_copies[w];
  }
  for (int i = i0; i < i1; ++i) {
    const int f = copy_at[i], page = f ? -1 : open_page(i);
    if (page >= 0) p.refs_out[page] = 1;    // its one holder
    copy_at[i] = before;
    before += f;
  }
  __syncthreads();
  auto copied = [&](int i) { return (i + 1 < p.N ? copy_at[i + 1] : wanted) != copy_at[i]; };
  const FreePages range(p.pages, warp, PLAN_WARPS);
  const int free_here = range.each(refs_of, lane, [](int, int, bool, int) {});
  if (lane == 0) w_free[warp] = free_here;
  __syncthreads();
  int free_before = 0, all_free = 0;
  for (int w = 0; w < PLAN_WARPS; ++w) {
    if (w < warp) free_before += w_free[w];
    all_free += w_free[w];
  }
  const bool fits = wanted <= all_free;
  const int missing = fits ? 0 : wanted - all_free;
  if (!fits) {                              // (rare) the counts as they were; the new rows are empty
    for (int i = warp; i < p.N; i += PLAN_WARPS) {
      const int b = parent(i);
      if (b >= 0) count(b, pages_of(length(b)) - (copied(i) ? 1 : 0), -1);
    }
    for (int b = warp; b < p.B; b += PLAN_WARPS) count(b, pages_of(length(b)), 1);
    __syncthreads();
    all_free = 0;
    const int back = range.each(refs_of, lane, [](int, int, bool, int) {});
    if (lane == 0) w_free[warp] = back;
    __syncthreads();
    for (int w = 0; w < PLAN_WARPS; ++w) all_free += w_free[w];
  }
  if (tid == 0) {
    if (!fits) atomicOr(&g_dev_error, DEVERR_NO_PAGES);
    if (p.info) {
      p.info[0] = missing;
      p.info[1] = all_free - (fits ? wanted : 0);
    }
  }
  // ---- the new rows -------------------------------------------------------------------------------------------------------------
  for (int i = warp; i < p.N; i += PLAN_WARPS) {
    const int b = fits ? parent(i) : -1, n = b < 0 ? 0 : length(b);
    const int kept = pages_of(n) - (n && copied(i) ? 1 : 0), all = pages_of(n);
    for (int j = lane; j < p.width; j += 32)
      if (j < kept || j >= all) p.table_out[i * p.out_stride + j] = j < kept ? __ldg(p.table + b * p.table_stride + j) : -1;
    if (lane == 0) p.lens_out[i] = n;
  }
  if (fits && free_before < wanted && free_here)
    range.each(refs_of, lane, [&](int page, int, bool free, int at) {
      const int rank = free_before + at;
      if (!free || rank >= wanted) return;
      const int i = taker_of(copy_at, p.N, rank);
      p.table_out[i * p.out_stride + (length(parent(i)) >> p.page_shift)] = page;
      p.refs_out[page] = 1;
    });
}

// The copies: row i's last page, where it is not its parent's. CTA (i, part): the part's layers' K and V pages.
__global__ void __launch_bounds__(256) paged_copy_kernel(const __grid_constant__ ForkParams p) {
  const int i = blockIdx.x, P = 1 << p.page_shift;
  grid_dep_wait();
  grid_dep_launch();
  const int n = __ldg(p.lens_out + i), fill = n & (P - 1), b = __ldg(p.parents + i);
  if (fill == 0 || b < 0 || b >= p.B) return;
  const int j = n >> p.page_shift;
  if (j >= p.width) return;
  const int src = __ldg(p.table + b * p.table_stride + j), dst = __ldg(p.table_out + i * p.out_stride + j);
  if (src == dst || src < 0 || dst < 0 || src >= p.pages || dst >= p.pages) return;
  const int per_row = p.row_bytes / 16, per_head = fill * per_row, all = p.n_kv * per_head;
  for (int l = blockIdx.y; l < 2 * p.layers; l += p.parts) {
    const size_t page0 = (size_t)(l >> 1) * p.pages;
    uint8_t* pool = l & 1 ? p.v : p.k;
    const size_t rows = (size_t)p.n_kv << p.page_shift;
    const uint4* from = reinterpret_cast<const uint4*>(pool + (page0 + src) * rows * p.row_bytes);
    uint4* to = reinterpret_cast<uint4*>(pool + (page0 + dst) * rows * p.row_bytes);
    for (int x0 = threadIdx.x; x0 < all; x0 += 4 * 256) {   // four vectors a thread on their way
      uint4 v[4];
      int at[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int x = min(x0 + k * 256, all - 1), h = x / per_head;
        at[k] = h * (P * per_row) + x - h * per_head;
        v[k] = ldg_stream(from + at[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (x0 + k * 256 < all) to[at[k]] = v[k];
    }
    if (p.ks) {
      float* scales = l & 1 ? p.vs : p.ks;
      for (int x = threadIdx.x; x < p.n_kv * fill; x += 256) {
        const int h = x / fill;
        const size_t at = ((size_t)h << p.page_shift) + x - h * fill;
        scales[(page0 + dst) * rows + at] = scales[(page0 + src) * rows + at];
      }
    }
  }
}

}  // namespace qk

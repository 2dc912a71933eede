// C entry points of the paged-serving operators (paged.cuh, attention_few.cuh, attention_tc.cuh). Included by qwen3_b200.cu, whose
// argument-check and launch helpers it uses.
#pragma once
#include <mutex>

// the shim packs these structs field by field
static_assert(sizeof(qk_paged_cache_t) == 14 * 8 && sizeof(qk_paged_qkv_t) == 30 * 8 && sizeof(qk_paged_kv_read_t) == 20 * 8 &&
                  sizeof(qk_ragged_attention_t) == 30 * 8,
              "argument structs have 8-byte fields only");

namespace {

// The checks every paged entry point shares, and the cache as the kernels take it.
int paged_cache(PagedCache* c, const qk_paged_cache_t& a, bool lens) {
  if (!a.k_pages || !a.v_pages || !a.cu_rows || !a.block_table || (lens && !a.seq_lens)) return fail(QK_EINVAL, "null pointer argument");
  if (a.kv_fp8 && (!a.k_scale || !a.v_scale)) return fail(QK_EINVAL, "an e4m3 cache needs its row scales");
  if (a.page_size != 16 && a.page_size != 32 && a.page_size != 64 && a.page_size != 128)
    return fail(QK_EINVAL, "page_size=%lld (16, 32, 64 or 128)", a.page_size);
  if (a.n_pages < 1 || a.n_kv < 1 || a.n_kv > 1024 || a.batch < 0 || a.batch > 65536)
    return fail(QK_EINVAL, "n_pages=%lld n_kv=%lld batch=%lld", a.n_pages, a.n_kv, a.batch);
  // rows are counted in 32 bits (bytes are not)
  if (a.n_pages > 0x7fffffffll / (a.n_kv * a.page_size)) return fail(QK_EINVAL, "a pool of more than 2^31 - 1 rows");
  // (stride 0: every sequence reads the one row)
  if (a.table_width < 1 || (a.table_stride != 0 && a.table_stride < a.table_width) || a.table_stride > 0x7fffffffll ||
      a.table_width > 0x3fffffffll / a.page_size)
    return fail(QK_EINVAL, "table_width=%lld table_stride=%lld", a.table_width, a.table_stride);
  if (!aligned(a.k_pages, 16) || !aligned(a.v_pages, 16) || !aligned(a.k_scale, 16) || !aligned(a.v_scale, 16))
    return fail(QK_EINVAL, "pages and scales must be 16-byte aligned");
  c->k = static_cast<uint8_t*>(const_cast<void*>(a.k_pages));
  c->v = static_cast<uint8_t*>(const_cast<void*>(a.v_pages));
  c->ks = const_cast<float*>(a.k_scale);
  c->vs = const_cast<float*>(a.v_scale);
  c->table = a.block_table;
  c->cu = a.cu_rows;
  c->seq_lens = a.seq_lens;
  c->B = (int)a.batch;
  c->n_kv = (int)a.n_kv;
  c->n_pages = (int)a.n_pages;
  c->page_shift = 31 - __builtin_clz((unsigned)a.page_size);
  c->table_width = (int)a.table_width;
  c->table_stride = (int)a.table_stride;
  return QK_OK;
}

// A dimension of one has no stride of its own: whatever it says, it is taken for that of contiguous rows.
long long own_stride(long long size, long long stride, long long contiguous) { return size == 1 ? contiguous : stride; }
bool row_strides(long long a, long long b) { return a >= 0 && b >= 0 && a % 8 == 0 && b % 8 == 0 && a < (1ll << 40) && b < (1ll << 40); }

// Whether no two of an output's rows of 128 values share one: row t, head h at t * row + h * head. Strides that are not
// negative meet only where t grows and h shrinks, so each distance of heads is held against the nearest of rows.
bool rows_apart(long long rows, long long heads, long long row, long long head) {
  if (rows > 1 && row < HEAD_DIM) return false;
  if (head >= HEAD_DIM && (rows <= 1 || row >= (heads - 1) * head + HEAD_DIM)) return true;   // heads within rows
  for (long long h = 1; h < heads; ++h) {
    const long long at = h * head, t = rows > 1 ? std::min(at / row, rows - 1) : 0;
    if (at - t * row < HEAD_DIM) return false;
    if (t + 1 < rows && (t + 1) * row - at < HEAD_DIM) return false;
  }
  return true;
}

// What both attention entry points check: heads, strides (elements), alignment, scale, workspace.
int ragged_common(RaggedParams* p, const qk_ragged_attention_t& a) {
  const long long n_kv = a.cache.n_kv;
  if (!a.q || !a.out || !a.workspace) return fail(QK_EINVAL, "null pointer argument");
  if (a.rows < 0 || a.rows > 0x7fffffffll / 64 || n_kv < 1 || n_kv > 1024 || a.n_q < 1 || a.n_q % n_kv || a.n_q / n_kv > 32)
    return fail(QK_EINVAL, "rows=%lld n_q=%lld n_kv=%lld (1 to 32 query heads per KV head)", a.rows, a.n_q, n_kv);
  const float scale = (float)a.scale;
  if (!(scale > 1e-30f) || !(scale < 1e30f)) return fail(QK_EINVAL, "scale=%g must be positive", a.scale);
  if (a.max_q < 1) return fail(QK_EINVAL, "max_q=%lld", a.max_q);
  p->q_row = own_stride(a.rows, a.q_row, a.n_q * HEAD_DIM);
  p->q_head = own_stride(a.n_q, a.q_head, HEAD_DIM);
  p->out_row = own_stride(a.rows, a.out_row, a.n_q * HEAD_DIM);
  p->out_head = own_stride(a.n_q, a.out_head, HEAD_DIM);
  if (!aligned(a.q, 16) || !aligned(a.out, 16) || !row_strides(p->q_row, p->q_head) || !row_strides(p->out_row, p->out_head))
    return fail(QK_EINVAL, "q and out rows and heads must start on 16-byte boundaries");
  if (!rows_apart(a.rows, a.n_q, p->out_row, p->out_head))
    return fail(QK_EINVAL, "rows of out overlap: row stride %lld, head stride %lld", p->out_row, p->out_head);
  if (a.workspace_bytes < qk_ragged_attention_workspace_bytes() || !aligned(a.workspace, 256))
    return fail(QK_EINVAL, "workspace of %lld bytes: %lld needed, 256-byte aligned", a.workspace_bytes, qk_ragged_attention_workspace_bytes());
  p->q = static_cast<const bf16*>(a.q);
  p->out = static_cast<bf16*>(a.out);
  p->T = (int)a.rows;
  p->n_q = (int)a.n_q;
  p->group = (int)(a.n_q / n_kv);
  p->scale = scale;
  return QK_OK;
}

// TMA map of a page pool as [n_pages * n_kv * page_size] rows: box {128 bytes, box_rows}, 128-byte swizzle.
int encode_pool_map(CUtensorMap* map, const void* pool, long long rows, bool fp8, int box_rows) {
  auto enc = tensor_map_encoder();
  if (!enc) return fail(QK_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dims[2] = {HEAD_DIM, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)HEAD_DIM * (fp8 ? 1 : 2)};
  const cuuint32_t box[2] = {fp8 ? 128u : 64u, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(pool),
                         dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(QK_EINVAL, "cuTensorMapEncodeTiled failed for a page pool (CUresult %d)", (int)r);
  return QK_OK;
}

// The attention workspace: counters, partial sums and their (m, l) pairs, two a CTA, of each kernel (the two of a call
// overlap).
constexpr int RAGGED_MAX_CTAS = 160;
struct RaggedWorkspace {
  int few_counters[256], tc_counters[256];
  float few_ml[RAGGED_MAX_CTAS * 2 * 16 * 2], tc_ml[RAGGED_MAX_CTAS * 2 * 256 * 2];
  float few_part[RAGGED_MAX_CTAS * 2 * 16 * HEAD_DIM], tc_part[RAGGED_MAX_CTAS * 2 * 256 * HEAD_DIM];
};

// Held over the launches of a call. The tensor-core kernel of a mixed batch skips its wait for what precedes the few-row
// kernel: another thread's call on the same stream must not get in between, or two of them would run at once on one workspace.
std::mutex& workspace_mutex(const void* workspace) {
  static std::mutex mu[16];
  return mu[(reinterpret_cast<uintptr_t>(workspace) >> 8) % 16];
}

template <bool FP8, int NT>
int launch_few(const RaggedParams& r, int strict, void* workspace, cudaStream_t stream) {
  FewParams p = {};
  const int box = std::min(1 << r.c.page_shift, FewShape<FP8, NT>::KEYS);
  const long long rows = ((long long)r.c.n_pages * r.c.n_kv) << r.c.page_shift;
  if (int e = encode_pool_map(&p.tm_k, r.c.k, rows, FP8, box)) return e;
  if (int e = encode_pool_map(&p.tm_v, r.c.v, rows, FP8, box)) return e;
  RaggedWorkspace* ws = static_cast<RaggedWorkspace*>(workspace);
  p.r = r;
  p.part = ws->few_part;
  p.ml = ws->few_ml;
  p.counters = ws->few_counters;
  p.strict = strict;
  auto k = few_attention_kernel<FP8, NT>;
  const int smem = (int)sizeof(FewSmem<FP8, NT>);
  if (int e = ensure_smem((const void*)k, smem)) return e;
  return launch(k, dim3(std::min(device_sms(), RAGGED_MAX_CTAS)), dim3(FewShape<FP8, NT>::THREADS), smem, stream, p);
}

// TMA map of rows [T][heads][128] bf16 with any strides: box {64 dims, box_heads, box_rows}, 128-byte swizzle, rows past T
// zero-filled.
int encode_rows_map(CUtensorMap* map, const void* base, int heads, int T, long long head_stride, long long row_stride, int box_heads, int box_rows) {
  auto enc = tensor_map_encoder();
  if (!enc) return fail(QK_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dims[3] = {HEAD_DIM, (cuuint64_t)heads, (cuuint64_t)T};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(QK_EINVAL, "cuTensorMapEncodeTiled failed for rows with strides %lld and %lld (CUresult %d)", row_stride, head_stride, (int)r);
  return QK_OK;
}

template <int SRC, int MODE = TC_WHOLE>
int launch_tc(const RaggedParams& r, int min_rows, bool after, void* workspace, cudaStream_t stream, const SharedParams& x = {}) {
  TcAttnParams p = {};
  if (int e = encode_rows_map(&p.tm_q, r.q, r.n_q, r.T, r.q_head, r.q_row, r.group, (MODE == TC_PREFIX ? 32 : 128) / r.group)) return e;
  if (SRC == SRC_PACKED) {
    if (int e = encode_rows_map(&p.tm_k, r.k, r.c.n_kv, r.T, r.kv_head, r.kv_row, 1, TCA_KEYS)) return e;
    if (int e = encode_rows_map(&p.tm_v, r.v, r.c.n_kv, r.T, r.kv_head, r.kv_row, 1, TCA_KEYS)) return e;
  } else {
    const int box = std::min(1 << r.c.page_shift, TCA_KEYS);
    const long long rows = ((long long)r.c.n_pages * r.c.n_kv) << r.c.page_shift;
    if (SRC == SRC_PAGED) {   // (e4m3 tiles come by untiled copies)
      if (int e = encode_pool_map(&p.tm_k, r.c.k, rows, false, box)) return e;
      if (int e = encode_pool_map(&p.tm_v, r.c.v, rows, false, box)) return e;
    }
  }
  RaggedWorkspace* ws = static_cast<RaggedWorkspace*>(workspace);
  p.r = r;
  p.part = ws->tc_part;
  p.ml = ws->tc_ml;
  p.counters = ws->tc_counters;
  p.min_rows = min_rows;
  p.after = after;
  p.seqs = MODE == TC_PREFIX ? x.G : r.c.B;
  p.x = x;
  if (MODE == TC_PREFIX) p.part = x.part, p.ml = x.part_ml;
  auto k = tc_attention_kernel<SRC, MODE>;
  const int smem = (int)sizeof(TcAttnSmem<SRC, MODE>);
  if (int e = ensure_smem((const void*)k, smem)) return e;
  return launch_as(after || g_pdl, k, dim3(std::min(device_sms(), RAGGED_MAX_CTAS)), dim3(TcShape<SRC>::THREADS), smem, stream, p);
}

int warp_grid(long long warps, dim3* grid) {   // 8 warps a CTA
  const long long n = (warps + 7) / 8;
  if (n > 0x7fffffff / 8) return fail(QK_EINVAL, "%lld warps are too many", warps);
  *grid = dim3((unsigned)n);
  return QK_OK;
}

// paged_qkv's warps an SM before a warp takes more than one pair of heads: 1,655 rows of 24 heads take 6.4 us in a graph with
// 16, 8.5 with 8 and 9.1 with 32; 16 rows of 48 heads have a pair each either way.
constexpr int QKV_WARPS = 16;
}  // namespace

extern "C" {

int qk_paged_qkv(const qk_paged_qkv_t* args, qk_stream_t stream) {
  if (!args) return fail(QK_EINVAL, "null pointer argument");
  const qk_paged_qkv_t& a = *args;
  PagedQkvParams p = {};
  if (!a.qkv || !a.cos_tab || !a.sin_tab || !a.q_out) return fail(QK_EINVAL, "null pointer argument");
  if ((a.q_norm == nullptr) != (a.k_norm == nullptr)) return fail(QK_EINVAL, "q_norm and k_norm go together");
  if (a.rows < 0 || a.rows > 0x7fffffffll / 64 || a.n_q < 1 || a.n_q > 4096) return fail(QK_EINVAL, "rows=%lld n_q=%lld", a.rows, a.n_q);
  if (a.rot_half < 8 || a.rot_half > HEAD_DIM / 2 || a.rot_half % 8)
    return fail(QK_EINVAL, "rotary dims %lld must be a multiple of 16, at most %d", 2 * a.rot_half, HEAD_DIM);
  if (a.max_pos < 1 || a.max_pos > 0x7fffffffll) return fail(QK_EINVAL, "max_pos=%lld", a.max_pos);
  if (int r = paged_cache(&p.c, a.cache, true)) return r;
  const long long w_qkv = (a.n_q + 2 * p.c.n_kv) * HEAD_DIM, w_q = a.n_q * HEAD_DIM, w_k = (long long)p.c.n_kv * HEAD_DIM;
  p.qkv_stride = own_stride(a.rows, a.qkv_stride, w_qkv);
  p.q_stride = own_stride(a.rows, a.q_stride, w_q);
  p.k_stride = own_stride(a.rows, a.k_stride, w_k);
  if (p.qkv_stride < w_qkv || p.q_stride < w_q || (a.k_out && p.k_stride < w_k) || !row_strides(p.qkv_stride, p.q_stride) ||
      !row_strides(p.k_stride, 0))
    return fail(QK_EINVAL, "rows overlap or do not start on 16-byte boundaries: qkv_stride=%lld q_stride=%lld k_stride=%lld",
                a.qkv_stride, a.q_stride, a.k_stride);
  if (!aligned(a.qkv, 16) || !aligned(a.q_out, 16) || !aligned(a.k_out, 16) || !aligned(a.q_norm, 16) || !aligned(a.k_norm, 16) ||
      !aligned(a.cos_tab, 16) || !aligned(a.sin_tab, 16))
    return fail(QK_EINVAL, "qkv, q_out, k_out, norms and tables must start on 16-byte boundaries");
  if (a.rows == 0 || p.c.B == 0) return QK_OK;
  p.qkv = static_cast<const bf16*>(a.qkv);
  p.q_out = static_cast<bf16*>(a.q_out);
  p.k_out = static_cast<bf16*>(a.k_out);
  p.q_norm = static_cast<const bf16*>(a.q_norm);
  p.k_norm = static_cast<const bf16*>(a.k_norm);
  p.cos = a.cos_tab;
  p.sin = a.sin_tab;
  p.T = (int)a.rows;
  p.n_q = (int)a.n_q;
  p.max_pos = (int)a.max_pos;
  p.half = (int)a.rot_half;
  p.eps = (float)a.eps;
  const long long pairs = (a.n_q + 1) / 2 + 2 * ((p.c.n_kv + 1) / 2);
  p.span = (int)std::min(pairs, std::max(1ll, a.rows * pairs / ((long long)device_sms() * QKV_WARPS)));
  dim3 grid;
  if (int r = warp_grid(a.rows * ((pairs + p.span - 1) / p.span), &grid)) return r;
  auto k = a.cache.kv_fp8 ? (a.interleaved ? paged_qkv_kernel<true, true> : paged_qkv_kernel<true, false>)
                          : (a.interleaved ? paged_qkv_kernel<false, true> : paged_qkv_kernel<false, false>);
  return launch(k, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), p);
}

int qk_paged_kv_read(const qk_paged_kv_read_t* args, qk_stream_t stream) {
  if (!args) return fail(QK_EINVAL, "null pointer argument");
  const qk_paged_kv_read_t& a = *args;
  PagedReadParams p = {};
  if (!a.k_out || !a.v_out) return fail(QK_EINVAL, "null pointer argument");
  if (a.rows < 0 || a.rows > 0x7fffffffll / 64) return fail(QK_EINVAL, "rows=%lld", a.rows);
  if (int r = paged_cache(&p.c, a.cache, false)) return r;
  p.row_stride = own_stride(a.rows, a.row_stride, (long long)p.c.n_kv * HEAD_DIM);
  p.head_stride = own_stride(p.c.n_kv, a.head_stride, HEAD_DIM);
  if (p.row_stride < HEAD_DIM || !row_strides(p.row_stride, p.head_stride) || !rows_apart(a.rows, p.c.n_kv, p.row_stride, p.head_stride) ||
      !aligned(a.k_out, 16) || !aligned(a.v_out, 16))
    return fail(QK_EINVAL, "row_stride=%lld head_stride=%lld: rows must not overlap and start on 16-byte boundaries", a.row_stride, a.head_stride);
  if (a.rows == 0 || p.c.B == 0) return QK_OK;
  p.starts = a.starts;
  p.k_out = static_cast<bf16*>(a.k_out);
  p.v_out = static_cast<bf16*>(a.v_out);
  p.T = (int)a.rows;
  dim3 grid;
  if (int r = warp_grid(a.rows, &grid)) return r;
  return launch(a.cache.kv_fp8 ? paged_kv_read_kernel<true> : paged_kv_read_kernel<false>, grid, dim3(256), 0,
                static_cast<cudaStream_t>(stream), p);
}

long long qk_ragged_attention_workspace_bytes(void) { return sizeof(RaggedWorkspace); }

int qk_paged_attention(const qk_ragged_attention_t* args, qk_stream_t stream) {
  if (!args) return fail(QK_EINVAL, "null pointer argument");
  RaggedParams p = {};
  if (int r = ragged_common(&p, *args)) return r;
  if (int r = paged_cache(&p.c, args->cache, true)) return r;
  if (p.T == 0 || p.c.B == 0) return QK_OK;
  const bool fp8 = args->cache.kv_fp8 != 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long rows = args->max_q * p.group;
  std::lock_guard<std::mutex> together(workspace_mutex(args->workspace));
  if (rows <= 8) return fp8 ? launch_few<true, 1>(p, 1, args->workspace, st) : launch_few<false, 1>(p, 1, args->workspace, st);
  if (rows <= 16) return fp8 ? launch_few<true, 2>(p, 1, args->workspace, st) : launch_few<false, 2>(p, 1, args->workspace, st);
  // More: the sequences with up to 8 query rows per KV head (those that decode beside a chunk), and the others behind them on
  // the tensor cores, which take a few rows too at the matrix unit's time for 128. 17 to 32 rows in the few-row kernel
  // took longer (16 sequences of up to 8 tokens at up to 16k: 183 us against 118; 8 at up to 400: 22 against 15), 9 to 16
  // take less (103 against 115 for 16 sequences of up to 4 tokens at up to 16k, 82 against 126 over e4m3 pages; 21 against 34
  // for 4 at up to 4k; 15 against 14 for 8 at up to 400).
  // From 9 query heads per KV head on no sequence has that few.
  const bool few = p.group <= 8;
  if (few)
    if (int e = fp8 ? launch_few<true, 1>(p, 0, args->workspace, st) : launch_few<false, 1>(p, 0, args->workspace, st)) return e;
  return fp8 ? launch_tc<SRC_PAGED_FP8>(p, 9, few, args->workspace, st) : launch_tc<SRC_PAGED>(p, 9, few, args->workspace, st);
}

int qk_packed_attention(const qk_ragged_attention_t* args, qk_stream_t stream) {
  if (!args) return fail(QK_EINVAL, "null pointer argument");
  const qk_ragged_attention_t& a = *args;
  RaggedParams p = {};
  if (int r = ragged_common(&p, a)) return r;
  if (!a.k || !a.v || !a.cache.cu_rows) return fail(QK_EINVAL, "null pointer argument");
  if (a.cache.batch < 0 || a.cache.batch > 65536) return fail(QK_EINVAL, "batch=%lld", a.cache.batch);
  p.kv_row = own_stride(a.rows, a.kv_row, a.cache.n_kv * HEAD_DIM);
  p.kv_head = own_stride(a.cache.n_kv, a.kv_head, HEAD_DIM);
  if (!aligned(a.k, 16) || !aligned(a.v, 16) || !row_strides(p.kv_row, p.kv_head))
    return fail(QK_EINVAL, "k and v rows and heads must start on 16-byte boundaries");
  if (p.T == 0 || a.cache.batch == 0) return QK_OK;
  p.k = static_cast<const bf16*>(a.k);
  p.v = static_cast<const bf16*>(a.v);
  p.c.cu = a.cache.cu_rows;
  p.c.B = (int)a.cache.batch;
  p.c.n_kv = (int)a.cache.n_kv;
  std::lock_guard<std::mutex> together(workspace_mutex(a.workspace));
  return launch_tc<SRC_PACKED>(p, 0, false, args->workspace, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

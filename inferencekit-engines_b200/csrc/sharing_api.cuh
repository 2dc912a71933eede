// C entry points of the operators for sequences that share pages (paged_plan.cuh, beam.cuh, the shared prefix of the attention
// kernels). Included by qwen3_b200.cu behind paged_api.cuh, whose helpers it uses.
#pragma once

static_assert(sizeof(qk_paged_plan_t) == 21 * 8 && sizeof(qk_paged_fork_t) == 22 * 8 && sizeof(qk_beam_select_t) == 14 * 8 &&
                  sizeof(qk_shared_attention_t) == 33 * 8,
              "argument structs have 8-byte fields only");

namespace {

bool apart(const void* a, long long a_bytes, const void* b, long long b_bytes) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  return !a || !b || a_bytes <= 0 || b_bytes <= 0 || x + a_bytes <= y || y + b_bytes <= x;
}
// Bytes that `rows` table rows reach over.
long long table_bytes(long long rows, long long width, long long stride) { return rows < 1 ? 0 : ((rows - 1) * stride + width) * 4; }

int pool_shape(long long n_pages, long long page_size, int* shift) {
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return fail(QK_EINVAL, "page_size=%lld (16, 32, 64 or 128)", page_size);
  if (n_pages < 1 || n_pages > 0x7fffffffll / page_size) return fail(QK_EINVAL, "n_pages=%lld", n_pages);
  *shift = 31 - __builtin_clz((unsigned)page_size);
  return QK_OK;
}
int table_shape(long long rows, long long width, long long stride, long long page_size, bool may_repeat) {
  if (rows < 0 || rows > PLAN_MAX_BATCH) return fail(QK_EINVAL, "%lld sequences: at most %d", rows, PLAN_MAX_BATCH);
  if (width < 1 || width > 0x3fffffffll / page_size || stride > 0x7fffffffll || !(stride >= width || (may_repeat && stride == 0)))
    return fail(QK_EINVAL, "table_width=%lld table_stride=%lld", width, stride);
  return QK_OK;
}

// The attention workspace, the prefixes' pieces and the own keys'; then the rows' sums.
struct SharedWorkspace {
  RaggedWorkspace base;
  float prefix_ml[RAGGED_MAX_CTAS * 2 * 256 * 2], prefix_part[RAGGED_MAX_CTAS * 2 * 256 * HEAD_DIM];
  float2 own_ml[OWN_MAX_GRID * 2 * 16];
  float own_part[OWN_MAX_GRID * 2 * 16 * HEAD_DIM];
};
constexpr long long shared_fixed_bytes() { return ((long long)sizeof(SharedWorkspace) + 255) / 256 * 256; }

template <bool FP8, int NT>
int launch_own(const RaggedParams& r, int strict, const SharedParams& x, cudaStream_t stream) {
  OwnParams p = {};
  const int box = std::min(1 << r.c.page_shift, OwnShape<FP8, NT>::KEYS);
  const long long rows = ((long long)r.c.n_pages * r.c.n_kv) << r.c.page_shift;
  if (int e = encode_pool_map(&p.tm_k, r.c.k, rows, FP8, box)) return e;
  if (int e = encode_pool_map(&p.tm_v, r.c.v, rows, FP8, box)) return e;
  p.r = r;
  p.x = x;
  p.strict = strict;
  auto k = own_attention_kernel<FP8, NT>;
  const int smem = (int)sizeof(OwnSmem<FP8, NT>);
  if (int e = ensure_smem((const void*)k, smem)) return e;
  return launch(k, dim3(std::min(std::min(device_sms(), RAGGED_MAX_CTAS) * OWN_WARPS, OWN_MAX_GRID)), dim3(32), smem, stream, p);
}

// The sequences' own keys, the prefixes, their sums: each launch starts beside its forerunner.
template <bool FP8>
int shared_launches(const RaggedParams& p, const qk_ragged_attention_t& a, const SharedParams& x, cudaStream_t st) {
  constexpr int SRC = FP8 ? SRC_PAGED_FP8 : SRC_PAGED;
  void* ws = a.workspace;
  const long long rows = a.max_q * p.group;
  std::lock_guard<std::mutex> together(workspace_mutex(ws));
  // sequences of up to OWN_MAX_ROWS query rows a KV head, and the others on the tensor cores
  const int strict = rows <= OWN_MAX_ROWS;
  // (blocks of 8 rows are the quicker ones; a second block of a prefix's 16 comes out of the L2 cache, which several groups fill:
  // one group of 4 behind 4,096 keys takes 23 us with 8 and 25 with 16, 8 such groups over e4m3 pages 49 and 41)
  if (int e = rows <= 8 && x.G == 1 ? launch_own<FP8, 1>(p, strict, x, st) : launch_own<FP8, 2>(p, strict, x, st)) return e;
  if (!strict)
    if (int e = launch_tc<SRC, TC_OWN>(p, OWN_MAX_ROWS + 1, true, ws, st, x)) return e;
  if (int e = launch_tc<SRC, TC_PREFIX>(p, 0, true, ws, st, x)) return e;
  MergeParams m = {};
  m.x = x;
  m.out = p.out, m.out_row = p.out_row, m.out_head = p.out_head, m.n_q = p.n_q, m.rows = p.T * p.n_q;
  return launch_as(true, prefix_merge_kernel, dim3((m.rows + 3) / 4), dim3(256), 0, st, m);
}

// A launch of one cluster of `ctas` CTAs.
template <typename... KArgs, typename... Args>
int launch_cluster(void (*kernel)(KArgs...), int ctas, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)ctas, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_pdl ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e == cudaSuccess ? QK_OK : cuda_fail(e, "kernel launch");
}
// One CTA for small work, eight for what takes longer than their barriers cost.
int plan_ctas(long long pages, long long batch, long long rows) { return pages > 8192 || batch > 128 || rows > 4096 ? 8 : 1; }

}  // namespace

extern "C" {

int qk_paged_plan(const qk_paged_plan_t* args, qk_stream_t stream) {
  if (!args) return fail(QK_EINVAL, "null pointer argument");
  const qk_paged_plan_t& a = *args;
  PlanParams p = {};
  // (an array without elements may be null)
  if (!a.refs || !a.refs_out || !a.cu_rows || (a.batch && (!a.lens || !a.fresh || !a.block_table || !a.table_out || !a.seq_lens)))
    return fail(QK_EINVAL, "null pointer argument");
  if (a.n_groups && (!a.groups || !a.shared)) return fail(QK_EINVAL, "groups and shared go together");
  if (int r = pool_shape(a.n_pages, a.page_size, &p.page_shift)) return r;
  if (a.n_groups < 0 || a.n_groups > PLAN_MAX_BATCH) return fail(QK_EINVAL, "n_groups=%lld: at most %d", a.n_groups, PLAN_MAX_BATCH);
  if (a.rows < -1 || a.rows > 0x7fffffffll / 64 || ((a.slots || a.positions) && a.rows < 0)) return fail(QK_EINVAL, "rows=%lld", a.rows);
  const bool in_place = a.table_out == a.block_table;
  const long long stride = own_stride(a.batch, a.table_stride, a.table_width), out = own_stride(a.batch, a.out_stride, a.table_width);
  if (int r = table_shape(a.batch, a.table_width, stride, a.page_size, !in_place)) return r;
  if (int r = table_shape(a.batch, a.table_width, out, a.page_size, false)) return r;
  if (in_place && stride != out) return fail(QK_EINVAL, "a table planned in place has one stride, not %lld and %lld", stride, out);
  const long long old_bytes = table_bytes(a.batch, a.table_width, stride), new_bytes = table_bytes(a.batch, a.table_width, out);
  if ((!in_place && !apart(a.block_table, old_bytes, a.table_out, new_bytes)) ||
      (a.refs_out != a.refs && !apart(a.refs, a.n_pages * 4, a.refs_out, a.n_pages * 4)) || !apart(a.lens, a.batch * 4, a.seq_lens, a.batch * 4) ||
      !apart(a.fresh, a.batch * 4, a.seq_lens, a.batch * 4))
    return fail(QK_EINVAL, "outputs overlap inputs (the tables and the counts may be planned in place as a whole)");
  p.refs = a.refs, p.refs_out = a.refs_out;
  p.table = a.block_table, p.table_out = a.table_out;
  p.lens = a.lens, p.fresh = a.fresh, p.cu = a.cu_rows, p.seq_lens = a.seq_lens;
  p.slots = a.slots, p.positions = a.positions, p.groups = a.groups, p.shared = a.shared, p.info = a.info;
  p.table_stride = stride, p.out_stride = out;
  p.B = (int)a.batch, p.width = (int)a.table_width, p.pages = (int)a.n_pages, p.T = (int)a.rows, p.G = (int)a.n_groups;
  const int smem = (int)sizeof(PlanSmem) + (2 * p.B + 1) * 4;
  if (int r = ensure_smem((const void*)paged_plan_kernel, smem)) return r;
  return launch_cluster(paged_plan_kernel, plan_ctas(p.pages, p.B, p.T), dim3(PLAN_THREADS), smem, static_cast<cudaStream_t>(stream), p);
}

int qk_paged_fork(const qk_paged_fork_t* args, qk_stream_t stream) {
  if (!args) return fail(QK_EINVAL, "null pointer argument");
  const qk_paged_fork_t& a = *args;
  ForkParams p = {};
  if (!a.refs || !a.refs_out || !a.k_pages || !a.v_pages || (a.batch && (!a.lens || !a.block_table)) ||
      (a.rows && (!a.parents || !a.table_out || !a.lens_out)))
    return fail(QK_EINVAL, "null pointer argument");
  if (a.kv_fp8 && (!a.k_scale || !a.v_scale)) return fail(QK_EINVAL, "an e4m3 cache needs its row scales");
  if (int r = pool_shape(a.n_pages, a.page_size, &p.page_shift)) return r;
  if (a.layers < 1 || a.layers > 4096 || a.n_kv < 1 || a.n_kv > 1024 || a.n_pages > 0x7fffffffll / (a.n_kv * a.page_size))
    return fail(QK_EINVAL, "layers=%lld n_kv=%lld n_pages=%lld", a.layers, a.n_kv, a.n_pages);
  if (!aligned(a.k_pages, 16) || !aligned(a.v_pages, 16)) return fail(QK_EINVAL, "pages must be 16-byte aligned");
  const long long stride = own_stride(a.batch, a.table_stride, a.table_width), out = own_stride(a.rows, a.out_stride, a.table_width);
  if (int r = table_shape(a.batch, a.table_width, stride, a.page_size, true)) return r;
  if (int r = table_shape(a.rows, a.table_width, out, a.page_size, false)) return r;
  if (!apart(a.block_table, table_bytes(a.batch, a.table_width, stride), a.table_out, table_bytes(a.rows, a.table_width, out)) ||
      (a.refs_out != a.refs && !apart(a.refs, a.n_pages * 4, a.refs_out, a.n_pages * 4)) || !apart(a.lens, a.batch * 4, a.lens_out, a.rows * 4) ||
      !apart(a.parents, a.rows * 4, a.lens_out, a.rows * 4))
    return fail(QK_EINVAL, "outputs overlap inputs (only the counts may be updated in place)");
  p.refs = a.refs, p.refs_out = a.refs_out;
  p.table = a.block_table, p.table_out = a.table_out;
  p.lens = a.lens, p.lens_out = a.lens_out, p.parents = a.parents, p.info = a.info;
  p.k = static_cast<uint8_t*>(a.k_pages), p.v = static_cast<uint8_t*>(a.v_pages);
  p.ks = a.kv_fp8 ? a.k_scale : nullptr, p.vs = a.kv_fp8 ? a.v_scale : nullptr;
  p.table_stride = stride, p.out_stride = out;
  p.B = (int)a.batch, p.N = (int)a.rows, p.width = (int)a.table_width, p.pages = (int)a.n_pages;
  p.layers = (int)a.layers, p.n_kv = (int)a.n_kv, p.row_bytes = a.kv_fp8 ? HEAD_DIM : 2 * HEAD_DIM;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int smem = (int)sizeof(PlanSmem) + p.N * 4;
  if (int r = ensure_smem((const void*)paged_fork_kernel, smem)) return r;
  if (int r = launch(paged_fork_kernel, dim3(1), dim3(PLAN_THREADS), smem, st, p)) return r;
  if (p.N == 0) return QK_OK;
  // a layer's K or V page at a time, where that leaves 32 CTAs an SM (53 us with 8 for 8 requests of 8 beams and 36 layers, 43 with 32)
  p.parts = (int)std::max(1ll, std::min(2ll * p.layers, 32ll * device_sms() / p.N));
  return launch_as(true, paged_copy_kernel, dim3(p.N, p.parts), dim3(256), 0, st, p);   // (its CTAs are there when the tables are)
}

// The chunks' sums and lists; as many chunks as a call of these sizes may make, of rows of either type.
long long qk_beam_workspace_bytes(long long rows, long long vocab, long long k) {
  if (rows < 0 || rows > 65536 || vocab < 1 || vocab > BEAM_MAX_VOCAB || k < 1 || k > BEAM_MAX_K) return -1;
  return std::max(256ll, rows * beam_min_chunks((int)vocab, 4) * (8 * k + 8));
}

int qk_beam_select(const qk_beam_select_t* args, qk_stream_t stream) {
  if (!args) return fail(QK_EINVAL, "null pointer argument");
  const qk_beam_select_t& a = *args;
  BeamParams p = {};
  if ((a.rows && (!a.logits || !a.scores)) || !a.cu_rows || (a.batch && (!a.out_scores || !a.out_parents || !a.out_tokens)) || !a.workspace)
    return fail(QK_EINVAL, "null pointer argument");
  if (a.rows < 0 || a.rows > 65536 || a.batch < 0 || a.batch > PLAN_MAX_BATCH) return fail(QK_EINVAL, "rows=%lld batch=%lld", a.rows, a.batch);
  if (a.vocab < 1 || a.vocab > BEAM_MAX_VOCAB || a.k < 1 || a.k > BEAM_MAX_K)
    return fail(QK_EINVAL, "vocab=%lld (at most %d) k=%lld (at most %d)", a.vocab, BEAM_MAX_VOCAB, a.k, BEAM_MAX_K);
  const int size = a.fp32 ? 4 : 2;
  p.row_stride = own_stride(a.rows, a.row_stride, a.vocab);
  if (!aligned(a.logits, size) || p.row_stride < 0 || p.row_stride > (1ll << 40)) return fail(QK_EINVAL, "row_stride=%lld", a.row_stride);
  const long long need = qk_beam_workspace_bytes(a.rows, a.vocab, a.k);
  if (a.workspace_bytes < need || !aligned(a.workspace, 256))
    return fail(QK_EINVAL, "workspace of %lld bytes: %lld needed, 256-byte aligned", a.workspace_bytes, need);
  if (a.batch == 0) return QK_OK;
  p.logits = a.logits, p.scores = a.scores, p.cu = a.cu_rows;
  p.out_scores = a.out_scores, p.out_parents = a.out_parents, p.out_tokens = a.out_tokens;
  p.B = (int)a.batch, p.R = (int)a.rows, p.V = (int)a.vocab, p.K = (int)a.k;
  p.chunks = beam_min_chunks(p.V, size);
  p.granules = (beam_granules(p.V, size) + p.chunks - 1) / p.chunks;
  const size_t all = (size_t)p.R * p.chunks;
  p.grid = beam_grid((long long)all, device_sms());
  p.keys = static_cast<unsigned long long*>(a.workspace);
  p.ml = reinterpret_cast<float2*>(p.keys + all * p.K);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  std::lock_guard<std::mutex> together(workspace_mutex(a.workspace));   // (another thread's chunks would take the lists' place)
  if (all) {
    auto k = a.fp32 ? beam_chunk_kernel<float> : beam_chunk_kernel<bf16>;
    if (int r = ensure_smem((const void*)k, (int)sizeof(BeamChunkSmem))) return r;
    if (int r = launch(k, dim3(p.grid), dim3(BEAM_THREADS), sizeof(BeamChunkSmem), st, p)) return r;
  }
  const int lists = (int)std::min((size_t)BEAM_MAX_USED, (size_t)std::min(p.R, BEAM_MAX_ROWS) * p.chunks), smem = (int)sizeof(BeamMergeSmem) + lists * p.K * 4;
  if (int r = ensure_smem((const void*)beam_merge_kernel, smem)) return r;
  return launch_as(all || g_pdl, beam_merge_kernel, dim3(p.B), dim3(BEAM_THREADS), smem, st, p);
}

long long qk_shared_attention_workspace_bytes(long long rows, long long n_q) {
  if (rows < 0 || rows > 0x7fffffffll / 64 || n_q < 1 || n_q > 32768 || rows > 0x7fffffffll / n_q) return -1;
  return shared_fixed_bytes() + (rows * n_q + SHARED_BLOCK - 1) / SHARED_BLOCK * (long long)sizeof(SharedRows);
}

int qk_shared_attention(const qk_shared_attention_t* args, qk_stream_t stream) {
  if (!args) return fail(QK_EINVAL, "null pointer argument");
  const qk_shared_attention_t& a = *args;
  RaggedParams p = {};
  if (a.n_groups && (!a.groups || !a.shared)) return fail(QK_EINVAL, "null pointer argument");
  if (a.n_groups < 0 || a.n_groups > 65536) return fail(QK_EINVAL, "n_groups=%lld", a.n_groups);
  if (int r = ragged_common(&p, a.att)) return r;
  if (int r = paged_cache(&p.c, a.att.cache, true)) return r;
  const long long need = qk_shared_attention_workspace_bytes(a.att.rows, a.att.n_q);
  if (need < 0 || a.att.workspace_bytes < need) return fail(QK_EINVAL, "workspace of %lld bytes: %lld needed", a.att.workspace_bytes, need);
  if (p.T == 0 || p.c.B == 0) return QK_OK;
  if (a.n_groups == 0) return qk_paged_attention(&a.att, stream);
  SharedParams x = {};
  x.groups = a.groups, x.shared = a.shared, x.G = (int)a.n_groups;
  char* ws = static_cast<char*>(a.att.workspace);
  SharedWorkspace* fixed = static_cast<SharedWorkspace*>(a.att.workspace);
  x.part = fixed->prefix_part, x.part_ml = fixed->prefix_ml;
  x.own_part = fixed->own_part, x.own_part_ml = fixed->own_ml;
  x.rows = reinterpret_cast<SharedRows*>(ws + shared_fixed_bytes());
  return a.att.cache.kv_fp8 ? shared_launches<true>(p, a.att, x, static_cast<cudaStream_t>(stream))
                            : shared_launches<false>(p, a.att, x, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

// Entry points of the operators on a paged key/value cache: argument checks, tensor maps and launches.
// Included by w4a4_lib.cu, whose helpers it uses.
#pragma once

namespace {

namespace kv = w4a4::kv;
namespace pdec = w4a4::pdec;
namespace ppre = w4a4::ppre;
namespace csum = w4a4::csum;
namespace evict = w4a4::evict;

// Rows of `row` elements at i * s0 + j * s1, i < n0, j < n1: one of the strides covers all that the other reaches.
bool rows_apart(long long s0, long long n0, long long s1, long long n1, long long row) {
  if (n0 <= 1 || n1 <= 1) return (n0 <= 1 || s0 >= row) && (n1 <= 1 || s1 >= row);
  return s0 >= s1 ? s1 >= row && s0 >= s1 * (n1 - 1) + row : s0 >= row && s1 >= s0 * (n0 - 1) + row;
}

// The same of three strides.
bool pages_apart(const long long* st, const w4a4_paged_kv* c) {
  struct Axis { long long stride, n; } a[3] = {{st[0], c->n_pages}, {st[1], c->n_kv_heads}, {st[2], c->page_size}};
  std::sort(a, a + 3, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
  long long reach = c->head_dim;
  for (const Axis& x : a) {
    if (x.n <= 1) continue;
    if (x.stride < reach) return false;
    reach += x.stride * (x.n - 1);
  }
  return true;
}

int check_cache(const w4a4_paged_kv* c) {
  CHECK_ARG(c != nullptr, "cache is NULL");
  CHECK_ARG(c->dtype == W4A4_F16 || c->dtype == W4A4_BF16, "cache dtype %d is neither W4A4_F16 nor W4A4_BF16", c->dtype);
  CHECK_ARG(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128, got %d", c->head_dim);
  CHECK_ARG(c->page_size >= 16 && c->page_size % 16 == 0, "page_size must be a positive multiple of 16, got %d", c->page_size);
  CHECK_ARG(c->n_kv_heads >= 1 && c->n_pages >= 1, "n_kv_heads %d and n_pages %d must be positive", c->n_kv_heads, c->n_pages);
  CHECK_ARG(c->n_seqs >= 0 && c->max_pages >= 0, "n_seqs %d and max_pages %d must not be negative", c->n_seqs, c->max_pages);
  CHECK_ARG((long long)c->max_pages * c->page_size < (1LL << 31) - 1024, "a sequence of %d pages of %d slots is too long",
            c->max_pages, c->page_size);
  CHECK_ARG(c->k_pages && c->v_pages && (c->block_table || c->n_seqs == 0 || c->max_pages == 0), "NULL cache pointer");
  CHECK_ARG(c->table_stride >= c->max_pages, "table_stride (%lld) must be >= max_pages (%d)", c->table_stride, c->max_pages);
  for (int i = 0; i < 3; ++i) {
    CHECK_ARG(c->k_strides[i] > 0 && c->v_strides[i] > 0 && c->k_strides[i] < (1LL << 38) && c->v_strides[i] < (1LL << 38),
              "cache strides must be positive and below 2^38 elements");
    if (c->k_strides[i] % 8 || c->v_strides[i] % 8)
      return fail(W4A4_ERR_ALIGNMENT, "cache strides must be multiples of 8 elements");
  }
  CHECK_ARG(pages_apart(c->k_strides, c) && pages_apart(c->v_strides, c), "slots of the cache overlap");
  if (!aligned(c->k_pages, 16) || !aligned(c->v_pages, 16) || !aligned(c->block_table, 4))
    return fail(W4A4_ERR_ALIGNMENT, "cache pointers must be 16-byte aligned");
  return W4A4_OK;
}

kv::Cache device_cache(const w4a4_paged_kv* c) {
  kv::Cache d;
  d.k = c->k_pages;
  d.v = c->v_pages;
  d.k_page = c->k_strides[0]; d.k_head = c->k_strides[1]; d.k_slot = c->k_strides[2];
  d.v_page = c->v_strides[0]; d.v_head = c->v_strides[1]; d.v_slot = c->v_strides[2];
  d.table = c->block_table;
  d.table_stride = c->table_stride;
  d.n_pages = c->n_pages;
  d.page = c->page_size;
  d.n_kv = c->n_kv_heads;
  d.dim = c->head_dim;
  d.n_seqs = c->n_seqs;
  d.max_pages = c->max_pages;
  return d;
}

kv::Seqs device_seqs(const w4a4_paged_kv* c, const int32_t* cu, const int32_t* lengths, int T, int max_q) {
  kv::Seqs s;
  s.cu = cu;
  s.lengths = lengths;
  s.n = c->n_seqs;
  s.T = T;
  s.max_slots = c->max_pages * c->page_size;
  s.max_q = max_q;
  return s;
}

// Row strides of a (T, heads, dim) operand: the heads of a token do not overlap, nor does a head in two tokens.
int check_rows(const char* what, const void* ptr, long long tok, long long head, int T, int n_heads, int dim) {
  CHECK_ARG(ptr != nullptr, "%s is NULL", what);
  CHECK_ARG(head >= dim || n_heads == 1, "%s: head stride %lld is below head_dim %d", what, head, dim);
  CHECK_ARG(tok >= dim || T == 1, "%s: token stride %lld is below head_dim %d", what, tok, dim);
  if (!aligned(ptr, 16) || tok % 8 || head % 8)
    return fail(W4A4_ERR_ALIGNMENT, "%s must be 16-byte aligned with strides that are multiples of 8 elements", what);
  return W4A4_OK;
}

int check_sizes(const w4a4_paged_kv* c, int T, int n_heads) {
  CHECK_ARG(T >= 0, "T must not be negative, got %d", T);
  CHECK_ARG(n_heads >= 1 && n_heads % c->n_kv_heads == 0, "n_heads (%d) must be a positive multiple of n_kv_heads (%d)", n_heads,
            c->n_kv_heads);
  return W4A4_OK;
}

int check_seqs(const w4a4_paged_kv* c, const int32_t* cu, const int32_t* lengths, int T, int n_heads) {
  const int rc = check_sizes(c, T, n_heads);
  if (rc) return rc;
  CHECK_ARG(c->n_seqs == 0 || (cu && lengths), "cu_seqlens or lengths is NULL");
  if (!aligned(cu, 4) || !aligned(lengths, 4)) return fail(W4A4_ERR_ALIGNMENT, "cu_seqlens and lengths must be 4-byte aligned");
  return W4A4_OK;
}

// Slots of one copy box: the largest power of two up to `tile` that divides a page, so that no box leaves its page.
int box_slots(int page, int tile) {
  int b = page & -page;
  return b < tile ? b : tile;
}

// 4-D map {element, slot, head, page} of keys or values, boxes of 64 elements x `box` slots, 128-byte swizzle.
int make_cache_map(CUtensorMap* m, const w4a4_paged_kv* c, bool values, int box) {
  const long long* st = values ? c->v_strides : c->k_strides;
  cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size, (cuuint64_t)c->n_kv_heads, (cuuint64_t)c->n_pages};
  cuuint64_t strides[3] = {(cuuint64_t)st[2] * 2, (cuuint64_t)st[1] * 2, (cuuint64_t)st[0] * 2};
  cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = encode_map(m, c->dtype == W4A4_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                          values ? c->v_pages : c->k_pages, dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(W4A4_ERR_LAUNCH, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return W4A4_OK;
}

// 3-D map {element, head, token} of queries, boxes of 64 elements x `heads` x `toks`, 128-byte swizzle: the rows of a
// box lie token by token, in each the heads.
int make_query_map(CUtensorMap* m, const void* q, long long tok, long long head, int T, int n_heads, int dim, int dtype, int heads, int toks) {
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)n_heads, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)(n_heads == 1 ? dim : head) * 2, (cuuint64_t)(T == 1 ? (long long)n_heads * dim : tok) * 2};
  cuuint32_t boxes[3] = {64, (cuuint32_t)heads, (cuuint32_t)toks};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = encode_map(m, dtype == W4A4_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                          const_cast<void*>(q), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(W4A4_ERR_LAUNCH, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return W4A4_OK;
}

template <typename F16K, typename BF16K>
auto by_type(int dtype, F16K a, BF16K b) { return dtype == W4A4_F16 ? a : b; }

// ------------------------------------------------------------------ attention plan
// Kernels and workspace (counters, then the parts of either kernel) of a call; host values only.
struct AttnPlan {
  bool few, many;             // the kernel for few rows, the one for many
  int few_rows;               // a sequence with at most this many rows goes to the former
  int toks;                   // tokens of a row tile of the latter
  size_t few_parts, many_parts, joins, total;
};
// A sequence with up to this many rows (new tokens x heads of a group) goes to the kernel for few rows: one row tile of it
// where there are many (sequence, key/value head) pairs, else two, the second of which reads keys and values again.  The
// kernel for many rows reads them once but has three launches.  Measured at 8 key/value heads, dim 128, few against many
// rows, with 20 and with 32 rows: one history of 8191 24 to 29 us, 26 to 29; 2 up to 8191 24 to 30, 26 to 31; 4 40 to 42, 42 to 41;
// 8 64 to 55, 80 to 55; 32 178 to 145, 214 to 142; 4 up to 512 15 to 20, 16 to 20; 8 21 to 21, 27 to 21; 64 62 to 52, 79 to 53.
constexpr int ATTN_MANY_PAIRS = 64;
int attn_few_rows(const w4a4_paged_kv* c) {
  return (long long)c->n_seqs * c->n_kv_heads >= ATTN_MANY_PAIRS ? pdec::ROWS : 2 * pdec::ROWS;
}

AttnPlan attn_plan(const w4a4_paged_kv* c, int T, int n_heads, int max_q, int sm_count) {
  AttnPlan a{};
  const int group = n_heads / c->n_kv_heads, few_rows = attn_few_rows(c);
  a.many = (long long)max_q * group > few_rows && group <= ppre::ROWS;
  a.few = !a.many || c->n_seqs > 1;                        // one sequence: whatever its length, one kernel
  a.few_rows = !a.many ? 0x7fffffff : a.few ? few_rows : 0;
  a.toks = a.many ? ppre::ROWS / group : 0;
  size_t off = W4A4_ATTENTION_STATE_BYTES;
  a.few_parts = off;
  if (a.few) off += round_up((size_t)2 * sm_count * (c->head_dim == 128 ? pdec::Layout<128>::PART : pdec::Layout<64>::PART) * 4, 256);
  a.many_parts = off;
  if (a.many) off += (size_t)2 * sm_count * (c->head_dim == 128 ? ppre::Layout<128>::PART : ppre::Layout<64>::PART) * 4;
  a.joins = off;
  if (a.many) off += (size_t)sm_count * sizeof(ppre::Join);
  a.total = off;
  return a;
}

int weight_sums(const w4a4_paged_kv* cache, const void* q, long long q_tok_stride, long long q_head_stride,
                const int32_t* cu_seqlens, const int32_t* lengths, const float* lse, float* sums, long long sums_seq_stride,
                long long sums_head_stride, int T, int n_heads, int max_q_len, float scale, bool fresh, void* stream) {
  begin_call();
  int rc = check_cache(cache);
  if (!rc) rc = check_seqs(cache, cu_seqlens, lengths, T, n_heads);
  if (rc) return rc;
  CHECK_ARG(max_q_len >= 0, "max_q_len must not be negative, got %d", max_q_len);
  CHECK_ARG(scale > 0.f && scale < 3e38f, "scale must be positive and finite, got %g", (double)scale);
  const int group = n_heads / cache->n_kv_heads;
  if (group > csum::MAX_COLS) return fail(W4A4_ERR_UNSUPPORTED, "%d heads share a key/value head; at most %d", group, csum::MAX_COLS);
  const long long slots = (long long)cache->max_pages * cache->page_size;
  CHECK_ARG((sums_head_stride >= slots || cache->n_kv_heads == 1) && (sums_seq_stride >= slots || cache->n_seqs <= 1),
            "sums strides (%lld, %lld) are below the %lld slots of a row", sums_seq_stride, sums_head_stride, slots);
  CHECK_ARG(slots == 0 || rows_apart(sums_seq_stride, cache->n_seqs, sums_head_stride, cache->n_kv_heads, slots), "rows of sums overlap");
  if (T == 0 || cache->n_seqs == 0 || max_q_len == 0 || slots == 0) return W4A4_OK;
  rc = check_rows("q", q, q_tok_stride, q_head_stride, T, n_heads, cache->head_dim);
  if (rc) return rc;
  CHECK_ARG(lse && sums, "lse or sums is NULL");
  if (!aligned(lse, 4) || !aligned(sums, 4)) return fail(W4A4_ERR_ALIGNMENT, "lse and sums must be 4-byte aligned");
  max_q_len = max_q_len < T ? max_q_len : T;
  // the narrowest product that takes all rows of the longest sequence, 128 at most
  const long long rows = (long long)max_q_len * group;
  const int cols = rows >= csum::MAX_COLS ? csum::MAX_COLS : (int)((rows + 15) / 16 * 16);
  // steps of a unit are counted in 32 bits
  const long long row_tiles = ((long long)max_q_len + cols / group - 1) / (cols / group);
  if ((slots + csum::TILE - 1) / csum::TILE * row_tiles > (1LL << 30))
    return fail(W4A4_ERR_UNSUPPORTED, "%d new tokens over %lld slots are too many for one call", max_q_len, slots);
  DeviceInfo* dev = nullptr;
  rc = current_device(&dev);
  if (rc) return rc;
  csum::Params p;
  p.c = device_cache(cache);
  p.s = device_seqs(cache, cu_seqlens, lengths, T, max_q_len);
  p.lse = lse;
  p.sums = sums;
  p.sums_seq = sums_seq_stride;
  p.sums_head = sums_head_stride;
  p.n_heads = n_heads;
  p.group = group;
  p.box = box_slots(cache->page_size, csum::TILE);
  p.cols = cols;
  p.toks = cols / group;
  p.scale_log2 = scale * kv::LOG2E;
  p.fresh = fresh;
  CUtensorMap tk, tq;
  rc = make_cache_map(&tk, cache, false, p.box);
  if (!rc) rc = make_query_map(&tq, q, q_tok_stride, q_head_stride, T, n_heads, cache->head_dim, cache->dtype, group, p.toks);
  if (rc) return rc;
  const bool d128 = cache->head_dim == 128;
  auto launch = [&](auto k64h, auto k64b, auto k128h, auto k128b, size_t smem) {
    auto kern = d128 ? by_type(cache->dtype, k128h, k128b) : by_type(cache->dtype, k64h, k64b);
    return launch_ex(kern, dim3((unsigned)dev->sm_count), dim3(csum::THREADS), smem, static_cast<cudaStream_t>(stream), 1, tk, tq, p);
  };
  constexpr int N = csum::NARROW, M = csum::MAX_COLS;
  const cudaError_t e =
      p.cols <= N ? launch(csum::cache_sums_kernel<__half, 64, N>, csum::cache_sums_kernel<__nv_bfloat16, 64, N>,
                           csum::cache_sums_kernel<__half, 128, N>, csum::cache_sums_kernel<__nv_bfloat16, 128, N>,
                           d128 ? csum::smem_bytes<128, N>() : csum::smem_bytes<64, N>())
                  : launch(csum::cache_sums_kernel<__half, 64, M>, csum::cache_sums_kernel<__nv_bfloat16, 64, M>,
                           csum::cache_sums_kernel<__half, 128, M>, csum::cache_sums_kernel<__nv_bfloat16, 128, M>,
                           d128 ? csum::smem_bytes<128, M>() : csum::smem_bytes<64, M>());
  if (e != cudaSuccess) return fail(W4A4_ERR_LAUNCH, "weight sums kernel launch: %s", cudaGetErrorString(e));
  return W4A4_OK;
}

}  // namespace

extern "C" {

int w4a4_qkv_rope_cache(const w4a4_paged_kv* cache, const void* qkv, long long ld_qkv, const int32_t* cu_seqlens,
                        const int32_t* lengths, const float* cos, const float* sin, int max_pos, int rot_dim,
                        const void* q_norm, const void* k_norm, float eps, int interleaved, const int32_t* offsets,
                        void* q_out, long long q_tok_stride, long long q_head_stride, int T, int n_heads, void* stream) {
  begin_call();
  int rc = check_cache(cache);
  if (!rc) rc = check_seqs(cache, cu_seqlens, lengths, T, n_heads);
  if (rc) return rc;
  CHECK_ARG(rot_dim >= 0 && rot_dim <= cache->head_dim && rot_dim % 16 == 0, "rot_dim must be a multiple of 16 up to head_dim, got %d", rot_dim);
  CHECK_ARG(rot_dim == 0 || (cos && sin), "cos or sin is NULL");
  CHECK_ARG(max_pos >= 0, "max_pos must not be negative, got %d", max_pos);
  if (!aligned(offsets, 4)) return fail(W4A4_ERR_ALIGNMENT, "offsets must be 4-byte aligned");
  if (T == 0 || cache->n_seqs == 0) return W4A4_OK;
  CHECK_ARG(qkv != nullptr, "qkv is NULL");
  CHECK_ARG(T == 1 || ld_qkv >= (long long)(n_heads + 2 * cache->n_kv_heads) * cache->head_dim, "ld_qkv (%lld) is below the width of a row", ld_qkv);
  rc = check_rows("q_out", q_out, q_tok_stride, q_head_stride, T, n_heads, cache->head_dim);
  if (rc) return rc;
  CHECK_ARG(rows_apart(q_tok_stride, T, q_head_stride, n_heads, cache->head_dim), "rows of q_out overlap");
  if (!aligned(qkv, 16) || ld_qkv % 8 || !aligned(cos, 16) || !aligned(sin, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16))
    return fail(W4A4_ERR_ALIGNMENT, "qkv, cos, sin and the norm weights must be 16-byte aligned");
  DeviceInfo* dev = nullptr;
  rc = current_device(&dev);
  if (rc) return rc;
  kv::RopeParams p;
  p.c = device_cache(cache);
  p.s = device_seqs(cache, cu_seqlens, lengths, T, T);
  p.qkv = qkv;
  p.ld_qkv = ld_qkv;
  p.q_out = q_out;
  p.q_tok = q_tok_stride;
  p.q_head = q_head_stride;
  p.cos = cos;
  p.sin = sin;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.offsets = offsets;
  p.n_heads = n_heads;
  p.rot = rot_dim;
  p.max_pos = max_pos;
  p.interleaved = interleaved != 0;
  p.eps = eps;
  // one token a block while blocks are few, for the latency of a decode step; then four, which pay for the chain to
  // the page number once
  p.toks = T > 8 * dev->sm_count ? 4 : T > 4 * dev->sm_count ? 2 : 1;
  auto pick = [&](auto k64h, auto k64b, auto k128h, auto k128b) { return cache->head_dim == 128 ? by_type(cache->dtype, k128h, k128b) : by_type(cache->dtype, k64h, k64b); };
  auto kern = interleaved ? pick(kv::qkv_rope_kernel<__half, 64, kv::ROPE_PAIRS>, kv::qkv_rope_kernel<__nv_bfloat16, 64, kv::ROPE_PAIRS>,
                                 kv::qkv_rope_kernel<__half, 128, kv::ROPE_PAIRS>, kv::qkv_rope_kernel<__nv_bfloat16, 128, kv::ROPE_PAIRS>)
              : rot_dim == cache->head_dim
                  ? pick(kv::qkv_rope_kernel<__half, 64, kv::ROPE_HALVES>, kv::qkv_rope_kernel<__nv_bfloat16, 64, kv::ROPE_HALVES>,
                         kv::qkv_rope_kernel<__half, 128, kv::ROPE_HALVES>, kv::qkv_rope_kernel<__nv_bfloat16, 128, kv::ROPE_HALVES>)
                  : pick(kv::qkv_rope_kernel<__half, 64, kv::ROPE_APART>, kv::qkv_rope_kernel<__nv_bfloat16, 64, kv::ROPE_APART>,
                         kv::qkv_rope_kernel<__half, 128, kv::ROPE_APART>, kv::qkv_rope_kernel<__nv_bfloat16, 128, kv::ROPE_APART>);
  cudaError_t e = launch_ex(kern, dim3((unsigned)((T + p.toks - 1) / p.toks)), dim3(kv::ROPE_THREADS), 0, static_cast<cudaStream_t>(stream), 1, p);
  if (e != cudaSuccess) return fail(W4A4_ERR_LAUNCH, "rope kernel launch: %s", cudaGetErrorString(e));
  return W4A4_OK;
}

size_t w4a4_paged_attention_workspace_bytes(const w4a4_paged_kv* cache, int T, int n_heads, int max_q_len) {
  begin_call();
  if (check_cache(cache) || check_sizes(cache, T, n_heads)) return 0;
  if (max_q_len < 0) {
    fail(W4A4_ERR_BAD_ARG, "max_q_len must not be negative, got %d", max_q_len);
    return 0;
  }
  DeviceInfo* dev = nullptr;
  if (current_device(&dev)) return 0;
  return attn_plan(cache, T, n_heads, max_q_len < T ? max_q_len : T, dev->sm_count).total;
}

int w4a4_paged_attention(const w4a4_paged_kv* cache, const void* q, long long q_tok_stride, long long q_head_stride,
                         const int32_t* cu_seqlens, const int32_t* lengths, void* out, long long out_tok_stride,
                         long long out_head_stride, float* lse, int T, int n_heads, int max_q_len, float scale,
                         void* workspace, size_t workspace_bytes, void* stream) {
  begin_call();
  int rc = check_cache(cache);
  if (!rc) rc = check_seqs(cache, cu_seqlens, lengths, T, n_heads);
  if (rc) return rc;
  CHECK_ARG(max_q_len >= 0, "max_q_len must not be negative, got %d", max_q_len);
  CHECK_ARG(scale > 0.f && scale < 3e38f, "scale must be positive and finite, got %g", (double)scale);
  if (T == 0 || cache->n_seqs == 0 || max_q_len == 0) return W4A4_OK;
  rc = check_rows("q", q, q_tok_stride, q_head_stride, T, n_heads, cache->head_dim);
  if (!rc) rc = check_rows("out", out, out_tok_stride, out_head_stride, T, n_heads, cache->head_dim);
  if (rc) return rc;
  CHECK_ARG(rows_apart(out_tok_stride, T, out_head_stride, n_heads, cache->head_dim), "rows of out overlap");
  if (!aligned(lse, 4)) return fail(W4A4_ERR_ALIGNMENT, "lse must be 4-byte aligned");
  DeviceInfo* dev = nullptr;
  rc = current_device(&dev);
  if (rc) return rc;
  max_q_len = max_q_len < T ? max_q_len : T;
  const AttnPlan plan = attn_plan(cache, T, n_heads, max_q_len, dev->sm_count);
  if (workspace == nullptr || workspace_bytes < plan.total)
    return fail(W4A4_ERR_WORKSPACE, "workspace of %zu bytes required, got %zu", plan.total, workspace_bytes);
  if (!aligned(workspace, 16)) return fail(W4A4_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  if (dev->sm_count > pdec::MAX_RUNS) return fail(W4A4_ERR_UNSUPPORTED, "%d SMs", dev->sm_count);
  std::lock_guard<std::recursive_mutex> together(dev->launches);
  char* ws = static_cast<char*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool d128 = cache->head_dim == 128;
  const int group = n_heads / cache->n_kv_heads;

  if (plan.few) {
    pdec::Params p;
    p.c = device_cache(cache);
    p.s = device_seqs(cache, cu_seqlens, lengths, T, max_q_len);
    p.q = q;
    p.q_tok = q_tok_stride;
    p.q_head = q_head_stride;
    p.out = out;
    p.o_tok = out_tok_stride;
    p.o_head = out_head_stride;
    p.lse = lse;
    p.arrived = reinterpret_cast<int*>(ws);
    p.parts = reinterpret_cast<float*>(ws + plan.few_parts);
    p.n_heads = n_heads;
    p.group = group;
    p.box = box_slots(cache->page_size, pdec::TILE);
    p.max_rows = plan.few_rows;
    p.scale_log2 = scale * kv::LOG2E;
    CUtensorMap tk, tv;
    rc = make_cache_map(&tk, cache, false, p.box);
    if (!rc) rc = make_cache_map(&tv, cache, true, p.box);
    if (rc) return rc;
    // (with at most eight rows in any sequence half of the row tile's registers and arithmetic fall away)
    auto pick = [&](auto k64h, auto k64b, auto k128h, auto k128b) { return d128 ? by_type(cache->dtype, k128h, k128b) : by_type(cache->dtype, k64h, k64b); };
    auto kern = (long long)max_q_len * group <= 8
                    ? pick(pdec::paged_decode_kernel<__half, 64, 1>, pdec::paged_decode_kernel<__nv_bfloat16, 64, 1>,
                           pdec::paged_decode_kernel<__half, 128, 1>, pdec::paged_decode_kernel<__nv_bfloat16, 128, 1>)
                    : pick(pdec::paged_decode_kernel<__half, 64, 2>, pdec::paged_decode_kernel<__nv_bfloat16, 64, 2>,
                           pdec::paged_decode_kernel<__half, 128, 2>, pdec::paged_decode_kernel<__nv_bfloat16, 128, 2>);
    cudaError_t e = launch_ex(kern, dim3((unsigned)dev->sm_count), dim3(pdec::THREADS), d128 ? pdec::smem_bytes<128>() : pdec::smem_bytes<64>(),
                              st, 1, tk, tv, p, (uint32_t)0);
    if (e != cudaSuccess) return fail(W4A4_ERR_LAUNCH, "decode attention kernel launch: %s", cudaGetErrorString(e));
  }
  if (plan.many) {
    ppre::Params p;
    p.c = device_cache(cache);
    p.s = device_seqs(cache, cu_seqlens, lengths, T, max_q_len);
    p.out = out;
    p.o_tok = out_tok_stride;
    p.o_head = out_head_stride;
    p.lse = lse;
    p.parts = reinterpret_cast<float*>(ws + plan.many_parts);
    p.joins = ws + plan.joins;
    p.n_heads = n_heads;
    p.group = group;
    p.box = box_slots(cache->page_size, ppre::TILE);
    p.toks = plan.toks;
    p.min_rows = plan.few_rows;
    p.scale_log2 = scale * kv::LOG2E;
    CUtensorMap tk, tv, tq;
    rc = make_cache_map(&tk, cache, false, p.box);
    if (!rc) rc = make_cache_map(&tv, cache, true, p.box);
    if (!rc) rc = make_query_map(&tq, q, q_tok_stride, q_head_stride, T, n_heads, cache->head_dim, cache->dtype, group, p.toks);
    if (rc) return rc;
    auto kern = d128 ? by_type(cache->dtype, ppre::paged_prefill_kernel<__half, 128>, ppre::paged_prefill_kernel<__nv_bfloat16, 128>)
                     : by_type(cache->dtype, ppre::paged_prefill_kernel<__half, 64>, ppre::paged_prefill_kernel<__nv_bfloat16, 64>);
    cudaError_t e = launch_ex(kern, dim3((unsigned)dev->sm_count), dim3(ppre::THREADS),
                              d128 ? ppre::smem_bytes<128>() : ppre::smem_bytes<64>(), st, 1, tk, tv, tq, p);
    if (e != cudaSuccess) return fail(W4A4_ERR_LAUNCH, "prompt attention kernel launch: %s", cudaGetErrorString(e));
    auto join = d128 ? by_type(cache->dtype, ppre::paged_join_kernel<__half, 128>, ppre::paged_join_kernel<__nv_bfloat16, 128>)
                     : by_type(cache->dtype, ppre::paged_join_kernel<__half, 64>, ppre::paged_join_kernel<__nv_bfloat16, 64>);
    e = launch_ex(join, dim3((unsigned)dev->sm_count, 2 * ppre::ROWS / ppre::JOIN_ROWS), dim3(ppre::JOIN_THREADS), 0, st, 1, p);
    if (e != cudaSuccess) return fail(W4A4_ERR_LAUNCH, "attention join kernel launch: %s", cudaGetErrorString(e));
  }
  return W4A4_OK;
}

int w4a4_cache_weight_sums(const w4a4_paged_kv* cache, const void* q, long long q_tok_stride, long long q_head_stride,
                           const int32_t* cu_seqlens, const int32_t* lengths, const float* lse, float* sums,
                           long long sums_seq_stride, long long sums_head_stride, int T, int n_heads, int max_q_len,
                           float scale, void* stream) {
  return weight_sums(cache, q, q_tok_stride, q_head_stride, cu_seqlens, lengths, lse, sums, sums_seq_stride, sums_head_stride, T,
                     n_heads, max_q_len, scale, false, stream);
}

int w4a4_cache_weight_sums_fresh(const w4a4_paged_kv* cache, const void* q, long long q_tok_stride, long long q_head_stride,
                                 const int32_t* cu_seqlens, const int32_t* lengths, const float* lse, float* sums,
                                 long long sums_seq_stride, long long sums_head_stride, int T, int n_heads, int max_q_len,
                                 float scale, void* stream) {
  if (T == 0 || max_q_len == 0) {
    begin_call();
    return fail(W4A4_ERR_BAD_ARG, "no new token: nothing would be written");
  }
  return weight_sums(cache, q, q_tok_stride, q_head_stride, cu_seqlens, lengths, lse, sums, sums_seq_stride, sums_head_stride, T,
                     n_heads, max_q_len, scale, true, stream);
}

int w4a4_cache_evict(const w4a4_paged_kv* cache, const w4a4_paged_kv* into, const int32_t* lengths, const float* sums,
                     long long sums_seq_stride, long long sums_head_stride, int budget, int n_sink, int n_recent,
                     int32_t* kept, int32_t* new_lengths, float* new_sums, void* stream) {
  begin_call();
  int rc = check_cache(cache);
  if (!rc) rc = check_cache(into);
  if (rc) return rc;
  CHECK_ARG(into->n_seqs == cache->n_seqs && into->n_kv_heads == cache->n_kv_heads && into->head_dim == cache->head_dim &&
                into->dtype == cache->dtype, "the caches differ in sequences, heads, head_dim or dtype");
  CHECK_ARG(n_sink >= 0 && n_recent >= 0 && (long long)n_sink + n_recent <= budget, "n_sink (%d) and n_recent (%d) must not be negative and fit budget (%d)",
            n_sink, n_recent, budget);
  CHECK_ARG(budget >= 1 && budget <= (long long)into->max_pages * into->page_size, "budget (%d) must be 1 .. %lld, the slots of a sequence",
            budget, (long long)into->max_pages * into->page_size);
  const long long slots = (long long)cache->max_pages * cache->page_size;
  CHECK_ARG((sums_head_stride >= slots || cache->n_kv_heads == 1) && (sums_seq_stride >= slots || cache->n_seqs <= 1),
            "sums strides (%lld, %lld) are below the %lld slots of a row", sums_seq_stride, sums_head_stride, slots);
  if (cache->n_seqs == 0) return W4A4_OK;
  CHECK_ARG(lengths && sums && kept && new_lengths && new_sums, "NULL tensor pointer");
  if (!aligned(lengths, 4) || !aligned(sums, 4) || !aligned(kept, 4) || !aligned(new_lengths, 4) || !aligned(new_sums, 4))
    return fail(W4A4_ERR_ALIGNMENT, "lengths, sums and the outputs must be 4-byte aligned");
  DeviceInfo* dev = nullptr;
  rc = current_device(&dev);
  if (rc) return rc;
  const long long units = (long long)cache->n_seqs * cache->n_kv_heads;
  if (units > (1 << 24)) return fail(W4A4_ERR_UNSUPPORTED, "%lld sequences x heads", units);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  evict::SelectParams s;
  s.lengths = lengths;
  s.sums = sums;
  s.sums_seq = sums_seq_stride;
  s.sums_head = sums_head_stride;
  s.kept = kept;
  s.new_lengths = new_lengths;
  s.new_sums = new_sums;
  s.n_kv = cache->n_kv_heads;
  s.max_slots = (int)slots;
  s.new_slots = into->max_pages * into->page_size;
  s.budget = budget;
  s.sink = n_sink;
  s.recent = n_recent;
  cudaError_t e = launch_ex(evict::evict_select_kernel, dim3((unsigned)units), dim3(evict::SELECT_THREADS), 0, st, 1, s);
  if (e != cudaSuccess) return fail(W4A4_ERR_LAUNCH, "eviction selection kernel launch: %s", cudaGetErrorString(e));
  evict::MoveParams m;
  m.from = device_cache(cache);
  m.to = device_cache(into);
  m.kept = kept;
  m.new_lengths = new_lengths;
  m.budget = budget;
  // Caches that share memory: slot j may be the same place in both, so rows go in order and one block takes them all.
  auto span = [](const w4a4_paged_kv* c, bool v) {
    const long long* t = v ? c->v_strides : c->k_strides;
    return (size_t)2 * ((c->n_pages - 1) * t[0] + (c->n_kv_heads - 1) * t[1] + (c->page_size - 1) * t[2] + c->head_dim);
  };
  auto overlap = [&](const w4a4_paged_kv* a, bool av, const w4a4_paged_kv* b, bool bv) {
    const char* x = static_cast<const char*>(av ? a->v_pages : a->k_pages);
    const char* y = static_cast<const char*>(bv ? b->v_pages : b->k_pages);
    return x < y + span(b, bv) && y < x + span(a, av);
  };
  const bool shared = overlap(cache, false, into, false) || overlap(cache, true, into, true) || overlap(cache, false, into, true) ||
                      overlap(cache, true, into, false);
  m.in_place = cache->k_pages == into->k_pages && cache->v_pages == into->v_pages && cache->block_table == into->block_table &&
               cache->table_stride == into->table_stride && cache->page_size == into->page_size &&
               !memcmp(cache->k_strides, into->k_strides, sizeof cache->k_strides) &&
               !memcmp(cache->v_strides, into->v_strides, sizeof cache->v_strides);
  const long long slices = units * (2 * cache->head_dim / 8 / evict::MOVE_CHUNKS);
  m.parts = 1;
  m.rows_per_part = budget;
  if (!shared) {
    // one batch a block while that fills the card, then up to four: a block's first batch pays for three loads in a row
    int batches = (int)(slices * budget / ((long long)evict::MOVE_ROWS * 8 * dev->sm_count));
    batches = batches < 1 ? 1 : batches > 4 ? 4 : batches;
    m.rows_per_part = batches * evict::MOVE_ROWS;
    m.parts = (budget + m.rows_per_part - 1) / m.rows_per_part;
  }
  const long long blocks = slices * m.parts;
  if (blocks > 2147483647LL) return fail(W4A4_ERR_UNSUPPORTED, "%lld blocks", blocks);
  e = launch_ex(evict::evict_move_kernel, dim3((unsigned)blocks), dim3(evict::MOVE_THREADS), 0, st, 1, m);
  if (e != cudaSuccess) return fail(W4A4_ERR_LAUNCH, "eviction move kernel launch: %s", cudaGetErrorString(e));
  return W4A4_OK;
}

}  // extern "C"

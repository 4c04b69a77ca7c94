// C ABI of the paged key-value cache and the token scores (include/nkimoe.h):
// argument checks in front of the launches of paged_store.cu, paged_copy.cu,
// paged_decode.cu, paged_prefill.cu, paged_tree.cu, accept.cu, logprobs.cu and sample.cu.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <vector>

#include "nkimoe.h"
#include "paged.cuh"

namespace nkimoe {

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

#define NKI_REQUIRE(cond, code, ...)             \
  do {                                           \
    if (!(cond)) return fail(code, __VA_ARGS__); \
  } while (0)

#define NKI_CUDA(call)                                                                            \
  do {                                                                                            \
    cudaError_t e_ = (call);                                                                      \
    if (e_ != cudaSuccess) return fail(NKIMOE_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_)); \
  } while (0)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

int check_heads(int n_heads, int n_kv_heads, int head_dim) {
  NKI_REQUIRE(n_heads > 0 && n_kv_heads > 0, NKIMOE_ERR_INVALID_ARG, "bad head counts");
  NKI_REQUIRE(head_dim == 128, NKIMOE_ERR_UNSUPPORTED, "head_dim %d (only 128 is supported)", head_dim);
  NKI_REQUIRE(n_heads % n_kv_heads == 0, NKIMOE_ERR_INVALID_ARG, "n_heads %d is not a multiple of n_kv_heads %d",
              n_heads, n_kv_heads);
  NKI_REQUIRE(n_heads / n_kv_heads <= 16, NKIMOE_ERR_UNSUPPORTED, "more than 16 query heads per kv head");
  NKI_REQUIRE(n_heads <= 65535, NKIMOE_ERR_UNSUPPORTED, "too many heads");
  return NKIMOE_OK;
}

// The cache arguments that every call shares (see include/nkimoe.h).
int check_cache(const void* k_pages, const void* v_pages, int64_t k_stride, int64_t v_stride, int64_t num_pages,
                int64_t page_size, const void* table, int64_t table_stride, int64_t max_pages, int n_kv,
                PagedCache* c) {
  NKI_REQUIRE(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128 || page_size == 256,
              NKIMOE_ERR_UNSUPPORTED, "page size %lld (16, 32, 64, 128 or 256)", (long long)page_size);
  NKI_REQUIRE(num_pages > 0 && num_pages <= 0x7fffffffLL && max_pages > 0, NKIMOE_ERR_INVALID_ARG, "bad page counts");
  NKI_REQUIRE(max_pages <= (1LL << 30) / page_size, NKIMOE_ERR_UNSUPPORTED, "sequences over 2^30 positions");
  const int64_t page = page_size * n_kv * 128;
  NKI_REQUIRE(k_stride >= page && v_stride >= page && k_stride % 8 == 0 && v_stride % 8 == 0, NKIMOE_ERR_INVALID_ARG,
              "page strides must be multiples of 8 elements and at least a page (%lld)", (long long)page);
  NKI_REQUIRE(table_stride >= max_pages, NKIMOE_ERR_INVALID_ARG, "page table rows overlap");
  NKI_REQUIRE(k_pages && v_pages && table, NKIMOE_ERR_INVALID_ARG, "null pointer");
  NKI_REQUIRE(aligned16(k_pages) && aligned16(v_pages) && aligned4(table), NKIMOE_ERR_INVALID_ARG,
              "pages must be 16-byte aligned, the page table 4-byte aligned");
  c->k = static_cast<__nv_bfloat16*>(const_cast<void*>(k_pages));
  c->v = static_cast<__nv_bfloat16*>(const_cast<void*>(v_pages));
  c->k_stride = k_stride;
  c->v_stride = v_stride;
  c->table = static_cast<const int*>(table);
  c->table_stride = table_stride;
  c->max_pages = static_cast<int>(max_pages);
  c->num_pages = static_cast<int>(num_pages);
  c->nkv = n_kv;
  c->page_shift = 0;
  while ((1 << c->page_shift) < page_size) ++c->page_shift;
  return NKIMOE_OK;
}

int check_window(int64_t window, int64_t sinks) {
  NKI_REQUIRE(window >= 0 && sinks >= 0, NKIMOE_ERR_INVALID_ARG, "window and sinks must not be negative");
  NKI_REQUIRE(window <= (1LL << 30) && sinks <= (1LL << 30), NKIMOE_ERR_UNSUPPORTED, "window or sinks over 2^30");
  return NKIMOE_OK;
}

int check_scale(float scale) {
  NKI_REQUIRE(scale > 0.f && scale <= 3e38f, NKIMOE_ERR_INVALID_ARG, "scale must be positive and finite");
  return NKIMOE_OK;
}

}  // namespace

}  // namespace nkimoe

using namespace nkimoe;

#define NKI_CHECK(call)                 \
  do {                                  \
    const int rc_ = (call);             \
    if (rc_ != NKIMOE_OK) return rc_;   \
  } while (0)

extern "C" {

int nkimoe_stream_capture_id(void* stream, unsigned long long* id) {
  NKI_REQUIRE(id, NKIMOE_ERR_INVALID_ARG, "null pointer");
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  unsigned long long got = 0;
  *id = 0;
  NKI_CUDA(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &st, &got));
  if (st == cudaStreamCaptureStatusActive) *id = got;
  return NKIMOE_OK;
}

int nkimoe_qk_norm_rope_store(const void* qkv, const void* q_weight, const void* k_weight, int w_dtype,
                              const int32_t* cu_seqlens, const int32_t* kv_lens, void* k_pages, void* v_pages,
                              int64_t k_page_stride, int64_t v_page_stride, int64_t num_pages, int64_t page_size,
                              const int32_t* page_table, int64_t table_stride, int64_t max_pages, void* q_out,
                              int64_t T, int64_t batch, int n_heads, int n_kv_heads, int head_dim, float rope_theta,
                              float eps, int* status, void* stream) {
  NKI_CHECK(check_heads(n_heads, n_kv_heads, head_dim));
  NKI_REQUIRE(T >= 0 && batch >= 0, NKIMOE_ERR_INVALID_ARG, "bad shape");
  NKI_REQUIRE(T <= 0x7fffffffLL && batch <= 0x7ffffffeLL, NKIMOE_ERR_UNSUPPORTED, "shape too large");
  NKI_REQUIRE(w_dtype == NKIMOE_F32 || w_dtype == NKIMOE_BF16, NKIMOE_ERR_INVALID_ARG, "bad weight dtype");
  NKI_REQUIRE(rope_theta > 0.f, NKIMOE_ERR_INVALID_ARG, "rope_theta must be positive");
  if (T == 0 || batch == 0) return NKIMOE_OK;
  PagedCache c;
  NKI_CHECK(check_cache(k_pages, v_pages, k_page_stride, v_page_stride, num_pages, page_size, page_table, table_stride,
                        max_pages, n_kv_heads, &c));
  NKI_REQUIRE(qkv && q_weight && k_weight && cu_seqlens && kv_lens && q_out && status, NKIMOE_ERR_INVALID_ARG,
              "null pointer");
  NKI_REQUIRE(aligned16(qkv) && aligned16(q_out) && aligned4(cu_seqlens) && aligned4(kv_lens) && aligned4(status),
              NKIMOE_ERR_INVALID_ARG, "qkv and q_out must be 16-byte aligned, lengths 4-byte aligned");
  NKI_CUDA(paged_store_launch(static_cast<const __nv_bfloat16*>(qkv), q_weight, k_weight, w_dtype, cu_seqlens, kv_lens,
                              c, static_cast<__nv_bfloat16*>(q_out), T, static_cast<int>(batch), n_heads, rope_theta,
                              eps, status, static_cast<cudaStream_t>(stream)));
  return NKIMOE_OK;
}

size_t nkimoe_paged_decode_attention_workspace_bytes(int64_t batch, int n_heads, int n_kv_heads, int64_t max_pages,
                                                     int64_t page_size) {
  if (batch <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || max_pages <= 0 || page_size <= 0 ||
      page_size > 256 || max_pages > (1LL << 30) / page_size || batch > 4096)
    return 0;
  return paged_decode_workspace_bytes(batch, n_heads, n_kv_heads, max_pages, static_cast<int>(page_size));
}

int nkimoe_paged_decode_attention(const void* qkv, const void* q_weight, const void* k_weight, int w_dtype,
                                  const int64_t* positions, int64_t pos_stride, void* k_pages, void* v_pages,
                                  int64_t k_page_stride, int64_t v_page_stride, int64_t num_pages, int64_t page_size,
                                  const int32_t* page_table, int64_t table_stride, int64_t max_pages, void* out,
                                  int64_t batch, int n_heads, int n_kv_heads, int head_dim, float rope_theta, float eps,
                                  float scale, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  NKI_CHECK(check_heads(n_heads, n_kv_heads, head_dim));
  NKI_CHECK(check_window(window, sinks));
  NKI_CHECK(check_scale(scale));
  NKI_REQUIRE(batch >= 0 && (pos_stride == 0 || pos_stride == 1), NKIMOE_ERR_INVALID_ARG, "bad shape");
  NKI_REQUIRE(batch <= 4096, NKIMOE_ERR_UNSUPPORTED, "more than 4096 sequences");
  NKI_REQUIRE(w_dtype == NKIMOE_F32 || w_dtype == NKIMOE_BF16, NKIMOE_ERR_INVALID_ARG, "bad weight dtype");
  NKI_REQUIRE(rope_theta > 0.f, NKIMOE_ERR_INVALID_ARG, "rope_theta must be positive");
  if (batch == 0) return NKIMOE_OK;
  PagedCache c;
  NKI_CHECK(check_cache(k_pages, v_pages, k_page_stride, v_page_stride, num_pages, page_size, page_table, table_stride,
                        max_pages, n_kv_heads, &c));
  NKI_REQUIRE(batch * n_kv_heads * ((max_pages * page_size + 63) / 64 + 6) < 0x7fff0000LL, NKIMOE_ERR_UNSUPPORTED,
              "batch and page table too large");
  NKI_REQUIRE(qkv && q_weight && k_weight && positions && out && workspace, NKIMOE_ERR_INVALID_ARG, "null pointer");
  NKI_REQUIRE(aligned16(qkv) && aligned16(out) && aligned16(workspace) &&
                  (reinterpret_cast<uintptr_t>(positions) & 7) == 0,
              NKIMOE_ERR_INVALID_ARG, "qkv, out and workspace must be 16-byte aligned, positions 8-byte aligned");
  const size_t need =
      paged_decode_workspace_bytes(batch, n_heads, n_kv_heads, max_pages, static_cast<int>(page_size));
  NKI_REQUIRE(workspace_bytes >= need, NKIMOE_ERR_WORKSPACE, "workspace %zu bytes < %zu", workspace_bytes, need);
  NKI_CUDA(paged_decode_launch(static_cast<const __nv_bfloat16*>(qkv), q_weight, k_weight, w_dtype,
                               reinterpret_cast<const long long*>(positions), pos_stride, c,
                               static_cast<__nv_bfloat16*>(out), static_cast<int>(batch), n_heads, rope_theta, eps,
                               scale, static_cast<int>(window), static_cast<int>(sinks), workspace,
                               static_cast<cudaStream_t>(stream)));
  return NKIMOE_OK;
}

size_t nkimoe_paged_prefill_attention_workspace_bytes(int64_t T, int64_t batch, int n_heads, int n_kv_heads,
                                                      int64_t max_pages, int64_t page_size) {
  if (T < 0 || batch < 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > 16 ||
      max_pages <= 0 || page_size <= 0 || page_size > 256 || max_pages > (1LL << 30) / page_size ||
      T > 0x7fffffffLL || batch > (1 << 24))
    return 0;
  return paged_prefill_workspace_bytes(T, batch, n_heads, n_kv_heads, max_pages, static_cast<int>(page_size));
}

int nkimoe_paged_prefill_attention(const void* q, int64_t q_row_stride, const void* k_pages, const void* v_pages,
                                   int64_t k_page_stride, int64_t v_page_stride, int64_t num_pages, int64_t page_size,
                                   const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                                   const int32_t* cu_seqlens, const int32_t* kv_lens, void* out, int64_t T,
                                   int64_t batch, int n_heads, int n_kv_heads, int head_dim, float scale,
                                   int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  NKI_CHECK(check_heads(n_heads, n_kv_heads, head_dim));
  NKI_CHECK(check_window(window, sinks));
  NKI_CHECK(check_scale(scale));
  NKI_REQUIRE(T >= 0 && batch >= 0, NKIMOE_ERR_INVALID_ARG, "bad shape");
  NKI_REQUIRE(T <= 0x7fffffffLL && batch <= (1 << 24), NKIMOE_ERR_UNSUPPORTED, "shape too large");
  if (T == 0 || batch == 0) return NKIMOE_OK;
  PagedCache c;
  NKI_CHECK(check_cache(k_pages, v_pages, k_page_stride, v_page_stride, num_pages, page_size, page_table, table_stride,
                        max_pages, n_kv_heads, &c));
  NKI_REQUIRE((T + batch) * n_kv_heads < 0x7fff0000LL, NKIMOE_ERR_UNSUPPORTED, "shape too large");
  // the key blocks (of 128 positions) of 256 pairs are added up in 32 bits
  NKI_REQUIRE(max_pages * page_size < (1LL << 30), NKIMOE_ERR_UNSUPPORTED, "page tables of 2^30 positions or more");
  NKI_REQUIRE(q && cu_seqlens && kv_lens && out && workspace, NKIMOE_ERR_INVALID_ARG, "null pointer");
  NKI_REQUIRE(q_row_stride >= static_cast<int64_t>(n_heads) * 128 && q_row_stride % 8 == 0, NKIMOE_ERR_INVALID_ARG,
              "query rows must be multiples of 8 elements apart and not overlap");
  NKI_REQUIRE(q_row_stride < (1LL << 38) && k_page_stride < (1LL << 38) && v_page_stride < (1LL << 38),
              NKIMOE_ERR_UNSUPPORTED, "stride too large");
  NKI_REQUIRE(aligned16(q) && aligned16(out) && aligned16(workspace) && aligned4(cu_seqlens) && aligned4(kv_lens),
              NKIMOE_ERR_INVALID_ARG, "q, out and workspace must be 16-byte aligned, lengths 4-byte aligned");
  const size_t need =
      paged_prefill_workspace_bytes(T, batch, n_heads, n_kv_heads, max_pages, static_cast<int>(page_size));
  NKI_REQUIRE(workspace_bytes >= need, NKIMOE_ERR_WORKSPACE, "workspace %zu bytes < %zu", workspace_bytes, need);
  NKI_CUDA(paged_prefill_launch(static_cast<const __nv_bfloat16*>(q), q_row_stride, cu_seqlens, kv_lens, c,
                                static_cast<__nv_bfloat16*>(out), T, static_cast<int>(batch), n_heads, scale,
                                static_cast<int>(window), static_cast<int>(sinks), workspace,
                                static_cast<cudaStream_t>(stream)));
  return NKIMOE_OK;
}

size_t nkimoe_paged_tree_attention_workspace_bytes(int64_t T, int64_t batch, int n_heads, int n_kv_heads,
                                                   int64_t max_pages, int64_t page_size) {
  if (T < 0 || batch < 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > 16 ||
      max_pages <= 0 || page_size <= 0 || page_size > 256 || max_pages > (1LL << 30) / page_size || T > (1 << 24) ||
      batch > (1 << 20))
    return 0;
  return paged_tree_workspace_bytes(T, batch, n_heads, n_kv_heads, max_pages, static_cast<int>(page_size));
}

int nkimoe_paged_tree_attention(const void* qkv, const void* q_weight, const void* k_weight, int w_dtype,
                                const int32_t* parents, const int32_t* cu_seqlens, const int32_t* kv_lens, void* k_pages,
                                void* v_pages, int64_t k_page_stride, int64_t v_page_stride, int64_t num_pages,
                                int64_t page_size, const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                                void* out, int64_t T, int64_t batch, int n_heads, int n_kv_heads, int head_dim,
                                float rope_theta, float eps, float scale, int64_t window, int64_t sinks,
                                void* workspace, size_t workspace_bytes, void* stream) {
  NKI_CHECK(check_heads(n_heads, n_kv_heads, head_dim));
  NKI_CHECK(check_window(window, sinks));
  NKI_CHECK(check_scale(scale));
  NKI_REQUIRE(T >= 0 && batch >= 0, NKIMOE_ERR_INVALID_ARG, "bad shape");
  NKI_REQUIRE(T <= (1 << 24) && batch <= (1 << 20), NKIMOE_ERR_UNSUPPORTED, "shape too large");
  NKI_REQUIRE(w_dtype == NKIMOE_F32 || w_dtype == NKIMOE_BF16, NKIMOE_ERR_INVALID_ARG, "bad weight dtype");
  NKI_REQUIRE(rope_theta > 0.f, NKIMOE_ERR_INVALID_ARG, "rope_theta must be positive");
  if (T == 0 || batch == 0) return NKIMOE_OK;
  PagedCache c;
  NKI_CHECK(check_cache(k_pages, v_pages, k_page_stride, v_page_stride, num_pages, page_size, page_table, table_stride,
                        max_pages, n_kv_heads, &c));
  // the places of all tiles are counted in 32 bits
  const int64_t tiles = (kTreeNodes + 128 / (n_heads / n_kv_heads) - 1) / (128 / (n_heads / n_kv_heads));
  NKI_REQUIRE(batch * tiles * n_kv_heads * ((max_pages * page_size + 127) / 128 + 2) < 0x7fff0000LL,
              NKIMOE_ERR_UNSUPPORTED, "batch and page table too large");
  NKI_REQUIRE(k_page_stride < (1LL << 38) && v_page_stride < (1LL << 38), NKIMOE_ERR_UNSUPPORTED, "stride too large");
  NKI_REQUIRE(qkv && q_weight && k_weight && parents && cu_seqlens && kv_lens && out && workspace,
              NKIMOE_ERR_INVALID_ARG, "null pointer");
  NKI_REQUIRE(aligned16(qkv) && aligned16(out) && aligned16(workspace) && aligned4(parents) && aligned4(cu_seqlens) &&
                  aligned4(kv_lens),
              NKIMOE_ERR_INVALID_ARG, "qkv, out and workspace must be 16-byte aligned, parents and lengths 4-byte aligned");
  const size_t need =
      paged_tree_workspace_bytes(T, batch, n_heads, n_kv_heads, max_pages, static_cast<int>(page_size));
  NKI_REQUIRE(workspace_bytes >= need, NKIMOE_ERR_WORKSPACE, "workspace %zu bytes < %zu", workspace_bytes, need);
  NKI_CUDA(paged_tree_launch(static_cast<const __nv_bfloat16*>(qkv), q_weight, k_weight, w_dtype, parents, cu_seqlens,
                             kv_lens, c, static_cast<__nv_bfloat16*>(out), T, static_cast<int>(batch), n_heads,
                             rope_theta, eps, scale, static_cast<int>(window), static_cast<int>(sinks), workspace,
                             static_cast<cudaStream_t>(stream)));
  return NKIMOE_OK;
}

int nkimoe_copy_pages(void* pages, int64_t planes, int64_t num_pages, int64_t page_bytes, const int32_t* src,
                      const int32_t* dst, int64_t n, void* stream) {
  NKI_REQUIRE(planes > 0 && num_pages > 0 && page_bytes > 0 && n >= 0, NKIMOE_ERR_INVALID_ARG, "bad shape");
  NKI_REQUIRE(page_bytes % 16 == 0, NKIMOE_ERR_UNSUPPORTED, "pages must be multiples of 16 bytes (%lld)",
              (long long)page_bytes);
  NKI_REQUIRE(planes <= (1 << 20) && num_pages <= 0x7fffffffLL && page_bytes <= (1LL << 24), NKIMOE_ERR_UNSUPPORTED,
              "pool too large");
  if (n == 0) return NKIMOE_OK;
  NKI_REQUIRE(pages && src && dst, NKIMOE_ERR_INVALID_ARG, "null pointer");
  NKI_REQUIRE(aligned16(pages), NKIMOE_ERR_INVALID_ARG, "pages must be 16-byte aligned");
  for (int64_t i = 0; i < n; ++i)
    NKI_REQUIRE(src[i] >= 0 && src[i] < num_pages && dst[i] >= 0 && dst[i] < num_pages, NKIMOE_ERR_INVALID_ARG,
                "pair %lld: page %d -> %d of %lld", (long long)i, src[i], dst[i], (long long)num_pages);
  // the copies run at the same time: a page that is written must be written
  // once and read by none
  // (1566 pairs in a pool of 3151: 2 us by a mark per page, 145 us by sorting,
  // which is left for pools so large that clearing the marks would cost more)
  try {
    if (num_pages <= 256 * n + (1 << 16)) {
      std::vector<char> written(static_cast<size_t>(num_pages), 0);
      for (int64_t i = 0; i < n; ++i) {
        NKI_REQUIRE(!written[dst[i]], NKIMOE_ERR_INVALID_ARG, "page %d is written twice", dst[i]);
        written[dst[i]] = 1;
      }
      for (int64_t i = 0; i < n; ++i)
        NKI_REQUIRE(!written[src[i]], NKIMOE_ERR_INVALID_ARG, "page %d is both read and written", src[i]);
    } else {
      std::vector<int32_t> to(dst, dst + n);
      std::sort(to.begin(), to.end());
      for (int64_t i = 1; i < n; ++i)
        NKI_REQUIRE(to[i] != to[i - 1], NKIMOE_ERR_INVALID_ARG, "page %d is written twice", to[i]);
      for (int64_t i = 0; i < n; ++i)
        NKI_REQUIRE(!std::binary_search(to.begin(), to.end(), src[i]), NKIMOE_ERR_INVALID_ARG,
                    "page %d is both read and written", src[i]);
    }
  } catch (...) {
    return fail(NKIMOE_ERR_INVALID_ARG, "out of host memory");
  }
  NKI_CUDA(copy_pages_launch(pages, planes, num_pages * page_bytes, page_bytes, src, dst, n,
                             static_cast<cudaStream_t>(stream)));
  return NKIMOE_OK;
}

size_t nkimoe_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top_n) {
  if (rows < 0 || vocab <= 0 || top_n < 0) return 0;
  return token_logprobs_workspace_bytes(rows, vocab, top_n);
}

int nkimoe_token_logprobs(const void* logits, int dtype, int64_t row_stride, const int64_t* tokens, int64_t rows,
                          int64_t vocab, int top_n, float* logprob, float* entropy, float* top_logprobs,
                          int64_t* top_ids, void* workspace, size_t workspace_bytes, void* stream) {
  NKI_REQUIRE(rows >= 0 && vocab > 0 && top_n >= 0 && row_stride >= 0, NKIMOE_ERR_INVALID_ARG, "bad shape");
  NKI_REQUIRE(dtype == NKIMOE_F32 || dtype == NKIMOE_BF16, NKIMOE_ERR_UNSUPPORTED, "logits must be fp32 or bf16");
  NKI_REQUIRE(top_n <= 32 && top_n <= vocab, NKIMOE_ERR_UNSUPPORTED, "top_n <= min(32, vocab) required (%d)", top_n);
  NKI_REQUIRE(vocab <= (1LL << 30) && rows <= (1LL << 25), NKIMOE_ERR_UNSUPPORTED, "shape too large");
  if (rows == 0) return NKIMOE_OK;
  NKI_REQUIRE(logits && tokens && logprob && entropy && workspace && (top_n == 0 || (top_logprobs && top_ids)),
              NKIMOE_ERR_INVALID_ARG, "null pointer");
  NKI_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype == NKIMOE_F32 ? 3 : 1)) == 0 &&
                  (reinterpret_cast<uintptr_t>(tokens) & 7) == 0 && aligned16(workspace),
              NKIMOE_ERR_INVALID_ARG, "logits and tokens must be aligned to their type, the workspace to 16 bytes");
  const size_t need = token_logprobs_workspace_bytes(rows, vocab, top_n);
  NKI_REQUIRE(workspace_bytes >= need, NKIMOE_ERR_WORKSPACE, "workspace %zu bytes < %zu", workspace_bytes, need);
  NKI_CUDA(token_logprobs_launch(logits, dtype, row_stride, reinterpret_cast<const long long*>(tokens), rows, vocab,
                                 top_n, logprob, entropy, top_logprobs, reinterpret_cast<long long*>(top_ids),
                                 workspace, static_cast<cudaStream_t>(stream)));
  return NKIMOE_OK;
}

int nkimoe_sample_tokens(const void* logits, int dtype, int64_t row_stride, const void* uniforms, int u_dtype,
                         const float* temperature, double temperature_all, const int32_t* top_k, int64_t top_k_all,
                         const float* top_p, double top_p_all, const float* min_p, double min_p_all, int64_t rows,
                         int64_t vocab, int64_t* tokens, float* logprob, void* stream) {
  NKI_REQUIRE(rows >= 0 && vocab > 0 && row_stride >= 0, NKIMOE_ERR_INVALID_ARG, "bad shape");
  NKI_REQUIRE(dtype == NKIMOE_F32 || dtype == NKIMOE_BF16, NKIMOE_ERR_UNSUPPORTED, "logits must be fp32 or bf16");
  NKI_REQUIRE(u_dtype == NKIMOE_F32 || u_dtype == NKIMOE_F64, NKIMOE_ERR_UNSUPPORTED, "uniforms must be fp32 or fp64");
  NKI_REQUIRE(vocab <= (1LL << 18) && rows <= (1LL << 25), NKIMOE_ERR_UNSUPPORTED, "vocab over 2^18 or rows over 2^25");
  NKI_REQUIRE(temperature || (temperature_all >= 0.0 && temperature_all < 1e300), NKIMOE_ERR_INVALID_ARG,
              "temperature must be finite and not negative");
  NKI_REQUIRE(top_p || (top_p_all >= 0.0 && top_p_all <= 1.0), NKIMOE_ERR_INVALID_ARG, "top_p must be in [0, 1]");
  NKI_REQUIRE(min_p || (min_p_all >= 0.0 && min_p_all <= 1.0), NKIMOE_ERR_INVALID_ARG, "min_p must be in [0, 1]");
  NKI_REQUIRE(top_k || top_k_all >= 0, NKIMOE_ERR_INVALID_ARG, "top_k must not be negative");
  if (rows == 0) return NKIMOE_OK;
  NKI_REQUIRE(logits && uniforms && tokens && logprob, NKIMOE_ERR_INVALID_ARG, "null pointer");
  NKI_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype == NKIMOE_F32 ? 3 : 1)) == 0 &&
                  (reinterpret_cast<uintptr_t>(uniforms) & (u_dtype == NKIMOE_F32 ? 3 : 7)) == 0 &&
                  (reinterpret_cast<uintptr_t>(tokens) & 7) == 0 && aligned4(logprob) && aligned4(temperature) &&
                  aligned4(top_k) && aligned4(top_p) && aligned4(min_p),
              NKIMOE_ERR_INVALID_ARG, "pointers must be aligned to their type");
  SampleSettings set;
  set.temperature = temperature;
  set.top_k = top_k;
  set.top_p = top_p;
  set.min_p = min_p;
  set.temperature_all = temperature_all;
  set.top_k_all = top_k_all;
  set.top_p_all = top_p_all;
  set.min_p_all = min_p_all;
  NKI_CUDA(sample_tokens_launch(logits, dtype, row_stride, uniforms, u_dtype == NKIMOE_F64, set, rows, vocab,
                                reinterpret_cast<long long*>(tokens), logprob, static_cast<cudaStream_t>(stream)));
  return NKIMOE_OK;
}

int nkimoe_accept_drafts(const int64_t* tokens, const int64_t* sampled, const int32_t* parents,
                         const int32_t* cu_seqlens, const int32_t* kv_lens, void* pages, int64_t planes,
                         int64_t num_pages, int64_t n_kv_heads, int64_t page_size, int64_t row_bytes,
                         const int32_t* page_table, int64_t table_stride, int64_t max_pages, int32_t* counts,
                         int32_t* path, int64_t* new_tokens, int64_t T, int64_t batch, int* status, void* stream) {
  NKI_REQUIRE(T >= 0 && batch >= 0 && planes > 0 && num_pages > 0 && n_kv_heads > 0 && page_size > 0 && row_bytes > 0 &&
                  max_pages > 0,
              NKIMOE_ERR_INVALID_ARG, "bad shape");
  NKI_REQUIRE(row_bytes % 16 == 0, NKIMOE_ERR_UNSUPPORTED, "rows must be multiples of 16 bytes (%lld)",
              (long long)row_bytes);
  NKI_REQUIRE(batch <= 65535 && T <= 0x7fffffffLL && planes <= (1 << 20) && num_pages <= 0x7fffffffLL &&
                  n_kv_heads <= 65535 && page_size <= (1 << 20) && row_bytes <= (1 << 14) &&
                  n_kv_heads * page_size * row_bytes <= (1LL << 30),
              NKIMOE_ERR_UNSUPPORTED, "shape too large");
  NKI_REQUIRE(max_pages <= (1LL << 30) / page_size, NKIMOE_ERR_UNSUPPORTED, "sequences over 2^30 positions");
  NKI_REQUIRE(table_stride >= max_pages, NKIMOE_ERR_INVALID_ARG, "page table rows overlap");
  if (T == 0 || batch == 0) {  // no paths; rows of no sequence
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (batch > 0 && counts) NKI_CUDA(cudaMemsetAsync(counts, 0, sizeof(int32_t) * batch, s));
    if (T > 0 && path) NKI_CUDA(cudaMemsetAsync(path, 0xff, sizeof(int32_t) * T, s));
    if (T > 0 && new_tokens) NKI_CUDA(cudaMemsetAsync(new_tokens, 0xff, sizeof(int64_t) * T, s));
    return NKIMOE_OK;
  }
  NKI_REQUIRE(tokens && sampled && parents && cu_seqlens && kv_lens && pages && page_table && counts && path &&
                  new_tokens && status,
              NKIMOE_ERR_INVALID_ARG, "null pointer");
  NKI_REQUIRE(aligned16(pages) && ((reinterpret_cast<uintptr_t>(tokens) | reinterpret_cast<uintptr_t>(sampled) |
                                    reinterpret_cast<uintptr_t>(new_tokens)) & 7) == 0 &&
                  aligned4(parents) && aligned4(cu_seqlens) && aligned4(kv_lens) && aligned4(page_table) &&
                  aligned4(counts) && aligned4(path) && aligned4(status),
              NKIMOE_ERR_INVALID_ARG, "pages must be 16-byte aligned, the others to their type");
  NKI_CUDA(accept_drafts_launch(reinterpret_cast<const long long*>(tokens), reinterpret_cast<const long long*>(sampled),
                                parents, cu_seqlens, kv_lens, pages, planes, num_pages, static_cast<int>(n_kv_heads),
                                static_cast<int>(page_size), static_cast<int>(row_bytes), page_table, table_stride,
                                static_cast<int>(max_pages), counts, path, reinterpret_cast<long long*>(new_tokens), T,
                                static_cast<int>(batch), status, static_cast<cudaStream_t>(stream)));
  return NKIMOE_OK;
}

}  // extern "C"

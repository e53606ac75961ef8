// The extern "C" boundary of the paged-cache operators: host-side checks, then the launchers.
#include <cstdarg>
#include <cstdio>

#include "launch.h"
#include "paged_records.cuh"

namespace ipe {
int report_failure(int status, const char* message);
}

namespace {

int fail(int status, const char* fmt, ...) {
  char text[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  return ipe::report_failure(status, text);
}

int finish(cudaError_t e, const char* name) {
  return e == cudaSuccess ? IPE_OK : fail(IPE_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

bool heads_fit(int q_heads, int kv_heads) {
  return q_heads >= 1 && kv_heads >= 1 && q_heads % kv_heads == 0 && q_heads / kv_heads <= 8;
}
bool page_size_fits(int page_size) { return page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128; }
// positions are 32-bit numbers in the kernels, and so is what they are rounded up to
bool pages_fit(int pages, int page_size) { return pages <= (1 << 27) / page_size; }

bool misaligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// The checks every paged entry point shares, and the kernels' view of the cache.
int paged_cache(const char* name, const void* k_pages, const void* v_pages, const int32_t* page_table,
                const int32_t* lengths, int64_t tokens, int sequences, int q_heads, int kv_heads, int64_t num_pages,
                int page_size, int max_pages, ipe::PagedCache* c) {
  if (!heads_fit(q_heads, kv_heads))
    return fail(IPE_ERR_UNSUPPORTED, "%s: %d query heads over %d KV heads: expected 1 to 8 query heads per KV head", name,
                q_heads, kv_heads);
  if (!page_size_fits(page_size))
    return fail(IPE_ERR_UNSUPPORTED, "%s: page_size %d is not 16, 32, 64 or 128", name, page_size);
  if (tokens < 0 || sequences < 0 || num_pages < 1 || max_pages < 1)
    return fail(IPE_ERR_ARGUMENT, "%s: bad sizes (%lld rows, %d sequences, %lld pages, %d per sequence)", name,
                static_cast<long long>(tokens), sequences, static_cast<long long>(num_pages), max_pages);
  // cache rows, (token, head) rows and units of 64 keys are 32-bit numbers in the kernels too; their byte offsets
  // are 64-bit
  if (tokens > INT32_MAX / q_heads || num_pages > INT32_MAX / (static_cast<int64_t>(kv_heads) * page_size) ||
      !pages_fit(max_pages, page_size) || sequences > (1 << 24) ||
      static_cast<int64_t>(sequences) * kv_heads > INT32_MAX / (static_cast<int64_t>(max_pages) * page_size / 64 + 1))
    return fail(IPE_ERR_UNSUPPORTED, "%s: sizes past the kernels' 32-bit row numbers", name);
  if (tokens == 0 || sequences == 0) return IPE_OK;
  if (!k_pages || !v_pages || !page_table || !lengths) return fail(IPE_ERR_ARGUMENT, "%s: null pointer", name);
  if (misaligned(k_pages, 16) || misaligned(v_pages, 16) || misaligned(page_table, 4) || misaligned(lengths, 4))
    return fail(IPE_ERR_ARGUMENT, "%s: pages must be 16-byte aligned, integers 4-byte", name);
  *c = ipe::PagedCache{};
  c->page_table = page_table;
  c->lengths = lengths;
  c->sequences = sequences;
  c->max_pages = max_pages;
  c->page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  c->kv_heads = kv_heads;
  c->num_pages = static_cast<int>(num_pages);
  c->err = ipe::device_error_word_ptr();
  return IPE_OK;
}

int rows_checks(const char* name, const void* q, const void* out) {
  if (!q || !out) return fail(IPE_ERR_ARGUMENT, "%s: null pointer", name);
  if (misaligned(q, 16) || misaligned(out, 16))
    return fail(IPE_ERR_ARGUMENT, "%s: q and out must be 16-byte aligned", name);
  return IPE_OK;
}

int workspace_checks(const char* name, const void* workspace, size_t bytes, size_t need) {
  if (need > 0 && (!workspace || misaligned(workspace, 256) || bytes < need))
    return fail(IPE_ERR_ARGUMENT, "%s: a 256-byte aligned workspace of %zu bytes is needed", name, need);
  return IPE_OK;
}

}  // namespace

extern "C" {

// Nothing for sizes that the entry points refuse: a caller allocates before it is told.
size_t ipe_paged_decode_attention_workspace(int sequences, int q_heads, int kv_heads) {
  if (sequences < 1 || !heads_fit(q_heads, kv_heads)) return 0;
  return ipe::paged_decode_workspace_bytes(sequences, q_heads, kv_heads);
}

size_t ipe_paged_prefill_attention_workspace(int64_t tokens, int sequences, int q_heads, int kv_heads) {
  if (tokens < 1 || sequences < 1 || !heads_fit(q_heads, kv_heads)) return 0;
  return ipe::paged_prefill_workspace_bytes(tokens, sequences, q_heads, kv_heads);
}

size_t ipe_shared_prefix_attention_workspace(int sequences, int q_heads, int kv_heads, int page_size, int prefix_count) {
  if (sequences < 1 || !heads_fit(q_heads, kv_heads) || !page_size_fits(page_size) || prefix_count < 0 ||
      !pages_fit(prefix_count, page_size))
    return 0;
  ipe::PagedCache c{};
  c.sequences = sequences;
  c.kv_heads = kv_heads;
  c.prefix_count = prefix_count;
  while ((1 << c.page_shift) < page_size) ++c.page_shift;
  return ipe::shared_prefix_workspace_bytes(c, q_heads);
}

int ipe_paged_qk_norm_rope_append(const void* qkv, int64_t tokens, int q_heads, int kv_heads,
                                  const void* q_norm_weight, const void* k_norm_weight, const void* cos_table,
                                  const void* sin_table, int table_dtype, int64_t table_rows,
                                  const int32_t* cu_tokens, const int32_t* lengths, const int32_t* page_table,
                                  int sequences, int max_pages, void* q_out, void* k_pages, void* v_pages,
                                  int64_t num_pages, int page_size, float eps, void* stream) {
  const char* name = "ipe_paged_qk_norm_rope_append";
  ipe::PagedCache c;
  if (int status = paged_cache(name, k_pages, v_pages, page_table, lengths, tokens, sequences, q_heads, kv_heads,
                               num_pages, page_size, max_pages, &c))
    return status;
  if ((table_dtype != 0 && table_dtype != 1) || table_rows < 1)
    return fail(IPE_ERR_ARGUMENT, "%s: %lld table rows of dtype %d", name, static_cast<long long>(table_rows), table_dtype);
  if (tokens == 0 || sequences == 0) return IPE_OK;
  if (!qkv || !q_norm_weight || !k_norm_weight || !cos_table || !sin_table || !cu_tokens || !q_out)
    return fail(IPE_ERR_ARGUMENT, "%s: null pointer", name);
  for (const void* p : {qkv, q_norm_weight, k_norm_weight, cos_table, sin_table, static_cast<const void*>(q_out)})
    if (misaligned(p, 16)) return fail(IPE_ERR_ARGUMENT, "%s: operands must be 16-byte aligned", name);
  if (misaligned(cu_tokens, 4)) return fail(IPE_ERR_ARGUMENT, "%s: cu_tokens must be 4-byte aligned", name);
  c.cu_tokens = cu_tokens;
  return finish(ipe::launch_paged_append(c, qkv, tokens, q_heads, q_norm_weight, k_norm_weight, cos_table, sin_table,
                                         table_dtype == 1, table_rows, q_out, k_pages, v_pages, eps,
                                         static_cast<cudaStream_t>(stream)),
                name);
}

int ipe_paged_decode_attention(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                               const int32_t* lengths, void* out, int sequences, int q_heads, int kv_heads,
                               int64_t num_pages, int page_size, int max_pages, void* workspace,
                               size_t workspace_bytes, void* stream) {
  const char* name = "ipe_paged_decode_attention";
  ipe::PagedCache c;
  if (int status = paged_cache(name, k_pages, v_pages, page_table, lengths, sequences, sequences, q_heads, kv_heads,
                               num_pages, page_size, max_pages, &c))
    return status;
  if (sequences == 0) return IPE_OK;
  if (int status = rows_checks(name, q, out)) return status;
  const size_t need = ipe::paged_decode_workspace_bytes(sequences, q_heads, kv_heads);
  if (int status = workspace_checks(name, workspace, workspace_bytes, need)) return status;
  return finish(ipe::launch_paged_decode(c, q, k_pages, v_pages, out, q_heads, workspace,
                                         static_cast<cudaStream_t>(stream)),
                name);
}

int ipe_paged_prefill_attention(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                                const int32_t* cu_tokens, const int32_t* lengths, void* out, int64_t tokens,
                                int sequences, int q_heads, int kv_heads, int64_t num_pages, int page_size,
                                int max_pages, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "ipe_paged_prefill_attention";
  ipe::PagedCache c;
  if (int status = paged_cache(name, k_pages, v_pages, page_table, lengths, tokens, sequences, q_heads, kv_heads,
                               num_pages, page_size, max_pages, &c))
    return status;
  if (tokens == 0 || sequences == 0) return IPE_OK;
  if (int status = rows_checks(name, q, out)) return status;
  if (!cu_tokens || misaligned(cu_tokens, 4)) return fail(IPE_ERR_ARGUMENT, "%s: cu_tokens", name);
  c.cu_tokens = cu_tokens;
  const size_t need = ipe::paged_prefill_workspace_bytes(tokens, sequences, q_heads, kv_heads);
  if (int status = workspace_checks(name, workspace, workspace_bytes, need)) return status;
  return finish(ipe::launch_paged_prefill(c, q, k_pages, v_pages, out, tokens, q_heads, workspace,
                                          static_cast<cudaStream_t>(stream)),
                name);
}

int ipe_shared_prefix_attention(const void* q, const void* k_pages, const void* v_pages, const int32_t* prefix_pages,
                                int prefix_count, const int32_t* page_table, const int32_t* lengths, void* out,
                                int sequences, int q_heads, int kv_heads, int64_t num_pages, int page_size,
                                int max_pages, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "ipe_shared_prefix_attention";
  ipe::PagedCache c;
  if (int status = paged_cache(name, k_pages, v_pages, page_table, lengths, sequences, sequences, q_heads, kv_heads,
                               num_pages, page_size, max_pages, &c))
    return status;
  if (prefix_count < 0 || prefix_count > max_pages)
    return fail(IPE_ERR_ARGUMENT, "%s: %d prefix pages of at most %d per sequence", name, prefix_count, max_pages);
  if (sequences == 0) return IPE_OK;
  if (int status = rows_checks(name, q, out)) return status;
  if (prefix_count > 0 && (!prefix_pages || misaligned(prefix_pages, 4)))
    return fail(IPE_ERR_ARGUMENT, "%s: prefix_pages", name);
  c.prefix_pages = prefix_pages;
  c.prefix_count = prefix_count;
  if (ipe::shared_keys_plan(c, q_heads).units > INT32_MAX)
    return fail(IPE_ERR_UNSUPPORTED, "%s: %d prefix pages for %d sequences are past the kernels' 32-bit numbers", name,
                prefix_count, sequences);
  const size_t need = ipe::shared_prefix_workspace_bytes(c, q_heads);
  if (int status = workspace_checks(name, workspace, workspace_bytes, need)) return status;
  return finish(ipe::launch_shared_prefix(c, q, k_pages, v_pages, out, q_heads, workspace,
                                          static_cast<cudaStream_t>(stream)),
                name);
}

}  // extern "C"

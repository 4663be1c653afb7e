// extern "C" entry points of the 4-bit paged cache: argument validation and
// launch.  Nothing here allocates or synchronises.
#include <cstdio>

#include "common.cuh"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "params.cuh"

namespace mi {

int capi_fail(int code, const char *msg);
int capi_select_device(const void *p);
int capi_cuda_status(cudaError_t e);
int capi_varlen_prefill_lifted(void *out, const void *query, const void *keys, const void *values,
                               int64_t kv_token_stride, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                               int32_t dtype, const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k,
                               int64_t num_seqs, int64_t num_tokens, int64_t num_kv_tokens, int32_t max_seqlen_q,
                               float scale, float p_lift, int32_t *dev_status, void *stream);

cudaError_t launch_mxfp4_store(const MxStoreParams &p, int dtype, int index_dtype, bool vec,
                               cudaStream_t stream);
cudaError_t launch_mxfp4_gather(const MxGatherParams &p, int dtype, int64_t num_seqs, int64_t max_context,
                                cudaStream_t stream);
cudaError_t launch_mxfp4_decode(const MxDecodeParams &p, int dtype, cudaStream_t stream);
bool mxfp4_decode_supported(int num_q_heads, int num_kv_heads, int head_dim, int64_t num_blocks, int block_size,
                            int64_t capacity);
size_t mxfp4_decode_workspace(int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int64_t capacity,
                              int sms);

bool mxfp4_prefill_supported(int dtype, int head_dim);
int mxfp4_prefill_splits(int64_t num_seqs, int64_t max_seqlen_q, int num_q_heads, int num_kv_heads,
                         int64_t capacity, int sms);
cudaError_t launch_mxfp4_prefill(const MxPrefillParams &p, int dtype, int head_dim, int64_t num_seqs,
                                 int64_t max_seqlen_q, cudaStream_t stream);

}  // namespace mi

using namespace mi;

namespace {

constexpr float kLog2eHost = 1.4426950408889634f;

bool known_dtype(int32_t dtype) {
  return dtype == MI_DTYPE_FLOAT32 || dtype == MI_DTYPE_FLOAT16 || dtype == MI_DTYPE_BFLOAT16;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What every entry point asks of a 4-bit cache.
int check_cache(int64_t num_blocks, int32_t block_size, int32_t num_kv_heads, int32_t head_dim) {
  if (num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || head_dim <= 0)
    return capi_fail(MI_ERR_INVALID, "cache dimensions must be positive");
  if (block_size % kMxGroup != 0)
    return capi_fail(MI_ERR_UNSUPPORTED, "a 4-bit cache needs a block_size that is a multiple of 16");
  if (head_dim % kMxBlock != 0 || head_dim > 256)
    return capi_fail(MI_ERR_UNSUPPORTED, "a 4-bit cache needs a head_dim that is a multiple of 32, at most 256");
  return MI_OK;
}

}  // namespace

extern "C" {

int64_t mi_mxfp4_page_bytes(int32_t block_size, int32_t head_dim) {
  if (const int s = check_cache(1, block_size, 1, head_dim)) return s;
  return static_cast<int64_t>(block_size / kMxGroup) * mx_group_bytes(head_dim);
}

int mi_store_kv_mxfp4(void *key_pages, void *value_pages, int64_t num_blocks, int32_t block_size,
                      int32_t num_kv_heads, int32_t head_dim, const void *slots, int32_t index_dtype,
                      const void *keys, const void *values, int32_t dtype, int64_t key_token_stride,
                      int64_t value_token_stride, int64_t num_tokens, int32_t *dev_status, void *stream) {
  if (!known_dtype(dtype)) return capi_fail(MI_ERR_INVALID, "unknown dtype");
  if (index_dtype != MI_INDEX_INT32 && index_dtype != MI_INDEX_INT64)
    return capi_fail(MI_ERR_INVALID, "index dtype must be int32 or int64");
  if (const int s = check_cache(num_blocks, block_size, num_kv_heads, head_dim)) return s;
  if (num_tokens < 0) return capi_fail(MI_ERR_INVALID, "num_tokens must be >= 0");
  if (key_token_stride < 0 || value_token_stride < 0)
    return capi_fail(MI_ERR_INVALID, "token strides must be >= 0");
  if (num_tokens / 8 + 1 >= (int64_t{1} << 31) / num_kv_heads)
    return capi_fail(MI_ERR_UNSUPPORTED, "too many tokens for one call");
  if (num_tokens == 0) return MI_OK;
  if (!key_pages || !value_pages || !keys || !values || !slots) return capi_fail(MI_ERR_INVALID, "null pointer");
  if (!aligned16(key_pages) || !aligned16(value_pages))
    return capi_fail(MI_ERR_ALIGNMENT, "pages must be 16-byte aligned");
  if (const int s = capi_select_device(key_pages)) return s;
  const int e = dtype == MI_DTYPE_FLOAT32 ? 4 : 2;
  MxStoreParams p = {};
  p.key_pages = static_cast<uint8_t *>(key_pages);
  p.value_pages = static_cast<uint8_t *>(value_pages);
  p.slots = slots;
  p.keys = keys;
  p.values = values;
  p.key_stride = key_token_stride;
  p.value_stride = value_token_stride;
  p.num_slots = num_blocks * block_size;
  p.num_tokens = num_tokens;
  p.block_size = block_size;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.status = dev_status;
  const bool vec = aligned16(keys) && aligned16(values) && key_token_stride * e % 16 == 0 &&
                   value_token_stride * e % 16 == 0;
  return capi_cuda_status(launch_mxfp4_store(p, dtype, index_dtype, vec, static_cast<cudaStream_t>(stream)));
}

int mi_gather_paged_kv_mxfp4(void *out_keys, void *out_values, const void *key_pages, const void *value_pages,
                             int64_t num_blocks, int32_t block_size, int32_t num_kv_heads, int32_t head_dim,
                             int32_t dtype, const int32_t *block_tables, int64_t block_table_stride,
                             const int32_t *cu_seqlens_k, int64_t num_seqs, int64_t out_rows,
                             int64_t max_context, int32_t *dev_status, void *stream) {
  if (!known_dtype(dtype)) return capi_fail(MI_ERR_INVALID, "unknown dtype");
  if (const int s = check_cache(num_blocks, block_size, num_kv_heads, head_dim)) return s;
  if (num_seqs < 0 || max_context < 0 || block_table_stride < 0 || out_rows < 0)
    return capi_fail(MI_ERR_INVALID, "negative sizes");
  if (num_seqs > 65535) return capi_fail(MI_ERR_UNSUPPORTED, "more than 65535 sequences in one call");
  if (num_seqs == 0 || max_context == 0 || out_rows == 0) return MI_OK;
  if (max_context / kMxGroup + 1 >= (int64_t{1} << 31) / num_kv_heads)
    return capi_fail(MI_ERR_UNSUPPORTED, "max_context too large for one call");
  if (!out_keys || !out_values || !key_pages || !value_pages || !block_tables || !cu_seqlens_k)
    return capi_fail(MI_ERR_INVALID, "null pointer");
  if (!aligned16(key_pages) || !aligned16(value_pages) || !aligned16(out_keys) || !aligned16(out_values))
    return capi_fail(MI_ERR_ALIGNMENT, "pages and outputs must be 16-byte aligned");
  if (const int s = capi_select_device(key_pages)) return s;
  MxGatherParams p = {};
  p.out_keys = out_keys;
  p.out_values = out_values;
  p.key_pages = static_cast<const uint8_t *>(key_pages);
  p.value_pages = static_cast<const uint8_t *>(value_pages);
  p.block_tables = block_tables;
  p.cu_seqlens_k = cu_seqlens_k;
  p.block_table_stride = block_table_stride;
  p.num_blocks = num_blocks;
  p.out_rows = out_rows;
  p.block_size = block_size;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.status = dev_status;
  return capi_cuda_status(
      launch_mxfp4_gather(p, dtype, num_seqs, max_context, static_cast<cudaStream_t>(stream)));
}

size_t mi_paged_decode_mxfp4_workspace_bytes(int64_t num_seqs, int64_t num_blocks, int32_t block_size,
                                             int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                             int32_t dtype, int64_t block_table_stride, int device) {
  if (num_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || block_table_stride <= 0 ||
      num_q_heads % num_kv_heads != 0 || check_cache(num_blocks, block_size, num_kv_heads, head_dim) != MI_OK)
    return 0;
  return mxfp4_decode_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, block_table_stride * block_size,
                                sm_count_of(device < 0 ? 0 : device));
}

int mi_paged_decode_mxfp4(void *out, const void *query, const void *key_pages, const void *value_pages,
                          int64_t num_blocks, int32_t block_size, int32_t num_q_heads, int32_t num_kv_heads,
                          int32_t head_dim, int32_t dtype, const int32_t *block_tables,
                          int64_t block_table_stride, const int32_t *context_lens, int64_t num_seqs,
                          float scale, void *workspace, size_t workspace_bytes, int32_t *dev_status,
                          void *stream) {
  if (!known_dtype(dtype)) return capi_fail(MI_ERR_INVALID, "unknown dtype");
  if (const int s = check_cache(num_blocks, block_size, num_kv_heads, head_dim)) return s;
  if (num_seqs < 0) return capi_fail(MI_ERR_INVALID, "num_seqs must be >= 0");
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0)
    return capi_fail(MI_ERR_INVALID, "num_q_heads must be divisible by num_kv_heads");
  if (block_table_stride < 0 || block_table_stride > INT32_MAX)
    return capi_fail(MI_ERR_INVALID, "block_table_stride out of range");
  if (num_seqs > 65535) return capi_fail(MI_ERR_UNSUPPORTED, "more than 65535 sequences in one call");
  if (num_q_heads > 65535) return capi_fail(MI_ERR_UNSUPPORTED, "more than 65535 query heads");
  if (!mxfp4_decode_supported(num_q_heads, num_kv_heads, head_dim, num_blocks, block_size,
                              block_table_stride * block_size))
    return capi_fail(MI_ERR_UNSUPPORTED, "pages or block table too large for one call");
  if (num_seqs == 0) return MI_OK;
  if (!out || !query || !key_pages || !value_pages || !block_tables || !context_lens)
    return capi_fail(MI_ERR_INVALID, "null pointer");
  if (!aligned16(key_pages) || !aligned16(value_pages) || !aligned16(query) || !aligned16(out))
    return capi_fail(MI_ERR_ALIGNMENT, "pages, query and out must be 16-byte aligned");
  if (const int s = capi_select_device(key_pages)) return s;
  const size_t need = mxfp4_decode_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim,
                                             block_table_stride * block_size, sm_count_current());
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return capi_fail(MI_ERR_INVALID, "workspace too small (see mi_paged_decode_mxfp4_workspace_bytes)");
  if (need > 0 && !aligned16(workspace)) return capi_fail(MI_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  MxDecodeParams p = {};
  p.out = out;
  p.query = query;
  p.key_pages = static_cast<const uint8_t *>(key_pages);
  p.value_pages = static_cast<const uint8_t *>(value_pages);
  p.block_tables = block_tables;
  p.context_lens = context_lens;
  p.workspace = need > 0 ? static_cast<float *>(workspace) : nullptr;  // unasked for: of any size, not written
  p.bt_stride = block_table_stride;
  p.num_blocks = num_blocks;
  p.num_seqs = num_seqs;
  p.block_size = block_size;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.scale_log2 = scale * kLog2eHost;
  p.status = dev_status;
  return capi_cuda_status(launch_mxfp4_decode(p, dtype, static_cast<cudaStream_t>(stream)));
}

static int prefill_splits(int64_t num_seqs, int64_t max_seqlen_q, int32_t num_q_heads, int32_t num_kv_heads,
                          int64_t max_context, int sms) {
  return mxfp4_prefill_splits(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads, max_context, sms);
}

static size_t prefill_workspace(int splits, int64_t num_tokens, int32_t num_q_heads, int32_t head_dim) {
  return splits <= 1 ? 0
                     : static_cast<size_t>(splits) * num_tokens * num_q_heads * (head_dim + 2) * sizeof(float);
}

size_t mi_paged_prefill_mxfp4_workspace_bytes(int64_t num_seqs, int64_t num_tokens, int64_t max_seqlen_q,
                                              int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                              int64_t max_context, int device) {
  if (num_seqs <= 0 || num_tokens <= 0 || max_seqlen_q <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      num_q_heads % num_kv_heads != 0 || head_dim <= 0 || max_context < 0)
    return 0;
  const int splits = prefill_splits(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads, max_context,
                                    sm_count_of(device < 0 ? 0 : device));
  return prefill_workspace(splits, num_tokens, num_q_heads, head_dim);
}

int mi_paged_prefill_mxfp4(void *out, const void *query, const void *key_pages, const void *value_pages,
                           int64_t num_blocks, int32_t block_size, int32_t num_q_heads, int32_t num_kv_heads,
                           int32_t head_dim, int32_t dtype, const int32_t *cu_seqlens_q,
                           const int32_t *cu_seqlens_k, const int32_t *block_tables, int64_t block_table_stride,
                           int64_t num_seqs, int64_t num_tokens, int64_t max_seqlen_q, int64_t max_context,
                           float scale, void *workspace, size_t workspace_bytes, int32_t *dev_status,
                           void *stream) {
  if (!known_dtype(dtype)) return capi_fail(MI_ERR_INVALID, "unknown dtype");
  if (const int s = check_cache(num_blocks, block_size, num_kv_heads, head_dim)) return s;
  if (num_seqs < 0 || num_tokens < 0 || max_context < 0 || block_table_stride < 0)
    return capi_fail(MI_ERR_INVALID, "negative sizes");
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0)
    return capi_fail(MI_ERR_INVALID, "num_q_heads must be divisible by num_kv_heads");
  if (!mxfp4_prefill_supported(dtype, head_dim))
    return capi_fail(MI_ERR_UNSUPPORTED, "prefill from the 4-bit cache takes fp32 up to head_dim 128; gather above");
  if (num_seqs > 65535 || num_kv_heads > 65535) return capi_fail(MI_ERR_UNSUPPORTED, "more than 65535 sequences or heads");
  if (num_seqs == 0 || num_tokens == 0) return MI_OK;
  if (max_seqlen_q <= 0) return capi_fail(MI_ERR_INVALID, "max_seqlen_q must be positive");
  // positions are 32 bits, and pages are looked up as many as three tiles of keys past the last
  if (max_seqlen_q > (int64_t{1} << 24) || max_seqlen_q * (num_q_heads / num_kv_heads) >= (int64_t{1} << 31) ||
      block_table_stride > (INT32_MAX - 256) / block_size)
    return capi_fail(MI_ERR_UNSUPPORTED, "sequence too long for one call");
  if (!out || !query || !key_pages || !value_pages || !cu_seqlens_q || !cu_seqlens_k || !block_tables)
    return capi_fail(MI_ERR_INVALID, "null pointer");
  if (!aligned16(key_pages) || !aligned16(value_pages) || !aligned16(query) || !aligned16(out))
    return capi_fail(MI_ERR_ALIGNMENT, "pages, query and out must be 16-byte aligned");
  if (const int s = capi_select_device(key_pages)) return s;
  const int splits = prefill_splits(num_seqs, max_seqlen_q, num_q_heads, num_kv_heads, max_context,
                                    sm_count_current());
  const size_t need = prefill_workspace(splits, num_tokens, num_q_heads, head_dim);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return capi_fail(MI_ERR_INVALID, "workspace too small (see mi_paged_prefill_mxfp4_workspace_bytes)");
  if (need > 0 && !aligned16(workspace)) return capi_fail(MI_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  MxPrefillParams p = {};
  p.out = out;
  p.query = query;
  p.key_pages = static_cast<const uint8_t *>(key_pages);
  p.value_pages = static_cast<const uint8_t *>(value_pages);
  p.block_tables = block_tables;
  p.cu_seqlens_q = cu_seqlens_q;
  p.cu_seqlens_k = cu_seqlens_k;
  p.workspace = need > 0 ? static_cast<float *>(workspace) : nullptr;
  p.bt_stride = block_table_stride;
  p.num_blocks = num_blocks;
  p.num_tokens = num_tokens;
  p.num_splits = splits;
  p.block_size = block_size;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads;
  p.scale_log2 = scale * kLog2eHost;
  p.status = dev_status;
  return capi_cuda_status(
      launch_mxfp4_prefill(p, dtype, head_dim, num_seqs, max_seqlen_q, static_cast<cudaStream_t>(stream)));
}

// K and V of kv_rows rows, each from a multiple of 256 bytes, then a byte per (sequence, kv head, group).
static size_t gathered_rows_bytes(int64_t kv_rows, int32_t num_kv_heads, int32_t head_dim, int32_t dtype) {
  const size_t bytes = static_cast<size_t>(kv_rows) * num_kv_heads * head_dim * (dtype == MI_DTYPE_FLOAT32 ? 4 : 2);
  return (bytes + 255) / 256 * 256;
}

size_t mi_paged_prefill_mxfp4_gathered_workspace_bytes(int64_t num_seqs, int64_t max_context, int64_t kv_rows,
                                                       int32_t num_kv_heads, int32_t head_dim, int32_t dtype) {
  if (num_seqs <= 0 || max_context <= 0 || kv_rows <= 0 || num_kv_heads <= 0 || head_dim <= 0 || !known_dtype(dtype))
    return 0;
  return 2 * gathered_rows_bytes(kv_rows, num_kv_heads, head_dim, dtype) +
         static_cast<size_t>(num_seqs) * num_kv_heads * ((max_context + kMxGroup - 1) / kMxGroup);
}

int mi_paged_prefill_mxfp4_gathered(void *out, const void *query, const void *key_pages, const void *value_pages,
                                    int64_t num_blocks, int32_t block_size, int32_t num_q_heads,
                                    int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                                    const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k,
                                    const int32_t *block_tables, int64_t block_table_stride, int64_t num_seqs,
                                    int64_t num_tokens, int32_t max_seqlen_q, int64_t max_context, int64_t kv_rows,
                                    float scale, void *workspace, size_t workspace_bytes, int32_t *dev_status,
                                    void *stream) {
  if (!known_dtype(dtype)) return capi_fail(MI_ERR_INVALID, "unknown dtype");
  if (const int s = check_cache(num_blocks, block_size, num_kv_heads, head_dim)) return s;
  if (num_seqs < 0 || num_tokens < 0 || max_context < 0 || kv_rows < 0 || block_table_stride < 0)
    return capi_fail(MI_ERR_INVALID, "negative sizes");
  if (num_q_heads <= 0 || num_q_heads % num_kv_heads != 0)
    return capi_fail(MI_ERR_INVALID, "num_q_heads must be divisible by num_kv_heads");
  if (num_seqs > 65535 || num_kv_heads > 65535) return capi_fail(MI_ERR_UNSUPPORTED, "more than 65535 sequences or heads");
  if (num_seqs == 0 || num_tokens == 0) return MI_OK;
  if (max_seqlen_q <= 0 || kv_rows == 0 || max_context == 0)
    return capi_fail(MI_ERR_INVALID, "max_seqlen_q, kv_rows and max_context must be positive");
  if (max_context / kMxGroup + 1 >= (int64_t{1} << 31) / num_kv_heads)
    return capi_fail(MI_ERR_UNSUPPORTED, "max_context too large for one call");
  if (!out || !query || !key_pages || !value_pages || !cu_seqlens_q || !cu_seqlens_k || !block_tables)
    return capi_fail(MI_ERR_INVALID, "null pointer");
  if (!aligned16(key_pages) || !aligned16(value_pages) || !aligned16(query) || !aligned16(out))
    return capi_fail(MI_ERR_ALIGNMENT, "pages, query and out must be 16-byte aligned");
  const size_t rows = gathered_rows_bytes(kv_rows, num_kv_heads, head_dim, dtype);
  if (workspace == nullptr ||
      workspace_bytes < mi_paged_prefill_mxfp4_gathered_workspace_bytes(num_seqs, max_context, kv_rows, num_kv_heads,
                                                                        head_dim, dtype))
    return capi_fail(MI_ERR_INVALID, "workspace too small (see mi_paged_prefill_mxfp4_gathered_workspace_bytes)");
  if (!aligned16(workspace)) return capi_fail(MI_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  if (const int s = capi_select_device(key_pages)) return s;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char *keys = static_cast<char *>(workspace), *values = keys + rows;
  // The tensor-core kernel multiplies what a row does not see by zero: sequences with blocks that this does not suit are
  // noted by the gather and done over from the pages (their tables have to be within that kernel's limit).
  const bool dense = mi_prefill_kernel_for(dtype, head_dim, num_q_heads, num_kv_heads, 0) == 2;
  const int64_t groups = (max_context + kMxGroup - 1) / kMxGroup;
  uint8_t *redo = nullptr;
  if (dense && max_seqlen_q <= (1 << 24) && block_table_stride <= (INT32_MAX - 256) / block_size)
    redo = reinterpret_cast<uint8_t *>(values + rows);
  MxGatherParams g = {};
  g.out_keys = keys;
  g.out_values = values;
  g.key_pages = static_cast<const uint8_t *>(key_pages);
  g.value_pages = static_cast<const uint8_t *>(value_pages);
  g.block_tables = block_tables;
  g.cu_seqlens_k = cu_seqlens_k;
  g.block_table_stride = block_table_stride;
  g.num_blocks = num_blocks;
  g.out_rows = kv_rows;
  g.redo = redo;
  g.redo_stride = groups;
  g.fill = static_cast<uint32_t>(groups);
  g.block_size = block_size;
  g.num_kv_heads = num_kv_heads;
  g.head_dim = head_dim;
  g.status = dev_status;
  if (const int s = capi_cuda_status(launch_mxfp4_gather(g, dtype, num_seqs, max_context, st))) return s;
  const float p_lift = dtype == MI_DTYPE_FLOAT16 ? 7.f : 0.f;  // small p keep their bits, as in the kernels on the pages
  if (const int s = capi_varlen_prefill_lifted(
          out, query, keys, values, static_cast<int64_t>(num_kv_heads) * head_dim, num_q_heads, num_kv_heads, head_dim, dtype,
          cu_seqlens_q, cu_seqlens_k, num_seqs, num_tokens, kv_rows, max_seqlen_q, scale, p_lift, dev_status, stream))
    return s;
  if (redo == nullptr) return MI_OK;
  MxPrefillParams p = {};
  p.out = out;
  p.query = query;
  p.key_pages = g.key_pages;
  p.value_pages = g.value_pages;
  p.block_tables = block_tables;
  p.cu_seqlens_q = cu_seqlens_q;
  p.cu_seqlens_k = cu_seqlens_k;
  p.redo = redo;
  p.redo_stride = groups;
  p.redo_groups = static_cast<int32_t>(groups);
  p.bt_stride = block_table_stride;
  p.num_blocks = num_blocks;
  p.num_tokens = num_tokens;
  p.num_splits = 1;
  p.block_size = block_size;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads;
  p.scale_log2 = scale * kLog2eHost;
  p.status = dev_status;
  return capi_cuda_status(launch_mxfp4_prefill(p, dtype, head_dim, num_seqs, max_seqlen_q, st));
}

}  // extern "C"

// C ABI of the decoding operators (declared in include/piper_b200.h): the
// quantised paged KV cache, attention of a drafted tree over it, and the
// tree's verification.  Argument checks and launches on the caller's stream,
// with no host synchronisation.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "host_api.h"
#include "kv_cache.cuh"
#include "piper_b200.h"
#include "tree_attention.cuh"
#include "verify_tree.cuh"

namespace {

using piper::host::fail;

int invalid(const std::string& msg) { return fail(PIPER_B200_ERR_INVALID_ARGUMENT, msg); }

int page_shift_of(int page_size) {
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  return shift;
}

int check_cache(const piper_b200_kv_cache_t* c) {
  if (c == nullptr || !c->key_codes || !c->key_scales || !c->value_codes || !c->value_scales || !c->block_table ||
      !c->lengths)
    return invalid("NULL pointer argument");
  if (c->head_dim != 64 && c->head_dim != 128)
    return invalid("head_dim must be 64 or 128, got " + std::to_string(c->head_dim));
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0)
    return invalid("page_size must be a power of two from 16 to 256, got " + std::to_string(c->page_size));
  if (c->pages <= 0 || c->kv_heads <= 0 || c->batch <= 0 || c->table_width <= 0)
    return invalid("pages, kv_heads, batch and table_width must be positive");
  if (c->kv_heads > 65535 || c->batch > 65535) return invalid("kv_heads and batch must be at most 65535");
  if (c->pages > 0x7fffffff / c->kv_heads) return invalid("pages * kv_heads must be below 2^31");
  if (c->table_stride < 0) return invalid("table_stride must not be negative");
  if (reinterpret_cast<uintptr_t>(c->key_codes) % 16 != 0 || reinterpret_cast<uintptr_t>(c->value_codes) % 16 != 0)
    return invalid("the cache's codes must be 16-byte aligned");
  return PIPER_B200_OK;
}

int check_dtype(int dtype) {
  if (dtype != PIPER_B200_FLOAT16 && dtype != PIPER_B200_BFLOAT16)
    return invalid("dtype must be PIPER_B200_FLOAT16 or PIPER_B200_BFLOAT16");
  return PIPER_B200_OK;
}

int use_device(int* sms = nullptr, unsigned long long* context = nullptr, int* device = nullptr) {
  int d = 0, s = 0;
  unsigned long long x = 0;
  const int rc = piper::host::ensure_device(&d, &x, &s);
  if (sms) *sms = s;
  if (context) *context = x;
  if (device) *device = d;
  return rc;
}

bool rows_aligned16(const void* p, const int64_t s[3]) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
}

// CTAs for `rows` rows of D/8 lanes each.
int row_blocks(int64_t rows, int d, unsigned* blocks) {
  const int64_t per = piper::kCacheThreads / (d / 8);
  const int64_t n = (rows + per - 1) / per;
  if (n > 0x7fffffff) return invalid("too many rows for one call");
  *blocks = static_cast<unsigned>(n);
  return PIPER_B200_OK;
}

template <typename T>
void launch_write(const piper::CacheRowsArgs& a, bool v16, const dim3& grid, cudaStream_t s) {
  if (a.c.head_dim == 64) {
    if (v16)
      piper::cache_write_kernel<T, 64, true><<<grid, piper::kCacheThreads, 0, s>>>(a);
    else
      piper::cache_write_kernel<T, 64, false><<<grid, piper::kCacheThreads, 0, s>>>(a);
  } else {
    if (v16)
      piper::cache_write_kernel<T, 128, true><<<grid, piper::kCacheThreads, 0, s>>>(a);
    else
      piper::cache_write_kernel<T, 128, false><<<grid, piper::kCacheThreads, 0, s>>>(a);
  }
}

template <typename T>
void launch_read(const piper::CacheRowsArgs& a, const dim3& grid, cudaStream_t s) {
  if (a.c.head_dim == 64)
    piper::cache_read_kernel<T, 64><<<grid, piper::kCacheThreads, 0, s>>>(a);
  else
    piper::cache_read_kernel<T, 128><<<grid, piper::kCacheThreads, 0, s>>>(a);
}

template <typename T>
void launch_tree(const piper::TreeArgs& a, cudaStream_t s) {
  const dim3 grid(a.nodes, a.heads, a.c.batch);
  if (a.c.head_dim == 64)
    piper::tree_attention_simple_kernel<T, 64><<<grid, 128, 0, s>>>(a);
  else
    piper::tree_attention_simple_kernel<T, 128><<<grid, 128, 0, s>>>(a);
}

}  // namespace

extern "C" int piper_b200_kv_cache_write(const piper_b200_kv_cache_t* cache, const void* key,
                                         const int64_t key_strides[3], const void* value,
                                         const int64_t value_strides[3], int dtype, int64_t tokens,
                                         const int32_t* counts, void* stream) {
  int rc = check_cache(cache);
  if (rc != PIPER_B200_OK) return rc;
  if ((rc = check_dtype(dtype)) != PIPER_B200_OK) return rc;
  if (!key || !value || !key_strides || !value_strides) return invalid("NULL pointer argument");
  if (tokens <= 0 || tokens > (int64_t(1) << 30)) return invalid("tokens must be in [1, 2^30]");
  piper::CacheRowsArgs a{};
  a.c = *cache;
  a.in[0] = key;
  a.in[1] = value;
  for (int i = 0; i < 3; ++i) {
    a.stride[0][i] = key_strides[i];
    a.stride[1][i] = value_strides[i];
  }
  a.counts = counts;
  a.tokens = tokens;
  a.page_shift = page_shift_of(cache->page_size);
  unsigned blocks = 0;
  if ((rc = row_blocks(tokens * cache->kv_heads, cache->head_dim, &blocks)) != PIPER_B200_OK) return rc;
  if ((rc = use_device()) != PIPER_B200_OK) return rc;
  const dim3 grid(blocks, static_cast<unsigned>(cache->batch));
  const bool v16 = rows_aligned16(key, key_strides) && rows_aligned16(value, value_strides);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PIPER_B200_FLOAT16)
    launch_write<__half>(a, v16, grid, s);
  else
    launch_write<__nv_bfloat16>(a, v16, grid, s);
  PIPER_HOST_CUDA(cudaGetLastError());
  return PIPER_B200_OK;
}

extern "C" int piper_b200_kv_cache_read(const piper_b200_kv_cache_t* cache, void* key_out, void* value_out, int dtype,
                                        int64_t tokens, const int32_t* counts, void* stream) {
  int rc = check_cache(cache);
  if (rc != PIPER_B200_OK) return rc;
  if ((rc = check_dtype(dtype)) != PIPER_B200_OK) return rc;
  if (!key_out || !value_out) return invalid("NULL pointer argument");
  if (reinterpret_cast<uintptr_t>(key_out) % 16 != 0 || reinterpret_cast<uintptr_t>(value_out) % 16 != 0)
    return invalid("outputs must be 16-byte aligned");
  if (tokens <= 0 || tokens > (int64_t(1) << 30)) return invalid("tokens must be in [1, 2^30]");
  piper::CacheRowsArgs a{};
  a.c = *cache;
  a.out[0] = key_out;
  a.out[1] = value_out;
  a.counts = counts;
  a.tokens = tokens;
  a.page_shift = page_shift_of(cache->page_size);
  unsigned blocks = 0;
  if ((rc = row_blocks(tokens * cache->kv_heads, cache->head_dim, &blocks)) != PIPER_B200_OK) return rc;
  if ((rc = use_device()) != PIPER_B200_OK) return rc;
  const dim3 grid(blocks, static_cast<unsigned>(cache->batch));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PIPER_B200_FLOAT16)
    launch_read<__half>(a, grid, s);
  else
    launch_read<__nv_bfloat16>(a, grid, s);
  PIPER_HOST_CUDA(cudaGetLastError());
  return PIPER_B200_OK;
}

extern "C" int piper_b200_kv_cache_keep(const piper_b200_kv_cache_t* cache, const int32_t* path, int64_t path_stride,
                                        int64_t nodes, const int32_t* counts, void* stream) {
  int rc = check_cache(cache);
  if (rc != PIPER_B200_OK) return rc;
  if (!path || !counts) return invalid("NULL pointer argument");
  if (nodes <= 0 || nodes > piper::kMaxNodes) return invalid("nodes must be in [1, 64], got " + std::to_string(nodes));
  if ((rc = use_device()) != PIPER_B200_OK) return rc;
  const dim3 grid(static_cast<unsigned>(cache->kv_heads), static_cast<unsigned>(cache->batch), 2);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int shift = page_shift_of(cache->page_size);
  if (cache->head_dim == 64)
    piper::cache_keep_kernel<64><<<grid, piper::kCacheThreads, 0, s>>>(*cache, path, path_stride,
                                                                       static_cast<int>(nodes), counts, shift);
  else
    piper::cache_keep_kernel<128><<<grid, piper::kCacheThreads, 0, s>>>(*cache, path, path_stride,
                                                                        static_cast<int>(nodes), counts, shift);
  PIPER_HOST_CUDA(cudaGetLastError());
  return PIPER_B200_OK;
}

extern "C" int piper_b200_tree_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t nodes,
                                                         int64_t head_dim, size_t* bytes) {
  if (bytes == nullptr) return invalid("bytes is NULL");
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || nodes <= 0 || head_dim <= 0)
    return invalid("sizes must be positive");
  *bytes = 0;
  return PIPER_B200_OK;
}

extern "C" int piper_b200_tree_attention(const piper_b200_kv_cache_t* cache, const void* query,
                                         const int64_t query_strides[3], void* out, int dtype, int64_t heads,
                                         int64_t nodes, const int64_t* tree_mask, int64_t mask_stride, double scale,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_cache(cache);
  if (rc != PIPER_B200_OK) return rc;
  if ((rc = check_dtype(dtype)) != PIPER_B200_OK) return rc;
  if (!query || !query_strides || !out) return invalid("NULL pointer argument");
  if (nodes <= 0 || nodes > piper::kMaxNodes) return invalid("nodes must be in [1, 64], got " + std::to_string(nodes));
  if (heads <= 0 || heads > 65535 || heads % cache->kv_heads != 0)
    return invalid("heads must be a multiple of kv_heads, at most 65535");
  if (!(std::isfinite(scale) && scale > 0.0)) return invalid("scale must be finite and positive");
  if (reinterpret_cast<uintptr_t>(out) % 16 != 0) return invalid("output must be 16-byte aligned");
  (void)workspace;
  (void)workspace_bytes;
  if ((rc = use_device()) != PIPER_B200_OK) return rc;
  piper::TreeArgs a{};
  a.c = *cache;
  a.query = query;
  for (int i = 0; i < 3; ++i) a.qs[i] = query_strides[i];
  a.out = out;
  a.mask = tree_mask;
  a.mask_stride = mask_stride;
  a.heads = static_cast<int>(heads);
  a.nodes = static_cast<int>(nodes);
  a.group = static_cast<int>(heads / cache->kv_heads);
  a.page_shift = page_shift_of(cache->page_size);
  a.scale_log2e = static_cast<float>(scale * 1.4426950408889634);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PIPER_B200_FLOAT16)
    launch_tree<__half>(a, s);
  else
    launch_tree<__nv_bfloat16>(a, s);
  PIPER_HOST_CUDA(cudaGetLastError());
  return PIPER_B200_OK;
}

extern "C" int piper_b200_verify_draft_tree(const float* target, const int64_t target_strides[2], const float* draft,
                                            const int64_t draft_strides[2], const int64_t* tokens,
                                            int64_t tokens_stride, const int32_t* parents, int64_t parents_stride,
                                            const float* uniform, int64_t uniform_stride, const float* noise,
                                            int64_t noise_stride, int64_t batch, int64_t nodes, int64_t vocab,
                                            int32_t* path, int32_t* count, int64_t* next_token, void* stream) {
  if (!target || !target_strides || !draft || !draft_strides || !tokens || !parents || !uniform || !noise || !path ||
      !count || !next_token)
    return invalid("NULL pointer argument");
  if (batch <= 0 || batch > 65535) return invalid("batch must be in [1, 65535]");
  if (nodes <= 0 || nodes > piper::kMaxNodes) return invalid("nodes must be in [1, 64], got " + std::to_string(nodes));
  if (vocab <= 0 || vocab > (int64_t(1) << 30)) return invalid("vocab must be in [1, 2^30]");
  int rc = use_device();
  if (rc != PIPER_B200_OK) return rc;
  piper::VerifyArgs a{};
  a.target = target;
  a.draft = draft;
  for (int i = 0; i < 2; ++i) {
    a.ts[i] = target_strides[i];
    a.ds[i] = draft_strides[i];
  }
  a.tokens = tokens;
  a.parents = parents;
  a.uniform = uniform;
  a.noise = noise;
  a.tokens_stride = tokens_stride;
  a.parents_stride = parents_stride;
  a.uniform_stride = uniform_stride;
  a.noise_stride = noise_stride;
  a.nodes = static_cast<int>(nodes);
  a.vocab = vocab;
  a.path = path;
  a.count = count;
  a.next = next_token;
  piper::verify_simple_kernel<<<static_cast<unsigned>(batch), piper::kVerifyThreads, 0,
                                static_cast<cudaStream_t>(stream)>>>(a);
  PIPER_HOST_CUDA(cudaGetLastError());
  return PIPER_B200_OK;
}

// C ABI of the decoding operators (declared in include/piper_b200.h): the
// quantised paged KV cache, attention of a drafted tree over it, and the
// tree's verification.  Argument checks and launches on the caller's stream,
// with no host synchronisation.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "host_api.h"
#include "kv_cache.cuh"
#include "piper_b200.h"
#include "tree_attention.cuh"
#include "tree_wide.cuh"
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
  if (reinterpret_cast<uintptr_t>(c->key_mean) % 16 != 0) return invalid("key_mean must be 16-byte aligned");
  return PIPER_B200_OK;
}

// The sizes of an attention call that do not come from the cache.
int check_rows(int64_t heads, int64_t kv_heads, int64_t nodes) {
  if (nodes <= 0 || nodes > piper::kMaxNodes) return invalid("nodes must be in [1, 64], got " + std::to_string(nodes));
  if (heads <= 0 || heads > 65535 || heads % kv_heads != 0)
    return invalid("heads must be a multiple of kv_heads, at most 65535");
  return PIPER_B200_OK;
}

int check_dtype(int dtype) {
  if (dtype != PIPER_B200_FLOAT16 && dtype != PIPER_B200_BFLOAT16)
    return invalid("dtype must be PIPER_B200_FLOAT16 or PIPER_B200_BFLOAT16");
  return PIPER_B200_OK;
}

int use_device() {
  piper::host::Device device;
  return piper::host::ensure_device(&device);
}

bool rows_aligned16(const void* p, const int64_t s[3]) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
}

// CTAs for `rows` rows of D/16 lanes each.
int row_blocks(int64_t rows, int d, unsigned* blocks) {
  const int64_t per = piper::kCacheThreads / (d / 16);
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

constexpr int kMaxDevices = 64;
std::mutex g_tree_mutex;
unsigned long long g_tree_context[kMaxDevices] = {};  // context whose kernels have their shared memory

// How one call is spread over the GPU.
struct TreePlan {
  int64_t grid = 0;
  size_t bytes = 0;  // of the workspace
  int row_tiles = 0;
  bool whole = false;
};

template <typename S>
TreePlan tree_plan(int64_t batch, int64_t kv_heads, int64_t rows, int64_t positions, int sms) {
  TreePlan p;
  p.row_tiles = static_cast<int>((rows + S::kRows - 1) / S::kRows);
  const int64_t segments = batch * kv_heads * p.row_tiles;
  const int64_t most = (positions + S::kKeys - 1) / S::kKeys;
  // Tables of a few tiles: a CTA for each (request, head, row tile), one launch and
  // nothing to merge.  Whole against shared segments, 32 over 8 heads of 128: one
  // request of 256 tokens 7.4 and 12.2 us, of 1000 11.5 and 12.8, of 2000 (16 tiles)
  // 18.6 and 13.3; 64 requests of 100 to 1000 26.8 and 28.5, of 100 to 2000 39.5 and
  // 37.5.
  p.whole = most <= 8 && segments < (int64_t(1) << 31);
  if (p.whole) {
    p.grid = segments;
    return p;
  }
  const int64_t slots = static_cast<int64_t>(sms) * S::kCtas;
  // No more CTAs than the segments have pairs of tiles: it takes as long as a full
  // grid, whose other CTAs find nothing to do, for less workspace.
  p.grid = most > 2 * slots / segments ? slots : std::max<int64_t>(1, segments * most / 2);
  p.bytes = static_cast<size_t>(p.grid) * 2 * S::kPart * 4;
  return p;
}

// The kernel for a number of query rows of a KV head: up to kMoreRows an mma
// tile of 8, 16 or that many rows on four warps, up to 128 a tcgen05 tile whose
// streams take alternate keys, more a pair of them over the same keys.  Both
// sides of the limits, 32 requests of 1000 to 8191 tokens, 8 KV heads of 128 (of
// 64): 8 and 16 rows 58 and 69 us (38 and 47); 24 rows on the mma tile 110, on the
// tcgen05 tile 161 (32 rows 93 and 143), which is as long for 32 rows (162; 64:
// 170).  One request of 131072 tokens: 128 rows 138 us, 132 on the pair 196.
enum class TreeKind { kEight, kSixteen, kMore, kAlternate, kPair };
template <int D>
constexpr int kMoreRows = D == 64 ? 32 : 24;
template <int D>
TreeKind tree_kind(int64_t rows) {
  if (rows <= kMoreRows<D>) return rows <= 8 ? TreeKind::kEight : rows <= 16 ? TreeKind::kSixteen : TreeKind::kMore;
  return rows <= 128 ? TreeKind::kAlternate : TreeKind::kPair;
}
constexpr int kFewGroups = 2;
template <int D, int ROWS>
using FewRows = piper::TreeTile<D, 4, kFewGroups, ROWS>;

template <int D>
TreePlan tree_plan(int64_t batch, int64_t kv_heads, int64_t rows, int64_t positions, int sms) {
  switch (tree_kind<D>(rows)) {
    case TreeKind::kEight: return tree_plan<FewRows<D, 8>>(batch, kv_heads, rows, positions, sms);
    case TreeKind::kSixteen: return tree_plan<FewRows<D, 16>>(batch, kv_heads, rows, positions, sms);
    case TreeKind::kMore: return tree_plan<FewRows<D, kMoreRows<D>>>(batch, kv_heads, rows, positions, sms);
    case TreeKind::kAlternate: return tree_plan<piper::WideTile<D, false>>(batch, kv_heads, rows, positions, sms);
    default: return tree_plan<piper::WideTile<D, true>>(batch, kv_heads, rows, positions, sms);
  }
}

int allow_smem(const void* kernel, int bytes) {
  PIPER_HOST_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return PIPER_B200_OK;
}

template <typename T, int D, int ROWS>
int set_up_few() {
  const void* kernel = reinterpret_cast<const void*>(piper::tree_attention_kernel<T, D, 4, kFewGroups, ROWS>);
  return allow_smem(kernel, FewRows<D, ROWS>::kAlloc);
}

template <typename T, int D, bool kShared>
int set_up_wide() {
  const void* kernel = reinterpret_cast<const void*>(piper::tree_wide_kernel<T, D, kShared>);
  return allow_smem(kernel, piper::WideTile<D, kShared>::kAlloc);
}

template <typename T, int D>
int set_up_instances() {
  int rc = set_up_few<T, D, 8>();
  if (rc != PIPER_B200_OK) return rc;
  if ((rc = set_up_few<T, D, 16>()) != PIPER_B200_OK) return rc;
  if ((rc = set_up_few<T, D, kMoreRows<D>>()) != PIPER_B200_OK) return rc;
  if ((rc = set_up_wide<T, D, false>()) != PIPER_B200_OK) return rc;
  return set_up_wide<T, D, true>();
}

int set_up_tree(const piper::host::Device& device) {
  std::lock_guard<std::mutex> lock(g_tree_mutex);
  if (device.context != 0 && g_tree_context[device.index] == device.context) return PIPER_B200_OK;
  int rc = PIPER_B200_OK;
  if ((rc = set_up_instances<__half, 64>()) != PIPER_B200_OK) return rc;
  if ((rc = set_up_instances<__half, 128>()) != PIPER_B200_OK) return rc;
  if ((rc = set_up_instances<__nv_bfloat16, 64>()) != PIPER_B200_OK) return rc;
  if ((rc = set_up_instances<__nv_bfloat16, 128>()) != PIPER_B200_OK) return rc;
  g_tree_context[device.index] = device.context;
  return PIPER_B200_OK;
}

template <typename T, int D, typename S, typename Kernel>
int launch_tree(piper::TreeArgs a, Kernel kernel, int threads, int sms, size_t workspace_bytes, cudaStream_t stream) {
  const TreePlan plan =
      tree_plan<S>(a.c.batch, a.c.kv_heads, a.rows, static_cast<int64_t>(a.c.table_width) << a.page_shift, sms);
  a.row_tiles = plan.row_tiles;
  a.whole = plan.whole;
  if (workspace_bytes < plan.bytes)
    return fail(PIPER_B200_ERR_WORKSPACE_TOO_SMALL, "workspace needs " + std::to_string(plan.bytes) + " bytes, got " +
                                                        std::to_string(workspace_bytes));
  if (plan.bytes > 0 && (a.parts == nullptr || reinterpret_cast<uintptr_t>(a.parts) % 256 != 0))
    return invalid("workspace must be 256-byte aligned and not NULL");
  const uint32_t box = static_cast<uint32_t>(std::min(a.c.page_size, 64));
  CUtensorMap key_map, value_map;
  const uint64_t outer = static_cast<uint64_t>(a.c.pages) * a.c.kv_heads;
  int rc = piper::host::encode_rows_map(&key_map, a.c.key_codes, D, a.c.page_size, outer, box);
  if (rc != PIPER_B200_OK) return rc;
  if ((rc = piper::host::encode_rows_map(&value_map, a.c.value_codes, D, a.c.page_size, outer, box)) != PIPER_B200_OK)
    return rc;
  kernel<<<static_cast<unsigned>(plan.grid), threads, S::kAlloc, stream>>>(key_map, value_map, a);
  PIPER_HOST_CUDA(cudaGetLastError());
  if (plan.whole || plan.grid == 1) return PIPER_B200_OK;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(plan.grid - 1), (std::min(a.rows, S::kRows) + 3) / 4);
  config.blockDim = dim3(128);
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  PIPER_HOST_CUDA(cudaLaunchKernelEx(&config, piper::tree_merge_kernel<T, D, S>, a, static_cast<int>(plan.grid)));
  return PIPER_B200_OK;
}

template <typename T, int D>
int launch_tree_rows(const piper::TreeArgs& a, int sms, size_t workspace_bytes, cudaStream_t stream) {
  switch (tree_kind<D>(a.rows)) {
    case TreeKind::kEight:
      return launch_tree<T, D, FewRows<D, 8>>(a, piper::tree_attention_kernel<T, D, 4, kFewGroups, 8>,
                                              FewRows<D, 8>::kThreads, sms, workspace_bytes, stream);
    case TreeKind::kSixteen:
      return launch_tree<T, D, FewRows<D, 16>>(a, piper::tree_attention_kernel<T, D, 4, kFewGroups, 16>,
                                               FewRows<D, 16>::kThreads, sms, workspace_bytes, stream);
    case TreeKind::kMore:
      return launch_tree<T, D, FewRows<D, kMoreRows<D>>>(a, piper::tree_attention_kernel<T, D, 4, kFewGroups, kMoreRows<D>>,
                                               FewRows<D, kMoreRows<D>>::kThreads, sms, workspace_bytes, stream);
    case TreeKind::kAlternate:
      return launch_tree<T, D, piper::WideTile<D, false>>(a, piper::tree_wide_kernel<T, D, false>,
                                                          piper::kWideThreads, sms, workspace_bytes, stream);
    default:
      return launch_tree<T, D, piper::WideTile<D, true>>(a, piper::tree_wide_kernel<T, D, true>, piper::kWideThreads,
                                                         sms, workspace_bytes, stream);
  }
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
  while (a.block_shift < 3 && (int64_t(2) << a.block_shift) <= tokens) ++a.block_shift;
  const int64_t block = int64_t(1) << a.block_shift;
  unsigned blocks = 0;
  if ((rc = row_blocks((tokens + block - 1) / block * block * cache->kv_heads, cache->head_dim, &blocks)) !=
      PIPER_B200_OK)
    return rc;
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
                                                         int64_t head_dim, int64_t positions, size_t* bytes) {
  if (bytes == nullptr) return invalid("bytes is NULL");
  if (batch <= 0 || kv_heads <= 0 || positions <= 0) return invalid("sizes must be positive");
  if (kv_heads > 65535 || batch > 65535) return invalid("kv_heads and batch must be at most 65535");
  if (positions > (int64_t(1) << 39)) return invalid("positions must be at most 2^39");  // the widest table, pages of 256
  const int rc = check_rows(heads, kv_heads, nodes);
  if (rc != PIPER_B200_OK) return rc;
  if (head_dim != 64 && head_dim != 128)
    return invalid("head_dim must be 64 or 128, got " + std::to_string(head_dim));
  int device = 0, sms = 148;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    cudaGetLastError();
    sms = 148;
  }
  const int64_t rows = heads / kv_heads * nodes;
  *bytes = head_dim == 64 ? tree_plan<64>(batch, kv_heads, rows, positions, sms).bytes
                          : tree_plan<128>(batch, kv_heads, rows, positions, sms).bytes;
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
  if ((rc = check_rows(heads, cache->kv_heads, nodes)) != PIPER_B200_OK) return rc;
  // (fp32 holds its product with log2(e) as a normal number.)
  if (!(scale >= 0x1p-126 && scale <= 0x1p127)) return invalid("scale must be from 2^-126 to 2^127");
  if (reinterpret_cast<uintptr_t>(out) % 16 != 0) return invalid("output must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(cache->key_scales) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(cache->value_scales) % 16 != 0)
    return invalid("the cache's scales must be 16-byte aligned");
  piper::host::Device device;
  if ((rc = piper::host::ensure_device(&device)) != PIPER_B200_OK) return rc;
  if ((rc = set_up_tree(device)) != PIPER_B200_OK) return rc;
  piper::TreeArgs a{};
  a.c = *cache;
  a.query = query;
  for (int i = 0; i < 3; ++i) a.qs[i] = query_strides[i];
  a.out = out;
  a.mask = tree_mask;
  a.mask_stride = mask_stride;
  a.parts = static_cast<float*>(workspace);
  a.status = device.status;
  a.wait_budget_ns = 2000000000ull;
  a.heads = static_cast<int>(heads);
  a.nodes = static_cast<int>(nodes);
  a.group = static_cast<int>(heads / cache->kv_heads);
  a.rows = a.group * a.nodes;
  a.page_shift = page_shift_of(cache->page_size);
  a.vec = reinterpret_cast<uintptr_t>(query) % 8 == 0 && query_strides[0] % 4 == 0 && query_strides[1] % 4 == 0 &&
          query_strides[2] % 4 == 0;
  a.scale_log2e = static_cast<float>(scale * 1.4426950408889634);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == PIPER_B200_FLOAT16)
    return cache->head_dim == 64 ? launch_tree_rows<__half, 64>(a, device.sms, workspace_bytes, s)
                                 : launch_tree_rows<__half, 128>(a, device.sms, workspace_bytes, s);
  return cache->head_dim == 64 ? launch_tree_rows<__nv_bfloat16, 64>(a, device.sms, workspace_bytes, s)
                               : launch_tree_rows<__nv_bfloat16, 128>(a, device.sms, workspace_bytes, s);
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
  piper::host::Device device;
  int rc = piper::host::ensure_device(&device);
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
  a.vec = reinterpret_cast<uintptr_t>(target) % 16 == 0 && reinterpret_cast<uintptr_t>(draft) % 16 == 0 &&
          reinterpret_cast<uintptr_t>(noise) % 16 == 0 && target_strides[0] % 4 == 0 && target_strides[1] % 4 == 0 &&
          draft_strides[0] % 4 == 0 && draft_strides[1] % 4 == 0 && noise_stride % 4 == 0;
  // CTAs a request: enough to fill the GPU, while each has 2048 words or more
  // (fewer are read in the time that a join takes).
  int ranks = 1;
  while (ranks < 8 && vocab > int64_t(ranks) * 2048 && batch * ranks < 2 * device.sms) ranks *= 2;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = static_cast<unsigned>(ranks);
  attribute.val.clusterDim.y = 1;
  attribute.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(ranks), static_cast<unsigned>(batch));
  config.blockDim = dim3(piper::kVerifyThreads);
  config.stream = static_cast<cudaStream_t>(stream);
  config.attrs = &attribute;
  config.numAttrs = 1;
  PIPER_HOST_CUDA(cudaLaunchKernelEx(&config, piper::verify_tree_kernel, a));
  return PIPER_B200_OK;
}

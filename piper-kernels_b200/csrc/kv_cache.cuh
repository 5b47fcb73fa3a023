// The quantised paged KV cache: writing new rows, reading rows back, and
// moving the accepted rows of a drafted tree together.  All three are bound
// by memory.
//
// A row is one token of one KV head: D codes q[d] and a scale s, standing for
// q[d] * s (plus the key mean for keys), with
//   s = max_d |x[d]| * fp32(1/127)   (1 for a row of zeros)
//   q[d] = round half to even (x[d] / s)
// in fp32 with IEEE rounding, x being the input minus the key mean.  A row
// with an infinity or a NaN gets a scale that is not finite, so all its values
// read back as NaN.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "piper_b200.h"
#include "prepass.cuh"

namespace piper {

constexpr int kCacheThreads = 256;
constexpr int kMaxNodes = 64;

// The row index (page * kv_heads + head) * page_size + offset of a position,
// or -1 where the table names none.
__device__ __forceinline__ int64_t cache_row(const piper_b200_kv_cache_t& c, int page_shift, int b, int head,
                                             int64_t position) {
  const int64_t column = position >> page_shift;
  if (position < 0 || column >= c.table_width) return -1;
  const int page = __ldg(c.block_table + b * c.table_stride + column);
  if (page < 0 || page >= c.pages) return -1;
  return ((static_cast<int64_t>(page) * c.kv_heads + head) << page_shift) + (position & (c.page_size - 1));
}

struct CacheRowsArgs {
  piper_b200_kv_cache_t c;
  const void* in[2];   // write: key, value
  int64_t stride[2][3];
  void* out[2];        // read: key, value
  const int32_t* counts;
  int64_t tokens;
  int page_shift;
};

// Codes of eight values, packed.
__device__ __forceinline__ uint2 row_codes(const float (&x)[8], float scale) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = max(-127, min(127, __float2int_rn(__fdiv_rn(x[i], scale))));
    w[i / 4] |= (static_cast<uint32_t>(q) & 0xffu) << (8 * (i % 4));
  }
  return make_uint2(w[0], w[1]);
}

// D/8 consecutive lanes hold a row, eight values each: K and V of one (token,
// head) per lane group.  grid (ceil(tokens * kv_heads / rows per CTA), batch);
// heads vary fastest, the order in which a projection leaves them.
template <typename T, int D, bool kVec16>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(CacheRowsArgs a) {
  constexpr int kLanes = D / 8;
  const int b = blockIdx.y;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kCacheThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int64_t token = row / a.c.kv_heads;
  const int head = static_cast<int>(row - token * a.c.kv_heads);
  int64_t n = a.tokens;
  if (a.counts != nullptr) n = min(n, static_cast<int64_t>(__ldg(a.counts + b)));
  const int64_t at = token < n ? cache_row(a.c, a.page_shift, b, head, __ldg(a.c.lengths + b) + token) : -1;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float x[8] = {};
    if (at >= 0) {
      const T* p = static_cast<const T*>(a.in[side]) + b * a.stride[side][0] + head * a.stride[side][1] +
                   token * a.stride[side][2] + lane * 8;
      unpack8<T>(load_raw8<T, kVec16>(p), x);
      if (side == 0 && a.c.key_mean != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __fsub_rn(x[i], __ldg(a.c.key_mean + head * D + lane * 8 + i));
      }
    }
    // The largest magnitude; fmaxf would drop a NaN, so the bits are compared
    // as integers (NaN above infinity above every finite magnitude).
    uint32_t amax = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (at < 0) continue;
    const float scale = amax == 0u ? 1.0f : __fmul_rn(__uint_as_float(amax), 1.0f / 127.0f);
    int8_t* codes = static_cast<int8_t*>(side == 0 ? a.c.key_codes : a.c.value_codes);
    *reinterpret_cast<uint2*>(codes + at * D + lane * 8) = row_codes(x, scale);
    if (lane == 0) (side == 0 ? a.c.key_scales : a.c.value_scales)[at] = scale;
  }
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// As cache_write_kernel, with tokens varying fastest: the outputs are
// contiguous [batch, kv_heads, tokens, D].
template <typename T, int D>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(CacheRowsArgs a) {
  constexpr int kLanes = D / 8;
  const int b = blockIdx.y;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kCacheThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int64_t head64 = row / a.tokens;
  if (head64 >= a.c.kv_heads) return;
  const int head = static_cast<int>(head64);
  const int64_t token = row - head64 * a.tokens;
  int64_t n = a.tokens;
  if (a.counts != nullptr) n = min(n, static_cast<int64_t>(__ldg(a.counts + b)));
  const int64_t at = token < n ? cache_row(a.c, a.page_shift, b, head, __ldg(a.c.lengths + b) + token) : -1;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float x[8] = {};
    if (at >= 0) {
      const int8_t* codes = static_cast<const int8_t*>(side == 0 ? a.c.key_codes : a.c.value_codes);
      const uint2 w = *reinterpret_cast<const uint2*>(codes + at * D + lane * 8);
      const float scale = (side == 0 ? a.c.key_scales : a.c.value_scales)[at];
      const int8_t* q = reinterpret_cast<const int8_t*>(&w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(static_cast<float>(q[i]), scale);
      if (side == 0 && a.c.key_mean != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(x[i], __ldg(a.c.key_mean + head * D + lane * 8 + i));
      }
    }
    uint4 w;
    w.x = pack2(x[0], x[1], T());
    w.y = pack2(x[2], x[3], T());
    w.z = pack2(x[4], x[5], T());
    w.w = pack2(x[6], x[7], T());
    const int64_t o = ((static_cast<int64_t>(b) * a.c.kv_heads + head) * a.tokens + token) * D + lane * 8;
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out[side]) + o) = w;
  }
}

// One CTA moves the rows of one (request, KV head), K then V: every source
// row is in registers before the barrier, every target row is written after
// it, because a row may be both.
template <int D>
__global__ void __launch_bounds__(kCacheThreads) cache_keep_kernel(piper_b200_kv_cache_t c, const int32_t* path,
                                                                   int64_t path_stride, int nodes,
                                                                   const int32_t* counts, int page_shift) {
  constexpr int kLanes = D / 16;                     // 16 codes each
  constexpr int kRows = kCacheThreads / kLanes;      // rows per pass
  constexpr int kPasses = (kMaxNodes + kRows - 1) / kRows;
  const int head = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x % kLanes;
  int8_t* codes = static_cast<int8_t*>(blockIdx.z == 0 ? c.key_codes : c.value_codes);
  float* scales = blockIdx.z == 0 ? c.key_scales : c.value_scales;
  const int kept = min(nodes, __ldg(counts + b));
  const int64_t length = __ldg(c.lengths + b);
  uint4 moved[kPasses];
  float scale[kPasses];
  int64_t to[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int j = static_cast<int>(threadIdx.x) / kLanes + p * kRows;
    to[p] = -1;
    if (j < 1 || j >= kept) continue;
    const int node = __ldg(path + b * path_stride + j);
    if (node < 0 || node >= nodes) continue;
    const int64_t from = cache_row(c, page_shift, b, head, length + node);
    if (from < 0) continue;
    to[p] = cache_row(c, page_shift, b, head, length + j);
    moved[p] = *reinterpret_cast<const uint4*>(codes + from * D + lane * 16);
    scale[p] = scales[from];
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    if (to[p] < 0) continue;
    *reinterpret_cast<uint4*>(codes + to[p] * D + lane * 16) = moved[p];
    if (lane == 0) scales[to[p]] = scale[p];
  }
}

}  // namespace piper

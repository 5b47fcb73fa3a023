// The quantised paged KV cache: writing new rows, reading rows back, and
// moving the accepted rows of a drafted tree together.  All three would be
// bound by memory.
//
// Measured (4 prompts of 5001 to 8192 tokens, 32 heads of 128, bf16): written in
// 181 us, read back in 156, where the copy rate allows 101 and 118 (the zeros that
// fill the shorter prompts included).  Writing takes 17 instructions a value, the
// near-tie test of the division-free rounding among them (both without it, which
// exact codes need, 304 us instead of 336; with IEEE division, and eight values a
// lane, 392), with the ALU pipe busy half the time and 43 % of an SM's warps
// resident.  Reading takes 10 with 87 % resident and the issue slots busy 42 % of the
// time: latency, of the table, the row and the key mean, which both kernels load
// again for every row.
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
  int block_shift;     // write: log2 of the tokens of a head that follow one another
};

// Codes of eight values, packed.  The prepass's division-free rounding needs
// the quotient to 2^-14: |x / s| <= 127 and an approximate reciprocal (2^-23)
// give 2^-15, while the scale and its reciprocal are normal numbers; other rows
// (nearly subnormal, or not finite) divide.
__device__ __forceinline__ uint2 row_codes(const float (&x)[8], float scale) {
  if (scale >= 0x1p-100f && scale <= 0x1p+121f) {
    float over;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(over) : "f"(scale));
    return pack_codes(x, scale, over);
  }
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = max(-127, min(127, __float2int_rn(__fdiv_rn(x[i], scale))));
    w[i / 4] |= (static_cast<uint32_t>(q) & 0xffu) << (8 * (i % 4));
  }
  return make_uint2(w[0], w[1]);
}

// Largest magnitude; a NaN wins.
__device__ __forceinline__ float amax3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight fp32 of the key mean.
__device__ __forceinline__ void mean8(const float* p, float (&m)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  m[0] = a.x, m[1] = a.y, m[2] = a.z, m[3] = a.w, m[4] = b.x, m[5] = b.y, m[6] = b.z, m[7] = b.w;
}

// Four codes as floats: the byte plus 128 under the exponent of 2^23.
__device__ __forceinline__ void codes_f32(uint32_t w, float (&x)[8], int at) {
  const uint32_t u = w ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[at + i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540u + i)) - 8388736.0f;
}

// (token, head) of the rows that a CTA takes, from row0 on.  `inner` varies
// fastest.  Divisions are of 32 bits where the rows' numbers are, and none for
// rows that stay near the first.
struct CacheRowWalk {
  int64_t outer0;
  unsigned inner0, inner;
  __device__ CacheRowWalk(int64_t row0, int64_t inner_count) {
    inner = static_cast<unsigned>(inner_count);
    outer0 = (row0 >> 32) == 0 ? static_cast<unsigned>(row0) / inner : row0 / inner_count;
    inner0 = static_cast<unsigned>(row0 - outer0 * inner_count);
  }
  __device__ __forceinline__ void at(unsigned ahead, int64_t* outer, unsigned* in) const {
    const unsigned x = inner0 + ahead, more = x < inner ? 0u : x - inner < inner ? 1u : x / inner;
    *outer = outer0 + more;
    *in = x - more * inner;
  }
};

// D/16 consecutive lanes hold K and V of one row (a token of a head), sixteen
// values of each a lane (four rows' loads in flight a thread took 457 us for the
// prompts above).  grid (ceil(rows / rows per CTA), batch).  Rows go by
// blocks of up to 8 tokens, then heads, then tokens: a projection leaves the heads of
// a token side by side, the cache has the tokens of a head side by side, and
// such a block is a kilobyte in both.
template <typename T, int D, bool kVec16>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(CacheRowsArgs a) {
  constexpr int kLanes = D / 16;
  constexpr int kRows = kCacheThreads / kLanes;
  const int b = blockIdx.y;
  const int lane = threadIdx.x % kLanes;
  const CacheRowWalk walk(static_cast<int64_t>(blockIdx.x) * kRows,
                          static_cast<int64_t>(a.c.kv_heads) << a.block_shift);
  int64_t n = a.tokens;
  if (a.counts != nullptr) n = min(n, static_cast<int64_t>(__ldg(a.counts + b)));
  const int64_t length = __ldg(a.c.lengths + b);
  int64_t token;
  unsigned head;
  walk.at(threadIdx.x / kLanes, &token, &head);
  token = (token << a.block_shift) + (head & ((1u << a.block_shift) - 1u));
  head >>= a.block_shift;
  uint4 raw[2][2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    raw[side][0] = raw[side][1] = make_uint4(0u, 0u, 0u, 0u);
    if (token < n) {
      const T* from = static_cast<const T*>(a.in[side]) + b * a.stride[side][0] + head * a.stride[side][1] +
                      token * a.stride[side][2] + lane * 16;
      raw[side][0] = load_raw8<T, kVec16>(from);
      raw[side][1] = load_raw8<T, kVec16>(from + 8);
    }
  }
  const int64_t at = token < n ? cache_row(a.c, a.page_shift, b, head, length + token) : -1;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float x[2][8];
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      unpack8<T>(raw[side][k], x[k]);
      if (side == 0 && a.c.key_mean != nullptr && at >= 0) {
        float m[8];
        mean8(a.c.key_mean + head * D + lane * 16 + k * 8, m);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = __fsub_rn(x[k][i], m[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; i += 2) amax = amax3(amax, x[k][i], x[k][i + 1]);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (at < 0) continue;
    const float scale = amax == 0.0f ? 1.0f : __fmul_rn(amax, 1.0f / 127.0f);
    int8_t* codes = static_cast<int8_t*>(side == 0 ? a.c.key_codes : a.c.value_codes);
    const uint2 lo = row_codes(x[0], scale), hi = row_codes(x[1], scale);
    *reinterpret_cast<uint4*>(codes + at * D + lane * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
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
  constexpr int kLanes = D / 16;
  constexpr int kRows = kCacheThreads / kLanes;
  const int b = blockIdx.y;
  const int lane = threadIdx.x % kLanes;
  const CacheRowWalk walk(static_cast<int64_t>(blockIdx.x) * kRows, a.tokens);
  int64_t n = a.tokens;
  if (a.counts != nullptr) n = min(n, static_cast<int64_t>(__ldg(a.counts + b)));
  const int64_t length = __ldg(a.c.lengths + b);
  int64_t head;
  unsigned token;
  walk.at(threadIdx.x / kLanes, &head, &token);
  const int64_t at = head < a.c.kv_heads && token < n
                         ? cache_row(a.c, a.page_shift, b, static_cast<int>(head), length + token)
                         : -1;
  uint4 w[2];
  float scale[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    if (at < 0) continue;
    const int8_t* codes = static_cast<const int8_t*>(side == 0 ? a.c.key_codes : a.c.value_codes);
    w[side] = *reinterpret_cast<const uint4*>(codes + at * D + lane * 16);
    scale[side] = (side == 0 ? a.c.key_scales : a.c.value_scales)[at];
  }
  if (head >= a.c.kv_heads) return;
  const int64_t o = ((static_cast<int64_t>(b) * a.c.kv_heads + head) * a.tokens + token) * D + lane * 16;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint4 y = make_uint4(0u, 0u, 0u, 0u);
      if (at >= 0) {
        float x[8];
        codes_f32(k == 0 ? w[side].x : w[side].z, x, 0);
        codes_f32(k == 0 ? w[side].y : w[side].w, x, 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(x[i], scale[side]);
        if (side == 0 && a.c.key_mean != nullptr) {
          float m[8];
          mean8(a.c.key_mean + head * D + lane * 16 + k * 8, m);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(x[i], m[i]);
        }
        y.x = pack2(x[0], x[1], T());
        y.y = pack2(x[2], x[3], T());
        y.z = pack2(x[4], x[5], T());
        y.w = pack2(x[6], x[7], T());
      }
      *reinterpret_cast<uint4*>(static_cast<T*>(a.out[side]) + o + k * 8) = y;
    }
  }
}

// One CTA moves the key rows of one (request, KV head), another its value rows
// (blockIdx.z): every source row is in registers before the barrier, every target
// row is written after it, because a row may be both.
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

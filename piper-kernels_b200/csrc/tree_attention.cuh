// Attention of a drafted tree's nodes over the quantised cache (simple form:
// one CTA per query row).
#pragma once

#include <math.h>

#include "kv_cache.cuh"

namespace piper {

struct TreeArgs {
  piper_b200_kv_cache_t c;
  const void* query;
  int64_t qs[3];
  void* out;
  const int64_t* mask;
  int64_t mask_stride;
  int heads, nodes, group, page_shift;
  float scale_log2e;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) tree_attention_simple_kernel(TreeArgs a) {
  constexpr int kPer = D / 32;
  const int node = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  const int kv = head / a.group;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const T* q = static_cast<const T*>(a.query) + b * a.qs[0] + head * a.qs[1] + node * a.qs[2] + lane * kPer;
  float qf[kPer], acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    qf[i] = to_f32<T>(q[i]);
    acc[i] = 0.0f;
  }
  const int64_t length = max(0, __ldg(a.c.lengths + b));
  const uint64_t mask = a.mask != nullptr ? static_cast<uint64_t>(a.mask[b * a.mask_stride + node])
                                          : (~0ull >> (63 - node));
  float m = -INFINITY, l = 0.0f;
  for (int64_t pos = warp; pos < length + a.nodes; pos += 4) {
    if (pos >= length && !((mask >> (pos - length)) & 1)) continue;
    const int64_t row = cache_row(a.c, a.page_shift, b, kv, pos);
    if (row < 0) continue;
    const int8_t* kc = static_cast<const int8_t*>(a.c.key_codes) + row * D + lane * kPer;
    const int8_t* vc = static_cast<const int8_t*>(a.c.value_codes) + row * D + lane * kPer;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) s += qf[i] * static_cast<float>(kc[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= a.c.key_scales[row] * a.scale_log2e;
    const float m_new = fmaxf(m, s);
    const float rescale = exp2f(m - m_new), p = exp2f(s - m_new);
    const float pv = p * a.c.value_scales[row];
    m = m_new;
    l = l * rescale + p;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * rescale + pv * static_cast<float>(vc[i]);
  }
  __shared__ float sm[4], sl[4], so[4][D];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) so[warp][lane * kPer + i] = acc[i];
  __syncthreads();
  if (threadIdx.x < D) {
    float top = -INFINITY;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, sm[w]);
    float o = 0.0f, total = 0.0f;
    for (int w = 0; w < 4; ++w) {
      if (sl[w] == 0.0f) continue;
      const float r = exp2f(sm[w] - top);
      total += sl[w] * r;
      o += so[w][threadIdx.x] * r;
    }
    const float y = total == 0.0f ? 0.0f : o / total;
    const int64_t at = ((static_cast<int64_t>(b) * a.heads + head) * a.nodes + node) * D + threadIdx.x;
    static_cast<T*>(a.out)[at] = static_cast<T>(y);
  }
}

}  // namespace piper

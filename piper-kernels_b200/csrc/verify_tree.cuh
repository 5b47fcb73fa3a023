// Rejection sampling over a drafted tree (simple form: one CTA per request).
#pragma once

#include <math.h>
#include <stdint.h>

namespace piper {

constexpr int kVerifyThreads = 1024;

struct VerifyArgs {
  const float* target;
  const float* draft;
  int64_t ts[2], ds[2];
  const int64_t* tokens;
  const int32_t* parents;
  const float* uniform;
  const float* noise;
  int64_t tokens_stride, parents_stride, uniform_stride, noise_stride;
  int nodes;
  int64_t vocab;
  int32_t* path;
  int32_t* count;
  int64_t* next;
};

// What is left of probability p after taking out the draft's q once for each
// of the n totals: max(r - q, 0) / total, or r where the total is zero.
__device__ __forceinline__ float rest_of(float p, float q, const float* totals, int n) {
  float r = p;
  for (int k = 0; k < n; ++k)
    if (totals[k] > 0.0f) r = __fdiv_rn(fmaxf(r - q, 0.0f), totals[k]);
  return r;
}

__global__ void __launch_bounds__(kVerifyThreads) verify_simple_kernel(VerifyArgs a) {
  __shared__ float totals[64];
  __shared__ float part[32];
  __shared__ float best_s[32];
  __shared__ int64_t best_i[32];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  int current = 0, rejected = 0, count = 1;
  int32_t* path = a.path + b * a.nodes;
  if (tid == 0) path[0] = 0;
  for (int i = 1; i < a.nodes; ++i) {
    const int64_t x = a.tokens[b * a.tokens_stride + i];
    if (a.parents[b * a.parents_stride + i] != current || x < 0 || x >= a.vocab) continue;
    const float* p = a.target + b * a.ts[0] + current * a.ts[1];
    const float* q = a.draft + b * a.ds[0] + current * a.ds[1];
    if (a.uniform[b * a.uniform_stride + i] * q[x] < rest_of(p[x], q[x], totals, rejected)) {
      if (tid == 0) path[count] = i;
      ++count;
      current = i;
      rejected = 0;
      continue;
    }
    float sum = 0.0f;
    for (int64_t v = tid; v < a.vocab; v += kVerifyThreads)
      sum += fmaxf(rest_of(p[v], q[v], totals, rejected) - q[v], 0.0f);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      float total = 0.0f;
      for (int w = 0; w < 32; ++w) total += part[w];
      totals[rejected] = total;
    }
    __syncthreads();
    ++rejected;
  }
  const float* p = a.target + b * a.ts[0] + current * a.ts[1];
  const float* q = a.draft + b * a.ds[0] + current * a.ds[1];
  float best = -1.0f;
  int64_t at = 0;
  for (int64_t v = tid; v < a.vocab; v += kVerifyThreads) {
    const float r = rejected == 0 ? p[v] : rest_of(p[v], q[v], totals, rejected);
    const float s = __fdiv_rn(r, a.noise[b * a.noise_stride + v]);
    if (s > best) {
      best = s;
      at = v;
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float s = __shfl_xor_sync(0xffffffffu, best, o);
    const int64_t j = __shfl_xor_sync(0xffffffffu, at, o);
    if (s > best || (s == best && j < at)) {
      best = s;
      at = j;
    }
  }
  if (lane == 0) {
    best_s[warp] = best;
    best_i[warp] = at;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 32; ++w)
      if (best_s[w] > best || (best_s[w] == best && best_i[w] < at)) {
        best = best_s[w];
        at = best_i[w];
      }
    a.next[b] = best < 0.0f ? 0 : at;
    a.count[b] = count;
  }
  for (int i = count + tid; i < a.nodes; i += kVerifyThreads) path[i] = -1;
}

}  // namespace piper

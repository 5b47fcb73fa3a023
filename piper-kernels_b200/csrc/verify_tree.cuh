// Rejection sampling over a drafted tree.
//
// A request's walk needs few numbers while it accepts: target[x] and draft[x]
// of each drafted token at its parent, which are fetched for all nodes at
// once.  A whole row is read only where the walk rejects: with r the rest of
// the target's distribution and q the draft's,
//   total = sum_v max(r[v] - q[v], 0),   r <- max(r - q, 0) / total
// before a further sibling can be tested, and at the end for the next token,
//   argmax_v r[v] / noise[v],
// which takes the last rejected draft out on the way: its total is not needed.
// The rest after several rejections is computed again from the rows and the
// totals, so that nothing is written back.  All is fp32; a total divides as its
// reciprocal multiplies (an IEEE division for each word and rejection made the
// passes twice as long), the last division, by the noise, is IEEE: equal
// quotients are equal, and go to the lowest index.
//
// A warp divides only near its best quotient (a division for every word: 6 us more
// in the largest case below).
//
// Bound: memory (12 bytes a word for the last pass), and with few requests the
// latency of the passes that follow one another.  A cluster of CTAs shares a
// request's vocabulary and joins its sums and maxima through distributed
// shared memory, in rank order (one CTA a request took four times as long).
//
// Measured: a chain of 8 over 32768 words 7.0 us; 16 trees of 16 over 50001 words
// (rows that start at any element) 12 us; 64 trees of 32 over 131072 words 43 us,
// where the mean request reads 1.7 to 1.8 MB: 0.4 of the copy rate, as 512 CTAs run
// in two turns and a request of four rejections takes four passes.  No faster: the
// noise fetched into L2 in advance (52 before, 53), half the loads under way and three
// CTAs on an SM (47), 1024 threads (64 against 52), one turn of 4 CTAs a request
// (60 against 51), passes made for no earlier rejection (45, with spills).
#pragma once

#include <cooperative_groups.h>
#include <math.h>
#include <stdint.h>

#include "kv_cache.cuh"

namespace piper {

constexpr int kVerifyThreads = 512;
constexpr int kVerifyUnroll = 4;  // 16-byte loads in flight of each row
constexpr int kVerifySingle = 8;  // 4-byte ones, where rows are not aligned
constexpr float kVerifyLeast = 0x1p-126f;  // the least total whose reciprocal is surely finite
constexpr float kVerifyUp = 0x1p64f;       // what a smaller one is scaled by
constexpr float kVerifyTold = 0x1p-64f;    // a quotient far above what fp32 rounds to zero

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
  int vec;  // rows of target, draft and noise allow 16-byte loads
  int32_t* path;
  int32_t* count;
  int64_t* next;
};

// What is left of probability p after taking out the draft's q n times:
// max(r - q, 0) over each total, given as reciprocals.  kSmall: a negative one is
// that of a subnormal total times kVerifyUp.
template <bool kSmall = false>
__device__ __forceinline__ float rest_of(float p, float q, const float* over, int n) {
  float r = p;
  for (int k = 0; k < n; ++k) {
    r = fmaxf(r - q, 0.0f);
    r = kSmall && over[k] < 0.0f ? r * kVerifyUp * -over[k] : r * over[k];
  }
  return r;
}

struct VerifyBest {
  float score;
  int at;
};
__device__ __forceinline__ VerifyBest verify_better(VerifyBest x, VerifyBest y) {
  return y.score > x.score || (y.score == x.score && y.at < x.at) ? y : x;
}

// Calls body(v, p, q, e) for this thread's words of [begin, end): the target's,
// the draft's and the noise's values (0 where a pass does not read them).
// `begin` is a multiple of 4.  After every few words a warp calls turn(), together.
template <bool kDraft, bool kNoise, typename Body, typename Turn>
__device__ __forceinline__ void verify_words(const VerifyArgs& a, const float* p, const float* q, const float* e,
                                             int begin, int end, Body body, Turn turn) {
  const int lane = threadIdx.x % 32;
  int v = begin + threadIdx.x;
  if (a.vec) {
    const int whole = begin + (end - begin) / 4 * 4;
    constexpr int kStep = kVerifyThreads * 4;
    for (int u = begin + threadIdx.x * 4; u - lane * 4 < whole; u += kStep * kVerifyUnroll) {
      float4 pw[kVerifyUnroll], qw[kVerifyUnroll], ew[kVerifyUnroll];
#pragma unroll
      for (int k = 0; k < kVerifyUnroll; ++k) {
        pw[k] = qw[k] = ew[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (u + k * kStep < whole) {
          pw[k] = __ldg(reinterpret_cast<const float4*>(p + u + k * kStep));
          if (kDraft) qw[k] = __ldg(reinterpret_cast<const float4*>(q + u + k * kStep));
          if (kNoise) ew[k] = __ldg(reinterpret_cast<const float4*>(e + u + k * kStep));
        }
      }
#pragma unroll
      for (int k = 0; k < kVerifyUnroll; ++k) {
        const int w = u + k * kStep;
        if (w < whole) {
          body(w, pw[k].x, qw[k].x, ew[k].x);
          body(w + 1, pw[k].y, qw[k].y, ew[k].y);
          body(w + 2, pw[k].z, qw[k].z, ew[k].z);
          body(w + 3, pw[k].w, qw[k].w, ew[k].w);
        }
        turn();
      }
    }
    v = whole + threadIdx.x;
  }
  for (; v - lane < end; v += kVerifyThreads * kVerifySingle) {
    float pw[kVerifySingle], qw[kVerifySingle], ew[kVerifySingle];
#pragma unroll
    for (int k = 0; k < kVerifySingle; ++k) {
      const int w = v + k * kVerifyThreads;
      pw[k] = qw[k] = ew[k] = 0.0f;
      if (w < end) {
        pw[k] = __ldg(p + w);
        if (kDraft) qw[k] = __ldg(q + w);
        if (kNoise) ew[k] = __ldg(e + w);
      }
    }
#pragma unroll
    for (int k = 0; k < kVerifySingle; ++k) {
      if (v + k * kVerifyThreads < end) body(v + k * kVerifyThreads, pw[k], qw[k], ew[k]);
      if (k % 4 == 3) turn();
    }
  }
}

// The passes over this thread's words of [begin, end) when a total was subnormal.
// Not inlined: they are rare, and their registers would be the others'.
__device__ __noinline__ float verify_small_sum(const float* p, const float* q, int begin, int end, const float* over,
                                               int n) {
  float sum = 0.0f;
  for (int v = begin + threadIdx.x; v < end; v += kVerifyThreads) {
    const float y = __ldg(q + v);
    sum += fmaxf(rest_of<true>(__ldg(p + v), y, over, n) - y, 0.0f);
  }
  return sum;
}
__device__ __noinline__ VerifyBest verify_small_best(const float* p, const float* q, const float* e, int begin,
                                                     int end, const float* over, int n, bool less) {
  VerifyBest best{-1.0f, 0};
  for (int v = begin + threadIdx.x; v < end; v += kVerifyThreads) {
    const float y = __ldg(q + v);
    const float r = rest_of<true>(__ldg(p + v), y, over, n);
    const float s = __fdiv_rn(less ? fmaxf(r - y, 0.0f) : r, __ldg(e + v));
    if (s > best.score) best = VerifyBest{s, v};
  }
  return best;
}

// grid (CTAs of a cluster, batch), a cluster to a request.
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_tree_kernel(VerifyArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int kWarps = kVerifyThreads / 32;
  __shared__ float node_p[kMaxNodes], node_q[kMaxNodes], node_u[kMaxNodes];
  __shared__ int node_parent[kMaxNodes];  // -1: absent
  __shared__ float over[kMaxNodes];
  __shared__ float warp_sum[kWarps], joined_sum[2];  // by turn
  __shared__ VerifyBest warp_best[kWarps], joined_best;
  const int64_t b = blockIdx.y;
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  // This CTA's words: a multiple of 4 to each rank.
  const int vocab = static_cast<int>(a.vocab);
  const int per = ((vocab + ranks - 1) / ranks + 3) / 4 * 4;
  const int begin = min(vocab, per * rank), end = min(vocab, begin + per);
  if (tid < kMaxNodes) {
    node_parent[tid] = -1;
    if (tid > 0 && tid < a.nodes) {
      const int64_t x = __ldg(reinterpret_cast<const long long*>(a.tokens) + b * a.tokens_stride + tid);
      const int parent = __ldg(a.parents + b * a.parents_stride + tid);
      if (x >= 0 && x < a.vocab && parent >= 0 && parent < tid) {
        node_parent[tid] = parent;
        node_p[tid] = __ldg(a.target + b * a.ts[0] + parent * a.ts[1] + x);
        node_q[tid] = __ldg(a.draft + b * a.ds[0] + parent * a.ds[1] + x);
        node_u[tid] = __ldg(a.uniform + b * a.uniform_stride + tid);
      }
    }
  }
  __syncthreads();
  // Every thread of the cluster takes the same walk.  A node's children, as
  // bits (they all come after it):
  auto children_of = [&](int node) {
    const uint64_t low = __ballot_sync(0xffffffffu, node_parent[lane] == node);
    const uint64_t high = __ballot_sync(0xffffffffu, node_parent[lane + 32] == node);
    return low | (high << 32);
  };
  int current = 0, rejected = 0, count = 1, turn = 0;
  int32_t* path = a.path + b * a.nodes;
  if (rank == 0 && tid == 0) path[0] = 0;
  uint64_t children = children_of(0);
  // Nothing is tested against the rest of the last rejection, and the next
  // token does not depend on its total: the last pass takes that draft out
  // without it, unless its scores come out too small to be told from nothing.
  bool open_end = false, may_end = true;
  // A total since the last accepted node was subnormal: such a walk takes the two
  // functions above (a second product for every word cost 5 % of the largest case,
  // loops in place 3 %, the branch 1.5 %).
  bool small = false;
  VerifyBest best;
  const float* er = a.noise + b * a.noise_stride;
  for (;;) {  // twice at most
    while (children != 0) {
      const int i = __ffsll(static_cast<long long>(children)) - 1;
      const float p = node_p[i], q = node_q[i];
      if (node_u[i] * q < rest_of<true>(p, q, over, rejected)) {
        if (rank == 0 && tid == 0) path[count] = i;
        ++count;
        current = i;
        rejected = 0;
        small = false;
        children = children_of(i);
        continue;
      }
      if (may_end && (children & (children - 1)) == 0) {
        open_end = true;
        break;
      }
      children &= children - 1;
      const float* pr = a.target + b * a.ts[0] + current * a.ts[1];
      const float* qr = a.draft + b * a.ds[0] + current * a.ds[1];
      float sum = 0.0f;
      if (!small) {
        verify_words<true, false>(
            a, pr, qr, nullptr, begin, end,
            [&](int, float x, float y, float) { sum += fmaxf(rest_of(x, y, over, rejected) - y, 0.0f); }, [] {});
      } else {
        sum = verify_small_sum(pr, qr, begin, end, over, rejected);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) warp_sum[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        float mine = 0.0f;
        for (int w = 0; w < kWarps; ++w) mine += warp_sum[w];
        joined_sum[turn] = mine;
      }
      cluster.sync();
      float total = 0.0f;
      for (int r = 0; r < ranks; ++r) total += *cluster.map_shared_rank(&joined_sum[turn], r);
      // The other turn's sums are written only after every rank has read these:
      // each passes the next cluster.sync after its reading.
      turn ^= 1;
      if (total > 0.0f) {  // else nothing would be left: rest stays as it was
        const bool subnormal = total < kVerifyLeast;
        if (tid == 0) over[rejected] = subnormal ? -1.0f / (total * kVerifyUp) : 1.0f / total;
        ++rejected;
        small |= subnormal;
      }
      __syncthreads();
    }
    const float* pr = a.target + b * a.ts[0] + current * a.ts[1];
    const float* qr = a.draft + b * a.ds[0] + current * a.ds[1];
    best = VerifyBest{-1.0f, 0};
    // Only a word near the warp's best is divided: r < score * e, by more than
    // the product's rounding, cannot win (nor does it tie).
    float bound = 0.0f;
    auto race = [&](int v, float r, float e) {
      if (!(r < bound * e)) {
        const float s = __fdiv_rn(r, e);
        if (s > best.score) best = VerifyBest{s, v};  // (a thread's words ascend)
        bound = fmaxf(bound, fminf(s, 0x1p127f) * 0x1.fffffp-1f);
      }
    };
    auto share = [&] { bound = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(bound))); };
    if (rejected == 0 && !open_end) {
      verify_words<false, true>(a, pr, qr, er, begin, end, [&](int v, float x, float, float e) { race(v, x, e); }, share);
    } else if (small) {
      best = verify_small_best(pr, qr, er, begin, end, over, rejected, open_end);
    } else {
      verify_words<true, true>(
          a, pr, qr, er, begin, end,
          [&](int v, float x, float y, float e) {
            const float r = rest_of(x, y, over, rejected);
            race(v, open_end ? fmaxf(r - y, 0.0f) : r, e);
          },
          share);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      best = verify_better(best, VerifyBest{__shfl_xor_sync(0xffffffffu, best.score, o),
                                            __shfl_xor_sync(0xffffffffu, best.at, o)});
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) best = verify_better(best, warp_best[w]);
      joined_best = best;
    }
    cluster.sync();
    if (!open_end) break;
    bool told = false;
    for (int r = 0; r < ranks; ++r) told |= cluster.map_shared_rank(&joined_best, r)->score > kVerifyTold;
    if (told) break;
    open_end = may_end = false;
    cluster.sync();  // every rank has read the scores that are written again
  }
  if (rank == 0) {
    if (tid == 0) {
      for (int r = 1; r < ranks; ++r) best = verify_better(best, *cluster.map_shared_rank(&joined_best, r));
      a.next[b] = best.score < 0.0f ? 0 : best.at;
      a.count[b] = count;
    }
    for (int i = count + tid; i < a.nodes; i += kVerifyThreads) path[i] = -1;
  }
  cluster.sync();  // shared memory stays until rank 0 has read it
}

}  // namespace piper

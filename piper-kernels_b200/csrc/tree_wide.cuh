// Attention of many query rows of a KV head (wide trees, large groups) over
// the quantised paged cache, on tcgen05.
//
// The mathematics, the units and the parts are those of tree_attention.cuh;
// here a tile is 128 keys and a product is a 128-row tcgen05 MMA with fp32
// accumulators in TMEM:
//   S = Q K^T   Q (fp16, scaled by row) and K from shared memory
//   O += W V    W (fp16 weights) from TMEM, over the spent scores; V from
//               shared memory with the head dimension contiguous
// kind::f16 needs 16-bit operands, so a warpgroup turns each tile's codes into
// fp16 between the TMA ring and the MMAs: 128 rows then pay for one
// conversion.
//
// Two streams of 128 TMEM lanes hide each other's latency: while one stream's
// softmax runs, the other's MMAs do.  kShared: the streams are rows 0-127 and
// 128-255 of the row tile over the same keys (more than 128 rows).  Otherwise
// they are alternate key tiles of the same 128 rows, joined at the end.
//
// Warps: 0-3 and 4-7 softmax of streams 0 and 1 (a thread owns a row), 8-11
// conversion (a thread owns a key), 12 fetches, 13 issues MMAs, 14 owns TMEM.
#pragma once

#include "tree_attention.cuh"

namespace piper {

constexpr int kWideThreads = 512;
// Register split (setmaxnreg), launch = 128 x 512: the softmax holds 128
// scores a thread.  128 * (2 * 192 + 72 + 56) = 65536.
constexpr int kWideLaunchRegs = 128;
constexpr int kWideRegsSoftmax = 192;
constexpr int kWideRegsConvert = 72;
constexpr int kWideRegsControl = 56;
static_assert(2 * kWideRegsSoftmax + kWideRegsConvert + kWideRegsControl <= 4 * kWideLaunchRegs,
              "setmaxnreg split exceeds the launch register allocation");

template <int D, bool kShared>
struct WideTile {
  static constexpr int kRows = kShared ? 256 : 128;
  static constexpr int kKeys = 128;
  static constexpr int kCtas = 1;
  static constexpr int kCodes = kKeys * D;          // one ring slot: K or V codes
  static constexpr int kHalf = kKeys * D * 2;       // one fp16 operand tile
  static constexpr int kQuery = (kShared ? 2 : 1) * kHalf;
  static constexpr int kBuffers = kShared ? 1 : 2;  // fp16 K and V tiles
  static constexpr int kScaleRing = 4;
  static constexpr int kOffQuery = 0;
  static constexpr int kOffK = kOffQuery + kQuery;
  static constexpr int kOffV = kOffK + kBuffers * kHalf;
  static constexpr int kOffScales = kOffV + kBuffers * kHalf;
  static constexpr int kOffState = kOffScales + kScaleRing * kKeys * 8;
  static constexpr int kOffRing = (kOffState + 3 * 128 * 4 + 1023) / 1024 * 1024;
  static constexpr int kFit = (225 * 1024 - kOffRing) / kCodes;
  static constexpr int kRing = kFit > 8 ? 8 : kFit;
  static constexpr int kAlloc = kOffRing + kRing * kCodes + 1024;
  static constexpr int kPart = kRows * (D + 2);
};
static_assert(WideTile<128, true>::kRing >= 3 && WideTile<128, false>::kRing >= 3, "ring too short");

// Descriptor of a B operand whose N (the head dimension) is contiguous: rows
// of 64 elements (128 bytes, SW128), 8 keys to a swizzle atom; blocks of 64
// head dimensions lie `block` bytes apart.
__device__ __forceinline__ uint64_t umma_desc_nmajor(uint32_t smem_addr, uint32_t block) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((block >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;
  return d;
}

// Walks a run's segments: (request, head, row tile) and the key tiles of it
// that the run has.
struct WideWalk {
  int b, hr, tile, tiles, count;
  int64_t left;
  bool all;
};
template <int kKeys>
__device__ __forceinline__ WideWalk wide_begin(const TreeRun& r) {
  WideWalk w;
  w.b = r.b;
  w.hr = r.hr;
  w.tile = r.tile;
  w.tiles = r.tiles;
  w.left = r.end - r.begin;
  w.count = static_cast<int>(min(static_cast<int64_t>(w.tiles - w.tile), w.left));
  w.all = w.tile == 0 && w.count == w.tiles;
  return w;
}
template <int kKeys>
__device__ __forceinline__ void wide_next(const TreeArgs& a, int per, WideWalk& w) {
  w.left -= w.count;
  if (w.left <= 0) return;
  w.tile = 0;
  if (++w.hr == per) {
    w.hr = 0;
    ++w.b;
    w.tiles = tree_tiles<kKeys>(a, w.b);
  }
  w.count = static_cast<int>(min(static_cast<int64_t>(w.tiles), w.left));
  w.all = w.count == w.tiles;
}

__device__ __forceinline__ float2 mul2(float2 x, float2 y) { return __fmul2_rn(x, y); }

// Query row `row` into shared memory at lane row r (K-major, SW128, blocks of
// 64 head dimensions), scaled to fp16; returns what undoes that, times the
// softmax scale.
template <typename T, int D>
__device__ __forceinline__ float wide_query_row(const TreeArgs& a, uint8_t* to, int b, int kv, int row, int r,
                                                bool store) {
  uint4 raw[D / 8];
  if (row < a.rows) {
    const T* p = static_cast<const T*>(a.query) + b * a.qs[0] + (kv * a.group + row / a.nodes) * a.qs[1] +
                 (row % a.nodes) * a.qs[2];
    if (a.vec) {
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint2 lo = __ldg(reinterpret_cast<const uint2*>(p) + 2 * c);
        const uint2 hi = __ldg(reinterpret_cast<const uint2*>(p) + 2 * c + 1);
        raw[c] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    } else {
#pragma unroll
      for (int c = 0; c < D / 8; ++c) raw[c] = load_raw8<T, false>(p + c * 8);
    }
  } else {
#pragma unroll
    for (int c = 0; c < D / 8; ++c) raw[c] = make_uint4(0u, 0u, 0u, 0u);
  }
  float up = 1.0f, factor = a.scale_log2e;
  if constexpr (!std::is_same<T, __half>::value) {
    uint32_t top = 0u;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      float x[8];
      unpack8<T>(raw[c], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    const uint32_t e = max(1u, min(253u, top >> 23));
    up = __uint_as_float((254u - e) << 23);
    factor = __uint_as_float(e << 23) * a.scale_log2e;
  }
  if (store) {
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      float x[8];
      unpack8<T>(raw[c], x);
      uint4 w;
      w.x = pack2(x[0] * up, x[1] * up, __half());
      w.y = pack2(x[2] * up, x[3] * up, __half());
      w.z = pack2(x[4] * up, x[5] * up, __half());
      w.w = pack2(x[6] * up, x[7] * up, __half());
      *reinterpret_cast<uint4*>(to + (c / 8) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = w;
    }
  }
  return factor;
}

// The keys of a tile that a row sees, 32 to a word.
__device__ __forceinline__ void wide_seen(uint32_t (&seen)[4], uint32_t goods, int box_shift, int open, uint64_t word) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int n = open - 32 * c;  // committed keys from this word's first on
    uint32_t bits = n >= 32 ? ~0u : n > 0 ? (1u << n) - 1u : 0u;
    if (n >= 0) {
      if (n < 32) bits |= static_cast<uint32_t>(word << n);
    } else if (n > -64) {
      bits |= static_cast<uint32_t>(word >> -n);
    }
    uint32_t there = 0u;
    if (box_shift >= 5) {
      there = (goods >> ((32 * c) >> box_shift)) & 1u ? ~0u : 0u;
    } else {
      there = ((goods >> (2 * c)) & 1u ? 0xffffu : 0u) | ((goods >> (2 * c + 1)) & 1u ? 0xffff0000u : 0u);
    }
    seen[c] = bits & there;
  }
}

template <typename T, int D, bool kShared>
__global__ void __launch_bounds__(kWideThreads, 1)
    tree_wide_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                     TreeArgs a) {
  using S = WideTile<D, kShared>;
  constexpr int kRing = S::kRing;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  __shared__ __align__(8) uint64_t ring_full[kRing], ring_empty[kRing], scale_full[S::kScaleRing],
      scale_empty[S::kScaleRing], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2],
      q_full[2], mma_done;
  __shared__ uint32_t valid[S::kScaleRing];
  __shared__ uint32_t abort_word, tmem_slot;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t abort_flag = smem_u32(&abort_word);
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(smem_u32(&ring_full[i]), 1);
      mbar_init(smem_u32(&ring_empty[i]), 4);
    }
    for (int i = 0; i < S::kScaleRing; ++i) {
      mbar_init(smem_u32(&scale_full[i]), 1);
      mbar_init(smem_u32(&scale_empty[i]), kShared ? 8 : 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&k_full[i]), 4);
      mbar_init(smem_u32(&k_empty[i]), 1);
      mbar_init(smem_u32(&v_full[i]), 4);
      mbar_init(smem_u32(&v_empty[i]), 1);
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&p_full[i]), 4);
      mbar_init(smem_u32(&o_done[i]), 1);
      mbar_init(smem_u32(&q_full[i]), 4);
    }
    mbar_init(smem_u32(&mma_done), 1);
    abort_word = 0u;
    fence_mbarrier_init();
  }
  if (warp == 14) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;
  const uint64_t budget = a.wait_budget_ns;
  const int per = a.c.kv_heads * a.row_tiles;
  const TreeRun run = tree_run<S::kKeys>(a);
  WideWalk w = wide_begin<S::kKeys>(run);
  const int box = min(a.c.page_size, 64);
  const int box_shift = min(a.page_shift, 6);
  const int boxes = S::kKeys >> box_shift;

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWideRegsSoftmax));
    const int x = warp / 4;
    const int r = tid % 128;
    const uint32_t lane_base = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t tm_s = tmem_base + lane_base + x * 128;
    const uint32_t tm_o = tmem_base + lane_base + 256 + x * 128;
    float* state = reinterpret_cast<float*>(smem + S::kOffState);
    bool ok = true;
    uint32_t jobs = 0;      // of this stream so far
    uint32_t done = 0;      // segments of this stream that had a job
    int64_t counter = 0;    // key tiles of the run so far
    int part = 0;
    while (w.left > 0) {
      const int kv = w.hr / a.row_tiles;
      const int row = (w.hr % a.row_tiles) * S::kRows + (kShared ? x * 128 : 0) + r;
      const int64_t length = max(0, __ldg(a.c.lengths + w.b));
      uint64_t word = 0;
      if (row < a.rows) {
        const int node = row % a.nodes;
        word = a.mask != nullptr ? static_cast<uint64_t>(__ldg(reinterpret_cast<const unsigned long long*>(
                                       a.mask + w.b * a.mask_stride + node)))
                                 : ~0ull >> (63 - node);
        word &= ~0ull >> (64 - a.nodes);
      }
      const float factor = wide_query_row<T, D>(a, smem + S::kOffQuery + (kShared ? x * S::kHalf : 0), w.b, kv, row, r,
                                                kShared || x == 0);
      if (kShared || x == 0) {
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&q_full[kShared ? x : 0]));
      }
      float m = -INFINITY, l = 0.0f, unit = 0.0f, inv = 0.0f;
      bool first_job = true;
      for (int j = kShared ? 0 : x; j < w.count; j += kShared ? 1 : 2) {
        const int64_t c = counter + j;
        const int entry = static_cast<int>(c % S::kScaleRing);
        if (ok) ok = mbar_wait_warp(smem_u32(&scale_full[entry]), static_cast<uint32_t>(c / S::kScaleRing) & 1, budget,
                                    a.status, kStatusTimeoutFull, abort_flag);
        if (ok) ok = mbar_wait_sleep_warp(smem_u32(&s_full[x]), jobs & 1, budget, a.status, kStatusTimeoutMma,
                                          abort_flag);
        ++jobs;
        if (!ok) continue;
        tc_fence_after();
        const uint32_t scales = sbase + S::kOffScales + entry * S::kKeys * 8;
        float2 y[64];
        {
          uint32_t t0[32], t1[32], t2[32], t3[32];
          tmem_ld32(tm_s, t0);
          tmem_ld32(tm_s + 32, t1);
          tmem_ld32(tm_s + 64, t2);
          tmem_ld32(tm_s + 96, t3);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            y[i] = make_float2(__uint_as_float(t0[2 * i]), __uint_as_float(t0[2 * i + 1]));
            y[16 + i] = make_float2(__uint_as_float(t1[2 * i]), __uint_as_float(t1[2 * i + 1]));
            y[32 + i] = make_float2(__uint_as_float(t2[2 * i]), __uint_as_float(t2[2 * i + 1]));
            y[48 + i] = make_float2(__uint_as_float(t3[2 * i]), __uint_as_float(t3[2 * i + 1]));
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float4 ks = lds128(scales + 16 * i);
          y[2 * i] = mul2(y[2 * i], make_float2(ks.x, ks.y));
          y[2 * i + 1] = mul2(y[2 * i + 1], make_float2(ks.z, ks.w));
        }
        const int64_t first = static_cast<int64_t>(w.tile + j) * S::kKeys;
        const uint32_t goods = valid[entry];
        const bool masked = first + S::kKeys > length || goods != (1u << boxes) - 1u;
        uint32_t seen[4];
        if (masked) {
          wide_seen(seen, goods, box_shift, static_cast<int>(max(min(length - first, int64_t(256)), int64_t(-256))),
                    word);
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            if (!((seen[i / 16] >> (2 * (i % 16))) & 1u)) y[i].x = -INFINITY;
            if (!((seen[i / 16] >> (2 * (i % 16) + 1)) & 1u)) y[i].y = -INFINITY;
          }
        }
        float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          top0 = fmax3(top0, y[i].x, y[i].y);
          top1 = fmax3(top1, y[i + 1].x, y[i + 1].y);
        }
        const float top = fmaxf(top0, top1);
        if ((top - m) * factor > kSlack) {
          const float shrink = ex2_approx((m - top) * factor);
          m = top;
          l *= shrink;
          unit *= shrink;
          inv = unit >= kUnitMin ? 1.0f / unit : 0.0f;
        }
        const float shift = m == -INFINITY ? 0.0f : -m * factor;
        const float2 f2 = make_float2(factor, factor), s2 = make_float2(shift, shift);
        float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
        float most0 = 0.0f, most1 = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float4 vs = lds128(scales + S::kKeys * 4 + 16 * i);
          float2 p = __ffma2_rn(y[2 * i], f2, s2);
          p.x = ex2_approx(p.x);
          p.y = ex2_approx(p.y);
          sum0 = __fadd2_rn(sum0, p);
          y[2 * i] = mul2(p, make_float2(vs.x, vs.y));
          float2 q = __ffma2_rn(y[2 * i + 1], f2, s2);
          q.x = ex2_approx(q.x);
          q.y = ex2_approx(q.y);
          sum1 = __fadd2_rn(sum1, q);
          y[2 * i + 1] = mul2(q, make_float2(vs.z, vs.w));
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            if (!((seen[i / 16] >> (2 * (i % 16))) & 1u)) y[i].x = 0.0f;
            if (!((seen[i / 16] >> (2 * (i % 16) + 1)) & 1u)) y[i].y = 0.0f;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&scale_empty[entry]));
        l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          most0 = fmax3(most0, y[i].x, y[i].y);
          most1 = fmax3(most1, y[i + 1].x, y[i + 1].y);
        }
        const float most = fmaxf(most0, most1);
        const bool over = most > unit * 256.0f;
        if (__any_sync(0xffffffffu, over)) {
          const float shrink = over ? unit / most : 1.0f;
          if (over) {
            unit = most;
            inv = most >= kUnitMin ? 1.0f / most : 0.0f;
          }
          // The stream's last numerator MMAs are complete: the scores of this
          // tile were committed after them.
          if (!first_job) {
            const float2 k2 = make_float2(shrink, shrink);
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
              uint32_t v[16];
              tmem_ld8(tm_o + d, v);
              tmem_ld8(tm_o + d + 8, v + 8);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 z = mul2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), k2);
                v[2 * i] = __float_as_uint(z.x);
                v[2 * i + 1] = __float_as_uint(z.y);
              }
              tmem_st8(tm_o + d, v);
              tmem_st8(tm_o + d + 8, v + 8);
            }
          }
        }
        first_job = false;
        const float2 i2 = make_float2(inv, inv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 z = mul2(y[8 * i + e], i2);
            h[e] = pack2(z.x, z.y, __half());
          }
          tmem_st8(tm_s + 8 * i, h);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[x]));
      }
      counter += w.count;
      // ---- the segment's end
      const bool mine = kShared || x < w.count;  // this stream had a job
      if (mine) {
        if (ok) ok = mbar_wait_sleep_warp(smem_u32(&o_done[x]), done & 1, budget, a.status, kStatusTimeoutMma,
                                          abort_flag);
        ++done;
        tc_fence_after();
      }
      m *= factor;
      float m1 = -INFINITY, l1 = 0.0f, unit1 = 0.0f;
      if constexpr (!kShared) {
        if (x == 1) {
          state[r] = mine ? m : -INFINITY;
          state[128 + r] = mine ? l : 0.0f;
          state[256 + r] = mine ? unit : 0.0f;
          tc_fence_before();
        }
        bar_sync(1, 256);
        if (x == 0) {
          tc_fence_after();
          m1 = state[r];
          l1 = state[128 + r];
          unit1 = state[256 + r];
        }
      }
      if (kShared || x == 0) {
        const bool two = !kShared && w.count > 1;
        const float whole_m = fmaxf(m, m1);
        const float ref = whole_m == -INFINITY ? 0.0f : whole_m;
        const float g0 = ex2_approx(m - ref), g1 = two ? ex2_approx(m1 - ref) : 0.0f;
        const float whole_l = l * g0 + l1 * g1;
        const float inv_l = whole_l == 0.0f ? 0.0f : 1.0f / whole_l;
        const float f0 = unit * g0 * (w.all ? inv_l : 1.0f), f1 = unit1 * g1 * (w.all ? inv_l : 1.0f);
        const int lr = (kShared ? x * 128 : 0) + r;  // row of the row tile
        float* to = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + part) * S::kPart;
        T* out = static_cast<T*>(a.out) +
                 ((static_cast<int64_t>(w.b) * a.heads + kv * a.group + row / a.nodes) * a.nodes + row % a.nodes) * D;
        if (!w.all && row < a.rows) {
          to[S::kRows * D + 2 * lr] = whole_m;
          to[S::kRows * D + 2 * lr + 1] = whole_l;
        }
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          uint32_t v[32], u[32];
          tmem_ld32(tm_o + d, v);
          if (two) tmem_ld32(tm_o + 128 + d, u);
          tmem_ld_wait();
          float z[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            z[i] = __uint_as_float(v[i]) * f0;
            if (two) z[i] += __uint_as_float(u[i]) * f1;
          }
          if (!ok || row >= a.rows) continue;
          if (w.all) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint4 h;
              h.x = pack2(z[i], z[i + 1], T());
              h.y = pack2(z[i + 2], z[i + 3], T());
              h.z = pack2(z[i + 4], z[i + 5], T());
              h.w = pack2(z[i + 6], z[i + 7], T());
              *reinterpret_cast<uint4*>(out + d + i) = h;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(to + lr * D + d + i) = make_float4(z[i], z[i + 1], z[i + 2], z[i + 3]);
          }
        }
        tc_fence_before();
      }
      if constexpr (!kShared) bar_sync(1, 256);
      part = 1;
      wide_next<S::kKeys>(a, per, w);
    }
  } else if (warp < 12) {
    // --------------------------------------------------------- conversion
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideRegsConvert));
    const int r = tid % 128;
    bool ok = true;
    uint32_t uses[2] = {0, 0};
    int64_t op = 0;
    while (w.left > 0) {
      for (int j = 0; ok && j < w.count; ++j) {
        const int buffer = kShared ? 0 : (j & 1);
        const uint32_t use = uses[buffer]++;
#pragma unroll 1
        for (int side = 0; ok && side < 2; ++side, ++op) {
          const int slot = static_cast<int>(op % kRing);
          ok = mbar_wait_warp(smem_u32(&ring_full[slot]), static_cast<uint32_t>(op / kRing) & 1, budget, a.status,
                              kStatusTimeoutFull, abort_flag) &&
               mbar_wait_sleep_warp(smem_u32(side == 0 ? &k_empty[buffer] : &v_empty[buffer]), (use & 1) ^ 1, budget,
                                    a.status, kStatusTimeoutMma, abort_flag);
          if (!ok) break;
          const uint32_t from = sbase + S::kOffRing + slot * S::kCodes;
          uint8_t* to = smem + (side == 0 ? S::kOffK : S::kOffV) + buffer * S::kHalf + r * 128;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const float4 raw = lds128(tile_chunk<D>(from, r, c));
            const uint32_t code[4] = {__float_as_uint(raw.x) ^ 0x80808080u, __float_as_uint(raw.y) ^ 0x80808080u,
                                      __float_as_uint(raw.z) ^ 0x80808080u, __float_as_uint(raw.w) ^ 0x80808080u};
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              h[2 * i] = codes_f16<0x4140>(code[i]);
              h[2 * i + 1] = codes_f16<0x4342>(code[i]);
            }
            uint8_t* block = to + (c / 4) * 16384;
            *reinterpret_cast<uint4*>(block + ((((c & 3) * 2) ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(block + ((((c & 3) * 2 + 1) ^ (r & 7)) << 4)) =
                make_uint4(h[4], h[5], h[6], h[7]);
          }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(smem_u32(&ring_empty[slot]));
            mbar_arrive(smem_u32(side == 0 ? &k_full[buffer] : &v_full[buffer]));
          }
        }
      }
      wide_next<S::kKeys>(a, per, w);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideRegsControl));
    if (warp == 12) {
      // ----------------------------------------------- fetching, a box a lane
      bool ok = true;
      int64_t op = 0, counter = 0;
      while (w.left > 0 && ok) {
        const int32_t* table = a.c.block_table + w.b * a.c.table_stride;
        const int head = w.hr / a.row_tiles;
        int have = -1, entry = -1;
        for (int j = 0; ok && j < w.count; ++j, ++counter) {
          const int64_t tile0 = static_cast<int64_t>(w.tile + j) * S::kKeys;
          const int64_t position = tile0 + static_cast<int64_t>(lane) * box;
          const int column = static_cast<int>(position >> a.page_shift);
          const int column0 = static_cast<int>(tile0 >> a.page_shift);
          const int column1 = static_cast<int>((tile0 + S::kKeys - 1) >> a.page_shift);
          if (have < 0 || column1 >= have + 32) {
            have = column0;
            entry = have + lane < a.c.table_width ? __ldg(table + have + lane) : -1;
          }
          const int page = __shfl_sync(0xffffffffu, entry, (column - have) & 31);
          const bool good = lane < boxes && column < a.c.table_width && page >= 0 && page < a.c.pages;
          const uint32_t goods = __ballot_sync(0xffffffffu, good);
          const int z = page * a.c.kv_heads + head;
          const int y = static_cast<int>(position & (a.c.page_size - 1));
          const int64_t at = (static_cast<int64_t>(z) << a.page_shift) + y;
          const int ring = static_cast<int>(counter % S::kScaleRing);
          ok = mbar_wait_sleep_warp(smem_u32(&scale_empty[ring]),
                                    (static_cast<uint32_t>(counter / S::kScaleRing) & 1) ^ 1, budget, a.status,
                                    kStatusTimeoutEmpty, abort_flag);
          if (!ok) break;
          if (lane == 0) {
            valid[ring] = goods;
            mbar_arrive_expect_tx(smem_u32(&scale_full[ring]), __popc(goods) * box * 8);
          }
          __syncwarp();
          if (good) {
            const uint32_t to = sbase + S::kOffScales + ring * S::kKeys * 8 + lane * box * 4;
            bulk_load(to, a.c.key_scales + at, box * 4, smem_u32(&scale_full[ring]));
            bulk_load(to + S::kKeys * 4, a.c.value_scales + at, box * 4, smem_u32(&scale_full[ring]));
          }
#pragma unroll 1
          for (int side = 0; ok && side < 2; ++side, ++op) {
            const int slot = static_cast<int>(op % kRing);
            const uint32_t bar = smem_u32(&ring_full[slot]);
            ok = mbar_wait_sleep_warp(smem_u32(&ring_empty[slot]), (static_cast<uint32_t>(op / kRing) & 1) ^ 1, budget,
                                      a.status, kStatusTimeoutEmpty, abort_flag);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(bar, __popc(goods) * box * D);
            __syncwarp();
            if (good)
              tma_load_3d(sbase + S::kOffRing + slot * S::kCodes + lane * box * D, side == 0 ? &key_map : &value_map,
                          bar, 0, y, z);
          }
        }
        wide_next<S::kKeys>(a, per, w);
      }
      // Every copy has landed before the CTA's shared memory goes.
      for (int64_t i = max(int64_t(0), op - kRing); i < op; ++i)
        mbar_wait_warp(smem_u32(&ring_full[i % kRing]), static_cast<uint32_t>(i / kRing) & 1, budget, a.status,
                       kStatusTimeoutDrain, 0u);
      if (!ok)
        for (int64_t i = max(int64_t(0), counter - S::kScaleRing); i < counter; ++i)
          mbar_wait_warp(smem_u32(&scale_full[i % S::kScaleRing]), static_cast<uint32_t>(i / S::kScaleRing) & 1, budget,
                         a.status, kStatusTimeoutDrain, 0u);
    } else if (warp == 13 && lane == 0) {
      // -------------------------------------------------------- MMA issue
      constexpr uint32_t kIdescQK = umma_idesc_f16(128, S::kKeys);
      constexpr uint32_t kIdescPV = umma_idesc_f16(128, D) | (1u << 16);  // B with N contiguous
      const uint64_t desc_q = umma_desc_kmajor(sbase + S::kOffQuery, 128);
      const uint64_t desc_k = umma_desc_kmajor(sbase + S::kOffK, 128);
      const uint64_t desc_v = umma_desc_nmajor(sbase + S::kOffV, 16384u);
      bool ok = true;
      uint32_t k_use[2] = {0, 0}, v_use[2] = {0, 0}, p_use[2] = {0, 0};
      uint32_t segment = 0;
      // A job is one stream's tile; a segment's jobs alternate between the
      // streams.  Shared keys: jobs 2i and 2i + 1 use tile i.
      auto scores = [&](int job) {
        const int x = job & 1;
        const int buffer = kShared ? 0 : x;
        if (!kShared || x == 0) {
          ok = mbar_wait(smem_u32(&k_full[buffer]), k_use[buffer] & 1, budget, a.status, kStatusTimeoutFull,
                         abort_flag);
          ++k_use[buffer];
          if (!ok) return;
          tc_fence_after();
        }
        const uint64_t q = desc_q + static_cast<uint64_t>((kShared ? x * S::kHalf : 0) >> 4);
        const uint64_t k = desc_k + static_cast<uint64_t>((buffer * S::kHalf) >> 4);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint64_t step = (i / 4) * (16384u >> 4) + (i % 4) * 2;
          umma_f16(tmem_base + x * 128, q + step, k + step, kIdescQK, i > 0 ? 1u : 0u);
        }
        umma_commit(smem_u32(&s_full[x]));
        if (!kShared || x == 1) umma_commit(smem_u32(&k_empty[buffer]));
      };
      while (w.left > 0 && ok) {
        const int jobs = kShared ? 2 * w.count : w.count;
        for (int x = 0; ok && x < (kShared ? 2 : 1); ++x)
          ok = mbar_wait(smem_u32(&q_full[x]), segment & 1, budget, a.status, kStatusTimeoutFull, abort_flag);
        ++segment;
        if (!ok) break;
        tc_fence_after();
        for (int job = 0; ok && job < 2 && job < jobs; ++job) scores(job);
        for (int job = 0; ok && job < jobs; ++job) {
          const int x = job & 1;
          const int buffer = kShared ? 0 : x;
          if (!kShared || x == 0) {
            ok = mbar_wait(smem_u32(&v_full[buffer]), v_use[buffer] & 1, budget, a.status, kStatusTimeoutFull,
                           abort_flag);
            ++v_use[buffer];
            if (!ok) break;
          }
          ok = mbar_wait(smem_u32(&p_full[x]), p_use[x] & 1, budget, a.status, kStatusTimeoutFull, abort_flag);
          ++p_use[x];
          if (!ok) break;
          tc_fence_after();
          const uint64_t v = desc_v + static_cast<uint64_t>((buffer * S::kHalf) >> 4);
#pragma unroll
          for (int i = 0; i < S::kKeys / 16; ++i)
            umma_f16_ts(tmem_base + 256 + x * 128, tmem_base + x * 128 + 8 * i, v + i * (2048u >> 4), kIdescPV,
                        job >= 2 || i > 0 ? 1u : 0u);
          if (!kShared || x == 1) umma_commit(smem_u32(&v_empty[buffer]));
          if (job + 2 < jobs)
            scores(job + 2);
          else
            umma_commit(smem_u32(&o_done[x]));
        }
        wide_next<S::kKeys>(a, per, w);
      }
      // Everything issued completes before TMEM is freed.
      umma_commit(smem_u32(&mma_done));
      mbar_wait(smem_u32(&mma_done), 0, budget, a.status, kStatusTimeoutMma, 0u);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 14) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace piper

// Attention of many query rows of a KV head (wide trees, large groups) over
// the quantised paged cache, on tcgen05.
//
// The mathematics, the units and the parts are those of tree_attention.cuh;
// here a tile is 128 keys and a product is a 128-row tcgen05 MMA with fp32
// accumulators in TMEM:
//   S = Q K^T   Q (fp16, scaled by row) and K from shared memory
//   O += W V    W (fp16 weights) from TMEM, over the spent scores; V from
//               shared memory with the head dimension contiguous
// kind::f16 needs 16-bit operands, so warps turn each tile's codes into fp16
// between the TMA ring and the MMAs: 128 rows or more pay for one conversion.
//
// Two streams of 128 TMEM lanes hide each other's latency: while one stream's
// softmax runs, the other's MMAs do.  kShared: the streams are rows 0-127 and
// 128-255 of the row tile over the same keys (more than 128 rows).  Otherwise
// they are alternate key tiles of the same 128 rows, joined at the end.
//
// A softmax warp takes its 16 rows' scores 32 columns at a time.  A row has one
// reference, the unit of its numerators and of its total: 2^unit is 2^6 to 2^15.9
// times smaller than the row's largest weight times its value scale, so that small
// weights have room in fp16 (kWideRoom), and moves only when 32 columns could
// outgrow that; then what is there already, the tile's first weights among it, is
// scaled down.
//
// Warps: 0-7 and 8-15 softmax of streams 0 and 1 (two for each 32 TMEM lanes),
// 16-17 conversion of K, 18-19 of V, 20 fetches, 21 issues MMAs, 22 owns
// TMEM.
//
// Measured: 16 nodes of 40 over 8 heads of 128 and 131072 tokens (80 rows) 130
// us, 330 TFLOP/s; 16 requests of 4000 to 8191 tokens, 47 nodes, 32 over 8 heads
// (188 rows) 186 us, 408 TFLOP/s.  The time hardly depends on the rows up to 128
// (131072 tokens: 25 rows 119 us, 40 rows 122, 128 rows 138; in pairs 132 rows 196,
// 256 rows 216).  What bounds it is a stream's chain of scores, weights and
// numerators, some 8500 cycles a tile with two tiles under way (tensor pipe busy 24
// and 27 % of the time, issue slots 45 and 44), and in it the fullest of an SM's four
// sub-partitions: rows fill TMEM lanes, and with them the warps of sub-partitions,
// from 0 up, so that 80 rows give one 132000 instructions and another 44000 (188
// rows: 178000 and 86000).  Tried and slower: a
// thread a row with all 128 scores in registers (204 us; one long unrolled
// body), half tiles with both halves' scores in TMEM (191 us; twice the
// hand-overs, and QK^T of 64 keys reads Q twice).
#pragma once

#include "tree_attention.cuh"

namespace piper {

// 23 warps at 80 registers: what a softmax warp needs without spilling in its
// loop (more columns at a time, or a look ahead, spilled and measured slower).
constexpr int kWideThreads = 736;
// log2 of a row's largest weight when its reference has just moved (less up to 1).
// The smallest step of fp16 is then 2^-30 of it or less.  A move holds its stream
// up, and the less the weights may grow the more there are: 131 us at 6 and below,
// 133 at 7, 135 at 8, 140 at 10 for the first case measured above.
constexpr float kWideRoom = 7.0f;

template <int D, bool kShared>
struct WideTile {
  static constexpr int kRows = kShared ? 256 : 128;
  static constexpr int kKeys = 128;
  static constexpr int kCtas = 1;
  static constexpr int kLead = 4;
  static constexpr int kCodes = kKeys * D;          // one ring slot: K or V codes
  static constexpr int kHalf = kKeys * D * 2;       // one fp16 operand tile
  static constexpr int kQuery = (kShared ? 2 : 1) * kHalf;
  static constexpr int kBuffers = kShared ? 1 : 2;  // fp16 K tiles (one V tile: a V tile is needed later)
  static constexpr int kScaleRing = 4;
  static constexpr int kEntry = kKeys * 8;          // scales of keys and of values
  static constexpr int kOffQuery = 0;
  static constexpr int kOffK = kOffQuery + kQuery;
  static constexpr int kOffV = kOffK + kBuffers * kHalf;
  static constexpr int kOffScales = kOffV + kHalf;
  static constexpr int kOffState = kOffScales + kScaleRing * kEntry;
  static constexpr int kOffRing = (kOffState + 256 * (3 * 4 + 8) + 1023) / 1024 * 1024;
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

__device__ __forceinline__ float2 mul2(float2 x, float2 y) { return __fmul2_rn(x, y); }

// Sixteen query rows, from row r0 of the stream (row `row0` of the KV head),
// into shared memory (K-major, SW128, blocks of 64 head dimensions), scaled to
// fp16, and what undoes that, times the softmax scale, into `factors`.  A warp
// reads a row at a time, eight in flight.
template <typename T, int D>
__device__ __forceinline__ void wide_query_rows(const TreeArgs& a, uint8_t* to, float* factors, int b, int kv, int row0,
                                                int r0) {
  constexpr int kPer = D / 32;  // elements a lane
  const int lane = threadIdx.x % 32;
  const int mine = row0 + r0 + (lane & 15);
  int64_t at = -1;
  if (mine < a.rows)
    at = b * a.qs[0] + (kv * a.group + mine / a.nodes) * a.qs[1] + (mine % a.nodes) * a.qs[2];
  const uint16_t* base = static_cast<const uint16_t*>(a.query) + lane * kPer;
#pragma unroll 1
  for (int k0 = 0; k0 < 16; k0 += 8) {
    uint32_t raw[8][kPer / 2];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t row_at = __shfl_sync(0xffffffffu, at, k0 + k);
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) raw[k][i] = 0u;
      if (row_at >= 0) {
        const uint16_t* p = base + row_at;
        if (a.vec) {
          if constexpr (kPer == 4) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
            raw[k][0] = w.x;
            raw[k][1] = w.y;
          } else {
            raw[k][0] = __ldg(reinterpret_cast<const uint32_t*>(p));
          }
        } else {
#pragma unroll
          for (int i = 0; i < kPer / 2; ++i)
            raw[k][i] = static_cast<uint32_t>(p[2 * i]) | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = r0 + k0 + k;
      float x[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint16_t e = static_cast<uint16_t>(raw[k][i / 2] >> (16 * (i % 2)));
        x[i] = to_f32<T>(*reinterpret_cast<const T*>(&e));
      }
      float up = 1.0f, factor = a.scale_log2e;
      if constexpr (!std::is_same<T, __half>::value) {
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < kPer; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        top = __reduce_max_sync(0xffffffffu, top);
        const uint32_t e = max(1u, min(253u, top >> 23));
        up = __uint_as_float((254u - e) << 23);
        factor = __uint_as_float(e << 23) * a.scale_log2e;
      }
      if (lane == 0) factors[r] = factor;
      const int chunk = lane * kPer / 8;
      uint8_t* p = to + (chunk / 8) * 16384 + r * 128 + (((chunk & 7) ^ (r & 7)) << 4) + (lane * kPer % 8) * 2;
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i)
        reinterpret_cast<uint32_t*>(p)[i] = pack2(x[2 * i] * up, x[2 * i + 1] * up, __half());
    }
  }
}

// Which of keys 32 c .. 32 c + 31 of a tile a row sees: the first `open` of the
// tile are committed, those after it follow `word`.
__device__ __forceinline__ uint32_t wide_seen(uint32_t goods, int box_shift, int open, uint64_t word, int c) {
  const int n = open - 32 * c;
  uint32_t bits = n >= 32 ? ~0u : n > 0 ? (1u << n) - 1u : 0u;
  if (n >= 0) {
    if (n < 32) bits |= static_cast<uint32_t>(word << n);
  } else if (n > -64) {
    bits |= static_cast<uint32_t>(word >> -n);
  }
  const uint32_t there = box_shift >= 5 ? ((goods >> ((32 * c) >> box_shift)) & 1u ? ~0u : 0u)
                                        : ((goods >> (2 * c)) & 1u ? 0xffffu : 0u) |
                                              ((goods >> (2 * c + 1)) & 1u ? 0xffff0000u : 0u);
  return bits & there;
}

// Scores of keys that a row does not see, by the two lowest bits.
__device__ __forceinline__ void hide(float2& y, uint32_t seen) {
  if (!(seen & 1u)) y.x = -INFINITY;
  if (!(seen & 2u)) y.y = -INFINITY;
}

__device__ __forceinline__ float2 f2_of(uint32_t x, uint32_t y) {
  return make_float2(__uint_as_float(x), __uint_as_float(y));
}

// New references of a lane's two rows, and by how much they moved.
struct WideMove {
  float2 unit, shrink;
};

// Moves the references to kWideRoom below the largest logarithm of a weight times
// its value scale in chunk c of a tile (bit 8 n + e of seen0 and seen1: column 8 n + e
// after the lane's first is seen), and scales down the tile's weights so far
// and `numerators` columns at tm_o.  Not inlined: it is rare, and its registers
// would be the common path's spills.
template <typename S>
__device__ __noinline__ WideMove wide_move(uint32_t tm_s, uint32_t tm_o, uint32_t scales, int c, float2 factor,
                                           float2 unit, uint32_t seen0, uint32_t seen1, int numerators) {
  const int t = threadIdx.x % 4;
  float most[2] = {-INFINITY, -INFINITY};
  const float factors[2] = {factor.x, factor.y};
  float units[2] = {unit.x, unit.y}, shrink[2] = {1.0f, 1.0f};
  const uint32_t seen[2] = {seen0, seen1};
  uint32_t v[16];
  tmem_ld_16x256b_x4(tm_s + 32 * c, v);
  tmem_ld_wait();
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float2 ks = lds64(scales + 128 * c + 32 * n + 8 * t);
    const float2 vs = lds64(scales + S::kKeys * 4 + 128 * c + 32 * n + 8 * t);
    const float lx = fmaxf(lg2_approx(fabsf(vs.x)), kScaleLogMin), ly = fmaxf(lg2_approx(fabsf(vs.y)), kScaleLogMin);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float zx = fmaf(__uint_as_float(v[4 * n + 2 * h]) * ks.x, factors[h], lx);
      const float zy = fmaf(__uint_as_float(v[4 * n + 2 * h + 1]) * ks.y, factors[h], ly);
      if ((seen[h] >> (8 * n)) & 1u) most[h] = fmaxf(most[h], zx);
      if ((seen[h] >> (8 * n + 1)) & 1u) most[h] = fmaxf(most[h], zy);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
    most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 2));
    const float to = most[h] - kWideRoom;
    if (to > units[h]) {
      // By whole powers of two: the weights that are in TMEM already stay exact.
      const float up = units[h] == kNoReference ? to : units[h] + ceilf(to - units[h]);
      shrink[h] = ex2_approx(units[h] - up);
      units[h] = up;
    }
  }
  tmem_st_wait();
#pragma unroll 1
  for (int d = 0; d < c; ++d) {
    uint32_t u[8];
    tmem_ld_16x128b_x4(tm_s + 16 * d, u);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // In fp32: fp16 has no factor below 2^-24, which a weight of 2^15 outlives.
      const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      u[i] = pack2(z.x * shrink[i & 1], z.y * shrink[i & 1], __half());
    }
    tmem_st_16x128b_x4(tm_s + 16 * d, u);
  }
  // (The stream's last numerator MMAs are complete: the scores of this tile
  // were committed after them.)
#pragma unroll 1
  for (int d = 0; d < numerators; d += 16) {
    uint32_t u[8];
    tmem_ld_16x256b_x2(tm_o + d, u);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * shrink[(i / 2) & 1]);
    tmem_st_16x256b_x2(tm_o + d, u);
  }
  tmem_st_wait();
  return WideMove{make_float2(units[0], units[1]), make_float2(shrink[0], shrink[1])};
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
      scale_empty[S::kScaleRing], k_full[2], k_empty[2], v_full, v_empty, s_full[2], p_full[2], o_done[2],
      q_full[2], mma_done;
  __shared__ uint32_t valid[S::kScaleRing];
  __shared__ uint32_t abort_word, tmem_slot;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t abort_flag = smem_u32(&abort_word);
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(smem_u32(&ring_full[i]), 1);
      mbar_init(smem_u32(&ring_empty[i]), 2);
    }
    for (int i = 0; i < S::kScaleRing; ++i) {
      mbar_init(smem_u32(&scale_full[i]), 1);
      mbar_init(smem_u32(&scale_empty[i]), kShared ? 16 : 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&k_full[i]), 2);
      mbar_init(smem_u32(&k_empty[i]), 1);
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&p_full[i]), 8);
      mbar_init(smem_u32(&o_done[i]), 1);
      mbar_init(smem_u32(&q_full[i]), 8);
    }
    mbar_init(smem_u32(&v_full), 2);
    mbar_init(smem_u32(&v_empty), 1);
    mbar_init(smem_u32(&mma_done), 1);
    abort_word = 0u;
    fence_mbarrier_init();
  }
  if (warp == 22) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;
  const uint64_t budget = a.wait_budget_ns;
  TreeRun w = tree_run<S>(a);
  const int box = min(a.c.page_size, 64);
  const int box_shift = min(a.page_shift, 6);
  const int boxes = S::kKeys >> box_shift;

  if (warp < 16) {
    // ------------------------------------------------------------ softmax
    const int x = warp / 8;              // stream
    const int half = (warp / 4) & 1;     // of the 32 TMEM lanes that the warp reaches
    const int lane0 = (warp % 4) * 32;   // the first of them
    const int g = lane / 4, t = lane % 4;
    const int r16 = lane0 + half * 16 + g;  // a lane has rows r16 and r16 + 8 of the stream
    const uint32_t tm_s = tmem_base + (static_cast<uint32_t>(lane0 + half * 16) << 16) + x * 128;
    const uint32_t tm_o = tmem_base + (static_cast<uint32_t>(lane0 + half * 16) << 16) + 256 + x * 128;
    float* totals = reinterpret_cast<float*>(smem + S::kOffState);  // [stream][128]
    float* units = totals + 256;
    float* factors = units + 256;
    uint64_t* words = reinterpret_cast<uint64_t*>(factors + 256);  // visible nodes
    const int own = kShared ? x * 128 : 0;  // of factors and words: alternate streams share their rows
    const int bar_id = kShared ? 1 + x : 1;
    constexpr int kBarThreads = kShared ? 256 : 512;
    bool ok = true;
    uint32_t jobs = 0;      // of this stream so far
    uint32_t done = 0;      // segments of this stream that had a job
    uint32_t counter = 0;   // key tiles of the run so far
    int part = 0;
    for (; w.left > 0; tree_next<S>(a, w)) {
      if (w.count == 0) continue;
      const int kv = w.hr / a.row_tiles;
      const int row0 = (w.hr % a.row_tiles) * S::kRows + (kShared ? x * 128 : 0);
      const int full_tiles = max(0, __ldg(a.c.lengths + w.b)) / S::kKeys;  // without drafted keys
      if (kShared || x == 0) {
        if (half == 0) {
          const int row = row0 + lane0 + lane;
          uint64_t word = 0;
          if (row < a.rows) {
            const int node = row % a.nodes;
            word = a.mask != nullptr ? static_cast<uint64_t>(__ldg(reinterpret_cast<const unsigned long long*>(
                                           a.mask + w.b * a.mask_stride + node)))
                                     : ~0ull >> (63 - node);
            word &= ~0ull >> (64 - a.nodes);
          }
          words[own + lane0 + lane] = word;
        }
        wide_query_rows<T, D>(a, smem + S::kOffQuery + (kShared ? x * S::kHalf : 0), factors + own, w.b, kv, row0,
                              (warp % 8) * 16);
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&q_full[kShared ? x : 0]));
      }
      bar_sync(bar_id, kBarThreads);
      // A row's reference `unit`: the logarithm of the numerators' unit, and of
      // the total's.
      float factor[2], unit[2], l[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        factor[h] = factors[own + r16 + 8 * h];
        unit[h] = kNoReference;
        l[h] = 0.0f;
      }
      // Warps whose rows are all past the last only take part in the hand-over.
      const bool idle = row0 + lane0 + half * 16 >= a.rows;
      bool first_job = true;
      for (int j = kShared ? 0 : x; j < w.count; j += kShared ? 1 : 2) {
        const uint32_t c0 = counter + j;
        const int entry = static_cast<int>(c0 % S::kScaleRing);
        if (ok) ok = mbar_wait_block_warp(smem_u32(&scale_full[entry]), (c0 / S::kScaleRing) & 1, budget, a.status,
                                          kStatusTimeoutFull, abort_flag);
        if (ok) ok = mbar_wait_block_warp(smem_u32(&s_full[x]), jobs & 1, budget, a.status, kStatusTimeoutMma,
                                          abort_flag);
        ++jobs;
        if (!ok) continue;
        tc_fence_after();
        if (!idle) {
          const uint32_t scales = sbase + S::kOffScales + entry * S::kEntry;
          const uint32_t goods = valid[entry];
          const bool masked = w.tile + j >= full_tiles || goods != (1u << boxes) - 1u;
          // Bit 8 n + e: column 32 c + 8 n + 2 t + e of row h is seen.
          auto seen_of = [&](int c, int h) {
            const int64_t open = max(0, __ldg(a.c.lengths + w.b)) - static_cast<int64_t>(w.tile + j) * S::kKeys;
            return wide_seen(goods, box_shift, static_cast<int>(max(min(open, int64_t(256)), int64_t(-256))),
                             words[own + r16 + 8 * h], c) >> (2 * t);
          };
          // The largest value scale of the tile, as a logarithm.  (NaN: 0; floats
          // that are not negative order as their bits.)
          const float4 four = lds128(scales + S::kKeys * 4 + 16 * lane);
          float reach = fmaxf(fmaxf(fmaxf(fabsf(four.x), fabsf(four.y)), fmaxf(fabsf(four.z), fabsf(four.w))), 0.0f);
          reach = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(reach)));
          const float reach_log = fmaxf(lg2_approx(reach), kScaleLogMin);
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
          // (A masked tile has a body of its own: branches inside would cut
          // the other's instructions into short chains.)
          auto weigh = [&](auto hidden) {
            bool moved = false;  // the references have, for this chunk
#pragma unroll 1
            for (int c = 0; c < 4;) {
              uint32_t v[16];
              tmem_ld_16x256b_x4(tm_s + 32 * c, v);
              float2 ks[4], vs[4];
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                ks[n] = lds64(scales + 128 * c + 32 * n + 8 * t);
                vs[n] = lds64(scales + S::kKeys * 4 + 128 * c + 32 * n + 8 * t);
              }
              tmem_ld_wait();
              uint32_t seen[2] = {~0u, ~0u};
              if constexpr (hidden.value) {
                seen[0] = seen_of(c, 0);
                seen[1] = seen_of(c, 1);
              }
              float2 y[4][2];
              float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
              for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  y[n][h] = mul2(f2_of(v[4 * n + 2 * h], v[4 * n + 2 * h + 1]), ks[n]);
                  if constexpr (hidden.value) hide(y[n][h], seen[h] >> (8 * n));
                  top[h] = fmax3(top[h], y[n][h].x, y[n][h].y);
                }
              // A weight times its value scale is at most 2^(top + reach_log - unit).
              if (!moved && __any_sync(0xffffffffu, fmaf(top[0], factor[0], reach_log - unit[0]) > kSlack ||
                                                        fmaf(top[1], factor[1], reach_log - unit[1]) > kSlack)) {
                const WideMove m = wide_move<S>(tm_s, tm_o, scales, c, make_float2(factor[0], factor[1]),
                                                make_float2(unit[0], unit[1]), seen[0], seen[1], first_job ? 0 : D);
                unit[0] = m.unit.x;
                unit[1] = m.unit.y;
                l[0] *= m.shrink.x;
                l[1] *= m.shrink.y;
                sum[0] = mul2(sum[0], make_float2(m.shrink.x, m.shrink.x));
                sum[1] = mul2(sum[1], make_float2(m.shrink.y, m.shrink.y));
                moved = true;  // and take the chunk again
                continue;
              }
              uint32_t p16[8];
#pragma unroll
              for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  float2 p = __ffma2_rn(y[n][h], make_float2(factor[h], factor[h]), make_float2(-unit[h], -unit[h]));
                  p.x = ex2_approx(p.x);
                  p.y = ex2_approx(p.y);
                  if constexpr (hidden.value) {  // (-infinity times a factor that underflowed is no number)
                    if (!((seen[h] >> (8 * n)) & 1u)) p.x = 0.0f;
                    if (!((seen[h] >> (8 * n + 1)) & 1u)) p.y = 0.0f;
                  }
                  sum[h] = __fadd2_rn(sum[h], p);
                  p = mul2(p, vs[n]);
                  uint32_t x16 = pack2(p.x, p.y, __half());
                  if constexpr (hidden.value)  // an unseen key's value scale may be anything
                    x16 &= ((seen[h] >> (8 * n)) & 1u ? 0xffffu : 0u) |
                           ((seen[h] >> (8 * n + 1)) & 1u ? 0xffff0000u : 0u);
                  p16[2 * n + h] = x16;
                }
              // Over spent scores: columns 16 c .. of chunk c / 2.
              tmem_st_16x128b_x4(tm_s + 16 * c, p16);
              moved = false;
              ++c;
            }
          };
          if (masked)
            weigh(std::true_type());
          else
            weigh(std::false_type());
#pragma unroll
          for (int h = 0; h < 2; ++h) l[h] += sum[h].x + sum[h].y;
          tmem_st_wait();
        }
        first_job = false;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&scale_empty[entry]));
          mbar_arrive(smem_u32(&p_full[x]));
        }
      }
      counter += w.count;
      // ---- the segment's end
      const bool mine = kShared || x < w.count;  // this stream had a job
      if (mine) {
        if (ok) ok = mbar_wait_block_warp(smem_u32(&o_done[x]), done & 1, budget, a.status, kStatusTimeoutMma,
                                          abort_flag);
        ++done;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (t == 0) {
          totals[x * 128 + r16 + 8 * h] = l[h];
          units[x * 128 + r16 + 8 * h] = unit[h] == kNoReference ? -INFINITY : unit[h];
        }
      }
      tc_fence_before();
      bar_sync(bar_id, kBarThreads);
      tc_fence_after();
      {
        // A thread writes its share of the head dimensions of one row.  The
        // warps that reach the row's lane: two, or four with both streams'.
        constexpr int kShare = D / (kShared ? 2 : 4);
        const int share = kShared ? half : 2 * x + half;
        const int s0 = kShared ? x : 0;  // the stream, or the first of two
        const bool two = !kShared && w.count > 1;
        const int r = lane0 + lane, row = row0 + r;
        const float unit0 = units[s0 * 128 + r], unit1 = two ? units[128 + r] : -INFINITY;
        const float whole_m = fmaxf(unit0, unit1);
        const float ref = whole_m == -INFINITY ? 0.0f : whole_m;
        const float g0 = ex2_approx(unit0 - ref), g1 = two ? ex2_approx(unit1 - ref) : 0.0f;
        const float whole_l = totals[s0 * 128 + r] * g0 + (two ? totals[128 + r] * g1 : 0.0f);
        const float over_l = !w.all ? 1.0f : whole_l == 0.0f ? 0.0f : 1.0f / whole_l;
        const float f0 = g0 * over_l, f1 = g1 * over_l;
        const int lr = s0 * 128 + r;  // row of the row tile
        const uint32_t from = tmem_base + (static_cast<uint32_t>(lane0) << 16) + 256 + s0 * 128;
        float* to = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + part) * S::kPart;
        if (!w.all && ok && share == 0 && row < a.rows) {
          to[S::kRows * D + 2 * lr] = whole_m;
          to[S::kRows * D + 2 * lr + 1] = whole_l;
        }
#pragma unroll 1
        for (int d = share * kShare; d < (share + 1) * kShare; d += 8) {
          uint32_t u0[8], u1[8];
          tmem_ld8(from + d, u0);
          if (two) tmem_ld8(from + 128 + d, u1);
          tmem_ld_wait();
          float z[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            z[i] = __uint_as_float(u0[i]) * f0;
            if (two) z[i] += __uint_as_float(u1[i]) * f1;
          }
          if (!ok || row >= a.rows) continue;
          if (w.all) {
            T* out = static_cast<T*>(a.out) + ((static_cast<int64_t>(w.b) * a.heads + kv * a.group + row / a.nodes) *
                                                   a.nodes + row % a.nodes) * D + d;
            uint4 h;
            h.x = pack2(z[0], z[1], T());
            h.y = pack2(z[2], z[3], T());
            h.z = pack2(z[4], z[5], T());
            h.w = pack2(z[6], z[7], T());
            *reinterpret_cast<uint4*>(out) = h;
          } else {
            *reinterpret_cast<float4*>(to + lr * D + d) = make_float4(z[0], z[1], z[2], z[3]);
            *reinterpret_cast<float4*>(to + lr * D + d + 4) = make_float4(z[4], z[5], z[6], z[7]);
          }
        }
        tc_fence_before();
      }
      // The numerators have been read, before any warp hands over the next
      // segment's first weights.
      if constexpr (!kShared) bar_sync(bar_id, kBarThreads);
      part = 1;
    }
  } else if (warp < 20) {
    // --------------------------------------------------------- conversion
    // Two warps turn K tiles, two V tiles: a V tile waits for the numerators
    // before it, which must not hold up the next K tile.
    const int side = (warp - 16) / 2;
    const int r = tid % 64;
    bool ok = true;
    uint32_t uses[2] = {0, 0};
    uint32_t op = side;
    while (w.left > 0) {
      for (int j = 0; ok && j < w.count; ++j, op += 2) {
        const int buffer = kShared || side == 1 ? 0 : (j & 1);
        const uint32_t use = uses[buffer]++;
        const uint32_t slot = op % kRing;
        ok = mbar_wait_block_warp(smem_u32(&ring_full[slot]), (op / kRing) & 1, budget, a.status, kStatusTimeoutFull,
                                  abort_flag) &&
             mbar_wait_block_warp(smem_u32(side == 0 ? &k_empty[buffer] : &v_empty), (use & 1) ^ 1, budget,
                                  a.status, kStatusTimeoutMma, abort_flag);
        if (!ok) break;
        const uint32_t from = sbase + S::kOffRing + slot * S::kCodes;
        uint8_t* to = smem + (side == 0 ? S::kOffK : S::kOffV) + buffer * S::kHalf;
#pragma unroll 1
        for (int row = r; row < S::kKeys; row += 64) {
          float4 raw[D / 16];
#pragma unroll
          for (int c = 0; c < D / 16; ++c) raw[c] = lds128(tile_chunk<D>(from, row, c));
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const uint32_t code[4] = {__float_as_uint(raw[c].x) ^ 0x80808080u, __float_as_uint(raw[c].y) ^ 0x80808080u,
                                      __float_as_uint(raw[c].z) ^ 0x80808080u, __float_as_uint(raw[c].w) ^ 0x80808080u};
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              h[2 * i] = codes_f16<0x4140>(code[i]);
              h[2 * i + 1] = codes_f16<0x4342>(code[i]);
            }
            uint8_t* block = to + row * 128 + (c / 4) * 16384;
            *reinterpret_cast<uint4*>(block + ((((c & 3) * 2) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(block + ((((c & 3) * 2 + 1) ^ (row & 7)) << 4)) =
                make_uint4(h[4], h[5], h[6], h[7]);
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&ring_empty[slot]));
          mbar_arrive(smem_u32(side == 0 ? &k_full[buffer] : &v_full));
        }
      }
      tree_next<S>(a, w);
    }
  } else {
    if (warp == 20) {
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
          ok = mbar_wait_block_warp(smem_u32(&scale_empty[ring]),
                                    (static_cast<uint32_t>(counter / S::kScaleRing) & 1) ^ 1, budget, a.status,
                                    kStatusTimeoutEmpty, abort_flag);
          if (!ok) break;
          if (lane == 0) {
            valid[ring] = goods;
            mbar_arrive_expect_tx(smem_u32(&scale_full[ring]), __popc(goods) * box * 8);
          }
          __syncwarp();
          if (good) {
            const uint32_t to = sbase + S::kOffScales + ring * S::kEntry + lane * box * 4;
            bulk_load(to, a.c.key_scales + at, box * 4, smem_u32(&scale_full[ring]));
            bulk_load(to + S::kKeys * 4, a.c.value_scales + at, box * 4, smem_u32(&scale_full[ring]));
          }
#pragma unroll 1
          for (int side = 0; ok && side < 2; ++side, ++op) {
            const int slot = static_cast<int>(op % kRing);
            const uint32_t bar = smem_u32(&ring_full[slot]);
            ok = mbar_wait_block_warp(smem_u32(&ring_empty[slot]), (static_cast<uint32_t>(op / kRing) & 1) ^ 1, budget,
                                      a.status, kStatusTimeoutEmpty, abort_flag);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(bar, __popc(goods) * box * D);
            __syncwarp();
            if (good)
              tma_load_3d(sbase + S::kOffRing + slot * S::kCodes + lane * box * D, side == 0 ? &key_map : &value_map,
                          bar, 0, y, z);
          }
        }
        tree_next<S>(a, w);
      }
      // Every copy has landed before the CTA's shared memory goes.
      for (int64_t i = max(int64_t(0), op - kRing); i < op; ++i)
        mbar_wait_block_warp(smem_u32(&ring_full[i % kRing]), static_cast<uint32_t>(i / kRing) & 1, budget, a.status,
                       kStatusTimeoutDrain, 0u);
      if (!ok)
        for (int64_t i = max(int64_t(0), counter - S::kScaleRing); i < counter; ++i)
          mbar_wait_block_warp(smem_u32(&scale_full[i % S::kScaleRing]), static_cast<uint32_t>(i / S::kScaleRing) & 1, budget,
                         a.status, kStatusTimeoutDrain, 0u);
    } else if (warp == 21 && lane == 0) {
      // -------------------------------------------------------- MMA issue
      constexpr uint32_t kIdescQK = umma_idesc_f16(128, S::kKeys);
      constexpr uint32_t kIdescPV = umma_idesc_f16(128, D) | (1u << 16);  // B with N contiguous
      const uint64_t desc_q = umma_desc_kmajor(sbase + S::kOffQuery, 128);
      const uint64_t desc_k = umma_desc_kmajor(sbase + S::kOffK, 128);
      const uint64_t desc_v = umma_desc_nmajor(sbase + S::kOffV, 16384u);
      bool ok = true;
      uint32_t k_use[2] = {0, 0}, v_use = 0, p_use[2] = {0, 0};
      uint32_t segment = 0;
      // A job is one stream's tile; a segment's jobs alternate between the
      // streams.  Shared keys: jobs 2i and 2i + 1 use tile i.
      auto scores = [&](int job) {
        const int x = job & 1;
        const int buffer = kShared ? 0 : x;
        if (!kShared || x == 0) {
          ok = mbar_wait_block(smem_u32(&k_full[buffer]), k_use[buffer] & 1, budget, a.status, kStatusTimeoutFull,
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
      for (; w.left > 0 && ok; tree_next<S>(a, w)) {
        if (w.count == 0) continue;
        const int jobs = kShared ? 2 * w.count : w.count;
        for (int x = 0; ok && x < (kShared ? 2 : 1); ++x)
          ok = mbar_wait_block(smem_u32(&q_full[x]), segment & 1, budget, a.status, kStatusTimeoutFull, abort_flag);
        ++segment;
        if (!ok) break;
        tc_fence_after();
        for (int job = 0; ok && job < 2 && job < jobs; ++job) scores(job);
        for (int job = 0; ok && job < jobs; ++job) {
          const int x = job & 1;
          if (!kShared || x == 0) {
            ok = mbar_wait_block(smem_u32(&v_full), v_use & 1, budget, a.status, kStatusTimeoutFull, abort_flag);
            ++v_use;
            if (!ok) break;
          }
          ok = mbar_wait_block(smem_u32(&p_full[x]), p_use[x] & 1, budget, a.status, kStatusTimeoutFull, abort_flag);
          ++p_use[x];
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < S::kKeys / 16; ++i)
            umma_f16_ts(tmem_base + 256 + x * 128, tmem_base + x * 128 + 8 * i, desc_v + i * (2048u >> 4), kIdescPV,
                        job >= 2 || i > 0 ? 1u : 0u);
          if (!kShared || x == 1) umma_commit(smem_u32(&v_empty));
          if (job + 2 < jobs)
            scores(job + 2);
          else
            umma_commit(smem_u32(&o_done[x]));
        }
      }
      // Everything issued completes before TMEM is freed.
      umma_commit(smem_u32(&mma_done));
      mbar_wait(smem_u32(&mma_done), 0, budget, a.status, kStatusTimeoutMma, 0u);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 22) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace piper

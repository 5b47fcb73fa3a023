// Attention of a drafted tree's nodes over the quantised paged cache.
//
// For a request and a KV head the `group * nodes` query rows that read that
// head are one small matrix Q.  With K codes k, V codes v and the row scales
// a (keys) and b (values), a row's output is
//   o = sum_j p_j b_j v_j / sum_j p_j,   p_j = exp(scale * a_j (q . k_j) - m)
// over the keys j that the row sees.  Reading the cache once (2 D + 8 bytes a
// key) bounds it while the rows are few: 16 rows need 64 products a byte.
//
// Up to 8 rows are the n of the products' m16n8k16: keys are the m of
// S^T = K Q^T and head dimensions that of O^T = V^T P^T, and the weights are
// transposed in registers between the two.  9 to 16 rows are the m, S = Q K^T
// and O = P V: for 8 rows that was half empty (110 against 94 us in the first
// case measured below).  Up to 24 (heads of 64: 32) rows are several blocks of
// 8 that share each converted fragment, as many as the numerators fit in
// registers.
//
// Products: fp16 tensor-core MMAs (m16n8k16, fp32 accumulators).  Codes are
// exact in fp16.  fp16 queries are used as they are; a bf16 row is scaled by
// a power of two to [1, 2) at its largest element, which loses only what lies
// 2^-25 and more below it.  A row has one reference, a logarithm `unit` that
// follows its largest p_j b_j: the total sums p_j / 2^unit, and the weights
// w_j = p_j b_j / 2^unit are rounded to fp16 (11 bits, against 8 or 11 of the
// output).  The reference moves, and the numerators with it, only when a
// weight would exceed 2^15.9, and then to 2^-10 of the largest: fp16 rounds
// weights below 2^-14 to steps of 2^-24, which is 2^-34 of the row's largest, so
// that the many small weights of a long context count beside a large one (a
// reference at the largest itself lost weights of 2^-25; the room costs nothing
// here).  Scores, weights, totals and numerators are fp32.
//
// Layout: a code of a page is the byte that a lane's fragment wants.  As 16-bit
// elements, ldmatrix gives lane (g, t) the bytes 4t .. 4t+3 of key g: the
// fragment's two pairs, if query elements are permuted alike.  ldmatrix.trans
// gives keys 2t, 2t+1 of bytes 2g, 2g+1: fragments of the even and of the odd
// head dimensions.  These are the b of 16 rows' products, and pairs of them the
// a of 8 rows'.  A byte becomes fp16 by a byte permute under 0x64 (1024 +
// code + 128) and one subtraction.
//
// Work: a segment is one (request, KV head, row tile); it has S::kLead units
// for its start and end (query rows, join), then a unit for each key tile.  The
// units of the whole batch are cut into equal runs, one for each CTA, so that
// ragged lengths balance (without the lead, runs of short requests took twice
// as long as the others: 187 against 141 us for 64 requests of 1 to 8192
// tokens).  A run that covers a segment writes its output; one that covers a
// part leaves its reference, total and numerator in the workspace, and
// tree_merge_kernel joins the parts.
//
// Measured (32 query over 8 KV heads of 128, pages of 64, one token each): 64
// requests of 1 to 8192 tokens 94 us, 5.9 TB/s or 0.92 of the copy rate; one
// request of 256 tokens 7.6 us.  24 heads of 64, 5 nodes, 32 requests of 333 to
// 4097 tokens in pages of 16: 57 us, 0.63 of the copy rate (pages of 64: 51), the
// ALU pipe busy 46 % and the issue slots 58 % of the time.  With 16 rows
// instructions bound it, 320 of some 660 for 32 keys a warp turning codes into
// fp16: 16 keys a warp took 131 us for 110.  32 requests of 1000 to 8191 tokens,
// 8 KV heads of 128: 8 rows 58 us, 16 rows 69, 24 rows 110; of 64: 38, 47, 32 rows
// 93.
#pragma once

#include <math.h>

#include <type_traits>

#include "kv_cache.cuh"
#include "sm100.cuh"

namespace piper {

constexpr float kSlack = 15.9f;         // log2 of the largest weight: fp16 holds less than 2^16
constexpr float kRoom = 10.0f;          // and of a row's largest one when its reference has just moved
constexpr float kScaleLogMin = -90.0f;  // smaller value scales count as 2^-90 in the references
constexpr float kNoReference = -1e30f;

struct TreeArgs {
  piper_b200_kv_cache_t c;
  const void* query;
  int64_t qs[3];
  void* out;
  const int64_t* mask;
  int64_t mask_stride;
  float* parts;      // [CTAs, 2] parts: rows x D numerators, then rows x (maximum, total)
  uint32_t* status;
  uint64_t wait_budget_ns;
  int heads, nodes, group, rows, row_tiles, page_shift;
  int whole;         // each CTA takes one whole (request, head, row tile)
  int vec;           // query rows allow 8-byte loads
  float scale_log2e;
};

// Tile of up to ROWS rows (16, or blocks of 8 that are the products' n): a warp takes 16 * GROUPS keys of it.
template <int D, int WARPS, int GROUPS, int ROWS>
struct TreeTile {
  static constexpr int kRows = ROWS;
  static constexpr int kKeys = 16 * GROUPS * WARPS;
  static constexpr int kThreads = 32 * (WARPS + 1);  // and one warp that fetches
  static constexpr int kCodes = kKeys * D;
  static constexpr int kScales = kKeys * 4;
  static constexpr int kStage = 2 * kCodes + 2 * kScales;
  static constexpr int kStageAlloc = (kStage + 1023) / 1024 * 1024;
  static constexpr bool kThin = ROWS != 16;
  static constexpr int kBlocks = kThin ? ROWS / 8 : 1;
  static constexpr int kJoinColumns = ROWS <= 16 ? 512 / ROWS : 16;
  static constexpr int kJoinStride = kJoinColumns + (ROWS <= 16 ? 16 : 4);  // floats; spreads rows over banks
  static constexpr int kJoin = WARPS * ROWS * kJoinStride * 4;
  static constexpr int kState = 2 * WARPS * kRows * 4;
  static constexpr bool kHeld = ROWS == 8;  // query fragments in registers
  static constexpr int kQuery = kHeld ? 0 : (D / 16) * 32 * ROWS;
  static constexpr int kFixed = kJoin + kState + kQuery + kRows * 8 + 512;
  // Per SM, what registers and stages allow.  8 rows of 128, 64 ragged requests as
  // above: two 94 us, three 110 (they spill).  8 rows of 64, 24 heads as above:
  // three 61 us, four 57, five 73.  16 rows of 64, 32 requests: two 52 us, three 47,
  // four 57.
  static constexpr int kCtas = D == 64 ? (ROWS == 8 ? 4 : ROWS == 16 ? 3 : 2) : 2;
  static constexpr int kLead = ROWS == 8 ? 3 : 4;  // a segment's start and end, in key tiles
  static constexpr int kFit = (227 * 1024 / kCtas - 1024 * 2 - kFixed) / kStageAlloc;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static constexpr int kAlloc = kStages * kStageAlloc + kFixed + 1024;
  static constexpr int kPart = kRows * (D + 2);  // floats of one part
};

// Key tiles of request b (at least one: it has a node).
template <int kKeys>
__device__ __forceinline__ int tree_tiles(const TreeArgs& a, int b) {
  const int64_t length = max(0, __ldg(a.c.lengths + b));
  const int64_t keys = min(length + a.nodes, static_cast<int64_t>(a.c.table_width) << a.page_shift);
  return static_cast<int>((keys + kKeys - 1) / kKeys);
}

// A run's place in the batch: `left` units from position `at` of segment
// (b, hr) on, hr being head * row_tiles + row tile; of the segment it has key
// tiles [tile, tile + count) of `tiles`.
struct TreeRun {
  int64_t left;
  int b, hr, at, tiles, tile, count;
  bool all;
};

// Units of the batch; every lane gets the result.
template <typename S>
__device__ __forceinline__ int64_t tree_units(const TreeArgs& a) {
  const int lane = threadIdx.x % 32;
  int64_t sum = 0;
  for (int b = lane; b < a.c.batch; b += 32) sum += S::kLead + tree_tiles<S::kKeys>(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum * (static_cast<int64_t>(a.c.kv_heads) * a.row_tiles);
}

// The request that unit u belongs to, its key tiles, and its first unit.
template <typename S>
__device__ __forceinline__ void tree_find(const TreeArgs& a, int64_t u, int* request, int* tiles, int64_t* first) {
  const int lane = threadIdx.x % 32;
  const int64_t per = static_cast<int64_t>(a.c.kv_heads) * a.row_tiles;
  int64_t base = 0;
  for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < a.c.batch ? tree_tiles<S::kKeys>(a, b) : 0;
    const int64_t mine = b < a.c.batch ? S::kLead + n : 0;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t below = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += below;
    }
    const unsigned past = __ballot_sync(0xffffffffu, u < base + upto * per);
    if (past != 0) {
      const int at = __ffs(past) - 1;
      *request = b0 + at;
      *tiles = __shfl_sync(0xffffffffu, n, at);
      *first = base + __shfl_sync(0xffffffffu, upto - mine, at) * per;
      return;
    }
    base += __shfl_sync(0xffffffffu, upto, 31) * per;
  }
  *request = a.c.batch;
  *tiles = 1;
  *first = base;
}

// CTAs that share the units: at least two key tiles' worth each (one request of
// 2000 tokens, 8 KV heads of 128: 13.3 us; at least four 14.8; at least one 12.0,
// and twice the workspace for tables of few tiles).
template <typename S>
__device__ __forceinline__ int64_t tree_ctas(int64_t units, int grid) {
  return max(static_cast<int64_t>(1), min(static_cast<int64_t>(grid), units / (S::kLead + 2)));
}
__device__ __forceinline__ int64_t tree_bound(int64_t units, int64_t ctas, int64_t i) { return units * i / ctas; }

// The key tiles of the run's segment, from its units.
template <typename S>
__device__ __forceinline__ void tree_range(TreeRun& r) {
  const int end = static_cast<int>(min(static_cast<int64_t>(S::kLead + r.tiles), r.at + r.left));
  r.tile = max(0, r.at - S::kLead);
  r.count = max(0, end - S::kLead) - r.tile;
  r.all = r.count == r.tiles;
}

template <typename S>
__device__ __forceinline__ TreeRun tree_run(const TreeArgs& a) {
  TreeRun r;
  const int per = a.c.kv_heads * a.row_tiles;
  r.at = 0;
  if (a.whole) {
    r.b = blockIdx.x / per;
    r.hr = blockIdx.x % per;
    r.tiles = tree_tiles<S::kKeys>(a, r.b);
    r.left = S::kLead + r.tiles;
  } else {
    const int64_t units = tree_units<S>(a);
    const int64_t ctas = tree_ctas<S>(units, gridDim.x);
    const int64_t begin = blockIdx.x < ctas ? tree_bound(units, ctas, blockIdx.x) : 0;
    r.left = blockIdx.x < ctas ? tree_bound(units, ctas, blockIdx.x + 1) - begin : 0;
    int64_t first = 0;
    tree_find<S>(a, begin, &r.b, &r.tiles, &first);
    const int length = S::kLead + r.tiles;
    r.hr = static_cast<int>((begin - first) / length);
    r.at = static_cast<int>((begin - first) % length);
  }
  tree_range<S>(r);
  if (r.left == 0) r.count = 0;
  return r;
}

// The run's next segment.
template <typename S>
__device__ __forceinline__ void tree_next(const TreeArgs& a, TreeRun& r) {
  r.left -= S::kLead + r.tiles - r.at;
  if (r.left <= 0) return;
  r.at = 0;
  if (++r.hr == a.c.kv_heads * a.row_tiles) {
    r.hr = 0;
    ++r.b;
    r.tiles = tree_tiles<S::kKeys>(a, r.b);
  }
  tree_range<S>(r);
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// This thread's arrival, once its earlier cp_async16 have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// An 8 x 8 matrix of 16-bit elements, a row's pair to each lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Two of the four codes in x (each plus 128), chosen by `select`, as fp16.
template <uint32_t select>
__device__ __forceinline__ uint32_t codes_f16(uint32_t x) {
  const uint32_t h = __byte_perm(x, 0x64646464u, select);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// Shared-memory address of 16-byte chunk `c` of row `r` of a tile that TMA
// wrote with the swizzle of D-byte rows.
template <int D>
__device__ __forceinline__ uint32_t tile_chunk(uint32_t base, int r, int c) {
  const int x = D == 128 ? (r & 7) : ((r >> 1) & 3);
  return base + r * D + ((c ^ x) << 4);
}

__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Four consecutive query elements as floats.
template <typename T>
__device__ __forceinline__ void query4(const T* p, bool vec, float (&x)[4]) {
  uint16_t e[4];
  if (vec) {
    *reinterpret_cast<uint2*>(e) = __ldg(reinterpret_cast<const uint2*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = reinterpret_cast<const uint16_t*>(p)[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(reinterpret_cast<const T*>(e)[i]);
}

// The fragments of query rows r0 + lane / 4 and, of two halves, that plus 8
// (zeros past the last row), scaled to fp16, and what undoes the scaling times the softmax
// scale.
template <typename T, int D, int HALVES = 2>
__device__ __forceinline__ void query_fragments(const TreeArgs& a, int b, int kv, int r0, uint32_t (&q)[D / 16][2 * HALVES],
                                                float (&factor)[HALVES]) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int half = 0; half < HALVES; ++half) {
    const int row = r0 + lane / 4 + 8 * half;
    float x[D / 16][4] = {};
    if (row < a.rows) {
      const int head = kv * a.group + row / a.nodes;
      const int node = row % a.nodes;
      const T* p = static_cast<const T*>(a.query) + b * a.qs[0] + head * a.qs[1] + node * a.qs[2] + (lane % 4) * 4;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) query4<T>(p + c * 16, a.vec, x[c]);
    }
    float up = 1.0f;
    factor[half] = a.scale_log2e;
    if constexpr (!std::is_same<T, __half>::value) {
      uint32_t top = 0u;
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[c][i]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t e = max(1u, min(253u, top >> 23));
      up = __uint_as_float((254u - e) << 23);
      factor[half] = __uint_as_float(e << 23) * a.scale_log2e;
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      q[c][half] = pack2(x[c][0] * up, x[c][1] * up, __half());
      q[c][half + HALVES] = pack2(x[c][2] * up, x[c][3] * up, __half());
    }
  }
}

template <typename T, int D, int WARPS, int GROUPS, int ROWS>
__global__ void __launch_bounds__(TreeTile<D, WARPS, GROUPS, ROWS>::kThreads, TreeTile<D, WARPS, GROUPS, ROWS>::kCtas)
    tree_attention_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                          TreeArgs a) {
  using S = TreeTile<D, WARPS, GROUPS, ROWS>;
  constexpr bool kThin = S::kThin, kHeld = S::kHeld;
  constexpr int kBlocks = S::kBlocks;
  constexpr int kSlots = 2 * kBlocks;  // rows of a thread
  constexpr int kN = kThin ? GROUPS * kBlocks : 2 * GROUPS;  // score fragments of a warp
  constexpr int kStages = S::kStages;
  constexpr int kChunks = D / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* join = reinterpret_cast<float*>(smem + kStages * S::kStageAlloc);
  float* state = reinterpret_cast<float*>(smem + kStages * S::kStageAlloc + S::kJoin);
  uint4* query = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(state) + S::kState);
  uint64_t* words = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(query) + S::kQuery);
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages];
  __shared__ uint32_t valid[kStages];
  __shared__ uint32_t abort_word;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t abort_flag = smem_u32(&abort_word);
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1 + 32);  // the codes' bytes, and each lane's scales
      mbar_init(smem_u32(&empty_bar[s]), WARPS);
    }
    abort_word = 0u;
    fence_mbarrier_init();
  }
  __syncthreads();
  // Lets tree_merge_kernel's CTAs be placed; they wait for this grid's end.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  TreeRun run = tree_run<S>(a);
  const int box = min(a.c.page_size, 64);
  const int box_shift = min(a.page_shift, 6);
  const int boxes = S::kKeys >> box_shift;

  if (warp == WARPS) {
    // ---- fetching warp: lane i brings box i of each tile's codes and four rows'
    // scales (a copy of a box's scales each, with pages of 16, made the copies so
    // many that they bound it: 65 us instead of 58).
    static_assert(S::kKeys == 32 * 4 && S::kBlocks <= WARPS, "a lane brings four rows' scales");
    int stage = 0, issued = 0;
    uint32_t phase = 1;  // a fresh barrier's previous phase counts as done
    bool ok = true;
    for (; run.left > 0 && ok; tree_next<S>(a, run)) {
      const int32_t* row = a.c.block_table + run.b * a.c.table_stride;
      const int head = run.hr / a.row_tiles;
      int have = -1, entry = -1;  // table columns [have, have + 32), one a lane
      for (int tile = run.tile; tile < run.tile + run.count && ok; ++tile) {
        const int64_t position = static_cast<int64_t>(tile) * S::kKeys + static_cast<int64_t>(lane) * box;
        const int column = static_cast<int>(position >> a.page_shift);
        const int column0 = static_cast<int>((static_cast<int64_t>(tile) * S::kKeys) >> a.page_shift);
        const int column1 =
            static_cast<int>((static_cast<int64_t>(tile) * S::kKeys + S::kKeys - 1) >> a.page_shift);
        if (have < 0 || column1 >= have + 32) {
          have = column0;
          entry = have + lane < a.c.table_width ? __ldg(row + have + lane) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, entry, (column - have) & 31);
        ok = mbar_wait_block_warp(smem_u32(&empty_bar[stage]), phase, a.wait_budget_ns, a.status, kStatusTimeoutEmpty,
                            abort_flag);
        if (!ok) break;
        const bool good = lane < boxes && column < a.c.table_width && page >= 0 && page < a.c.pages;
        const uint32_t goods = __ballot_sync(0xffffffffu, good);
        const uint32_t bar = smem_u32(&full_bar[stage]);
        if (lane == 0) {
          valid[stage] = goods;
          mbar_arrive_expect_tx(bar, __popc(goods) * box * 2 * D);
        }
        __syncwarp();
        const uint32_t base = smem_u32(smem + stage * S::kStageAlloc);
        const int z = page * a.c.kv_heads + head;
        const int y = static_cast<int>(position & (a.c.page_size - 1));
        if (good) {
          tma_load_3d(base + lane * box * D, &key_map, bar, 0, y, z);
          tma_load_3d(base + S::kCodes + lane * box * D, &value_map, bar, 0, y, z);
        }
        const int from = (4 * lane) >> box_shift;  // the box of this lane's four rows
        const int64_t at = (static_cast<int64_t>(__shfl_sync(0xffffffffu, z, from)) << a.page_shift) +
                           __shfl_sync(0xffffffffu, y, from) + (4 * lane & (box - 1));
        if ((goods >> from) & 1u) {
          cp_async16(base + 2 * S::kCodes + lane * 16, a.c.key_scales + at);
          cp_async16(base + 2 * S::kCodes + S::kScales + lane * 16, a.c.value_scales + at);
        }
        cp_async_arrive(bar);
        ++issued;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // Every copy has landed before the CTA's shared memory goes (the
    // consumers have waited for all of them unless something gave up).
    if (!ok)
      for (int i = max(0, issued - kStages); i < issued; ++i)
        mbar_wait_block_warp(smem_u32(&full_bar[i % kStages]), (i / kStages) & 1, a.wait_budget_ns, a.status,
                       kStatusTimeoutDrain, 0u);
    return;
  }

  // ---- computing warps: some keys of each tile, all rows.
  const int g = lane / 4, t = lane % 4;
  // Element x of score fragment n is row row_at(h), h = row_slot(n, x), and key
  // key_at(n, e), e = key_half(x), of the warp's.
  auto row_slot = [](int n, int x) { return kThin ? 2 * (n % kBlocks) + (x & 1) : x / 2; };
  auto key_half = [](int x) { return kThin ? x / 2 : (x & 1); };
  auto row_at = [&](int h) { return kThin ? 8 * (h / 2) + 2 * t + (h & 1) : g + 8 * h; };
  auto key_at = [&](int n, int e) { return kThin ? 16 * (n / kBlocks) + g + 8 * e : 8 * n + 2 * t + e; };
  // Over the lanes that hold the same rows.
  auto of_row = [&](float x, auto join2) {
#pragma unroll
    for (int o = kThin ? 4 : 1; o < (kThin ? 32 : 4); o <<= 1) x = join2(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
  };
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  int part = 0;
  for (; run.left > 0; tree_next<S>(a, run)) {
    if (run.count == 0) continue;
    const int b = run.b, kv = run.hr / a.row_tiles;
    const int row0 = (run.hr % a.row_tiles) * S::kRows;
    const bool all = run.all;
    const int64_t length = max(0, __ldg(a.c.lengths + b));
    float factor[kSlots];
    uint32_t held[kHeld ? kChunks : 1][2];
    uint2* query_pairs = reinterpret_cast<uint2*>(query);
    if constexpr (kThin) {
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        uint32_t q[kChunks][2];
        float mine[1];
        query_fragments<T, D, 1>(a, b, kv, row0 + 8 * k, q, mine);
#pragma unroll
        for (int h = 0; h < 2; ++h) factor[2 * k + h] = __shfl_sync(0xffffffffu, mine[0], 4 * row_at(h));
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          if constexpr (kHeld)
            held[c][0] = q[c][0], held[c][1] = q[c][1];
          else if (warp == k)
            query_pairs[(c * kBlocks + k) * 32 + lane] = make_uint2(q[c][0], q[c][1]);
        }
      }
    } else {
      // Every warp has the rows' factors; warp 0's fragments serve all (holding
      // them cost each thread 32 registers, and the SM a CTA).
      uint32_t q[kChunks][4];
      query_fragments<T, D>(a, b, kv, row0, q, factor);
      if (warp == 0) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) query[c * 32 + lane] = make_uint4(q[c][0], q[c][1], q[c][2], q[c][3]);
      }
    }
    if (tid < S::kRows) {
      const int row = row0 + tid;
      uint64_t word = 0;
      if (row < a.rows) {
        const int node = row % a.nodes;
        word = a.mask != nullptr ? static_cast<uint64_t>(__ldg(reinterpret_cast<const unsigned long long*>(
                                       a.mask + b * a.mask_stride + node)))
                                 : ~0ull >> (63 - node);
        word &= ~0ull >> (64 - a.nodes);
      }
      words[tid] = word;
    }
    bar_sync(1, WARPS * 32);
    float o[kThin ? kChunks * kBlocks : 2 * kChunks][4] = {};
    float unit[kSlots], l[kSlots];
#pragma unroll
    for (int h = 0; h < kSlots; ++h) unit[h] = kNoReference, l[h] = 0.0f;
    for (int tile = run.tile; tile < run.tile + run.count; ++tile) {
      if (ok) ok = mbar_wait_block_warp(smem_u32(&full_bar[stage]), phase, a.wait_budget_ns, a.status, kStatusTimeoutFull,
                                  abort_flag);
      if (ok) {
        const uint32_t base = smem_u32(smem + stage * S::kStageAlloc);
        const float* scales = reinterpret_cast<const float*>(smem + stage * S::kStageAlloc + 2 * S::kCodes);
        const int key0 = warp * 16 * GROUPS;
        const uint32_t goods = valid[stage];
        const int64_t first = static_cast<int64_t>(tile) * S::kKeys;
        const bool masked = first + S::kKeys > length || goods != (1u << boxes) - 1u;
        // ---- scores
        float y[kN][4] = {};
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint4 f[2];
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if constexpr (!kThin) f[x] = query[(c + x) * 32 + lane];
#pragma unroll
          for (int i = 0; i < GROUPS; ++i) {
            uint32_t k[4];
            ldmatrix4(tile_chunk<D>(base, key0 + 16 * i + (lane & 15), c + (lane >> 4)), k);
#pragma unroll
            for (int x = 0; x < 4; ++x) k[x] ^= 0x80808080u;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if constexpr (kThin) {
                const uint32_t keys[4] = {codes_f16<0x4140>(k[2 * x]), codes_f16<0x4140>(k[2 * x + 1]),
                                          codes_f16<0x4342>(k[2 * x]), codes_f16<0x4342>(k[2 * x + 1])};
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                  uint2 q;
                  if constexpr (kHeld)
                    q = make_uint2(held[c + x][0], held[c + x][1]);
                  else
                    q = query_pairs[((c + x) * kBlocks + n) * 32 + lane];
                  mma16816(y[i * kBlocks + n], keys, q.x, q.y);
                }
              } else {
                const uint32_t q[4] = {f[x].x, f[x].y, f[x].z, f[x].w};
#pragma unroll
                for (int n = 0; n < 2; ++n)
                  mma16816(y[2 * i + n], q, codes_f16<0x4140>(k[2 * x + n]), codes_f16<0x4342>(k[2 * x + n]));
              }
            }
          }
        }
        uint32_t w[GROUPS][kThin ? kSlots : 4];
        auto two = [&](const float* p, int n) {
          if constexpr (kThin) return make_float2(p[key_at(n, 0)], p[key_at(n, 1)]);
          return *reinterpret_cast<const float2*>(p + key_at(n, 0));
        };
        // A masked tile has a body of its own: selections would lengthen the
        // other's.
        auto weigh = [&](auto hidden) {
          uint32_t unseen = 0u;  // bit 4 n + x
          if constexpr (hidden.value) {
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = key0 + key_at(n, e);
                const int64_t j = first + key - length;
                const bool there = (goods >> (key >> box_shift)) & 1u;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  if (key_half(x) == e &&
                      !(there && (j < 0 || (j < a.nodes && ((words[row_at(row_slot(n, x))] >> (j & 63)) & 1u)))))
                    unseen |= 1u << (4 * n + x);
              }
          }
          float most[kSlots];
#pragma unroll
          for (int h = 0; h < kSlots; ++h) most[h] = -INFINITY;
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            const float2 ks = two(scales + key0, n);
            const float2 vs = two(scales + S::kKeys + key0, n);
            const float lv[2] = {fmaxf(lg2_approx(fabsf(vs.x)), kScaleLogMin), fmaxf(lg2_approx(fabsf(vs.y)), kScaleLogMin)};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              y[n][x] *= key_half(x) ? ks.y : ks.x;
              // A key that a row does not see may hold anything.
              if (hidden.value && ((unseen >> (4 * n + x)) & 1u)) y[n][x] = -INFINITY;
              float z = fmaf(y[n][x], factor[row_slot(n, x)], lv[key_half(x)]);
              if (hidden.value && ((unseen >> (4 * n + x)) & 1u)) z = -INFINITY;
              most[row_slot(n, x)] = fmaxf(most[row_slot(n, x)], z);
            }
          }
          bool above = false;
#pragma unroll
          for (int h = 0; h < kSlots; ++h) above |= most[h] - unit[h] > kSlack;
          if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int h = 0; h < kSlots; ++h) {
              most[h] = of_row(most[h], [](float u, float v) { return fmaxf(u, v); });
              const float to = most[h] - kRoom;
              // (The numerators' columns are rows as the scores' are.)
              const float shrink = to > unit[h] ? ex2_approx(unit[h] - to) : 1.0f;
              unit[h] = fmaxf(unit[h], to);
              l[h] *= shrink;
#pragma unroll
              for (int c = 0; c < static_cast<int>(sizeof(o) / sizeof(o[0])); ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  if (row_slot(c, x) == h) o[c][x] *= shrink;
            }
          }
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            const float2 vs = two(scales + S::kKeys + key0, n);
            float p[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int h = row_slot(n, x);
              // (An unseen key's value scale may be anything, and -infinity times a
              // factor that underflowed is no number.)
              const bool out = hidden.value && ((unseen >> (4 * n + x)) & 1u);
              p[x] = ex2_approx(fmaf(y[n][x], factor[h], -unit[h]));
              if (out) p[x] = 0.0f;
              l[h] += p[x];
              p[x] *= key_half(x) ? vs.y : vs.x;
              if (out) p[x] = 0.0f;
            }
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t pair = pack2(p[2 * z], p[2 * z + 1], __half());
              if constexpr (kThin)
                w[n / kBlocks][2 * (n % kBlocks) + z] = transpose8(pair);
              else
                w[n / 2][2 * (n & 1) + z] = pair;
            }
          }
        };
        if (masked)
          weigh(std::true_type());
        else
          weigh(std::false_type());
        // ---- numerators: even, then odd head dimensions of each chunk
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
#pragma unroll
          for (int i = 0; i < GROUPS; ++i) {
            uint32_t v[4];
            ldmatrix4_trans(tile_chunk<D>(base + S::kCodes, key0 + 16 * i + (lane & 15), c + (lane >> 4)), v);
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] ^= 0x80808080u;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if constexpr (kThin) {
                const uint32_t values[4] = {codes_f16<0x4240>(v[2 * x]), codes_f16<0x4341>(v[2 * x]),
                                            codes_f16<0x4240>(v[2 * x + 1]), codes_f16<0x4341>(v[2 * x + 1])};
#pragma unroll
                for (int n = 0; n < kBlocks; ++n)
                  mma16816(o[(c + x) * kBlocks + n], values, w[i][2 * n], w[i][2 * n + 1]);
              } else {
                mma16816(o[2 * (c + x)], w[i], codes_f16<0x4240>(v[2 * x]), codes_f16<0x4240>(v[2 * x + 1]));
                mma16816(o[2 * (c + x) + 1], w[i], codes_f16<0x4341>(v[2 * x]), codes_f16<0x4341>(v[2 * x + 1]));
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty_bar[stage]));
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    // ---- join the warps' parts: each row's reference and total, then the
    // numerators, kJoinColumns head dimensions at a time.
#pragma unroll
    for (int h = 0; h < kSlots; ++h) {
      l[h] = of_row(l[h], [](float u, float v) { return u + v; });
      if (unit[h] == kNoReference) unit[h] = -INFINITY;
      if ((kThin ? g : t) == 0) {
        state[warp * ROWS + row_at(h)] = unit[h];
        state[(WARPS + warp) * ROWS + row_at(h)] = l[h];
      }
    }
    bar_sync(1, WARPS * 32);
    // A row's reference (0 where it saw nothing) and total over the warps.
    auto joined = [&](int r, float* total) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, state[w * ROWS + r]);
      const float ref = top == -INFINITY ? 0.0f : top;
      *total = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) *total += state[(WARPS + w) * ROWS + r] * ex2_approx(state[w * ROWS + r] - ref);
      return top;
    };
    float share[kSlots];
    float* to = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + part) * S::kPart;
#pragma unroll
    for (int h = 0; h < kSlots; ++h) {
      float total;
      const float top = joined(row_at(h), &total);
      share[h] = ex2_approx(unit[h] - (top == -INFINITY ? 0.0f : top));
      if (!all && warp == 0 && (kThin ? g : t) == 0) {
        to[ROWS * D + 2 * row_at(h)] = top;
        to[ROWS * D + 2 * row_at(h) + 1] = total;
      }
    }
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += S::kJoinColumns) {
      float* mine = join + warp * ROWS * S::kJoinStride;
#pragma unroll
      for (int c = 0; c < S::kJoinColumns / 16; ++c)
#pragma unroll
        for (int h = 0; h < kSlots; ++h) {
          const float f = share[h];
          float* row = mine + row_at(h) * S::kJoinStride + c * 16;
          if constexpr (kThin) {
            const float(&both)[4] = o[(d0 / 16 + c) * kBlocks + h / 2];
            *reinterpret_cast<float2*>(row + 2 * g) = make_float2(both[h & 1] * f, both[2 + (h & 1)] * f);
          } else {
            const float(&even)[4] = o[2 * (d0 / 16 + c)];
            const float(&odd)[4] = o[2 * (d0 / 16 + c) + 1];
            *reinterpret_cast<float4*>(row + 4 * t) =
                make_float4(even[2 * h] * f, odd[2 * h] * f, even[2 * h + 1] * f, odd[2 * h + 1] * f);
          }
        }
      bar_sync(1, WARPS * 32);
      // Four columns a thread.
      for (int x = tid; x < ROWS * S::kJoinColumns / 4; x += WARPS * 32) {
        constexpr int kFours = S::kJoinColumns / 4;
        const int r = x / kFours, d = (x % kFours) * 4;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(join + (w * ROWS + r) * S::kJoinStride + d);
          sum.x += y.x;
          sum.y += y.y;
          sum.z += y.z;
          sum.w += y.w;
        }
        const int row = row0 + r;
        if (!all) {
          *reinterpret_cast<float4*>(to + r * D + d0 + d) = sum;
        } else if (row < a.rows) {
          float total;
          joined(r, &total);
          const float f = total == 0.0f ? 0.0f : 1.0f / total;
          const int64_t at =
              ((static_cast<int64_t>(b) * a.heads + kv * a.group + row / a.nodes) * a.nodes + row % a.nodes) * D;
          uint2 y;
          y.x = pack2(sum.x * f, sum.y * f, T());
          y.y = pack2(sum.z * f, sum.w * f, T());
          *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at + d0 + d) = y;
        }
      }
      bar_sync(1, WARPS * 32);
    }
    part = 1;
  }
}

// Joins the parts of every segment whose key tiles a boundary between two runs
// cuts.  CTA x looks at the boundary before run x + 1 and works if it is the
// first such one of its segment; a warp takes a row, and CTAs y share the
// rows.  A lane holds the maximum and total of one of 32 parts, so that the
// numerators' loads do not wait for one another.
template <typename T, int D, typename S>
__global__ void __launch_bounds__(128) tree_merge_kernel(TreeArgs a, int grid) {
  // (The lengths were there before the attention kernel began.)
  const int64_t units = tree_units<S>(a);
  const int64_t ctas = tree_ctas<S>(units, grid);
  const int64_t i = blockIdx.x + 1;
  const int64_t at = i < ctas ? tree_bound(units, ctas, i) : 0;
  int b = 0, tiles = 1;
  int64_t first = 0;
  tree_find<S>(a, at, &b, &tiles, &first);
  const int hr = static_cast<int>((at - first) / (S::kLead + tiles));
  const int64_t start = first + static_cast<int64_t>(hr) * (S::kLead + tiles);
  const int64_t begin = start + S::kLead, end = begin + tiles;  // its key tiles
  const int64_t before = i < ctas ? tree_bound(units, ctas, i - 1) : 0;
  // Every CTA waits, so that this grid does not end before the other.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (i >= ctas || at <= begin || before > begin) return;
  // Runs i - 1 to `last` have parts of it: `last` holds its last unit.
  int64_t last = ((end - 1) * ctas) / units;
  while (last + 1 < ctas && tree_bound(units, ctas, last + 1) < end) ++last;
  while (tree_bound(units, ctas, last) >= end) --last;
  const int count = static_cast<int>(last - (i - 1) + 1);
  const int lane = threadIdx.x % 32;
  const int kv = hr / a.row_tiles, row0 = (hr % a.row_tiles) * S::kRows;
  constexpr int kPer = D / 32;
  // Part k is run i - 1 + k's first one if the run starts in the segment.
  auto part_of = [&](int k) {
    return a.parts + ((i - 1 + k) * 2 + (k == 0 && before < start ? 1 : 0)) * S::kPart;
  };
  for (int r = blockIdx.y * 4 + threadIdx.x / 32; r < S::kRows && row0 + r < a.rows; r += 4 * gridDim.y) {
    float m = -INFINITY, l = 0.0f, o[kPer] = {};
    for (int k0 = 0; k0 < count; k0 += 32) {
      float pm = -INFINITY, pl = 0.0f;
      if (k0 + lane < count) {
        const float2 ml = *reinterpret_cast<const float2*>(part_of(k0 + lane) + S::kRows * D + 2 * r);
        pm = ml.x;
        pl = ml.y;
      }
      float top = pm;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      top = fmaxf(top, m);
      const float ref = top == -INFINITY ? 0.0f : top;
      const float pf = ex2_approx(pm - ref), f = ex2_approx(m - ref);
      float sum = pl * pf;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      m = top;
      l = l * f + sum;
#pragma unroll
      for (int x = 0; x < kPer; ++x) o[x] *= f;
      const int n = min(32, count - k0);
#pragma unroll 8
      for (int k = 0; k < n; ++k) {
        const float g = __shfl_sync(0xffffffffu, pf, k);
        const float* from = part_of(k0 + k) + r * D + lane * kPer;
        float v[kPer];
        if constexpr (kPer == 4)
          *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(from);
        else
          *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(from);
#pragma unroll
        for (int x = 0; x < kPer; ++x) o[x] = fmaf(v[x], g, o[x]);
      }
    }
    const int row = row0 + r;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(a.out) +
             ((static_cast<int64_t>(b) * a.heads + kv * a.group + row / a.nodes) * a.nodes + row % a.nodes) * D;
#pragma unroll
    for (int x = 0; x < kPer; x += 2)
      *reinterpret_cast<uint32_t*>(out + lane * kPer + x) = pack2(o[x] * f, o[x + 1] * f, T());
  }
}

}  // namespace piper

// Matrix products with the surrounding operator's arithmetic applied to the
// accumulators before anything reaches memory.
//
// A product is C[i, j] = sum_k A(i, k) * B(j, k) for i < m, j < n, k < depth,
// 16-bit operands (bf16 or fp16), fp32 accumulation.  Each operand lies in
// memory either with k contiguous ("k-major": element (i, k) at p[i * ld + k])
// or with i contiguous ("row-major": p[k * ld + i]), so the three products of a
// linear layer (forward, gradient of the input, gradient of the weight) read
// the tensors as they are.
//
// What happens to the accumulators is an epilogue: a struct whose methods a
// warp calls together, each lane for the row i it holds (`Lane::inside` where
// i < m):
//   Row begin(lane, i)                          per-row state
//   chunk(Row&, lane, i, j, float (&v)[32])     columns j .. j + 31 of row i
//   end(Row&, lane, i, part)                    after the lane's last chunk
// and, for products whose sums may be split or empty,
//   point(i, j, v)                              one value by itself
// A "paired" epilogue (kPaired) gets two accumulators for each column: those
// of B's rows j and pair_offset + j (gate and up).  The chunks of a tile's row
// are shared out to kColumnGroups lanes; `part` numbers these shares along C's
// columns.
// kSegment, stages: 0 leaves a tile's whole sum to the tensor cores.  Their
// adder cuts off what falls below the running sum's last place, 16 terms a step,
// so a sum of n steps comes out short by about n * 2^-24 * 0.22 (bf16) to 0.28
// (fp16) of itself, by up to 1.6 where all terms have one sign, and by nothing
// where no term is cut.  With kSegment the tensor cores sum that many stages at
// a time and the segments' sums join in registers by rounded additions.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>
#include <type_traits>

#include "runtime.cuh"
#include "tcgen05.cuh"
#include "vec.cuh"

namespace hprn {

struct Operand {
  const uint16_t* p = nullptr;
  int64_t ld = 0;
};

struct Product {
  Operand a, b;
  int64_t m = 0;      // rows of C
  int64_t n = 0;      // columns of C
  int64_t depth = 0;  // length of the sums
  int64_t pair_offset = 0;
};

constexpr int kChunk = 32;         // accumulators a thread hands to an epilogue at once
constexpr int kColumnGroups = 2;   // lanes that share a tile's row
constexpr int kScratchWords = 32 * 17;  // a warp's transposition buffer

struct Lane {
  uint32_t* scratch;  // kScratchWords words of the warp's own
  int lane;
  int32_t split;  // which share of a split sum the accumulators are
  bool inside;
};

// ---------------------------------------------------------------------------
// Rows of 16-bit values written a chunk at a time.  Where rows start on
// 16-byte boundaries a lane writes its 64 bytes as full 32- or 16-byte
// sectors.  Elsewhere (odd widths, ragged last chunks) the warp turns the
// chunk in shared memory, so that its lanes write neighbouring elements of one
// row: 2 sectors a store instead of 32.
struct Out16 {
  uint16_t* p = nullptr;
  int64_t ld = 0;
  int64_t n = 0;
  int32_t align = 2;  // of every row's start: 32, 16 or less

  Out16() = default;
  Out16(void* base, int64_t row_stride, int64_t cols) : p(static_cast<uint16_t*>(base)), ld(row_stride), n(cols) {
    for (int v : {32, 16})
      if (aligned(base, v) && (row_stride * 2) % v == 0) {
        align = v;
        break;
      }
  }

  template <typename T>
  __device__ __forceinline__ void store(const Lane& l, int64_t i, int64_t j, const float (&v)[kChunk]) const {
    uint32_t w[kChunk / 2];
#pragma unroll
    for (int k = 0; k < kChunk / 2; ++k) w[k] = pack2<T>(v[2 * k], v[2 * k + 1]);
    if (align >= 16 && j + kChunk <= n) {
      if (!l.inside) return;
      uint16_t* q = p + i * ld + j;
      if (align == 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Vec<32> o;
#pragma unroll
          for (int k = 0; k < 8; ++k) o.w[k] = w[8 * h + k];
          st_global<32>(q + 16 * h, o);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          Vec<16> o;
#pragma unroll
          for (int k = 0; k < 4; ++k) o.w[k] = w[4 * h + k];
          st_global<16>(q + 8 * h, o);
        }
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < kChunk / 2; ++k) l.scratch[l.lane * 17 + k] = w[k];
    const int count = __popc(__ballot_sync(~0u, l.inside));  // the inside lanes are the first ones
    __syncwarp();
    uint16_t* q = p + (i - l.lane) * ld + j + l.lane;
    const bool mine = j + l.lane < n;
    const uint16_t* e = reinterpret_cast<const uint16_t*>(l.scratch) + l.lane;
    for (int r = 0; r < count; ++r, q += ld)
      if (mine) *q = e[r * 34];
    __syncwarp();
  }
};

// The same for fp32 rows.
struct Out32 {
  float* p = nullptr;
  int64_t ld = 0;
  int64_t n = 0;
  int32_t align = 4;

  Out32() = default;
  Out32(float* base, int64_t row_stride, int64_t cols) : p(base), ld(row_stride), n(cols) {
    if (aligned(base, 32) && (row_stride * 4) % 32 == 0) align = 32;
  }

  __device__ __forceinline__ void store(const Lane& l, int64_t i, int64_t j, const float (&v)[kChunk]) const {
    if (align == 32 && j + kChunk <= n) {
      if (!l.inside) return;
      float* q = p + i * ld + j;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        Vec<32> o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o.w[k] = __float_as_uint(v[8 * h + k]);
        st_global<32>(q + 8 * h, o);
      }
      return;
    }
    // 16 columns at a time, two rows a store.
    const int count = __popc(__ballot_sync(~0u, l.inside));
    const int c = l.lane % 16, up = l.lane / 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < 16; ++k) l.scratch[l.lane * 17 + k] = __float_as_uint(v[16 * h + k]);
      __syncwarp();
      const bool mine = j + 16 * h + c < n;
      for (int r = up; r < count; r += 2)
        if (mine) p[(i - l.lane + r) * ld + j + 16 * h + c] = __uint_as_float(l.scratch[r * 17 + c]);
      __syncwarp();
    }
  }
};

// ---------------------------------------------------------------------------
// C itself, optionally summed over several products (the pieces of a long
// sum) in an fp32 buffer: `sum` holds the earlier pieces' total; `last` says
// whether this product finishes it.  The total is rounded to 16 bits once.
template <typename T>
struct StoreEpilogue {
  static constexpr bool kPaired = false;
  static constexpr int kSegment = 0;
  Out16 out;             // written by the last piece
  float* sum = nullptr;  // rows of sum_ld (a multiple of 32), or null when there is one piece
  int64_t sum_ld = 0;
  bool first = true;
  bool last = true;
  const float* scale = nullptr;  // one float that multiplies the total, or null

  struct Row {
    float scale;
  };
  __device__ __forceinline__ Row begin(const Lane&, int64_t) const { return Row{scale ? *scale : 1.0f}; }
  __device__ __forceinline__ void chunk(Row& s, const Lane& l, int64_t i, int64_t j, float (&v)[kChunk]) const {
    if (!(first && last) && l.inside) {
      float4* p = reinterpret_cast<float4*>(sum + i * sum_ld + j);
      if (!first) {
#pragma unroll
        for (int k = 0; k < kChunk / 4; ++k) {
          const float4 q = p[k];
          v[4 * k] += q.x, v[4 * k + 1] += q.y, v[4 * k + 2] += q.z, v[4 * k + 3] += q.w;
        }
      }
      if (!last) {
#pragma unroll
        for (int k = 0; k < kChunk / 4; ++k) p[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
      }
    }
    if (!last) return;
    if (scale) {
#pragma unroll
      for (int k = 0; k < kChunk; ++k) v[k] *= s.scale;
    }
    out.template store<T>(l, i, j, v);
  }
  __device__ __forceinline__ void end(Row&, const Lane&, int64_t, int64_t) const {}
  __device__ __forceinline__ void point(int64_t i, int64_t j, float v) const {
    float* p = sum + i * sum_ld + j;
    if (!first) v += *p;
    if (!last) *p = v;
    else out.p[i * out.ld + j] = pack1<T>(scale ? v * *scale : v);
  }
};

// The raw accumulators of one share of a split sum; join_splits adds the
// shares up and calls the product's own epilogue.
template <bool kPair>
struct SplitEpilogue {
  static constexpr bool kPaired = kPair;
  static constexpr int kSegment = 0;
  float* partial = nullptr;  // [splits][rows][ld]; a pair's second values follow its first
  int64_t ld = 0;            // columns of one value, a multiple of 32
  int64_t rows = 0;

  struct Row {
    float* p;
  };
  __device__ __forceinline__ float* at(int32_t split, int64_t i) const {
    return partial + ((split * rows + i) * (kPair ? 2 : 1)) * ld;
  }
  __device__ __forceinline__ Row begin(const Lane& l, int64_t i) const { return Row{at(l.split, l.inside ? i : 0)}; }
  __device__ __forceinline__ void chunk(Row& r, const Lane& l, int64_t, int64_t j, float (&v)[kChunk]) const {
    if (l.inside) put(r.p + j, v);
  }
  __device__ __forceinline__ void chunk(Row& r, const Lane& l, int64_t, int64_t j, float (&v)[kChunk],
                                        float (&u)[kChunk]) const {
    if (l.inside) put(r.p + j, v), put(r.p + ld + j, u);
  }
  __device__ __forceinline__ void end(Row&, const Lane&, int64_t, int64_t) const {}
  static __device__ __forceinline__ void put(float* p, const float (&v)[kChunk]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      Vec<32> o;
#pragma unroll
      for (int k = 0; k < 8; ++k) o.w[k] = __float_as_uint(v[8 * h + k]);
      st_global<32>(p + 8 * h, o);
    }
  }
};

// ---------------------------------------------------------------------------
// The kernel: a persistent grid of CTAs (or pairs of CTAs), each taking tiles
// of C (or shares of a tile's sum) in turn.  In a CTA
//   warp 0     one thread keeps a ring of shared-memory stages filled by TMA,
//              64 of the sum's terms a stage;
//   warp 1     (of the pair's first CTA) one thread issues the MMAs of a stage
//              as it arrives, into one of two TMEM accumulators;
//   warp 2     allocates and frees TMEM;
//   warps 4-11 hand the finished accumulator's rows to the epilogue, while the
//              next tile's MMAs fill the other one.
// Tiles are 128 rows x `cols` accumulator columns per CTA, or 256 x `cols` per
// pair.  A stage holds the rows of A that exist (at most 128, in eights); the
// MMA always reads 128, the rest being whatever follows in shared memory, and
// those rows of the accumulator are not looked at.
//
// Every wait has a limit (mbar_wait_bounded).  A role whose wait runs out
// says so (report_give_up) and stops; the others' waits then run out too,
// and the CTA ends after its copies and MMAs in flight.
constexpr int kDepthBlock = 64;  // 16-bit elements in a 128-byte row of a stage
constexpr int kMatmulThreads = 384;
constexpr int kMaxStages = 24;
// Shared memory the ring may take: 227 KB less the transposition buffers (8
// warps x 2176 bytes), the barriers and the ring's alignment.
constexpr int kRingBytes = 208 * 1024;
constexpr int kMatmulSmem = kRingBytes + 1024;
constexpr int kTmemColumns = 512;

struct MatmulArgs {
  int32_t tiles_m, tiles_n;
  int32_t splits;
  int32_t depth_blocks;
  int32_t cols;      // accumulator columns of a tile
  int32_t a_rows;    // rows of A in a CTA's stage (k-major), in eights
  int32_t stages;
  int32_t band;      // tile rows taken together
  int32_t pair_offset;
  int64_t m, n;
  Waits waits;
};

struct Item {
  int32_t tm, tn, split;
};
// The stages [first, last) of the sum that share `split` covers.
struct DepthRange {
  int32_t first, last;
};
__device__ __forceinline__ DepthRange depth_range(const MatmulArgs& a, int32_t split) {
  if (a.splits == 1) return DepthRange{0, a.depth_blocks};
  const int64_t n = a.depth_blocks;
  return DepthRange{static_cast<int32_t>(n * split / a.splits),
                    static_cast<int32_t>(n * (split + 1) / a.splits)};
}

// Item `t` of the order items are taken in: a tile's splits follow each other;
// tiles go in bands of `band` tile rows, down a band's columns first, so that
// the tiles in flight at one time cover a near-square part of C and share A's
// and B's rows in L2.
__device__ __forceinline__ Item item_at(const MatmulArgs& a, int32_t t) {
  Item r;
  const int32_t tile = t / a.splits;
  r.split = t - tile * a.splits;
  const int32_t band_tiles = a.band * a.tiles_n;
  const int32_t band = tile / band_tiles;
  const int32_t first = band * a.band;
  const int32_t rows = min(a.band, a.tiles_m - first);
  const int32_t in = tile - band * band_tiles;
  r.tm = first + in % rows;
  r.tn = in / rows;
  return r;
}

// One lane's share of a tile's row through the epilogue.  load(column, v)
// gives 32 accumulators from that accumulator column on.
template <typename E, typename Load>
__device__ __forceinline__ void run_epilogue(const E& epi, const Lane& l, int64_t i, int64_t j0, int64_t n,
                                             int cols, int group, int64_t part, Load&& load) {
  auto row = epi.begin(l, i);
#pragma unroll 1
  for (int c = group * kChunk; c < cols && j0 + c < n; c += kColumnGroups * kChunk) {
    float v[kChunk];
    if constexpr (E::kPaired) {
      float u[kChunk];
      load(c, v, cols + c, u);
      epi.chunk(row, l, i, j0 + c, v, u);
    } else {
      load(c, v);
      epi.chunk(row, l, i, j0 + c, v);
    }
    __syncwarp();
  }
  epi.end(row, l, i, part);
}

// The same for a sum in segments: a lane's share of the tile's row, held in
// 128 registers.  kUnrolled: the epilogue's code once a chunk, each on its own
// registers, else one copy of it that the chunks move up to.  The softmax sums
// fit unrolled (7 x 1024 x 32768: 19.7 us, moving 20.5; 2048 x 5120 x 100003:
// 1685, 1725); the logit gradients then spill 800 bytes (1023 x 2056 x 50001
// with both gradients: 843 us, moving 783).  Loads of 32 columns instead of 16
// spill 24 to 300 bytes more and are no faster.
constexpr int kLaneChunks = 256 / kChunk / kColumnGroups;

struct LaneSums {
  float v[kLaneChunks][kChunk];
  __device__ __forceinline__ static int column(int k, int group) { return (k * kColumnGroups + group) * kChunk; }
  // Adds the accumulators of one more segment (sets them, of the first).
  __device__ __forceinline__ void add(uint32_t acc, bool first, int cols, int group) {
#pragma unroll
    for (int k = 0; k < kLaneChunks; ++k) {
      const int c = column(k, group);
      if (c >= cols) break;
      if (first) {
        tmem_load_32(acc + c, v[k]);
        tmem_wait_load(v[k]);
        continue;
      }
#pragma unroll
      for (int h = 0; h < kChunk; h += 16) {
        float w[16];
        tmem_load_16(acc + c + h, w);
        tmem_wait_load(w);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[k][h + e] += w[e];
      }
    }
  }
  template <typename E>
  __device__ __forceinline__ void run(const E& epi, const Lane& l, int64_t i, int64_t j0, int64_t n, int cols,
                                      int group, int64_t part) {
    auto row = epi.begin(l, i);
    if constexpr (E::kUnrolled) {
#pragma unroll
      for (int k = 0; k < kLaneChunks; ++k) {
        const int c = column(k, group);
        if (c >= cols || j0 + c >= n) break;
        epi.chunk(row, l, i, j0 + c, v[k]);
        __syncwarp();
      }
    } else {
#pragma unroll 1
      for (int k = 0; k < kLaneChunks; ++k) {
        const int c = column(k, group);
        if (c >= cols || j0 + c >= n) break;
        epi.chunk(row, l, i, j0 + c, v[0]);
#pragma unroll
        for (int q = 1; q < kLaneChunks; ++q)
#pragma unroll
          for (int e = 0; e < kChunk; ++e) v[q - 1][e] = v[q][e];
        __syncwarp();
      }
    }
    epi.end(row, l, i, part);
  }
};

template <typename T, typename E, int kGroup, bool kAKMajor, bool kBKMajor>
__global__ void __launch_bounds__(kMatmulThreads, 1)
    matmul_tiles(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const MatmulArgs args, const E epi) {
  extern __shared__ unsigned char ring_mem[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 5];
  __shared__ uint32_t scratch[8 * kScratchWords];
  __shared__ uint32_t tmem_base;
  const uint32_t ring = (smem_u32(ring_mem) + 1023) & ~1023u;
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const uint32_t rank = kGroup == 2 ? cluster_rank() : 0;
  const int stages = args.stages;
  const uint32_t a_bytes = args.a_rows * 128, b_rows = args.cols / kGroup;
  const uint32_t stage_bytes = a_bytes + b_rows * 128;
  const int32_t c_cols = E::kPaired ? args.cols / 2 : args.cols;  // columns of C per tile
  auto full = [&](int s) { return smem_u32(&bars[s]); };
  auto empty = [&](int s) { return smem_u32(&bars[kMaxStages + s]); };
  auto acc_full = [&](int b) { return smem_u32(&bars[2 * kMaxStages + b]); };
  auto acc_empty = [&](int b) { return smem_u32(&bars[2 * kMaxStages + 2 + b]); };
  const uint32_t drained = smem_u32(&bars[2 * kMaxStages + 4]);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
    for (int b = 0; b < 2; ++b) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), 8 * kGroup);
    mbar_init(drained, 1);
    mbar_init_fence();
    prefetch_tensor_map(&map_a), prefetch_tensor_map(&map_b);
  }
  __syncwarp();
  if (warp == 2) tmem_alloc<kGroup>(smem_u32(&tmem_base), kTmemColumns);
  tmem_fence_before();
  __syncthreads();
  if constexpr (kGroup == 2) cluster_sync_all();
  tmem_fence_after();
  const uint32_t tmem = tmem_base;
  const int32_t items = args.tiles_m * args.tiles_n * args.splits;
  const int32_t first = blockIdx.x / kGroup, step = gridDim.x / kGroup;
  if (kBKMajor && warp == 0 && first < items) {
    // The first stages of B (the weight, in the products that end in an
    // operator's own output) into L2 while the preceding grid drains: 48 rows
    // of A against 2 x 14336 x 4096, launches back to back, 40.5 us instead of
    // 41.7.  (Asking for a tile's rows of B a kilobyte at a time, ahead of the
    // loads all along, took 74.)
    const Item it = item_at(args, first);
    const DepthRange range = depth_range(args, it.split);
    const int32_t half = kGroup == 2 ? static_cast<int32_t>(rank) : lane % 2;
    const int32_t y = it.tn * c_cols + (E::kPaired ? half * args.pair_offset
                                                   : kGroup == 2 ? half * static_cast<int32_t>(b_rows) : 0);
    const int32_t k = range.first + (kGroup == 1 && E::kPaired ? lane / 2 : lane);
    if (k < range.last && k < range.first + stages) tma_prefetch_2d(&map_b, k * kDepthBlock, y);
    __syncwarp();
  }
  pdl_wait();

  if (warp == 0) {
    // Loads.  A pair's stage completes on the first CTA's barrier, which
    // expects the bytes of both.
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    int64_t issued = 0;
    for (int32_t t = args.waits.stall ? items : first; t < items && ok; t += step) {
      const Item it = item_at(args, t);
      const int32_t row = it.tm * (128 * kGroup) + static_cast<int32_t>(rank) * 128;
      const int32_t col = it.tn * c_cols;
      const DepthRange range = depth_range(args, it.split);
      for (int32_t k = range.first; k < range.last; ++k) {
        if (!mbar_wait_warp(empty(s), phase ^ 1, args.waits.limit_ns)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t a = ring + s * stage_bytes, b = a + a_bytes;
          const uint32_t bar = kGroup == 2 ? map_shared(full(s), 0) : full(s);
          if (rank == 0) mbar_arrive_expect_tx(full(s), kGroup * stage_bytes);
          const int32_t x = k * kDepthBlock;
          if constexpr (kAKMajor) {
            tma_load_2d<kGroup>(a, &map_a, x, row, bar);
          } else {
            tma_load_2d<kGroup>(a, &map_a, row, x, bar);
            tma_load_2d<kGroup>(a + 8192, &map_a, row + 64, x, bar);
          }
          if constexpr (E::kPaired && kGroup == 2) {
            // The first CTA's half of the tile's columns are gates, the other's ups.
            tma_load_2d<kGroup>(b, &map_b, x, col + static_cast<int32_t>(rank) * args.pair_offset, bar);
          } else if constexpr (E::kPaired) {
            tma_load_2d<kGroup>(b, &map_b, x, col, bar);
            tma_load_2d<kGroup>(b + c_cols * 128, &map_b, x, col + args.pair_offset, bar);
          } else {
            const int32_t r = col + static_cast<int32_t>(rank * b_rows);
            if constexpr (kBKMajor) {
              tma_load_2d<kGroup>(b, &map_b, x, r, bar);
            } else {
              for (uint32_t c = 0; c < b_rows; c += 64)
                tma_load_2d<kGroup>(b + c * 128, &map_b, r + static_cast<int32_t>(c), x, bar);
            }
          }
        }
        __syncwarp();
        ++issued;
        if (++s == stages) s = 0, phase ^= 1;
      }
    }
    pdl_trigger();
    if (!ok) {
      if (lane == 0) report_give_up(args.waits);
      // The stages issued last and not known to have landed.
      if (rank == 0) {
        for (int j = 0; j < stages && j < issued; ++j) {
          if (--s < 0) s = stages - 1, phase ^= 1;
          mbar_wait_warp(full(s), phase, kWaitLimitNs / 16);
        }
      }
    }
  } else if (warp == 1 && rank == 0) {
    const uint32_t idesc = mma_descriptor(std::is_same<T, __nv_bfloat16>::value, !kAKMajor, !kBKMajor,
                                          128 * kGroup, args.cols);
    // 16 of the stage's 64 terms per MMA: 32 bytes along a k-major tile's
    // rows, two atoms of a row-major tile.  In descriptors, 16 bytes a unit.
    constexpr uint32_t kAStep = (kAKMajor ? 32 : 2048) / 16, kBStep = (kBKMajor ? 32 : 2048) / 16;
    const uint64_t a_desc = smem_descriptor(ring, kAKMajor ? 16 : 8192);
    const uint64_t b_desc = smem_descriptor(ring + a_bytes, kBKMajor ? 16 : 8192);
    int s = 0;
    uint32_t phase = 0;
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    for (int32_t t = first; t < items && ok; t += step) {
      const DepthRange range = depth_range(args, t % args.splits);
      for (int32_t begin = range.first; begin < range.last && ok;) {
        const int32_t end = E::kSegment > 0 ? min(begin + E::kSegment, range.last) : range.last;
        if (!mbar_wait_warp(acc_empty(buf), buf_phase ^ 1, args.waits.limit_ns)) {
          ok = false;
          break;
        }
        tmem_fence_after();
        const uint32_t d = tmem + buf * (kTmemColumns / 2);
        for (int32_t k = begin; k < end; ++k) {
          if (!mbar_wait_warp(full(s), phase, args.waits.limit_ns)) {
            ok = false;
            break;
          }
          tmem_fence_after();
          if (elect_one()) {
            const uint64_t a = a_desc + s * (stage_bytes / 16), b = b_desc + s * (stage_bytes / 16);
#pragma unroll
            for (int j = 0; j < kDepthBlock / 16; ++j)
              mma_f16<kGroup>(d, a + j * kAStep, b + j * kBStep, idesc, k > begin || j > 0);
            mma_commit<kGroup>(empty(s));
            if (k + 1 == end) mma_commit<kGroup>(acc_full(buf));
          }
          __syncwarp();
          if (++s == stages) s = 0, phase ^= 1;
        }
        if (++buf == 2) buf = 0, buf_phase ^= 1;
        begin = end;
      }
    }
    if (!ok) {
      if (elect_one()) {
        report_give_up(args.waits);
        mma_commit<kGroup>(drained);
      }
      __syncwarp();
      mbar_wait_warp(drained, 0, kWaitLimitNs / 16);
    }
  } else if (warp >= 4) {
    const int quarter = warp % 4, group = (warp - 4) / 4;
    Lane l{scratch + (warp - 4) * kScratchWords, lane, 0, false};
    int buf = 0;
    uint32_t phase = 0;
    for (int32_t t = first; t < items; t += step) {
      const Item it = item_at(args, t);
      const int64_t i = static_cast<int64_t>(it.tm) * (128 * kGroup) + rank * 128 + quarter * 32 + lane;
      const int64_t j0 = static_cast<int64_t>(it.tn) * c_cols;
      l.inside = i < args.m, l.split = it.split;
      const bool any = __any_sync(~0u, l.inside);
      // Waits for the accumulators that are due next; their address.
      auto take = [&](uint32_t& acc) {
        if (!mbar_wait_warp(acc_full(buf), phase, args.waits.limit_ns)) {
          if (lane == 0) report_give_up(args.waits);
          return false;
        }
        tmem_fence_after();
        acc = tmem + buf * (kTmemColumns / 2) + (static_cast<uint32_t>(quarter * 32) << 16);
        return true;
      };
      // Hands them back to the MMA warp.
      auto give = [&] {
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_shared(acc_empty(buf), 0));
        if (++buf == 2) buf = 0, phase ^= 1;
      };
      uint32_t acc = 0;
      const int64_t part = it.tn * kColumnGroups + group;
      if constexpr (E::kSegment > 0) {
        const DepthRange range = depth_range(args, it.split);
        LaneSums sums;
        bool ok = true;
        for (int32_t begin = range.first; begin < range.last; begin += E::kSegment) {
          if (!(ok = take(acc))) break;
          if (any) sums.add(acc, begin == range.first, c_cols, group);
          give();
        }
        if (!ok) break;
        if (any) sums.run(epi, l, i, j0, args.n, c_cols, group, part);
      } else {
        if (!take(acc)) break;
        if (any) {
          if constexpr (E::kPaired) {
            run_epilogue(epi, l, i, j0, args.n, c_cols, group, part,
                         [&](int c, float (&v)[kChunk], int c2, float (&u)[kChunk]) {
                           tmem_load_32(acc + c, v);
                           tmem_load_32(acc + c2, u);
                           tmem_wait_load(v);
                           tmem_wait_load(u);
                         });
          } else {
            run_epilogue(epi, l, i, j0, args.n, c_cols, group, part, [&](int c, float (&v)[kChunk]) {
              tmem_load_32(acc + c, v);
              tmem_wait_load(v);
            });
          }
        }
        give();
      }
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if constexpr (kGroup == 2) cluster_sync_all();
  tmem_fence_after();
  if (warp == 2) tmem_dealloc<kGroup>(tmem, kTmemColumns);
}

// Adds up a split sum's shares and hands each value to the epilogue's
// point(i, j, ...); without shares (splits 0: sums of no terms) the values are
// zeros.  A thread takes four neighbouring columns.
template <typename E>
__global__ void __launch_bounds__(256)
    join_splits(const E epi, const SplitEpilogue<E::kPaired> shares, int32_t splits, int64_t m, int64_t n) {
  pdl_wait();
  const int64_t per_row = (n + 3) / 4, count = m * per_row;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < count; e += step) {
    const int64_t i = e / per_row, j = (e - i * per_row) * 4;
    float v[2][4] = {};
#pragma unroll 4
    for (int32_t s = 0; s < splits; ++s) {
      const float* p = shares.at(s, i) + j;
#pragma unroll
      for (int h = 0; h < (E::kPaired ? 2 : 1); ++h) {
        const float4 q = *reinterpret_cast<const float4*>(p + h * shares.ld);
        v[h][0] += q.x, v[h][1] += q.y, v[h][2] += q.z, v[h][3] += q.w;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (j + k >= n) break;
      if constexpr (E::kPaired) epi.point(i, j + k, v[0][k], v[1][k]);
      else epi.point(i, j + k, v[0][k]);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.

// A [rows, cols] operand as TMA reads it best: the tensor itself, or a copy of
// it with aligned rows taken from the workspace.  TMA needs rows on 16-byte
// boundaries.  Where a k-major operand's rows start inside a 32-byte sector the
// product takes up to half as long again (4096 x 2056 x 32768: 577 us; rows
// 2064 long 382), a copy 4 bytes an element, so such rows are copied where each
// element meets `reads` >= 2000 rows of the other operand in such products.
class AlignedRows {
 public:
  AlignedRows(Workspace& ws, const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t reads)
      : src_(static_cast<const uint16_t*>(p)), rows_(rows), cols_(cols), src_ld_(ld), ld_(ld) {
    if (rows <= 1) ld_ = round_up(cols > 0 ? cols : 1, 8);
    if (rows <= 0 || cols <= 0) return;
    const bool split = rows > 1 && (!aligned(p, 32) || ld % 16 != 0);
    if (tma_rows(p, rows, ld) && !(split && reads >= 2000)) return;
    ld_ = round_up(cols, 16);
    copies_ = true;
    copy_ = ws.take<uint16_t>(rows * ld_);
  }
  const uint16_t* data() const { return copies_ ? copy_ : src_; }
  int64_t ld() const { return ld_; }
  // Makes the copies of a call's two operands, or of one.
  static int prepare(const AlignedRows& x, const AlignedRows& w, cudaStream_t stream, unsigned flags);
  int prepare(cudaStream_t stream, unsigned flags) const { return prepare(*this, *this, stream, flags); }

 private:
  const uint16_t* src_;
  int64_t rows_, cols_, src_ld_, ld_;
  bool copies_ = false;
  uint16_t* copy_ = nullptr;
};

// How a product is cut up.
struct Tiling {
  int group;   // CTAs per tile
  int cols;    // accumulator columns of a tile
  int splits;  // shares of a tile's sum
};

// Products the rule in matmul.cu is asked about.
struct TilingQuery {
  int64_t m, n, depth;
  bool paired;
  bool b_k_major;
  bool may_split;
};
Tiling choose_tiling(const TilingQuery& q);

// The tensor map of `rows` x `cols` 16-bit elements, boxes of box_rows x 64.
int encode_rows(CUtensorMap* map, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows,
                const char* what);

// A product with its tiling and, where its sums are split, the workspace for
// the shares.  kAKMajor / kBKMajor: how the operands lie.
template <bool kPaired, bool kAKMajor, bool kBKMajor>
class PlannedProduct {
 public:
  PlannedProduct(Workspace& ws, int64_t m, int64_t n, int64_t depth, bool may_split = true) {
    tiling_ = choose_tiling({m, n, depth, kPaired, kBKMajor, may_split});
    shares_.rows = m;
    shares_.ld = round_up(n, kChunk);
    if (tiling_.splits > 1)
      shares_.partial = ws.take<float>(tiling_.splits * m * shares_.ld * (kPaired ? 2 : 1));
  }
  int c_cols() const { return tiling_.cols / (kPaired ? 2 : 1); }
  // How many `part` numbers the epilogue's `end` sees.
  int64_t parts(int64_t n) const { return (n + c_cols() - 1) / c_cols() * kColumnGroups; }
  // Shares that a sum of `depth` terms is dealt out to: as planned, but each
  // has a stage.  A product may have less depth than its plan (the vocabulary's
  // last piece); a share without a stage would have no MMA to finish it.
  int shares(int64_t depth) const {
    const int64_t stages = (depth + kDepthBlock - 1) / kDepthBlock;
    return static_cast<int>(tiling_.splits < stages ? tiling_.splits : stages);
  }

  template <typename T, typename E>
  int launch(const Product& q, const E& epi, cudaStream_t stream, unsigned flags, const char* what) const {
    if (q.m <= 0 || q.n <= 0) return HPRN_OK;
    if (q.depth <= 0) return join(q, epi, 0, stream, flags, what);
    const int n = shares(q.depth);
    if (n == 1) return launch_shares<T>(q, epi, 1, stream, flags, what);
    const int st = launch_shares<T>(q, shares_, n, stream, flags, what);
    return st != HPRN_OK ? st : join(q, epi, n, stream, flags, what);
  }

  // The same for products planned without shares and with depth > 0, for
  // epilogues that have no point().
  template <typename T, typename E>
  int launch_whole(const Product& q, const E& epi, cudaStream_t stream, unsigned flags,
                   const char* what) const {
    if (q.m <= 0 || q.n <= 0) return HPRN_OK;
    return launch_shares<T>(q, epi, 1, stream, flags, what);
  }

 private:
  template <typename T, typename E>
  int launch_shares(const Product& q, const E& epi, int shares, cudaStream_t stream, unsigned flags,
                    const char* what) const {
    return tiling_.group == 2 ? tiles<T, 2>(q, epi, shares, stream, flags, what)
                              : tiles<T, 1>(q, epi, shares, stream, flags, what);
  }

  template <typename T, int kGroup, typename E>
  int tiles(const Product& q, const E& epi, int shares, cudaStream_t stream, unsigned flags,
            const char* what) const {
    const DeviceInfo* dev = nullptr;
    int st = current_device(&dev);
    if (st != HPRN_OK) return st;
    MatmulArgs args;
    const int64_t rows = 128 * kGroup;
    const int64_t tm = (q.m + rows - 1) / rows, tn = (q.n + c_cols() - 1) / c_cols();
    const int64_t items = tm * tn * shares;
    if (items > (int64_t{1} << 30)) return fail(HPRN_ERR_INVALID_ARGUMENT, "product too large for one launch");
    args.tiles_m = static_cast<int32_t>(tm), args.tiles_n = static_cast<int32_t>(tn);
    args.splits = shares;
    args.depth_blocks = static_cast<int32_t>((q.depth + kDepthBlock - 1) / kDepthBlock);
    if (shares < 1 || shares > args.depth_blocks)
      return fail(HPRN_ERR_INVALID_ARGUMENT, std::string(what) + ": a share of a sum without terms");
    args.cols = tiling_.cols;
    args.a_rows = kAKMajor && q.m < 128 ? static_cast<int32_t>(round_up(q.m, 8)) : 128;
    const int stage = args.a_rows * 128 + tiling_.cols / kGroup * 128;
    // The MMA reads 128 rows of A whatever the stage holds: keep those inside the ring.
    const int stages = (kRingBytes - (128 - args.a_rows) * 128) / stage;
    args.stages = stages < kMaxStages ? stages : kMaxStages;
    // Under the power cap, 4096 x 4096 x 28672 and 8192 x 4096 x 65536: 698 and
    // 3091 us with bands of 16 against 718 and 3169 with 8 (4: 734, 3328; 32:
    // 696, 3290); the gradients' products differ by less than 1% from 4 to 16.
    args.band = kAKMajor && kBKMajor ? 16 : 8;
    args.m = q.m, args.n = q.n, args.pair_offset = static_cast<int32_t>(q.pair_offset);
    if ((st = waits_of(dev, &args.waits, what)) != HPRN_OK) return st;
    CUtensorMap map_a, map_b;
    st = kAKMajor ? encode_rows(&map_a, q.a.p, q.m, q.depth, q.a.ld, args.a_rows, what)
                  : encode_rows(&map_a, q.a.p, q.depth, q.m, q.a.ld, kDepthBlock, what);
    if (st != HPRN_OK) return st;
    const int64_t b_rows = kPaired ? q.pair_offset + q.n : q.n;
    const int b_box = kPaired ? c_cols() : tiling_.cols / kGroup;
    st = kBKMajor ? encode_rows(&map_b, q.b.p, b_rows, q.depth, q.b.ld, b_box, what)
                  : encode_rows(&map_b, q.b.p, q.depth, b_rows, q.b.ld, kDepthBlock, what);
    if (st != HPRN_OK) return st;
    auto fn = matmul_tiles<T, E, kGroup, kAKMajor, kBKMajor>;
    if ((st = allow_smem(dev, reinterpret_cast<const void*>(fn), kMatmulSmem, what)) != HPRN_OK) return st;
    const int64_t most = dev->sm_count / kGroup;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(static_cast<unsigned>((items < most ? items : most) * kGroup), 1, 1);
    cfg.blockDim = dim3(kMatmulThreads, 1, 1);
    cfg.dynamicSmemBytes = kMatmulSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    if (kGroup == 2) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim.x = 2;
      attr[cfg.numAttrs].val.clusterDim.y = 1;
      attr[cfg.numAttrs].val.clusterDim.z = 1;
      ++cfg.numAttrs;
    }
    if (flags & HPRN_LAUNCH_PDL) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
      ++cfg.numAttrs;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, map_a, map_b, args, epi);
    if (e != cudaSuccess)
      return fail(HPRN_ERR_CUDA, std::string(what) + " launch failed: " + cudaGetErrorString(e));
    return ok();
  }

  template <typename E>
  int join(const Product& q, const E& epi, int splits, cudaStream_t stream, unsigned flags,
           const char* what) const {
    const int64_t ctas = (q.m * ((q.n + 3) / 4) + 255) / 256, most = 148 * 16;
    return launch_rows(join_splits<E>, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(256),
                       stream, flags, what, epi, shares_, splits, q.m, q.n);
  }

  Tiling tiling_;
  SplitEpilogue<kPaired> shares_;
};

}  // namespace hprn

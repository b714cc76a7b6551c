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
// What happens to a row of accumulators is an epilogue: a struct whose methods
// one thread calls for the row it holds, in order:
//   Row begin(i)                          per-row state
//   chunk(Row&, i, j, const float (&v)[32])   columns j .. j + 31 of row i
//   end(Row&, i, tile)                    after the tile's last chunk
// A "paired" epilogue (kPaired) gets two accumulators for each column: those
// of B's rows j and pair_offset + j (gate and up).
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

constexpr int kChunk = 32;  // accumulators a thread hands to an epilogue at once

// ---------------------------------------------------------------------------
// Columns j .. j + 31 of one row as 16-bit values: full 32-byte sectors where
// the row allows, element by element at a ragged edge.
template <typename T>
__device__ __forceinline__ void store_chunk(uint16_t* row, int64_t j, int64_t n,
                                            const float (&v)[kChunk]) {
  uint16_t* p = row + j;
  if (j + kChunk <= n && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Vec<32> o;
#pragma unroll
      for (int k = 0; k < 8; ++k) o.w[k] = pack2<T>(v[16 * h + 2 * k], v[16 * h + 2 * k + 1]);
      st_global<32>(p + 16 * h, o);
    }
  } else if (j + kChunk <= n && (reinterpret_cast<uintptr_t>(p) & 3) == 0) {
#pragma unroll
    for (int k = 0; k < kChunk / 2; ++k)
      reinterpret_cast<uint32_t*>(p)[k] = pack2<T>(v[2 * k], v[2 * k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < kChunk; ++k)
      if (j + k < n) p[k] = pack1<T>(v[k]);
  }
}

__device__ __forceinline__ void store_chunk_f32(float* row, int64_t j, int64_t n,
                                                const float (&v)[kChunk]) {
  float* p = row + j;
  if (j + kChunk <= n && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      Vec<32> o;
#pragma unroll
      for (int k = 0; k < 8; ++k) o.w[k] = __float_as_uint(v[8 * h + k]);
      st_global<32>(p + 8 * h, o);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kChunk; ++k)
      if (j + k < n) p[k] = v[k];
  }
}

// ---------------------------------------------------------------------------
// C itself, optionally summed over several products (the pieces of a long
// sum) in an fp32 buffer: `sum` holds the earlier pieces' total; `last` says
// whether this product finishes it.  The total is rounded to 16 bits once.
template <typename T>
struct StoreEpilogue {
  static constexpr bool kPaired = false;
  uint16_t* out = nullptr;  // rows of `ld` elements; written by the last piece
  int64_t ld = 0;
  int64_t n = 0;
  float* sum = nullptr;  // m x n, or null when there is one piece
  bool first = true;
  bool last = true;
  const float* scale = nullptr;  // one float that multiplies the total, or null

  struct Row {
    float scale;
  };
  __device__ __forceinline__ Row begin(int64_t) const { return Row{scale ? *scale : 1.0f}; }
  __device__ __forceinline__ void chunk(Row& s, int64_t i, int64_t j, const float (&acc)[kChunk]) const {
    float v[kChunk];
#pragma unroll
    for (int k = 0; k < kChunk; ++k) v[k] = acc[k];
    if (!first) {
      const float* p = sum + i * n + j;
      if (j + kChunk <= n && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
        for (int k = 0; k < kChunk; k += 4) {
          const float4 q = *reinterpret_cast<const float4*>(p + k);
          v[k] += q.x, v[k + 1] += q.y, v[k + 2] += q.z, v[k + 3] += q.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < kChunk; ++k)
          if (j + k < n) v[k] += p[k];
      }
    }
    if (!last) {
      store_chunk_f32(sum + i * n, j, n, v);
    } else {
#pragma unroll
      for (int k = 0; k < kChunk; ++k) v[k] *= s.scale;
      store_chunk<T>(out + i * ld, j, n, v);
    }
  }
  __device__ __forceinline__ void end(Row&, int64_t, int64_t) const {}
};

// ---------------------------------------------------------------------------
// The kernel: a persistent grid of CTAs (or pairs of CTAs), each taking tiles
// of C in turn.  In a CTA
//   warp 0    one thread keeps a ring of shared-memory stages filled by TMA,
//             64 of the sum's terms a stage;
//   warp 1    (of the pair's first CTA) one thread issues the MMAs of a stage
//             as it arrives, into one of two TMEM accumulators;
//   warp 2    allocates and frees TMEM;
//   warps 4-7 hand the finished accumulator's rows to the epilogue, one row a
//             thread, while the next tile's MMAs fill the other one.
// Tiles are 128 rows x kN columns per CTA, or 256 x kN per pair of CTAs.
//
// Every wait has a limit (mbar_wait_bounded).  A role whose wait runs out
// counts itself in `timeouts` and stops; the others' waits then run out too,
// and the CTA ends after its copies and MMAs in flight.
constexpr int kDepthBlock = 64;  // 16-bit elements in a 128-byte row of a stage
constexpr int kMatmulThreads = 256;

template <int kGroup, int kN>
struct Tile {
  static constexpr int kRows = 128 * kGroup;         // of C, per pair
  static constexpr int kABytes = 128 * 128;          // a CTA's part of A's stage
  static constexpr int kBRows = kN / kGroup;         // B's rows in a CTA's stage
  static constexpr int kBBytes = kBRows * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = (196 * 1024) / kStageBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + 1024;  // + alignment of the ring
  static constexpr int kTmemColumns = 2 * kN < 32 ? 32 : 2 * kN;
};

struct MatmulArgs {
  int32_t tiles_m, tiles_n;
  int32_t depth_blocks;
  int64_t m, n;
  int32_t pair_offset;
  unsigned* timeouts;
};

// Tile `t` of the order tiles are taken in: bands of kBand tile rows, down a
// band's columns first, so that the tiles in flight at one time cover a
// near-square part of C and share A's and B's rows in L2.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_at(const MatmulArgs& a, int32_t t, int32_t* tm, int32_t* tn) {
  const int32_t band_tiles = kBand * a.tiles_n;
  const int32_t band = t / band_tiles;
  const int32_t first = band * kBand;
  const int32_t rows = min(kBand, a.tiles_m - first);
  const int32_t in = t - band * band_tiles;
  *tm = first + in % rows;
  *tn = in / rows;
}

template <typename T, typename E, int kGroup, int kN, bool kAKMajor, bool kBKMajor>
__global__ void __launch_bounds__(kMatmulThreads, 1)
    matmul_tiles(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const MatmulArgs args, const E epi) {
  using L = Tile<kGroup, kN>;
  constexpr int kStages = L::kStages;
  constexpr int kCols = E::kPaired ? kN / 2 : kN;  // columns of C per tile
  static_assert(kBKMajor || L::kBRows % 64 == 0, "row-major tiles are blocks of 64 rows");
  extern __shared__ unsigned char ring_mem[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 5];
  __shared__ uint32_t tmem_base;
  const uint32_t ring = (smem_u32(ring_mem) + 1023) & ~1023u;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = kGroup == 2 ? cluster_rank() : 0;
  auto full = [&](int s) { return smem_u32(&bars[s]); };
  auto empty = [&](int s) { return smem_u32(&bars[kStages + s]); };
  auto acc_full = [&](int b) { return smem_u32(&bars[2 * kStages + b]); };
  auto acc_empty = [&](int b) { return smem_u32(&bars[2 * kStages + 2 + b]); };
  const uint32_t drained = smem_u32(&bars[2 * kStages + 4]);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
    for (int b = 0; b < 2; ++b) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), 4 * kGroup);
    mbar_init(drained, 1);
    mbar_init_fence();
    if (args.depth_blocks > 0) prefetch_tensor_map(&map_a), prefetch_tensor_map(&map_b);
  }
  __syncwarp();
  if (warp == 2) tmem_alloc<kGroup>(smem_u32(&tmem_base), L::kTmemColumns);
  tmem_fence_before();
  __syncthreads();
  if constexpr (kGroup == 2) cluster_sync_all();
  tmem_fence_after();
  const uint32_t tmem = tmem_base;
  pdl_wait();

  const int32_t tiles = args.tiles_m * args.tiles_n;
  const int32_t first = blockIdx.x / kGroup, step = gridDim.x / kGroup;

  if (warp == 0 && lane == 0) {
    // Loads.  A pair's stage completes on the first CTA's barrier, which
    // expects the bytes of both.
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    int64_t issued = 0;
    for (int32_t t = first; t < tiles && ok; t += step) {
      int32_t tm, tn;
      tile_at(args, t, &tm, &tn);
      const int32_t row = tm * L::kRows + static_cast<int32_t>(rank) * 128;
      const int32_t col = tn * kCols;
      for (int32_t k = 0; k < args.depth_blocks; ++k) {
        if (!mbar_wait_bounded(empty(s), phase ^ 1)) {
          ok = false;
          break;
        }
        const uint32_t a = ring + s * L::kStageBytes, b = a + L::kABytes;
        const uint32_t bar = kGroup == 2 ? map_shared(full(s), 0) : full(s);
        if (rank == 0) mbar_arrive_expect_tx(full(s), kGroup * L::kStageBytes);
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
          tma_load_2d<kGroup>(b + L::kBBytes / 2, &map_b, x, col + args.pair_offset, bar);
        } else {
          const int32_t r = col + static_cast<int32_t>(rank) * L::kBRows;
          if constexpr (kBKMajor) {
            tma_load_2d<kGroup>(b, &map_b, x, r, bar);
          } else {
#pragma unroll
            for (int c = 0; c < L::kBRows / 64; ++c)
              tma_load_2d<kGroup>(b + c * 8192, &map_b, r + c * 64, x, bar);
          }
        }
        ++issued;
        if (++s == kStages) s = 0, phase ^= 1;
      }
    }
    pdl_trigger();
    if (!ok) {
      atomicAdd(args.timeouts, 1u);
      // The stages issued last and not known to have landed.
      if (rank == 0) {
        for (int j = 0; j < kStages && j < issued; ++j) {
          if (--s < 0) s = kStages - 1, phase ^= 1;
          mbar_wait_bounded(full(s), phase, kWaitLimitNs / 16);
        }
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    constexpr uint32_t idesc =
        mma_descriptor(std::is_same<T, __nv_bfloat16>::value, !kAKMajor, !kBKMajor, 128 * kGroup, kN);
    // 16 of the stage's 64 terms per MMA: 32 bytes along a k-major tile's
    // rows, two atoms of a row-major tile.
    constexpr uint32_t kAStep = kAKMajor ? 32 : 2048, kBStep = kBKMajor ? 32 : 2048;
    int s = 0;
    uint32_t phase = 0;
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    for (int32_t t = first; t < tiles && ok && args.depth_blocks > 0; t += step) {
      if (!mbar_wait_bounded(acc_empty(buf), buf_phase ^ 1)) {
        ok = false;
        break;
      }
      tmem_fence_after();
      const uint32_t d = tmem + buf * kN;
      for (int32_t k = 0; k < args.depth_blocks; ++k) {
        if (!mbar_wait_bounded(full(s), phase)) {
          ok = false;
          break;
        }
        tmem_fence_after();
        const uint32_t a = ring + s * L::kStageBytes, b = a + L::kABytes;
#pragma unroll
        for (int j = 0; j < kDepthBlock / 16; ++j)
          mma_f16<kGroup>(d, smem_descriptor(a + j * kAStep, kAKMajor ? 16 : 8192),
                          smem_descriptor(b + j * kBStep, kBKMajor ? 16 : 8192), idesc, k > 0 || j > 0);
        mma_commit<kGroup>(empty(s));
        if (++s == kStages) s = 0, phase ^= 1;
      }
      if (!ok) break;
      mma_commit<kGroup>(acc_full(buf));
      if (++buf == 2) buf = 0, buf_phase ^= 1;
    }
    if (!ok) {
      atomicAdd(args.timeouts, 1u);
      mma_commit<kGroup>(drained);
      mbar_wait_bounded(drained, 0, kWaitLimitNs / 16);
    }
  } else if (warp >= 4) {
    const int quarter = warp - 4;
    int buf = 0;
    uint32_t phase = 0;
    for (int32_t t = first; t < tiles; t += step) {
      int32_t tm, tn;
      tile_at(args, t, &tm, &tn);
      const int64_t i = static_cast<int64_t>(tm) * L::kRows + rank * 128 + quarter * 32 + lane;
      const int64_t j0 = static_cast<int64_t>(tn) * kCols;
      const bool any = args.depth_blocks > 0;
      if (any) {
        // Every lane waits for itself; a warp goes on together or not at all.
        const bool arrived = mbar_wait_bounded(acc_full(buf), phase);
        if (!__all_sync(~0u, arrived)) {
          if (lane == 0) atomicAdd(args.timeouts, 1u);
          break;
        }
        tmem_fence_after();
      }
      const uint32_t acc = tmem + buf * kN + (static_cast<uint32_t>(quarter * 32) << 16);
      const bool inside = i < args.m;
      typename E::Row row{};
      if (inside) row = epi.begin(i);
#pragma unroll 1
      for (int c = 0; c < kCols && j0 + c < args.n; c += kChunk) {
        float v[kChunk];
        if (any) {
          tmem_load_32(acc + c, v);
        } else {
#pragma unroll
          for (int k = 0; k < kChunk; ++k) v[k] = 0.f;
        }
        if constexpr (E::kPaired) {
          float u[kChunk];
          if (any) {
            tmem_load_32(acc + kCols + c, u);
            tmem_wait_load(v);
            tmem_wait_load(u);
          } else {
#pragma unroll
            for (int k = 0; k < kChunk; ++k) u[k] = 0.f;
          }
          if (inside) epi.chunk(row, i, j0 + c, v, u);
        } else {
          if (any) tmem_wait_load(v);
          if (inside) epi.chunk(row, i, j0 + c, v);
        }
        __syncwarp();
      }
      if (inside) epi.end(row, i, tn);
      if (any) {
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_shared(acc_empty(buf), 0));
        if (++buf == 2) buf = 0, phase ^= 1;
      }
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if constexpr (kGroup == 2) cluster_sync_all();
  tmem_fence_after();
  if (warp == 2) tmem_dealloc<kGroup>(tmem, L::kTmemColumns);
}

// ---------------------------------------------------------------------------
// Host side.

// The tile shape a product takes.
struct Tiling {
  int group;  // CTAs per tile
  int n;      // accumulator columns
};

template <typename E>
inline Tiling tiling_of(const Product&) {
  return Tiling{2, 256};
}

// Columns of C that one `end` call covers (how an epilogue with per-tile
// results sizes them).
template <typename E>
inline int64_t product_tiles(const Product& q) {
  const int cols = tiling_of<E>(q).n / (E::kPaired ? 2 : 1);
  return (q.n + cols - 1) / cols;
}

// TMA reads rows that start on 16-byte boundaries.
inline bool tma_rows(const void* p, int64_t rows, int64_t ld) {
  return aligned(p, 16) && (rows <= 1 || ld % 8 == 0);
}

// A [rows, cols] operand TMA can read: the tensor itself, or a copy of it with
// aligned rows taken from the workspace.
class AlignedRows {
 public:
  AlignedRows(Workspace& ws, const void* p, int64_t rows, int64_t cols, int64_t ld)
      : src_(static_cast<const uint16_t*>(p)), rows_(rows), cols_(cols), src_ld_(ld), ld_(ld) {
    if (rows <= 1) ld_ = round_up(cols > 0 ? cols : 1, 8);
    if (rows > 0 && cols > 0 && !tma_rows(p, rows, ld)) {
      ld_ = round_up(cols, 8);
      copies_ = true;
      copy_ = ws.take<uint16_t>(rows * ld_);
    }
  }
  int prepare(cudaStream_t stream, unsigned flags) const;
  const uint16_t* data() const { return copies_ ? copy_ : src_; }
  int64_t ld() const { return ld_; }

 private:
  const uint16_t* src_;
  int64_t rows_, cols_, src_ld_, ld_;
  bool copies_ = false;
  uint16_t* copy_ = nullptr;
};

// The tensor map of `rows` x `cols` 16-bit elements, boxes of box_rows x 64.
int encode_rows(CUtensorMap* map, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows,
                const char* what);
// The counter of waits that ran out, on the current device.
int timeout_counter(unsigned** out);
// Raises a kernel's dynamic shared memory limit, once per device.
int allow_smem(const DeviceInfo* dev, const void* fn, int bytes, const char* what);

template <typename T, typename E, int kGroup, int kN, bool kAKMajor, bool kBKMajor>
int launch_tiles(const Product& q, const E& epi, cudaStream_t stream, unsigned flags, const char* what) {
  using L = Tile<kGroup, kN>;
  const DeviceInfo* dev = nullptr;
  int st = current_device(&dev);
  if (st != HPRN_OK) return st;
  const int cols = E::kPaired ? kN / 2 : kN;
  MatmulArgs args;
  const int64_t tm = (q.m + L::kRows - 1) / L::kRows, tn = (q.n + cols - 1) / cols;
  if (tm * tn > (int64_t{1} << 30)) return fail(HPRN_ERR_INVALID_ARGUMENT, "product too large for one launch");
  args.tiles_m = static_cast<int32_t>(tm), args.tiles_n = static_cast<int32_t>(tn);
  args.depth_blocks = static_cast<int32_t>((q.depth + kDepthBlock - 1) / kDepthBlock);
  args.m = q.m, args.n = q.n, args.pair_offset = static_cast<int32_t>(q.pair_offset);
  if ((st = timeout_counter(&args.timeouts)) != HPRN_OK) return st;
  CUtensorMap map_a = {}, map_b = {};
  if (q.depth > 0) {
    st = kAKMajor ? encode_rows(&map_a, q.a.p, q.m, q.depth, q.a.ld, 128, what)
                  : encode_rows(&map_a, q.a.p, q.depth, q.m, q.a.ld, kDepthBlock, what);
    if (st != HPRN_OK) return st;
    const int64_t b_rows = E::kPaired ? q.pair_offset + q.n : q.n;
    const int b_box = E::kPaired ? kN / 2 : L::kBRows;
    st = kBKMajor ? encode_rows(&map_b, q.b.p, b_rows, q.depth, q.b.ld, b_box, what)
                  : encode_rows(&map_b, q.b.p, q.depth, b_rows, q.b.ld, kDepthBlock, what);
    if (st != HPRN_OK) return st;
  }
  auto fn = matmul_tiles<T, E, kGroup, kN, kAKMajor, kBKMajor>;
  if ((st = allow_smem(dev, reinterpret_cast<const void*>(fn), L::kSmemBytes, what)) != HPRN_OK) return st;
  const int64_t most = dev->sm_count / kGroup;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>((tm * tn < most ? tm * tn : most) * kGroup), 1, 1);
  cfg.blockDim = dim3(kMatmulThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kSmemBytes;
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

// kAKMajor / kBKMajor: how the operands lie, Operand::k_major at compile time.
template <typename T, bool kAKMajor, bool kBKMajor, typename E>
int launch_product(const Product& q, const E& epi, cudaStream_t stream, unsigned flags, const char* what) {
  return launch_tiles<T, E, 2, 256, kAKMajor, kBKMajor>(q, epi, stream, flags, what);
}

}  // namespace hprn

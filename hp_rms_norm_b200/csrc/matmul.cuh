// Matrix products with the surrounding operator's arithmetic applied to the
// accumulators before anything reaches memory.
//
// A product is C[i, j] = sum_k A(i, k) * B(j, k) for i < m, j < n, k < depth,
// 16-bit operands (bf16 or fp16), fp32 accumulation.  Each operand lies in
// memory either with k contiguous ("k-major": element (i, k) at p[i * ld + k])
// or with i contiguous ("row-major in i": p[k * ld + i]), so the three products
// of a linear layer (forward, gradient of the input, gradient of the weight)
// read the tensors as they are.
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

#include "runtime.cuh"
#include "vec.cuh"

namespace hprn {

struct Operand {
  const uint16_t* p = nullptr;
  int64_t ld = 0;
  bool k_major = true;
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
// The simplest kernel that is right for every operand: fp32 products of a
// 64 x 64 tile, 16 deep, in shared memory.
constexpr int kTile = 64;
constexpr int kDepth = 16;

template <typename T, typename E>
__global__ void __launch_bounds__(256) matmul_tile(Product q, E epi) {
  __shared__ float as[kDepth][kTile + 1];
  __shared__ float bs[kDepth][kTile + 1];
  __shared__ float cs[kTile][kTile + 1];
  constexpr int kCols = E::kPaired ? kTile / 2 : kTile;  // columns of C per tile
  const int64_t i0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const int64_t j0 = static_cast<int64_t>(blockIdx.x) * kCols;
  const int tid = threadIdx.x;
  const int tx = tid % 16, ty = tid / 16;
  pdl_wait();
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < q.depth; k0 += kDepth) {
    for (int e = tid; e < kTile * kDepth; e += 256) {
      const int ra = q.a.k_major ? e / kDepth : e % kTile;
      const int ka = q.a.k_major ? e % kDepth : e / kTile;
      const int64_t i = i0 + ra, k = k0 + ka;
      float v = 0.f;
      if (i < q.m && k < q.depth)
        v = unpack1<T>(q.a.p[q.a.k_major ? i * q.a.ld + k : k * q.a.ld + i]);
      as[ka][ra] = v;
      const int rb = q.b.k_major ? e / kDepth : e % kTile;
      const int kb = q.b.k_major ? e % kDepth : e / kTile;
      const bool second = E::kPaired && rb >= kCols;
      int64_t j = j0 + (second ? rb - kCols : rb);
      const int64_t kk = k0 + kb;
      v = 0.f;
      if (j < q.n && kk < q.depth) {
        if (second) j += q.pair_offset;
        v = unpack1<T>(q.b.p[q.b.k_major ? j * q.b.ld + kk : kk * q.b.ld + j]);
      }
      bs[kb][rb] = v;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) a[x] = as[k][ty * 4 + x], b[x] = bs[k][tx + 16 * x];
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = fmaf(a[x], b[y], acc[x][y]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) cs[ty * 4 + x][tx + 16 * y] = acc[x][y];
  __syncthreads();
  if (tid >= kTile || i0 + tid >= q.m) return;
  const int64_t i = i0 + tid;
  auto row = epi.begin(i);
  for (int c = 0; c < kCols; c += kChunk) {
    if (j0 + c >= q.n) break;
    float v[kChunk];
#pragma unroll
    for (int k = 0; k < kChunk; ++k) v[k] = cs[tid][c + k];
    if constexpr (E::kPaired) {
      float u[kChunk];
#pragma unroll
      for (int k = 0; k < kChunk; ++k) u[k] = cs[tid][kCols + c + k];
      epi.chunk(row, i, j0 + c, v, u);
    } else {
      epi.chunk(row, i, j0 + c, v);
    }
  }
  epi.end(row, i, blockIdx.x);
}

// Columns of C that one `end` call covers (how an epilogue with per-tile
// results sizes them).
template <typename E>
inline int64_t product_tiles(int64_t n) {
  const int cols = E::kPaired ? kTile / 2 : kTile;
  return (n + cols - 1) / cols;
}

template <typename T, typename E>
int launch_product(const Product& q, const E& epi, cudaStream_t stream, const char* what) {
  const dim3 grid(static_cast<unsigned>(product_tiles<E>(q.n)),
                  static_cast<unsigned>((q.m + kTile - 1) / kTile));
  matmul_tile<T, E><<<grid, 256, 0, stream>>>(q, epi);
  return check_launch(what);
}

}  // namespace hprn

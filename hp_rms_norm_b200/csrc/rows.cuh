// What the row kernels of gated_norm.cu and int8.cu share: vectors of 16-bit
// elements as pairs of floats, and sums over the threads that hold a row.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "vec.cuh"

namespace hprn {

// The elements of a vector in pairs; a vector of one element is a pair with a 0.
template <int VEC>
struct Pairs {
  static constexpr int kCount = VEC >= 4 ? VEC / 4 : 1;
};

template <typename T, int VEC>
__device__ __forceinline__ float2 pair_of(const Vec<VEC>& v, int e) {
  if constexpr (VEC == 2) return make_float2(unpack1<T>(v.h), 0.f);
  else return unpack2<T>(v.w[e]);
}

template <typename T, int VEC>
__device__ __forceinline__ void set_pair(Vec<VEC>& v, int e, float2 f) {
  if constexpr (VEC == 2) v.h = pack1<T>(f.x);
  else v.w[e] = pack2<T>(f.x, f.y);
}

// Pair e of the vector that starts at p.
template <typename T, int VEC>
__device__ __forceinline__ float2 load_pair(const uint16_t* p, int e) {
  if constexpr (VEC == 2) return make_float2(unpack1<T>(*p), 0.f);
  else return unpack2<T>(reinterpret_cast<const uint32_t*>(p)[e]);
}

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The sum over the `warps` warps from `first_warp` that hold a row, the same
// bits in every thread.  Every thread of the CTA calls it where warps > 1; a
// row's next sum takes another buffer `part`.
__device__ __forceinline__ float row_sum(float v, float* part, int warps, int first_warp) {
  v = warp_total(v);
  if (warps == 1) return v;
  const int lane = threadIdx.x % 32;
  if (lane == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  return warp_total(lane < warps ? part[first_warp + lane] : 0.f);
}

}  // namespace hprn

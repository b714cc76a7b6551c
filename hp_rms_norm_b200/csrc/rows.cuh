// What the row kernels of gated_norm.cu and int8.cu share: vectors of 16-bit
// elements as pairs of floats, sums over the threads that hold a row, and rows that
// start anywhere.
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

// ---------------------------------------------------------------------------
// Rows that start anywhere: vectors of eight elements by the 16-byte granules of
// memory that they lie in, two loads and a shift instead of eight loads.

// Elements o to o + 7 of the sixteen in w, into w[0..3]; o the same in a warp.
__device__ __forceinline__ void shift_down(uint32_t (&w)[8], int o) {
  if (o & 4) {
#pragma unroll
    for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
  }
  if (o & 2) {
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
  }
  if (o & 1) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
  }
}

__host__ __device__ __forceinline__ int granule_offset(const void* row) {
  return static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / 2;
}

// Zeros for the elements of vector v behind a row of n.
__device__ __forceinline__ void clear_tail(uint32_t (&w)[4], int v, int n) {
  const int left = n - 8 * v;
  if (left >= 8) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = 2 * k >= left ? 0 : 2 * k + 1 >= left ? w[k] & 0xffffu : w[k];
}

// A row of n elements and whether the granules its ends lie in may be read whole.
struct LooseRow {
  const uint16_t* p;
  int n;
  bool low, high;
};
// Row i of `rows` with a stride between them: the granules reach into the rows beside
// it, but not out of the tensor.  A row's last warp has lanes behind its end; what they
// read is thrown away, so `high` asks for room for all of them (where each lane asks
// for itself 3084 x 5001 forward takes 54 us for 50).
__host__ __device__ __forceinline__ LooseRow loose_row(const uint16_t* base, int64_t i, int64_t rows, int64_t stride,
                                                       int n) {
  const uint16_t* p = base + i * stride;
  const int lanes = (n + 255) & ~255;  // the elements of whole warps
  return LooseRow{p, n, granule_offset(p) <= i * stride, (rows - 1 - i) * stride >= lanes - n + 8};
}

// How vector v of a row is read: by its granule, whose first element is 8 v - o of the
// row, and the next one, or else by those of its elements that lie before the row's end.
__host__ __device__ __forceinline__ bool reads_granule(const LooseRow& r, int o, int v) {
  // (What a granule behind the row's last whole one holds of the next row, or of
  // nothing.)
  return (v > 0 || o == 0 || r.low) && (r.high || 8 * (v + (o > 0 ? 2 : 1)) - o <= r.n);
}
__host__ __device__ __forceinline__ bool reads_next(const LooseRow& r, int o, int v) {
  return o > 0 && 8 * (v + 1) - o < r.n;
}

// Elements 8 v to 8 v + 7, zeros past the row's end.
__device__ __forceinline__ void load_loose(uint32_t (&out)[4], const LooseRow& r, int v) {
  const int o = granule_offset(r.p);
  const uint4* g = reinterpret_cast<const uint4*>(r.p - o) + v;
  if (reads_granule(r, o, v)) {
    const uint4 a = *g;
    uint32_t w[8] = {a.x, a.y, a.z, a.w, 0, 0, 0, 0};
    if (o > 0) {
      if (reads_next(r, o, v)) {
        const uint4 b = g[1];
        w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
      }
      shift_down(w, o);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = w[k];
    clear_tail(out, v, r.n);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int j = 8 * v + 2 * k;
    const uint32_t lo = j < r.n ? r.p[j] : 0, hi = j + 1 < r.n ? r.p[j + 1] : 0;
    out[k] = lo | hi << 16;
  }
}

// What of a warp's 256 neighbouring units (elements, or bytes) of a row of n lies in
// granules of eight that are not whole: up to seven before the first whole one, up to
// seven behind the last.  Lanes 0 to 15 take one each.
struct LooseEdge {
  int unit, lane, at;  // of the row; the lane that has it, its place there
  bool mine;
};
__device__ __forceinline__ LooseEdge loose_edge(int n, int v, int o) {
  const int lane = threadIdx.x % 32, first = 8 * (v - lane), last = min(n, first + 256);
  const int head = min(first + ((8 - o) & 7), last), tail = max(last - ((last + o) & 7), head);
  const int j = lane < 8 ? first + lane : tail + lane - 8;
  return LooseEdge{j, (j - first) / 8, j & 7, lane < 8 ? j < head : lane < 16 && j < last};
}

// Elements 8 v to 8 v + 7 of a row of n, v neighbouring in neighbouring lanes: the
// granules inside a warp's span whole, put together with the lane before, what is
// over at its ends by an element a lane.  Whole warps whose first lane is inside
// the row; v may lie past it.  (Ends stored by the lanes that hold them, element by
// element: 3084 x 1001 forward 13.6 us, now 12.2.)
__device__ __forceinline__ void store_loose(uint16_t* row, int n, int v, const uint32_t (&w)[4]) {
  const int o = granule_offset(row), lane = threadIdx.x % 32;
  const LooseEdge edge = loose_edge(n, v, o);
  uint32_t both[8], over = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    both[4 + k] = w[k], both[k] = __shfl_up_sync(~0u, w[k], 1);
    const uint32_t other = __shfl_sync(~0u, w[k], edge.lane);
    over = edge.at / 2 == k ? other : over;
  }
  if (edge.mine) row[edge.unit] = static_cast<uint16_t>(edge.at & 1 ? over >> 16 : over);
  if (o > 0) shift_down(both, 8 - o);
  else both[0] = w[0], both[1] = w[1], both[2] = w[2], both[3] = w[3];
  if ((lane > 0 || o == 0) && 8 * v - o + 8 <= n)
    *reinterpret_cast<uint4*>(row + 8 * v - o) = make_uint4(both[0], both[1], both[2], both[3]);
}

}  // namespace hprn

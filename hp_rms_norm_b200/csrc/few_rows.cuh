// Products of few rows with a large weight.  The weight's bytes bound them, so it is
// read straight into registers, without the pipeline of stages (matmul.cuh) whose
// filling and draining costs 6 us.  A CTA takes 16 or 32 rows of the weight; its
// warps take shares of the sums in blocks of 128 bytes, the loads of several in
// flight; the products are mma.sync's 16 weight rows x 8 rows of x x 32 bytes.  A
// lane's 32 bytes of a block are the terms that the instruction wants of it in some
// order, the same for both operands, which is all that a sum needs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "vec.cuh"

namespace hprn {

constexpr int kFewWarps = 8;

struct FewOperands {
  const uint8_t* x;  // rows of `bytes`
  const uint8_t* w;
  int64_t x_ld, w_ld;  // in bytes
  int32_t rows, channels, bytes;
  int32_t first_wave;  // CTAs that are resident at once
};

// What the sums are held in, and the instruction.
template <typename T>
struct FewMma {
  using Sum = float;
  // Blocks that the tensor cores sum before a rounded addition: 512 terms, as the
  // tiles of the softmax operators (vocabulary.cuh).
  static constexpr int kSegment = 8;
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
};
template <>
__device__ __forceinline__ void FewMma<__nv_bfloat16>::mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                           uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void FewMma<__half>::mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
struct FewMma<int8_t> {
  using Sum = int;
  static constexpr int kSegment = 0;  // exact
  static __device__ __forceinline__ void mma(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// A CTA's share of the sums: [warp][row of x][weight row].
template <typename T, int kTiles, int kWide>
using FewSums = typename FewMma<T>::Sum[kFewWarps][8 * kTiles][16 * kWide + 1];

// The CTA's products with the 16 kWide weight rows from `channel` on: each warp's
// share into `sums`, which the caller adds up after this (a barrier is its end).
// kTiles: tiles of 8 rows of x.
// kAlign: what every row's start and length are multiples of, 16 or 8 bytes.
template <typename T, int kTiles, int kWide, int kAlign>
__device__ __forceinline__ void few_products(const FewOperands& a, int channel, FewSums<T, kTiles, kWide>& sums) {
  using Sum = typename FewMma<T>::Sum;
  constexpr int kBlocks = kWide == 1 ? 2 : 1;  // blocks whose loads are in flight together
  constexpr int kSegment = FewMma<T>::kSegment;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  // The first rows into L2 while the preceding grid drains.
  if (blockIdx.x < a.first_wave && threadIdx.x < 16 * kWide && channel + threadIdx.x < a.channels)
    prefetch_l2(a.w + (channel + threadIdx.x) * a.w_ld, a.bytes);
  pdl_wait();
  const uint64_t once = policy_evict_first(), keep = policy_evict_last();
  const uint8_t* w0 = a.w + (channel + g) * a.w_ld;
  Sum acc[kTiles][kWide][4] = {}, total[kTiles][kWide][4] = {};
  auto load = [&](uint32_t (&v)[8], const uint8_t* p, int at, bool there, bool stream) {
    constexpr int kWords = kAlign / 4;
#pragma unroll
    for (int h = 0; h < 8 / kWords; ++h) {
      Vec<kAlign> q = {};
      if (there && at + kAlign * h < a.bytes) {
        if (stream) q = ld_stream<kAlign>(p + at + kAlign * h, once);
        else q = ld_weight<kAlign>(p + at + kAlign * h, keep);
      }
#pragma unroll
      for (int k = 0; k < kWords; ++k) v[kWords * h + k] = q.w[k];
    }
  };
  auto join = [&] {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
#pragma unroll
      for (int m = 0; m < kWide; ++m) {
#pragma unroll
        for (int k = 0; k < 4; ++k) total[i][m][k] += acc[i][m][k], acc[i][m][k] = 0;
      }
    }
  };
  int summed = 0;
  for (int block = warp; block * 128 < a.bytes; block += kFewWarps * kBlocks) {
    uint32_t w[kBlocks][2 * kWide][8];
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
#pragma unroll
      for (int m = 0; m < 2 * kWide; ++m)
        load(w[u][m], w0 + 8 * m * a.w_ld, (block + u * kFewWarps) * 128 + 32 * t, channel + g + 8 * m < a.channels, true);
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      uint32_t x[kBlocks][8];
#pragma unroll
      for (int u = 0; u < kBlocks; ++u)
        load(x[u], a.x + (8 * i + g) * a.x_ld, (block + u * kFewWarps) * 128 + 32 * t, 8 * i + g < a.rows, false);
#pragma unroll
      for (int u = 0; u < kBlocks; ++u) {
#pragma unroll
        for (int m = 0; m < kWide; ++m) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t q[4] = {w[u][2 * m][2 * j], w[u][2 * m + 1][2 * j], w[u][2 * m][2 * j + 1],
                                   w[u][2 * m + 1][2 * j + 1]};
            FewMma<T>::mma(acc[i][m], q, x[u][2 * j], x[u][2 * j + 1]);
          }
        }
      }
    }
    if constexpr (kSegment > 0) {
      if ((summed += kBlocks) >= kSegment) join(), summed = 0;
    }
  }
  if constexpr (kSegment > 0) join();
  pdl_trigger();
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
#pragma unroll
    for (int m = 0; m < kWide; ++m) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        sums[warp][8 * i + 2 * t + k % 2][16 * m + g + k / 2 * 8] = kSegment > 0 ? total[i][m][k] : acc[i][m][k];
    }
  }
  __syncthreads();
}

}  // namespace hprn

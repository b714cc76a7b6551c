// Fifth-generation tensor cores (tcgen05) and tiled TMA loads for sm_100a,
// inline PTX: the instructions the matrix products are made of.
//
// One thread issues an MMA; its operands are tiles in shared memory named by
// descriptors, its fp32 accumulators lie in tensor memory (TMEM, 128 lanes x 512
// columns per SM) and are read back 32 lanes a warp.  With cta_group::2 a pair
// of CTAs (a cluster of two) works on one 256-row tile: each holds its 128 rows
// of A and of the accumulators and half of B's rows, so B is read from L2 once
// for both.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "bulk.cuh"

namespace hprn {

// ---------------------------------------------------------------------------
// Clusters.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

// The address, in the cluster's shared window, of `addr` in CTA `rank`.
__device__ __forceinline__ uint32_t map_shared(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

// One arrival on a barrier anywhere in the cluster.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// A whole warp waits; the answer is the same in every lane, which lets the
// compiler keep what depends on it in uniform registers.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, uint64_t limit_ns = kWaitLimitNs) {
  return __all_sync(~0u, mbar_wait_bounded(bar, parity, limit_ns));
}

// ---------------------------------------------------------------------------
// Tiled TMA load of one box: coordinates in elements, x along the contiguous
// dimension; elements outside the tensor arrive as zeros and count as bytes.
// `bar` is in the issuing CTA (kGroup 1) or in either CTA of the pair.
template <int kGroup>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y,
                                            uint32_t bar) {
  if constexpr (kGroup == 2) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  }
}

// Asks L2 for a box: a hint, no bytes arrive anywhere.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y)
               : "memory");
}

__device__ __forceinline__ void prefetch_tensor_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ---------------------------------------------------------------------------
// TMEM allocation: whole warps, `columns` a power of two from 32.
template <int kGroup>
__device__ __forceinline__ void tmem_alloc(uint32_t result, uint32_t columns) {
  if constexpr (kGroup == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(result),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(result),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}

template <int kGroup>
__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t columns) {
  if constexpr (kGroup == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}

// Order tcgen05 operations with barriers between threads.
__device__ __forceinline__ void tmem_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 columns of this warp's 32 lanes, one lane a thread.  The values may be
// used after tmem_wait_load().
__device__ __forceinline__ void tmem_load_32(uint32_t addr, float (&v)[32]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]),
        "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
        "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr)
      : "memory");
}
// The same for 16 columns.
__device__ __forceinline__ void tmem_load_16(uint32_t addr, float (&v)[16]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15])
      : "r"(addr)
      : "memory");
}
// The load's registers pass through the wait, so nothing reads them before it.
template <int N>
__device__ __forceinline__ void tmem_wait_load(float (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int k = 0; k < N; ++k) asm volatile("" : "+f"(v[k]));
}

// ---------------------------------------------------------------------------
// MMA.  Operand tiles are 64 elements (128 bytes) wide rows in the 128-byte
// swizzle that TMA writes; 8 rows make an atom of 1024 bytes.
//   k-major tile:  a row is 64 values of k for one row of the operand;
//                  atoms of 8 operand rows follow each other (stride 1024).
//   row-major tile: a row is 64 operand rows for one k; atoms of 8 k follow
//                  each other (stride 1024), blocks of 64 operand rows are
//                  `block_bytes` apart (the "leading" offset).
// Fields: address / 16 in bits 0-13, leading offset / 16 in 16-29, stride / 16
// in 32-45, descriptor version 1 in 46-47, layout in 61-63 (2: 128-byte swizzle).
__device__ __forceinline__ uint64_t smem_descriptor(uint32_t addr, uint32_t block_bytes) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(block_bytes >> 4) << 16) |
         (uint64_t{1024 >> 4} << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}

// Instruction descriptor of kind::f16: fp32 accumulators, both operands bf16
// (1) or fp16 (0), `row_major` bits where an operand is not k-major, tile n x m.
__host__ __device__ constexpr uint32_t mma_descriptor(bool bf16, bool a_row_major, bool b_row_major, int m, int n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) |
         ((a_row_major ? 1u : 0u) << 15) | ((b_row_major ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <int kGroup>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if constexpr (kGroup == 2) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
  }
}

// One arrival on `bar` (at the same offset in both CTAs of a pair) once every
// MMA this thread issued so far is done.
template <int kGroup>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (kGroup == 2) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
  }
}

}  // namespace hprn

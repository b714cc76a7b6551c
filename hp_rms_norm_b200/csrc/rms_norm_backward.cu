// Gradients of RMSNorm, y_j = x_j w_j inv, inv = rsqrt(mean(x^2) + eps), for a
// gradient D of y, with n_j = x_j inv:
//   dx_j = inv (w_j D_j - n_j mean_k(w_k D_k n_k)) [+ E_j]
//   dw_j = sum over rows of D_j n_j
// E is the gradient that reaches x another way: in a pre-norm block x is the
// updated residual, which the next layer reads as well.  For the fused add
// (residual += input; y = RMSNorm(residual) w) x is the updated residual and
// dx is the gradient of both the input and the residual.
//
// All sums are fp32; dx and dw are rounded to 16 bits once.
//
// Memory-bound: x, D (and E) in, dx out, 6 (8) bytes per element.  norm_grad_rows
// reads them once: rows wait in shared memory, several deep, between memory
// and the two passes over them; dw's sums over a CTA's rows stay in registers,
// and the CTAs' sums are joined by a second kernel.  Rows too long for that
// (see norm_grad_plan) are read twice, by norm_grad_stats and norm_grad_columns.
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "bulk.cuh"
#include "runtime.cuh"
#include "vec.cuh"

namespace hprn {

struct NormGradArgs {
  uint16_t* dx;
  uint16_t* dw;
  const uint16_t* dy;
  const uint16_t* x;
  const uint16_t* w;
  const uint16_t* extra;  // E, or null
  int64_t rows, hidden;
  int64_t dx_stride, dy_stride, x_stride, extra_stride;
  float eps;
  float2* stats;   // per row: {inv, mean_k(w_k D_k n_k)}
  float* partial;  // [groups, partial_ld]: dw's sums over a group's rows
  int64_t partial_ld;
  int64_t groups;
  int row_threads, row_groups, slots;  // of norm_grad_rows
  bool weight_staged;                  // in shared memory
  bool dense;                          // every tensor's rows follow each other
  Waits waits;
};

// Both of a pair's sums over a warp: the lower half warp adds up .x, the upper
// .y, one shuffle a step instead of two.  The lower lanes return the sum of .x,
// the upper ones that of .y.
__device__ __forceinline__ float half_sum(float v) {
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
__device__ __forceinline__ float warp_halves(float2 v) {
  const bool lower = threadIdx.x % 32 < 16;
  const float mine = lower ? v.x : v.y, other = lower ? v.y : v.x;
  return half_sum(mine + __shfl_xor_sync(~0u, other, 16));
}

__device__ __forceinline__ void group_barrier(int barrier, int warps) {
  if (warps == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
}

// Both sums over the `warps` (at most 32) warps from `first_warp` that hold a
// row, which meet at hardware barrier `barrier`.  `part` is one of two buffers that calls
// alternate between, so one barrier a call is enough.
__device__ __forceinline__ float2 row_sum2(float2 v, float (*part)[32], int warp, int warps, int barrier,
                                           int first_warp) {
  const int lane = threadIdx.x % 32;
  float s = warp_halves(v);
  if (warps > 1) {
    if (lane % 16 == 0) part[lane / 16][warp] = s;
    group_barrier(barrier, warps);
    const int k = lane % 16;
    s = k < warps ? part[lane / 16][first_warp + k] : 0.f;
    if (k + 16 < warps) s += part[lane / 16][first_warp + k + 16];
    s = half_sum(s);
  } else {
    __syncwarp();
  }
  return make_float2(__shfl_sync(~0u, s, 0), __shfl_sync(~0u, s, 16));
}

constexpr int kMostRowGroups = 16;
constexpr int kMostSlots = 4;

__device__ __forceinline__ void lds4(uint32_t (&w)[4], uint32_t addr) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t lds1(uint32_t addr) {
  uint32_t w;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(addr));
  return w;
}
__device__ __forceinline__ void sts_half(uint32_t addr, uint16_t h) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"(h) : "memory");
}

// A CTA is `groups` groups of `row_threads` threads, and one warp more; a group
// works on one row at a time, each thread on the same W words (pairs of
// elements) of every row.  A group's rows arrive in a ring of `slots` row
// buffers in shared memory, which the extra warp keeps filled by bulk copies.
//   kVectors: every row of every tensor starts on a 16-byte boundary and hidden
// is a multiple of 8.  Rows that follow each other come in one copy; threads
// take vectors of eight elements.
//   Else a row is copied with the 16-byte granules it lies in, so that it starts
// as far into its buffer as it does into its first granule (the first and the
// last row's elements in granules that reach out of the tensor come by
// ordinary loads); threads take single words, neighbouring threads
// neighbouring ones, put together from two where the row starts on an odd element.
//
// Registers hold dw's sums (2 W floats) and, up to 8 words, w D between the
// two passes (held at 16 words it spilled: 4096 x 16384 106 us instead of 93).
// 4096 x 8192 with E: 48.0 us (0.87 of a copy of the same bytes),
// against 55.8 with the rows themselves in registers, which spilled or kept
// one row a CTA in flight.  4096 x 5001 with E: 73 us, bound by issue, against
// 155 with rows copied element by element.
//
// A wait that runs out (mbar_wait_bounded) ends its group after the copies
// still in flight, and says so (report_give_up); the rows it had not finished
// keep their dx.
constexpr int kNormThreads = 512;

template <typename T, int W, bool EXTRA, bool kVectors>
__global__ void __launch_bounds__(kNormThreads + 32, 1) norm_grad_rows(NormGradArgs a) {
  constexpr int kVecs = W / 4;
  constexpr int kTensors = EXTRA ? 3 : 2;
  constexpr bool kHold = W <= 8;
  extern __shared__ __align__(128) unsigned char row_mem[];
  __shared__ __align__(8) uint64_t full[kMostSlots], empty[kMostSlots];
  __shared__ float part[2][2][32];  // a group's warps follow those of the groups before it
  __shared__ int gave_up[kMostRowGroups];
  const int tid = threadIdx.x, row_threads = a.row_threads, groups = a.row_groups;
  const int workers = groups * row_threads;
  const bool copier = tid >= workers;
  const int group = copier ? tid - workers : tid / row_threads, in = copier ? 0 : tid - group * row_threads;
  const int warps = row_threads / 32, barrier = 1 + group;
  const int hidden = static_cast<int>(a.hidden), nvec = (hidden + 7) / 8;
  const int words = (hidden + 1) / 2;
  // A slot: `groups` rows of x, then of D, then of E; `pitch` bytes a row.
  const uint32_t row_bytes = static_cast<uint32_t>(nvec) * 16, pitch = row_bytes + (kVectors ? 0 : 16);
  const uint32_t tensor_bytes = pitch * groups, slot_bytes = tensor_bytes * kTensors;
  const uint32_t w_row = smem_u32(row_mem), slots_at = w_row + (a.weight_staged ? row_bytes : 0);
  const uint32_t ring = slots_at + group * pitch;
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * groups + group;
  const uint64_t pol = policy_evict_first();
  // The tensors' rows `i`, in a slot's order.
  auto row_of = [&](int t, int64_t i) {
    return t == 0 ? a.x + i * a.x_stride : t == 1 ? a.dy + i * a.dy_stride : a.extra + i * a.extra_stride;
  };
  const int lane = tid % 32;
  // Bytes of the rows that a round of the CTA has of one tensor.
  auto round_bytes = [&](int64_t base) {
    return static_cast<uint32_t>(min(static_cast<int64_t>(groups), a.rows - base)) * row_bytes;
  };
  if (copier) {
    if (lane < groups) gave_up[lane] = 0;
    if (lane == 0) {
      for (int s = 0; s < a.slots; ++s) {
        mbar_init(smem_u32(&full[s]), 1);
        mbar_init(smem_u32(&empty[s]), groups * warps);
      }
      mbar_init_fence();
    }
    {
      // The first rows, into L2, while the preceding grid drains.
      for (int s = 0; s < a.slots; ++s) {
        const int64_t i = first - group + s * step + lane;
        if (lane < groups && i < a.rows)
          for (int t = 0; t < kTensors; ++t) prefetch_l2(row_of(t, i), static_cast<uint64_t>(hidden) * 2);
      }
    }
  }
  __syncthreads();
  pdl_wait();

  if (copier) {
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int64_t base = a.waits.stall ? a.rows : static_cast<int64_t>(blockIdx.x) * groups; base < a.rows;
         base += step) {
      ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&empty[slot]), phase ^ 1, a.waits.limit_ns));
      if (!ok) break;
      const uint32_t bar = smem_u32(&full[slot]), to = slots_at + slot * slot_bytes;
      const int64_t next = base + a.slots * step;  // few buffers: asked into L2
      if (kVectors && a.dense) {
        const uint32_t bytes = round_bytes(base);
        if (lane == 0) mbar_arrive_expect_tx(bar, bytes * kTensors);
        __syncwarp();
        if (lane < kTensors) {
          bulk_load(to + lane * tensor_bytes, row_of(lane, base), bytes, bar, pol);
          if (a.slots < 3 && next < a.rows) prefetch_l2(row_of(lane, next), round_bytes(next));
        }
      } else {
        const bool mine = lane < groups && base + lane < a.rows;
        const int64_t i = base + lane;
        const unsigned char* from[kTensors];
        uint32_t bytes[kTensors], at[kTensors], total = 0;
#pragma unroll
        for (int t = 0; t < kTensors; ++t) {
          bytes[t] = 0;
          if (!mine) continue;
          const unsigned char* p = reinterpret_cast<const unsigned char*>(row_of(t, i));
          const uint32_t off = kVectors ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
          at[t] = to + t * tensor_bytes + lane * pitch;
          // Granules [lo, hi) of the row's span, from its first one.
          const uint32_t end = off + static_cast<uint32_t>(hidden) * 2;
          uint32_t lo = 0, hi = (end + 15) & ~15u;
          // Granules that reach out of the tensor are left out, their elements
          // of this row stored one by one.
          const int64_t stride = t == 0 ? a.x_stride : t == 1 ? a.dy_stride : a.extra_stride;
          if (off > i * stride * 2) lo = 16;
          if (hi - end > (a.rows - 1 - i) * stride * 2) hi -= 16;
          hi = max(hi, lo);
          const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
          if (lo > 0)
            for (int j = 0; j < hidden && off + 2 * j < lo; ++j) sts_half(at[t] + off + 2 * j, q[j]);
          if (hi < end)
            for (int j = hi > off ? static_cast<int>(hi - off) / 2 : 0; j < hidden; ++j)
              sts_half(at[t] + off + 2 * j, q[j]);
          from[t] = p - off + lo, at[t] += lo, bytes[t] = hi - lo, total += bytes[t];
        }
        // The stores above, in this round and in earlier ones of this buffer, before
        // the bulk copies that write there by another proxy.
        if constexpr (!kVectors) fence_proxy_async_smem();
        total = __reduce_add_sync(~0u, total);
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(bar, total);
        __syncwarp();
#pragma unroll
        for (int t = 0; t < kTensors; ++t) {
          if (bytes[t] > 0) bulk_load(at[t], from[t], bytes[t], bar, pol);
          if (a.slots < 3 && lane < groups && next + lane < a.rows)
            prefetch_l2(row_of(t, next + lane), static_cast<uint64_t>(hidden) * 2);
        }
      }
      if (++slot == a.slots) slot = 0, phase ^= 1;
    }
    if (!ok) {
      if (lane == 0) report_give_up(a.waits);
      for (int k = 0; k < a.slots; ++k) {  // copies still in flight
        if (--slot < 0) slot = a.slots - 1, phase ^= 1;
        mbar_wait_bounded(smem_u32(&full[slot]), phase, kWaitLimitNs / 16);
      }
    }
    __syncwarp();
    if (groups > 1) {
      __syncthreads();
      __syncthreads();
    }
    return;
  }

  float2 acc[W];
#pragma unroll
  for (int k = 0; k < W; ++k) acc[k] = make_float2(0.f, 0.f);
  // Every group writes the same weight row, pairs with eight a thread in flight,
  // and reads it after its own barrier.
  if (a.weight_staged) {
    uint32_t* q = reinterpret_cast<uint32_t*>(row_mem);
    for (int j0 = in; j0 < nvec * 4; j0 += 8 * row_threads) {
      uint32_t w[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = 2 * (j0 + u * row_threads);
        const uint32_t lo = j < hidden ? ld_stream<2>(a.w + j, pol).h : 0;
        const uint32_t hi = j + 1 < hidden ? ld_stream<2>(a.w + j + 1, pol).h : 0;
        w[u] = lo | hi << 16;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (j0 + u * row_threads < nvec * 4) q[j0 + u * row_threads] = w[u];
    }
  }
  group_barrier(barrier, warps);
  pdl_trigger();
  const uint64_t keep = policy_evict_last();
  // Words 4 k to 4 k + 3 of this thread's: one vector, or one word every row_threads.
  auto inside = [&](int k) { return kVectors ? in + k * row_threads < nvec : in + 4 * k * row_threads < words; };
  auto word_at = [&](int k, int e) { return in + (4 * k + e) * row_threads; };
  auto load_weight = [&](uint32_t (&w)[4], int k) {
    if constexpr (!kVectors) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = word_at(k, e) < words ? lds1(w_row + word_at(k, e) * 4) : 0;
    } else if (a.weight_staged) {
      lds4(w, w_row + (in + k * row_threads) * 16);
    } else {
      const Vec<16> q = ld_weight<16>(a.w + (in + k * row_threads) * 8, keep);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = q.w[e];
    }
  };
  // The same of a row that starts at shared address `at`.
  auto load_row = [&](uint32_t (&w)[4], uint32_t at, int k) {
    if constexpr (kVectors) {
      lds4(w, at + (in + k * row_threads) * 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = word_at(k, e);
        w[e] = 0;
        if (j >= words) continue;
        if (at & 2) w[e] = __funnelshift_r(lds1(at - 2 + 4 * j), lds1(at + 2 + 4 * j), 16);
        else w[e] = lds1(at + 4 * j);
        if (2 * j + 1 == hidden) w[e] &= 0xffffu;
      }
    }
  };
  auto offset_of = [&](const uint16_t* p) {
    return kVectors ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
  };

  const float scale = 1.0f / static_cast<float>(hidden);
  int slot = 0, turn = 0;
  uint32_t phase = 0;
  for (int64_t i = first; i < a.rows; i += step) {
    const uint32_t at = ring + slot * slot_bytes;
    const uint32_t xs = at + offset_of(row_of(0, i)), ds = at + tensor_bytes + offset_of(row_of(1, i));
    const uint32_t es = EXTRA ? at + 2 * tensor_bytes + offset_of(row_of(2, i)) : 0;
    if (!mbar_wait_bounded(smem_u32(&full[slot]), phase, a.waits.limit_ns)) gave_up[group] = 1;
    float2 ss = make_float2(0.f, 0.f), sd = ss;
    float2 wd[kHold ? W : 1];  // w D, for both passes
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      if (!inside(k)) break;
      uint32_t x[4], d[4], w[4];
      load_row(x, xs, k);
      load_row(d, ds, k);
      load_weight(w, k);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 xf = unpack2<T>(x[e]), p = mul_pair<T>(w[e], d[e]);
        ss = __ffma2_rn(xf, xf, ss);
        sd = __ffma2_rn(p, xf, sd);
        if constexpr (kHold) wd[4 * k + e] = p;
      }
    }
    const float2 s =
        row_sum2(make_float2(ss.x + ss.y, sd.x + sd.y), part[turn], tid / 32, warps, barrier, group * warps);
    if (*static_cast<volatile int*>(&gave_up[group])) {
      // The copier may have issued its last row and left without a wait.
      if (in == 0) report_give_up(a.waits);
      break;
    }
    const float inv = rsqrtf(s.x * scale + a.eps), mean = s.y * inv * scale;
    const float2 inv2 = make_float2(inv, inv), minus = make_float2(-mean * inv, -mean * inv);
    uint16_t* dx = a.dx + i * a.dx_stride;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      if (!inside(k)) break;
      uint32_t x[4], d[4], w[4], e4[4];
      load_row(x, xs, k);
      load_row(d, ds, k);
      if constexpr (!kHold) load_weight(w, k);
      if constexpr (EXTRA) load_row(e4, es, k);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 n = __fmul2_rn(unpack2<T>(x[e]), inv2);
        acc[4 * k + e] = __ffma2_rn(unpack2<T>(d[e]), n, acc[4 * k + e]);
        float2 p;
        if constexpr (kHold) p = wd[4 * k + e];
        else p = mul_pair<T>(w[e], d[e]);
        float2 g = __ffma2_rn(p, inv2, __fmul2_rn(n, minus));
        if constexpr (EXTRA) g = __fadd2_rn(g, unpack2<T>(e4[e]));
        x[e] = pack2<T>(g.x, g.y);
      }
      if constexpr (kVectors) {
        *reinterpret_cast<uint4*>(dx + (in + k * row_threads) * 8) = make_uint4(x[0], x[1], x[2], x[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = word_at(k, e);
          uint16_t* q = dx + 2 * j;
          if (j >= words) continue;
          if (2 * j + 1 < hidden && (reinterpret_cast<uintptr_t>(q) & 2) == 0) {
            *reinterpret_cast<uint32_t*>(q) = x[e];
          } else {
            q[0] = static_cast<uint16_t>(x[e]);
            if (2 * j + 1 < hidden) q[1] = static_cast<uint16_t>(x[e] >> 16);
          }
        }
      }
    }
    __syncwarp();
    if (tid % 32 == 0) mbar_arrive(smem_u32(&empty[slot]));
    turn ^= 1;
    if (++slot == a.slots) slot = 0, phase ^= 1;
  }
  // The groups' sums meet in shared memory (every copy has landed); the first
  // group writes the CTA's.
  if (groups > 1) {
    __syncthreads();
    float2* sums = reinterpret_cast<float2*>(row_mem);
#pragma unroll
    for (int k = 0; k < W; ++k) sums[k * workers + tid] = acc[k];
    __syncthreads();
    if (group > 0) return;
    for (int g = 1; g < groups; ++g) {
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] = __fadd2_rn(acc[k], sums[k * workers + g * row_threads + tid]);
    }
  }
  // (partial's rows are padded to whole vectors.)
  float* out = a.partial + blockIdx.x * static_cast<int64_t>(nvec) * 8;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    if (!inside(k)) break;
    if constexpr (kVectors) {
      Vec<32> q;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        q.w[2 * e] = __float_as_uint(acc[4 * k + e].x);
        q.w[2 * e + 1] = __float_as_uint(acc[4 * k + e].y);
      }
      st_global<32>(out + (in + k * row_threads) * 8, q);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (word_at(k, e) < words) reinterpret_cast<float2*>(out)[word_at(k, e)] = acc[4 * k + e];
    }
  }
}

// Rows too long for norm_grad_rows (more than 32768 elements, or about 28,150 off
// 16-byte boundaries with E) in two readings of single elements, bound by the
// loads in flight: 4096 x 32769 with E 476 us, 0.35 of a copy's rate, where
// 32768 takes 277.
//
// One CTA per row: the row's two sums.
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_stats(NormGradArgs a) {
  pdl_wait();
  __shared__ float part[2][32];
  const int64_t i = blockIdx.x;
  const uint16_t* x = a.x + i * a.x_stride;
  const uint16_t* dy = a.dy + i * a.dy_stride;
  float2 s = make_float2(0.f, 0.f);
  for (int64_t j = threadIdx.x; j < a.hidden; j += blockDim.x) {
    const float v = unpack1<T>(x[j]);
    s.x = fmaf(v, v, s.x);
    s.y = fmaf(unpack1<T>(a.w[j]) * unpack1<T>(dy[j]), v, s.y);
  }
  s = row_sum2(s, part, threadIdx.x / 32, 8, 1, 0);
  if (threadIdx.x == 0) {
    const float inv = rsqrtf(s.x / static_cast<float>(a.hidden) + a.eps);
    a.stats[i] = make_float2(inv, s.y * inv / static_cast<float>(a.hidden));
  }
}

// A group of rows x blockDim columns per CTA: dx, and the group's part of dw.
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_columns(NormGradArgs a) {
  pdl_wait();
  const int64_t j = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (j >= a.hidden) return;
  const float w = unpack1<T>(a.w[j]);
  float sum = 0.f;
  for (int64_t i = blockIdx.y; i < a.rows; i += a.groups) {
    const float2 st = a.stats[i];
    const float n = unpack1<T>(a.x[i * a.x_stride + j]) * st.x;
    const float d = unpack1<T>(a.dy[i * a.dy_stride + j]);
    sum = fmaf(d, n, sum);
    float g = st.x * (w * d - n * st.y);
    if (a.extra) g += unpack1<T>(a.extra[i * a.extra_stride + j]);
    a.dx[i * a.dx_stride + j] = pack1<T>(g);
  }
  a.partial[blockIdx.y * a.partial_ld + j] = sum;
}

// dw from the groups' sums: 32 columns a CTA, its 8 warps taking groups in turn.
// (256 threads, so that the CTAs fit beside norm_grad_rows' and wait there for
// its end.)
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_weight(NormGradArgs a) {
  __shared__ float part[8][32];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  pdl_trigger();
  pdl_wait();
  float sum = 0.f;
  if (j < a.hidden) {
#pragma unroll 10
    for (int64_t g = ty; g < a.groups; g += 8) sum += a.partial[g * a.partial_ld + j];
  }
  part[ty][tx] = sum;
  __syncthreads();
  if (ty > 0 || j >= a.hidden) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) sum += part[k][tx];
  a.dw[j] = pack1<T>(sum);
}

// How norm_grad_rows takes the rows: words (of two elements) a thread, threads a
// row, rows a CTA works on at once, row buffers each, and CTAs (also dw's
// partial sums).  words 0: rows that are read twice.
constexpr int kNormSmem = 220 * 1024;
struct NormGradPlan {
  int words, row_threads, row_groups, slots, smem;
  bool vectors, weight_staged;
  int64_t ctas;
};

// One CTA per SM.  The words a thread decide how many of the CTA's 512 threads
// have work: a row takes as many as it has, and as many rows go at once as have
// threads and two buffers each.  The fewest words that employ 416 threads or
// more win, else the most threads; 4 words (the shortest way through a row)
// only for rows up to 1024 elements or few rows: 4096 x 4096 with E takes
// 25.5 us with 8 words and two rows at once, 30.7 with 4 and one; 4096 x 1024
// 13.7 with 4, 14.8 with 8; 512 x 4096 9.6 with 4, 10.5 with 8; 4096 x 16448
// 95 with 20 words and 416 threads, about 160 with 32 and 288.  The weight is kept in shared memory beside the rows unless that
// leaves them fewer than two buffers.
NormGradPlan norm_grad_plan(const NormGradArgs& a) {
  auto fits = [&](const void* p, int64_t stride) { return !p || tma_rows(p, a.rows, stride); };
  const bool vectors = a.hidden % 8 == 0 && fits(a.x, a.x_stride) && fits(a.dy, a.dy_stride) &&
                       fits(a.dx, a.dx_stride) && fits(a.extra, a.extra_stride);
  const int64_t nvec = (a.hidden + 7) / 8, row = nvec * 16, pairs = (a.hidden + 1) / 2;
  const int64_t slot = (row + (vectors ? 0 : 16)) * (a.extra ? 3 : 2);
  NormGradPlan best{};
  best.ctas = a.rows < 64 ? a.rows : 64;
  for (int words : {4, 8, 12, 16, 20, 24, 32}) {
    const int64_t threads = round_up(vectors ? (nvec + words / 4 - 1) / (words / 4) : (pairs + words - 1) / words, 32);
    const bool few = a.rows <= 4 * 148;
    if (threads > kNormThreads || (words == 4 && threads > 128 && !few)) continue;
    int64_t groups = kNormThreads / threads;
    while (groups > 1 && row + 2 * groups * slot > kNormSmem) --groups;
    int64_t slots = (kNormSmem - row) / (groups * slot);
    const bool staged = slots >= 2 || !vectors || !aligned(a.w, 16);
    if (!staged) slots = kNormSmem / (groups * slot);
    if (slots < 1) break;
    if (threads * groups <= best.row_threads * best.row_groups) continue;
    NormGradPlan p{};
    p.vectors = vectors, p.weight_staged = staged;
    p.words = words, p.row_threads = static_cast<int>(threads), p.row_groups = static_cast<int>(groups);
    p.slots = static_cast<int>(slots < kMostSlots ? slots : kMostSlots);
    const int64_t ring = (staged ? row : 0) + groups * p.slots * slot;
    const int64_t sums = groups > 1 ? words * threads * groups * 8 : 0;
    p.smem = static_cast<int>(ring > sums ? ring : sums);
    const int64_t need = (a.rows + groups - 1) / groups;
    p.ctas = need < 148 ? need : 148;
    best = p;
    if (few || threads * groups >= 416) break;
  }
  return best;
}

template <typename T, bool EXTRA, bool kVectors>
void (*norm_grad_kernel(int words))(NormGradArgs) {
  switch (words) {
    case 4: return norm_grad_rows<T, 4, EXTRA, kVectors>;
    case 8: return norm_grad_rows<T, 8, EXTRA, kVectors>;
    case 12: return norm_grad_rows<T, 12, EXTRA, kVectors>;
    case 16: return norm_grad_rows<T, 16, EXTRA, kVectors>;
    case 20: return norm_grad_rows<T, 20, EXTRA, kVectors>;
    case 24: return norm_grad_rows<T, 24, EXTRA, kVectors>;
    default: return norm_grad_rows<T, 32, EXTRA, kVectors>;
  }
}

template <typename T>
int launch_norm_grad(const NormGradArgs& a, const NormGradPlan& p, const DeviceInfo* dev, cudaStream_t stream,
                     unsigned flags) {
  const char* what = "rms_norm_backward";
  int st = HPRN_OK;
  if (a.rows > 0 && p.words > 0) {
    auto fn = p.vectors ? (a.extra ? norm_grad_kernel<T, true, true>(p.words) : norm_grad_kernel<T, false, true>(p.words))
                     : (a.extra ? norm_grad_kernel<T, true, false>(p.words) : norm_grad_kernel<T, false, false>(p.words));
    if ((st = allow_smem(dev, reinterpret_cast<const void*>(fn), kNormSmem, what)) != HPRN_OK) return st;
    st = launch_rows_smem(fn, dim3(static_cast<unsigned>(p.ctas)),
                          dim3(static_cast<unsigned>(p.row_threads * p.row_groups + 32)), p.smem, stream, flags, what, a);
  } else if (a.rows > 0) {
    const unsigned cols = static_cast<unsigned>((a.hidden + 255) / 256);
    st = launch_rows(norm_grad_stats<T>, dim3(static_cast<unsigned>(a.rows)), dim3(256), stream, flags, what, a);
    if (st != HPRN_OK) return st;
    st = launch_rows(norm_grad_columns<T>, dim3(cols, static_cast<unsigned>(a.groups)), dim3(256), stream,
                     flags, what, a);
  }
  if (st != HPRN_OK) return st;
  return launch_rows(norm_grad_weight<T>, dim3(static_cast<unsigned>((a.hidden + 31) / 32)), dim3(256), stream,
                     flags, what, a);
}

}  // namespace hprn

extern "C" int hprn_rms_norm_backward(void* grad_input, void* grad_weight, const void* grad_out,
                                      const void* input, const void* weight,
                                      const void* grad_residual, int64_t rows, int64_t hidden,
                                      int64_t grad_input_row_stride, int64_t grad_out_row_stride,
                                      int64_t input_row_stride, int64_t grad_residual_row_stride,
                                      double eps, int dtype, void* workspace,
                                      int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (dtype != HPRN_DTYPE_BF16 && dtype != HPRN_DTYPE_FP16)
    return fail(HPRN_ERR_UNSUPPORTED_DTYPE, "dtype must be kFloat16 or kBFloat16");
  if (rows < 0 || hidden < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "sizes must be >= 0");
  if (rows > kMaxExtent || hidden > kMaxExtent)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows and hidden must be at most 2^30");
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  if (rows > 1 && (grad_input_row_stride < hidden || grad_out_row_stride < hidden ||
                   input_row_stride < hidden || (grad_residual && grad_residual_row_stride < hidden)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  NormGradArgs a{};
  a.dx = static_cast<uint16_t*>(grad_input), a.dw = static_cast<uint16_t*>(grad_weight);
  a.dy = static_cast<const uint16_t*>(grad_out), a.x = static_cast<const uint16_t*>(input);
  a.w = static_cast<const uint16_t*>(weight), a.extra = static_cast<const uint16_t*>(grad_residual);
  a.rows = rows, a.hidden = hidden;
  a.dx_stride = grad_input_row_stride, a.dy_stride = grad_out_row_stride;
  a.x_stride = input_row_stride, a.extra_stride = grad_residual_row_stride;
  a.eps = static_cast<float>(eps);
  const NormGradPlan plan = norm_grad_plan(a);
  a.groups = plan.ctas, a.row_threads = plan.row_threads;
  a.dense = rows <= 1 || (input_row_stride == hidden && grad_out_row_stride == hidden &&
                          (!grad_residual || grad_residual_row_stride == hidden));
  a.row_groups = plan.row_groups, a.slots = plan.slots, a.weight_staged = plan.weight_staged;
  Workspace ws(workspace, *workspace_bytes);
  a.stats = ws.take<float2>(plan.words > 0 ? 0 : rows);
  a.partial_ld = round_up(hidden, 8);
  a.partial = ws.take<float>(a.groups * a.partial_ld);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (hidden == 0) return ok();
  if (!grad_weight || !weight || (rows > 0 && (!grad_input || !grad_out || !input)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(grad_input, 2) || !aligned(grad_weight, 2) || !aligned(grad_out, 2) ||
      !aligned(input, 2) || !aligned(weight, 2) || !aligned(grad_residual, 2))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(grad_input, rows, hidden, grad_input_row_stride),
                       extent16(grad_weight, 1, hidden, hidden)};
  const Extent ins[] = {extent16(grad_out, rows, hidden, grad_out_row_stride),
                      extent16(input, rows, hidden, input_row_stride), extent16(weight, 1, hidden, hidden),
                      extent16(grad_residual, rows, hidden, grad_residual_row_stride)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  int st = current_device(&dev);
  if (st != HPRN_OK) return st;
  if ((st = waits_of(dev, &a.waits, "rms_norm_backward")) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == HPRN_DTYPE_BF16 ? launch_norm_grad<__nv_bfloat16>(a, plan, dev, cs, flags)
                                  : launch_norm_grad<__half>(a, plan, dev, cs, flags);
}

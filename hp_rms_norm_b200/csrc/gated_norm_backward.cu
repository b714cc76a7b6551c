// Gradients of the norms on both sides of a gated block (gated_norm.cu):
//   t = a r + g y,  y_j = x_j inv_x p_j (y = x without p),  out_j = t_j inv_t w_j
// With D the gradient of out, E that of t from its other uses, n = t inv_t,
// m = x inv_x (m = x and p = 1 without p), means over a row:
//   dt = inv_t (w D - n mean(w D n)) + E
//   dr = a dt,  dg = sum of dt m p over what shares the gate,
//   dx = inv_x (p g dt - m mean(p g dt m)),  dp = sum over rows of g dt m,
//   dw = sum over rows of D n
// t is read as the forward call wrote it, rounded to 16 bits: the unrounded sum would
// have to be kept in 32 bits, 4 bytes an element more to write and read, or made again
// from the old residual, which an update in place has overwritten.  In bf16 the gradients
// are 2.3e-3 from 64 bits for it, where 1.7e-3 is their own rounding.
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "bulk.cuh"
#include "gated_norm.cuh"
#include "rows.cuh"
#include "runtime.cuh"
#include "vec.cuh"

namespace hprn {

struct BlockGradArgs {
  uint16_t *dx, *dr, *dp, *dw, *dg;  // dp, dg: or null
  const uint16_t *d, *e, *x, *t, *p, *w, *g;  // e, p, g: or null
  int64_t dx_stride, dr_stride, dg_stride, d_stride, e_stride, x_stride, t_stride, g_stride;
  int64_t rows, hidden;
  int64_t rows_per_gate, gates;
  bool gate_row;  // the gate is a row of `hidden` values
  bool gate_each;  // ... of its own for every row
  float scale, eps;
  float4* stats;      // per row: {inv_t, mean(w D n), inv_x, mean(p g dt m)}
  float* gate_sums;   // per row: sum of dt m p, where the gate is one value
  // Sums over the rows of a part (`parts` for each gate where the gate is a
  // shared row, else `parts` in all): of D n, and of dt m where the gate is a
  // shared row, else of g dt m.
  float *dw_parts, *m_parts;
  int64_t parts, part_rows, parts_ld;
  // Of block_grad_rows: what a row's buffer holds (t, D, and x, E, g where they are
  // needed; their places in it, or -1), and how its threads are dealt out.
  const uint16_t* src[5];
  int64_t src_stride[5];
  int tensors, x_at, e_at, g_at;
  int row_threads, row_groups, slots;
  uint32_t ring_at;  // in shared memory
  bool staged;       // w and p are in shared memory, before the ring
  bool e_direct;     // E is read where it is, not through the ring
  int64_t ctas, runs;
  bool own_runs;  // of the groups of a CTA
  bool dense;  // every tensor's rows follow each other
  Waits waits;
};

// ---------------------------------------------------------------------------
// Rows read once: memory-bound, 8 bytes of an element in and 4 out with E and x.
//
// A CTA works on a run of neighbouring rows, `row_groups` at a time, each by
// row_threads threads, a thread always on the same W words (pairs of elements).
//   Where a gate's row is shared by few rows, more than two gates a CTA, each group has
// a run of its own: the sums for a gate are then one row for each run that meets it,
// where groups that share a run each write a row for every gate of it (gates of two rows,
// 65536 x 512: 67 MiB of workspace for 579, 3.9 ms for 10.3; of 64 rows 246 us for 347).
// With more rows a gate a CTA's rows are better copied together (65536 x 128, gates of
// 512 rows: 85 us, with runs of their own 127).
// One warp more brings the rows into a ring of `slots` buffers in shared memory by
// bulk copies.  Two sums over the row's threads lie between three passes over the
// buffer: the means of squares and of w D n; then dt, and with it dr, dg, the sums
// over rows, and the mean of p g dt m; then dx.  The second sum and the next row's
// first one meet at one barrier (4096 x 8192 with E: 80 us, its bytes at a copy's rate
// 61).  The sums over rows (D n, and dt m or g dt m) stay in registers, 4 W floats, as
// do w, p and a gate row that rows share up to 12 words a thread (of more they are in
// shared memory).  Where a run reaches into another gate's rows, the sums for the gate
// are written out and started anew.
//   kVectors: every row of every tensor starts on a 16-byte boundary and hidden is
// a multiple of 8.  Else a row is copied with the 16-byte granules it lies in
// (elements in granules that reach out of the tensor one by one), and a vector put
// together from two (12 x 257 rows of 1001, fp16: 34 us).
//
// A wait that runs out (mbar_wait_bounded) ends its group after the copies in
// flight, and says so (report_give_up).
// Threads that work on rows, by their words: what their registers leave room for (96,
// 128 and 168 each).
__host__ __device__ constexpr int block_threads(int words) { return words <= 4 ? 608 : words <= 8 ? 480 : 352; }
constexpr int kBlockSmem = 220 * 1024;
constexpr int kBlockSlots = 4;
constexpr int kBlockGroups = 16;

__device__ __forceinline__ void team_barrier(int barrier, int threads) {
  if (threads == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}

// The sums of four values over the `warps` (at most 24) warps from `first_warp` that
// hold a row, which meet at hardware barrier `barrier`; `part` alternates between two
// buffers.  In a warp each lane goes on with half of its values twice, 6 shuffles for
// the 20 of four sums by themselves; eight lanes each add up one value's sums of the
// warps.
__device__ __forceinline__ void team_sums(float (&v)[4], float4* part, int warps, int first_warp, int barrier) {
  const int lane = threadIdx.x % 32;
  const bool upper = lane & 16, odd = lane & 8;
  float a = upper ? v[2] : v[0], b = upper ? v[3] : v[1];
  a += __shfl_xor_sync(~0u, upper ? v[0] : v[2], 16);
  b += __shfl_xor_sync(~0u, upper ? v[1] : v[3], 16);
  float s = odd ? b : a;
  s += __shfl_xor_sync(~0u, odd ? a : b, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (warps > 1) {
    float* sums = reinterpret_cast<float*>(part);
    if (lane % 8 == 0) sums[threadIdx.x / 32 * 4 + lane / 8] = s;
    team_barrier(barrier, warps * 32);
    const int k = lane % 8;
    const float* q = sums + (first_warp + k) * 4 + lane / 8;
    s = k < warps ? q[0] : 0.f;
    if (k + 8 < warps) s += q[32];
    if (k + 16 < warps) s += q[64];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = __shfl_sync(~0u, s, 8 * k);
}

__device__ __forceinline__ void shared_words(uint32_t (&w)[4], uint32_t addr) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(addr));
}
__device__ __forceinline__ void set_shared_words(uint32_t addr, const uint32_t (&w)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
               : "memory");
}
__device__ __forceinline__ void set_shared_half(uint32_t addr, uint16_t h) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"(h) : "memory");
}

// The first row of run c (no more runs than rows: none is empty); row i lies in run
// ((i + 1) runs - 1) / rows.
__device__ __forceinline__ int run_start(const BlockGradArgs& a, int64_t c) {
  return static_cast<int>(a.rows * min(c, a.runs) / a.runs);
}
__device__ __forceinline__ int64_t run_of(const BlockGradArgs& a, int64_t i) { return ((i + 1) * a.runs - 1) / a.rows; }

// kGate: kOneGate a gate of one value a row, or none (1); kChannels one row of values
// for all rows; kGateRow rows of values that rows share, kGateRuns with own runs;
// kGateEach one for every row.
enum GateKind { kOneGate, kChannels, kGateRow, kGateRuns, kGateEach };

template <typename T, int W, bool kVectors, bool kPost, int kGate>
__global__ void __launch_bounds__(block_threads(W) + 32, 1) block_grad_rows(BlockGradArgs a) {
  constexpr int kVecs = W / 4;
  constexpr bool kOwnRuns = kGate == kGateRuns, kSharedRow = kGate == kGateRow || kOwnRuns;
  constexpr bool kHold = W <= 12;
  static_assert(kHold || kVectors, "vectors of loose rows are read by two threads");
  extern __shared__ __align__(128) unsigned char row_mem[];
  __shared__ __align__(8) uint64_t full[kBlockSlots], empty[kBlockSlots];
  __shared__ float4 part[2][block_threads(W) / 32];
  __shared__ int gave_up[kBlockGroups];
  const int tid = threadIdx.x, row_threads = a.row_threads, groups = a.row_groups;
  const int workers = groups * row_threads;
  const bool copier = tid >= workers;
  const int group = copier ? 0 : tid / row_threads, in = copier ? 0 : tid - group * row_threads;
  const int warps = row_threads / 32, barrier = 1 + group;
  const int hidden = static_cast<int>(a.hidden), nvec = (hidden + 7) / 8;
  // A buffer: `groups` rows of each tensor in turn, `pitch` bytes a row.
  const uint32_t row_bytes = static_cast<uint32_t>(nvec) * 16, pitch = row_bytes + (kVectors ? 0 : 16);
  const uint32_t tensor_bytes = pitch * groups, slot_bytes = tensor_bytes * a.tensors;
  const uint32_t staged = smem_u32(row_mem), ring = staged + a.ring_at;
  // A group's rows, `step` apart; its run, its own or the CTA's.  A lane of the copying
  // warp has a group's.
  const int lane = tid % 32, member = copier ? lane : group, step = kOwnRuns ? 1 : groups;
  const int64_t run = kOwnRuns ? static_cast<int64_t>(blockIdx.x) * groups + min(member, groups - 1) : blockIdx.x;
  const int begin = run_start(a, run), end = run_start(a, run + 1);
  const int first = kOwnRuns ? begin : begin + member;
  if (copier) {
    if (lane < groups) gave_up[lane] = 0;
    if (lane == 0) {
      for (int s = 0; s < a.slots; ++s) {
        mbar_init(smem_u32(&full[s]), 1);
        mbar_init(smem_u32(&empty[s]), groups * warps);
      }
      mbar_init_fence();
    }
    // The first rows, into L2, while the preceding grid drains.
    const int ahead = kOwnRuns ? min(end, first + a.slots) : min(end, first + 1);
    if (lane < (kOwnRuns ? groups : groups * a.slots))
      for (int i = first; i < ahead; ++i)
        for (int t = 0; t < a.tensors; ++t)
          prefetch_l2(a.src[t] + static_cast<int64_t>(i) * a.src_stride[t], static_cast<uint64_t>(hidden) * 2);
  }
  __syncthreads();
  pdl_wait();

  if (copier) {
    const uint64_t pol = policy_evict_first();
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    // (Runs differ by a row at most: only a last round has groups without one.)
    // The lane's row: `base` and, in a run that groups share, its own behind it.
    const int longest = kOwnRuns ? __reduce_max_sync(~0u, end - begin) : end - begin;
    const int behind = kOwnRuns ? 0 : lane;
    for (int done = a.waits.stall ? longest : 0; done < longest; done += step) {
      ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&empty[slot]), phase ^ 1, a.waits.limit_ns));
      if (!ok) break;
      const uint32_t bar = smem_u32(&full[slot]), to = ring + slot * slot_bytes;
      // With few buffers a later round's rows are asked into L2.
      const int base = begin + done, next = base + a.slots * step;
      const bool mine = lane < groups && base + behind < end;
      if (kVectors && !kOwnRuns && a.dense) {
        const int here = min(groups, end - base);
        const uint32_t bytes = static_cast<uint32_t>(here) * row_bytes;
        if (lane == 0) mbar_arrive_expect_tx(bar, bytes * a.tensors);
        __syncwarp();
        if (lane < a.tensors) {
          bulk_load(to + lane * tensor_bytes, a.src[lane] + base * a.src_stride[lane], bytes, bar, pol);
          if (a.slots < 3 && next < end)
            prefetch_l2(a.src[lane] + next * a.src_stride[lane],
                        static_cast<uint64_t>(min(groups, end - next)) * row_bytes);
        }
      } else {
        const int64_t i = base + behind;
        const unsigned char* from[5];
        uint32_t bytes[5], at[5], total = 0;
#pragma unroll
        for (int t = 0; t < 5; ++t) {
          bytes[t] = 0;
          if (!mine || t >= a.tensors) continue;
          const int64_t stride = a.src_stride[t];
          const unsigned char* p = reinterpret_cast<const unsigned char*>(a.src[t] + i * stride);
          const uint32_t off = kVectors ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
          at[t] = to + t * tensor_bytes + lane * pitch;
          // Granules [lo, hi) of the row's span, from its first one; those that
          // reach out of the tensor are left out, their elements of this row stored
          // one by one.
          const uint32_t stop = off + static_cast<uint32_t>(hidden) * 2;
          uint32_t lo = 0, hi = (stop + 15) & ~15u;
          if (off > i * stride * 2) lo = 16;
          if (hi - stop > (a.rows - 1 - i) * stride * 2) hi -= 16;
          hi = max(hi, lo);
          const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
          if (lo > 0)
            for (int j = 0; j < hidden && off + 2 * j < lo; ++j) set_shared_half(at[t] + off + 2 * j, q[j]);
          if (hi < stop)
            for (int j = hi > off ? static_cast<int>(hi - off) / 2 : 0; j < hidden; ++j)
              set_shared_half(at[t] + off + 2 * j, q[j]);
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
        for (int t = 0; t < 5; ++t) {
          if (bytes[t] > 0) bulk_load(at[t], from[t], bytes[t], bar, pol);
          if (a.slots < 3 && t < a.tensors && lane < groups && next + behind < end)
            prefetch_l2(a.src[t] + (next + behind) * a.src_stride[t], static_cast<uint64_t>(hidden) * 2);
        }
      }
      if (a.e_direct && mine)
        prefetch_l2(a.e + (base + behind) * a.e_stride, static_cast<uint64_t>(hidden) * 2);
      if (++slot == a.slots) slot = 0, phase ^= 1;
    }
    if (!ok) {
      if (lane == 0) report_give_up(a.waits);
      for (int k = 0; k < a.slots; ++k) {  // copies still in flight
        if (--slot < 0) slot = a.slots - 1, phase ^= 1;
        mbar_wait_bounded(smem_u32(&full[slot]), phase, kWaitLimitNs / 16);
      }
    }
    return;
  }
  pdl_trigger();

  // This thread's vector k.  (Of loose rows, what the whole warp has some of: lanes
  // past the end work on zeros.)
  auto inside = [&](int k) { return (kVectors ? in : in - lane) + k * row_threads < nvec; };
  const uint64_t keep = policy_evict_last();
  // Of a row in memory.
  auto load_weight = [&](uint32_t (&w)[4], const uint16_t* p, int k) {
    if constexpr (kVectors) {
      const Vec<16> q = ld_weight<16>(p + (in + k * row_threads) * 8, keep);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = q.w[e];
    } else {
      load_loose(w, LooseRow{p, hidden, false, false}, in + k * row_threads);
    }
  };
  // Of a row in shared memory that starts at `at`.
  auto load_row = [&](uint32_t (&w)[4], uint32_t at, int k) {
    if constexpr (kVectors) {
      shared_words(w, at + (in + k * row_threads) * 16);
    } else {
      const int v = in + k * row_threads, o = static_cast<int>(at & 15) / 2;
      if (v >= nvec) {
        w[0] = w[1] = w[2] = w[3] = 0;
        return;
      }
      uint32_t lo[4], hi[4] = {};
      shared_words(lo, (at & ~15u) + v * 16);
      if (o > 0) shared_words(hi, (at & ~15u) + v * 16 + 16);
      uint32_t both[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      shift_down(both, o);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = both[e];
      clear_tail(w, v, hidden);
    }
  };
  auto store_row = [&](uint16_t* row, int k, const uint32_t (&w)[4]) {
    if constexpr (kVectors) *reinterpret_cast<uint4*>(row + (in + k * row_threads) * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    else store_loose(row, hidden, in + k * row_threads, w);
  };

  // Weights (0 w, 1 p, 2 a shared gate row): in registers, in shared memory, or (the
  // gate row of many words a thread) where they are.
  uint32_t held[kHold ? 3 : 1][kHold ? W : 1];
  auto take_weight = [&](int which, const uint16_t* p) {
    if constexpr (kHold) {
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        if (!inside(k)) break;
        uint32_t w[4];
        load_weight(w, p, k);
#pragma unroll
        for (int e = 0; e < 4; ++e) held[which][4 * k + e] = w[e];
      }
    } else if (a.staged && (which < 2 || kGate == kChannels)) {
      for (int v = tid; v < nvec; v += workers)
        reinterpret_cast<uint4*>(row_mem)[which * nvec + v] = *reinterpret_cast<const uint4*>(p + v * 8);
    }
  };
  auto weight = [&](uint32_t (&w)[4], int which, const uint16_t* p, int k) {
    if constexpr (kHold) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = held[which][4 * k + e];
    } else if (a.staged && (which < 2 || kGate == kChannels)) {
      shared_words(w, staged + (which * nvec + in + k * row_threads) * 16);
    } else {
      load_weight(w, p, k);
    }
  };
  take_weight(0, a.w);
  if constexpr (kPost) take_weight(1, a.p);
  if constexpr (kGate == kChannels) take_weight(2, a.g);
  if (!kHold && a.staged) team_barrier(15, workers);

  float2 acc_w[W], acc_m[W];
#pragma unroll
  for (int k = 0; k < W; ++k) acc_w[k] = acc_m[k] = make_float2(0.f, 0.f);
  // Sums over rows, to a row of vectors.
  auto write_sums = [&](const float2 (&acc)[W], float* out) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      if (in + k * row_threads >= nvec) break;
      Vec<32> q;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        q.w[2 * e] = __float_as_uint(acc[4 * k + e].x);
        q.w[2 * e + 1] = __float_as_uint(acc[4 * k + e].y);
      }
      st_global<32>(out + (in + k * row_threads) * 8, q);
    }
  };
  // The groups' sums meet in shared memory (the ring, done with), the first group
  // writes them.
  auto join_sums = [&](float2 (&acc)[W], float* out) {
    if (groups > 1) {
      float2* sums = reinterpret_cast<float2*>(row_mem);
      team_barrier(15, workers);
#pragma unroll
      for (int k = 0; k < W; ++k) sums[k * workers + tid] = acc[k];
      team_barrier(15, workers);
      if (group > 0) return;
      for (int g = 1; g < groups; ++g) {
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k] = __fadd2_rn(acc[k], sums[k * workers + g * row_threads + tid]);
      }
    }
    write_sums(acc, out);
  };

  const float scale = 1.0f / static_cast<float>(hidden);
  const float2 residual_scale = make_float2(a.scale, a.scale);
  const bool one_gate = kGate == kOneGate && a.g;
  const int rows_per_gate = static_cast<int>(a.rows_per_gate);
  int slot = 0, turn = 0, held_gate = -1, gate_at = begin / rows_per_gate;
  uint32_t phase = 0;
  float sums[4] = {0.f, 0.f, 0.f, 0.f};  // of t^2, w D t and x^2 of the coming row, of p g dt x of the last one
  // A group's sums for the gates of its run before gate k: those for the one that its
  // rows had, zeros for the others.
  auto finish_gates = [&](int k) {
    for (; gate_at < k; ++gate_at) {
      const int64_t at = run + gate_at;
      write_sums(acc_m, a.m_parts + (kOwnRuns ? at : at * groups + group) * a.parts_ld);
#pragma unroll
      for (int q = 0; q < W; ++q) acc_m[q] = make_float2(0.f, 0.f);
    }
  };
  // Held or put back: p dt, times g where that is a row.
  float2 u[kHold ? W : 1];
  int64_t last = -1;  // the row whose last pass is due; its buffer, and what its sums are multiplied by
  uint32_t last_at = 0, last_bar = 0;
  float last_by = 0.f, last_inv = 0.f;
  for (int64_t i = first;; i += step) {
    const bool more = i < end;
    const uint32_t at = ring + slot * slot_bytes + group * pitch;
    auto start_of = [&](int t) {
      return at + t * tensor_bytes +
             (kVectors ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.src[t] + i * a.src_stride[t]) & 15));
    };
    uint32_t ts = 0, ds = 0, xs = 0;
    if (more) {
      // First pass.
      ts = start_of(0), ds = start_of(1);
      if (a.x_at >= 0) xs = start_of(a.x_at);
      if (!mbar_wait_bounded(smem_u32(&full[slot]), phase, a.waits.limit_ns)) gave_up[group] = 1;
      float2 st = make_float2(0.f, 0.f), sd = st, sx = st;
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        if (!inside(k)) break;
        uint32_t t[4], d[4], w[4], x[4];
        load_row(t, ts, k);
        load_row(d, ds, k);
        weight(w, 0, a.w, k);
        if constexpr (kPost) load_row(x, xs, k);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 tf = unpack2<T>(t[e]);
          st = __ffma2_rn(tf, tf, st);
          sd = __ffma2_rn(mul_pair<T>(w[e], d[e]), tf, sd);
          if constexpr (kPost) sx = fma_pair<T>(x[e], x[e], sx);
        }
      }
      sums[0] = st.x + st.y, sums[1] = sd.x + sd.y, sums[2] = sx.x + sx.y;
    }
    if (more || (last >= 0 && (kPost || one_gate))) {
      team_sums(sums, part[turn], warps, group * warps, barrier);
      turn ^= 1;
    }
    if (last >= 0) {
      // The row before's last pass:
      //   dx = inv_x (p g dt - m mean(p g dt m)) = u by - x inv_x^2 mean(u x by)
      if (one_gate && in == 0) a.gate_sums[last] = sums[3] * last_inv;
      if constexpr (kPost) {
        const float b = -sums[3] * last_by * last_inv * last_inv * scale;
        const float2 back = make_float2(b, b), by = make_float2(last_by, last_by);
        uint16_t* dx = a.dx + last * a.dx_stride;
        const uint32_t x_at = last_at + a.x_at * tensor_bytes +
            (kVectors ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.src[a.x_at] + last * a.src_stride[a.x_at]) & 15));
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
          if (!inside(k)) break;
          uint32_t x[4], ux[4], uy[4], o[4];
          load_row(x, x_at, k);
          if constexpr (!kHold) {
            shared_words(ux, last_at + (in + k * row_threads) * 16);
            shared_words(uy, last_at + tensor_bytes + (in + k * row_threads) * 16);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float2 pgdt;
            if constexpr (kHold) pgdt = u[4 * k + e];
            else pgdt = make_float2(__uint_as_float(ux[e]), __uint_as_float(uy[e]));
            const float2 v = __ffma2_rn(pgdt, by, __fmul2_rn(unpack2<T>(x[e]), back));
            o[e] = pack2<T>(v.x, v.y);
          }
          store_row(dx, k, o);
        }
        // The words put into the buffer, before the next copies into it.
        if constexpr (!kHold) fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(last_bar);
    }
    if (!more) break;
    if (*static_cast<volatile int*>(&gave_up[group])) {
      // The copier may have issued its last row and left without a wait.
      if (in == 0) report_give_up(a.waits);
      break;
    }
    const uint16_t* gate_row = a.g;
    if constexpr (kSharedRow) {
      const int k = static_cast<int>(i) / rows_per_gate;
      gate_row = a.g + k * a.g_stride;
      if (k != held_gate) {
        finish_gates(k);
        take_weight(2, gate_row);
        held_gate = k;
      }
    }
    // Second pass: dt = w D inv_t + (E - t mean inv_t^2); the sums over a row leave
    // inv_x out.
    const float inv_t = rsqrtf(sums[0] * scale + a.eps), mean = sums[1] * inv_t * scale;
    const float inv_x = kPost ? rsqrtf(sums[2] * scale + a.eps) : 1.f;
    float by = inv_x;
    if constexpr (kGate == kOneGate) {
      if (a.g) by *= unpack1<T>(a.g[(static_cast<uint32_t>(i) / static_cast<uint32_t>(rows_per_gate)) * a.g_stride]);
    }
    const float2 inv_t2 = make_float2(inv_t, inv_t), minus = make_float2(-mean * inv_t * inv_t, -mean * inv_t * inv_t);
    const float2 m_by = make_float2(by, by);
    float2 su = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      if (!inside(k)) break;
      uint32_t t[4], d[4], w[4], x[4] = {}, e4[4] = {}, g[4], p[4], out_r[4], out_g[4];
      if (a.e_direct) load_loose(e4, loose_row(a.e, i, a.rows, a.e_stride, hidden), in + k * row_threads);
      load_row(t, ts, k);
      load_row(d, ds, k);
      weight(w, 0, a.w, k);
      if (a.x_at >= 0) load_row(x, xs, k);
      if (a.e_at >= 0) load_row(e4, start_of(a.e_at), k);
      if constexpr (kPost) weight(p, 1, a.p, k);
      if constexpr (kGate == kGateEach) load_row(g, start_of(a.g_at), k);
      if constexpr (kSharedRow || kGate == kChannels) weight(g, 2, gate_row, k);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 dt = __ffma2_rn(mul_pair<T>(w[e], d[e]), inv_t2, __ffma2_rn(unpack2<T>(t[e]), minus, unpack2<T>(e4[e])));
        acc_w[4 * k + e] = __ffma2_rn(mul_pair<T>(d[e], t[e]), inv_t2, acc_w[4 * k + e]);
        const float2 xf = unpack2<T>(x[e]), q = __fmul2_rn(dt, xf);
        float2 pdt = dt;
        if constexpr (kGate == kOneGate) {
          acc_m[4 * k + e] = __ffma2_rn(q, m_by, acc_m[4 * k + e]);
          if constexpr (kPost) pdt = __fmul2_rn(dt, unpack2<T>(p[e]));
        } else {
          if constexpr (kGate == kGateEach)
            acc_m[4 * k + e] = __ffma2_rn(__fmul2_rn(q, unpack2<T>(g[e])), m_by, acc_m[4 * k + e]);
          else
            acc_m[4 * k + e] = __ffma2_rn(q, m_by, acc_m[4 * k + e]);
          if constexpr (kPost) pdt = __fmul2_rn(dt, mul_pair<T>(p[e], g[e]));
          else pdt = __fmul2_rn(dt, unpack2<T>(g[e]));
        }
        su = __ffma2_rn(pdt, xf, su);
        const float2 r = __fmul2_rn(dt, residual_scale);
        out_r[e] = pack2<T>(r.x, r.y);
        if constexpr (kGate == kGateEach) {
          float2 v = __fmul2_rn(q, m_by);
          if constexpr (kPost) v = __fmul2_rn(v, unpack2<T>(p[e]));
          out_g[e] = pack2<T>(v.x, v.y);
        }
        if constexpr (!kPost) {
          const float2 v = kGate == kOneGate ? __fmul2_rn(pdt, m_by) : pdt;
          t[e] = pack2<T>(v.x, v.y);
        } else if constexpr (kHold) {
          u[4 * k + e] = pdt;
        } else {
          t[e] = __float_as_uint(pdt.x), d[e] = __float_as_uint(pdt.y);
        }
      }
      store_row(a.dr + i * a.dr_stride, k, out_r);
      if constexpr (kGate == kGateEach) store_row(a.dg + i * a.dg_stride, k, out_g);
      if constexpr (!kPost) {
        store_row(a.dx + i * a.dx_stride, k, t);
      } else if constexpr (!kHold) {
        set_shared_words(ts + (in + k * row_threads) * 16, t);
        set_shared_words(ds + (in + k * row_threads) * 16, d);
      }
    }
    sums[3] = su.x + su.y;
    last = i, last_at = at, last_bar = smem_u32(&empty[slot]), last_by = by, last_inv = inv_x;
    if (++slot == a.slots) slot = 0, phase ^= 1;
  }
  // Buffers of a last round with fewer rows than groups are nobody's any more.
  if constexpr (kSharedRow) finish_gates((end - 1) / rows_per_gate + 1);
  else join_sums(acc_m, a.m_parts + blockIdx.x * a.parts_ld);
  join_sums(acc_w, a.dw_parts + blockIdx.x * a.parts_ld);
}

// The weights' and a shared gate row's gradients from block_grad_rows' sums: 32
// columns a CTA.  Its 16 warps share out the CTAs' sums; where rows of the gate
// are few they share out each one's sums as well, else they take gates in turn.
constexpr int kRunWarps = 16;

template <typename T>
__global__ void __launch_bounds__(32 * kRunWarps) block_grad_runs(BlockGradArgs a) {
  __shared__ float sums[2][kRunWarps][32];
  pdl_wait();
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  const bool shared_row = a.gate_row && !a.gate_each, in = j < a.hidden;
  const int ctas = static_cast<int>(a.ctas);
  float sw = 0.f, sp = 0.f;
  if (in) {
#pragma unroll 10
    for (int c = ty; c < ctas; c += kRunWarps) sw += a.dw_parts[c * a.parts_ld + j];
  }
  if (!shared_row) {
    if (in) {
#pragma unroll 10
      for (int c = ty; c < ctas; c += kRunWarps) sp += a.m_parts[c * a.parts_ld + j];
    }
  } else {
    const float p = in && a.p ? unpack1<T>(a.p[j]) : 1.f;
    const bool together = a.gates <= 2;
    const int groups = a.gates > 1 && !a.own_runs ? a.row_groups : 1;
    for (int64_t k = together ? 0 : ty; k < a.gates; k += together ? 1 : kRunWarps) {
      // The sums of the runs that the gate's rows lie in follow each other.
      const int64_t first = (run_of(a, k * a.rows_per_gate) + k) * groups;
      const int64_t end = (run_of(a, (k + 1) * a.rows_per_gate - 1) + k + 1) * groups;
      float sm = 0.f;
      if (in) {
#pragma unroll 10
        for (int64_t e = first + (together ? ty : 0); e < end; e += together ? kRunWarps : 1) sm += a.m_parts[e * a.parts_ld + j];
      }
      if (together) {
        __syncthreads();
        sums[0][ty][tx] = sm;
        __syncthreads();
        if (ty > 0) continue;
#pragma unroll
        for (int q = 1; q < kRunWarps; ++q) sm += sums[0][q][tx];
      }
      if (!in) continue;
      sp = fmaf(unpack1<T>(a.g[k * a.g_stride + j]), sm, sp);
      a.dg[k * a.dg_stride + j] = pack1<T>(sm * p);
    }
    __syncthreads();
  }
  sums[0][ty][tx] = sw, sums[1][ty][tx] = sp;
  __syncthreads();
  if (ty > 0 || !in) return;
#pragma unroll
  for (int k = 1; k < kRunWarps; ++k) sw += sums[0][k][tx], sp += sums[1][k][tx];
  a.dw[j] = pack1<T>(sw);
  if (a.dp) a.dp[j] = pack1<T>(sp);
}

// ---------------------------------------------------------------------------
// Rows that block_grad_rows has no variant for, read twice, element by element: from
// 16897 elements, from 8449 where they start anywhere, from 14081 with a gate for every
// element, of which two buffers have no room (us: 4096 x 9001 384, x 10001 411, x 16383
// 718; 4096 x 16384 with a full gate 813, where one row for all takes 239 in the ring).

// The values of one element of row i that the sums and outputs are made of.
template <typename T>
struct BlockGradElement {
  float d, e, n, m, p, g, wd;
  __device__ __forceinline__ BlockGradElement(const BlockGradArgs& a, int64_t i, int64_t j, const uint16_t* gate,
                                         float inv_t, float inv_x) {
    d = unpack1<T>(a.d[i * a.d_stride + j]);
    e = a.e ? unpack1<T>(a.e[i * a.e_stride + j]) : 0.f;
    n = unpack1<T>(a.t[i * a.t_stride + j]) * inv_t;
    m = unpack1<T>(a.x[i * a.x_stride + j]) * inv_x;
    p = a.p ? unpack1<T>(a.p[j]) : 1.f;
    g = gate ? unpack1<T>(gate[a.gate_row ? j : 0]) : 1.f;
    wd = unpack1<T>(a.w[j]) * d;
  }
  __device__ __forceinline__ float dt(float inv_t, float mean) const { return inv_t * (wd - n * mean) + e; }
};

template <typename T>
__device__ __forceinline__ const uint16_t* gate_of(const BlockGradArgs& a, int64_t i) {
  return a.g ? a.g + (static_cast<uint32_t>(i) / static_cast<uint32_t>(a.rows_per_gate)) * a.g_stride : nullptr;
}

// One CTA per row: the row's means.
template <typename T>
__global__ void __launch_bounds__(256) block_grad_stats(BlockGradArgs a) {
  __shared__ float part[4][32];
  pdl_wait();
  const int64_t i = blockIdx.x;
  const uint16_t* gate = gate_of<T>(a, i);
  const float inv_hidden = 1.f / static_cast<float>(a.hidden);
  float st = 0.f, sx = 0.f, sd = 0.f;
  for (int64_t j = threadIdx.x; j < a.hidden; j += 256) {
    const BlockGradElement<T> v(a, i, j, gate, 1.f, 1.f);
    st = fmaf(v.n, v.n, st), sx = fmaf(v.m, v.m, sx), sd = fmaf(v.wd, v.n, sd);
  }
  st = row_sum(st, part[0], 8, 0), sx = row_sum(sx, part[1], 8, 0), sd = row_sum(sd, part[2], 8, 0);
  const float inv_t = rsqrtf(st * inv_hidden + a.eps), inv_x = a.p ? rsqrtf(sx * inv_hidden + a.eps) : 1.f;
  const float mean = sd * inv_t * inv_hidden;
  float s = 0.f;
  for (int64_t j = threadIdx.x; j < a.hidden; j += 256) {
    const BlockGradElement<T> v(a, i, j, gate, inv_t, inv_x);
    s = fmaf(v.dt(inv_t, mean) * v.p * (a.gate_row ? v.g : 1.f), v.m, s);
  }
  s = row_sum(s, part[3], 8, 0);
  if (threadIdx.x != 0) return;
  if (a.gate_sums) a.gate_sums[i] = s;
  if (gate && !a.gate_row) s *= unpack1<T>(gate[0]);
  a.stats[i] = make_float4(inv_t, mean, inv_x, a.p ? s * inv_hidden : 0.f);
}

// A part of the rows x 256 columns per CTA: the rows' outputs, the part's sums.
template <typename T>
__global__ void __launch_bounds__(256) block_grad_columns(BlockGradArgs a) {
  pdl_wait();
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (j >= a.hidden) return;
  const bool shared_row = a.gate_row && !a.gate_each;
  const int64_t gates = shared_row ? a.gates : 1, rows = shared_row ? a.rows_per_gate : a.rows;
  for (int64_t part = blockIdx.y; part < gates * a.parts; part += gridDim.y) {
    const int64_t first = part / a.parts * rows, in = part % a.parts * a.part_rows;
    const int64_t end = first + min(rows, in + a.part_rows);
    float sw = 0.f, sm = 0.f;
    for (int64_t i = first + in; i < end; ++i) {
      const float4 st = a.stats[i];
      const BlockGradElement<T> v(a, i, j, gate_of<T>(a, i), st.x, st.z);
      const float dt = v.dt(st.x, st.y);
      a.dr[i * a.dr_stride + j] = pack1<T>(a.scale * dt);
      a.dx[i * a.dx_stride + j] = pack1<T>(a.p ? st.z * (v.p * v.g * dt - v.m * st.w) : v.g * dt);
      sw = fmaf(v.d, v.n, sw);
      sm = fmaf(shared_row ? dt : v.g * dt, v.m, sm);
      if (a.gate_each) a.dg[i * a.dg_stride + j] = pack1<T>(dt * v.m * v.p);
    }
    a.dw_parts[part * a.parts_ld + j] = sw;
    a.m_parts[part * a.parts_ld + j] = sm;
  }
}

// The weights' and a shared gate row's gradients from the parts' sums: 32
// columns a CTA, its 8 warps taking gates (or, where there are none, parts) in
// turn.
template <typename T>
__global__ void __launch_bounds__(256) block_grad_join(BlockGradArgs a) {
  __shared__ float sums[2][8][32];
  pdl_wait();
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + tx;
  const bool shared_row = a.gate_row && !a.gate_each;
  float sw = 0.f, sp = 0.f;
  if (j < a.hidden) {
    if (shared_row) {
      const float p = a.p ? unpack1<T>(a.p[j]) : 1.f;
      for (int64_t k = ty; k < a.gates; k += 8) {
        float sm = 0.f;
        for (int64_t part = k * a.parts; part < (k + 1) * a.parts; ++part) {
          sw += a.dw_parts[part * a.parts_ld + j];
          sm += a.m_parts[part * a.parts_ld + j];
        }
        sp = fmaf(unpack1<T>(a.g[k * a.g_stride + j]), sm, sp);
        a.dg[k * a.dg_stride + j] = pack1<T>(sm * p);
      }
    } else {
      for (int64_t part = ty; part < a.parts; part += 8) {
        sw += a.dw_parts[part * a.parts_ld + j];
        sp += a.m_parts[part * a.parts_ld + j];
      }
    }
  }
  sums[0][ty][tx] = sw, sums[1][ty][tx] = sp;
  __syncthreads();
  if (ty > 0 || j >= a.hidden) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) sw += sums[0][k][tx], sp += sums[1][k][tx];
  a.dw[j] = pack1<T>(sw);
  if (a.dp) a.dp[j] = pack1<T>(sp);
}

// The gradients of gates of one value: one CTA adds up the rows that share one.
template <typename T>
__global__ void __launch_bounds__(256) block_grad_gates(BlockGradArgs a) {
  __shared__ float part[32];
  pdl_wait();
  for (int64_t k = blockIdx.x; k < a.gates; k += gridDim.x) {
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < a.rows_per_gate; i += 256) s += a.gate_sums[k * a.rows_per_gate + i];
    s = row_sum(s, part, 8, 0);
    if (threadIdx.x == 0) a.dg[k * a.dg_stride] = pack1<T>(s);
    __syncthreads();
  }
}

namespace {

// How block_grad_rows takes the rows; words 0 where it does not.
struct BlockGradPlan {
  int words, smem;
  bool vectors;
};

BlockGradPlan plan_block_grad(BlockGradArgs& a) {
  BlockGradPlan plan{};
  plan.vectors = a.hidden % 8 == 0 && tma_rows(a.dx, a.rows, a.dx_stride) && tma_rows(a.dr, a.rows, a.dr_stride) &&
                 tma_rows(a.t, a.rows, a.t_stride) && tma_rows(a.d, a.rows, a.d_stride) &&
                 tma_rows(a.x, a.rows, a.x_stride) && (!a.e || tma_rows(a.e, a.rows, a.e_stride)) &&
                 aligned(a.w, 16) && aligned(a.p, 16) &&
                 (!a.gate_each || (tma_rows(a.dg, a.rows, a.dg_stride) && tma_rows(a.g, a.rows, a.g_stride))) &&
                 (!a.gate_row || a.gate_each || tma_rows(a.g, a.gates, a.g_stride));
  if (a.rows <= 0 || a.hidden <= 0) return plan;
  const int64_t nvec = (a.hidden + 7) / 8;
  // Two buffers at least: a row's last pass waits for the next one's first.  Where E
  // leaves no room for them it stays outside.
  for (int direct = 0; direct < (a.e ? 2 : 1); ++direct) {
    a.tensors = 0, a.x_at = a.e_at = a.g_at = -1, a.e_direct = direct;
    auto add = [&](const uint16_t* p, int64_t stride) {
      a.src[a.tensors] = p, a.src_stride[a.tensors] = a.rows > 1 ? stride : a.hidden;
      return a.tensors++;
    };
    add(a.t, a.t_stride);
    add(a.d, a.d_stride);
    if (a.p || a.g) a.x_at = add(a.x, a.x_stride);
    if (a.e && !direct) a.e_at = add(a.e, a.e_stride);
    if (a.gate_each) a.g_at = add(a.g, a.g_stride);
    a.dense = true;
    for (int k = 0; k < a.tensors; ++k) a.dense = a.dense && a.src_stride[k] == a.hidden;
    const int64_t slot = (nvec * 16 + (plan.vectors ? 0 : 16)) * a.tensors;
    for (int words : {4, 8, 12, 24}) {
      if (words > 12 && !plan.vectors) break;
      const int64_t threads = round_up((nvec + words / 4 - 1) / (words / 4), 32);
      if (threads > block_threads(words) || (words == 4 && threads > 128)) continue;
      int64_t groups = block_threads(words) / threads;
      if (groups > 14) groups = 14;  // a hardware barrier each, and one for all
      if (groups > a.rows) groups = a.rows;
      // (Places for w, p and the gate's row.)
      const int64_t weights = words <= 12 ? 0 : (a.gate_row && a.gates == 1 ? 3 : 2) * nvec * 16;
      while (groups > 1 && weights + 2 * groups * slot > kBlockSmem) --groups;
      const bool staged = weights > 0 && weights + 2 * groups * slot <= kBlockSmem;
      int64_t slots = (kBlockSmem - (staged ? weights : 0)) / (groups * slot);
      if (slots > kBlockSlots) slots = kBlockSlots;
      if (slots < 2) continue;
      plan.words = words;
      a.row_threads = static_cast<int>(threads), a.row_groups = static_cast<int>(groups), a.slots = static_cast<int>(slots);
      a.staged = staged, a.ring_at = static_cast<uint32_t>(staged ? weights : 0);
      const int64_t ring = a.ring_at + slots * groups * slot, joined = groups > 1 ? words * threads * groups * 8 : 0;
      plan.smem = static_cast<int>(ring > joined ? ring : joined);
      const int64_t need = (a.rows + groups - 1) / groups;
      // (A B200's SMs, as in the tilings: workspaces are sized without a device.)
      a.ctas = need < 148 ? need : 148;
      a.runs = a.ctas;
      a.own_runs = a.gate_row && !a.gate_each && a.gates > 2 * a.ctas;
      if (a.own_runs) a.runs = a.ctas * groups < a.rows ? a.ctas * groups : a.rows;
      break;
    }
    if (plan.words > 0) break;
  }
  return plan;
}

template <typename T, bool kVectors, bool kPost, int kGate>
void (*block_grad_kernel(int words))(BlockGradArgs) {
  switch (words) {
    case 4: return block_grad_rows<T, 4, kVectors, kPost, kGate>;
    case 8: return block_grad_rows<T, 8, kVectors, kPost, kGate>;
    case 12: return block_grad_rows<T, 12, kVectors, kPost, kGate>;
  }
  if constexpr (kVectors) return block_grad_rows<T, 24, true, kPost, kGate>;
  return nullptr;
}
template <typename T, bool kVectors>
void (*block_grad_kernel(const BlockGradArgs& a, int words))(BlockGradArgs) {
  const int gate = !a.gate_row ? kOneGate : a.gate_each ? kGateEach : a.gates == 1 ? kChannels : a.own_runs ? kGateRuns : kGateRow;
  if (gate == kChannels)
    return a.p ? block_grad_kernel<T, kVectors, true, kChannels>(words) : block_grad_kernel<T, kVectors, false, kChannels>(words);
  if (gate == kOneGate)
    return a.p ? block_grad_kernel<T, kVectors, true, kOneGate>(words) : block_grad_kernel<T, kVectors, false, kOneGate>(words);
  if (gate == kGateRuns)
    return a.p ? block_grad_kernel<T, kVectors, true, kGateRuns>(words) : block_grad_kernel<T, kVectors, false, kGateRuns>(words);
  if (gate == kGateRow)
    return a.p ? block_grad_kernel<T, kVectors, true, kGateRow>(words) : block_grad_kernel<T, kVectors, false, kGateRow>(words);
  return a.p ? block_grad_kernel<T, kVectors, true, kGateEach>(words) : block_grad_kernel<T, kVectors, false, kGateEach>(words);
}

template <typename T>
int launch_backward(const BlockGradArgs& a, const BlockGradPlan& plan, const DeviceInfo* dev, cudaStream_t stream,
                    unsigned flags) {
  const char* what = "gated_add_rms_norm_backward";
  int st = HPRN_OK;
  if (plan.words > 0) {
    const auto fn = plan.vectors ? block_grad_kernel<T, true>(a, plan.words) : block_grad_kernel<T, false>(a, plan.words);
    if ((st = allow_smem(dev, reinterpret_cast<const void*>(fn), kBlockSmem, what)) != HPRN_OK) return st;
    st = launch_rows_smem(fn, dim3(static_cast<unsigned>(a.ctas)),
                          dim3(static_cast<unsigned>(a.row_threads * a.row_groups + 32)), plan.smem, stream, flags, what, a);
    if (st != HPRN_OK) return st;
  } else if (a.rows > 0) {
    st = launch_rows(block_grad_stats<T>, dim3(static_cast<unsigned>(a.rows)), dim3(256), stream, flags, what, a);
    if (st != HPRN_OK) return st;
    const int64_t parts = (a.gate_row && !a.gate_each ? a.gates : 1) * a.parts;
    st = launch_rows(block_grad_columns<T>,
                     dim3(static_cast<unsigned>((a.hidden + 255) / 256), static_cast<unsigned>(parts < 65535 ? parts : 65535)),
                     dim3(256), stream, flags, what, a);
    if (st != HPRN_OK) return st;
  }
  if (a.rows > 0 && a.gate_sums) {
    st = launch_rows(block_grad_gates<T>, dim3(static_cast<unsigned>(a.gates < 65535 ? a.gates : 65535)), dim3(256),
                     stream, flags, what, a);
    if (st != HPRN_OK) return st;
  }
  const dim3 columns(static_cast<unsigned>((a.hidden + 31) / 32));
  return plan.words > 0 ? launch_rows(block_grad_runs<T>, columns, dim3(32 * kRunWarps), stream, flags, what, a)
                        : launch_rows(block_grad_join<T>, columns, dim3(256), stream, flags, what, a);
}

}  // namespace
}  // namespace hprn

extern "C" {

int hprn_gated_add_rms_norm_backward(
    void* grad_input, void* grad_residual, void* grad_post_weight, void* grad_weight, void* grad_gate,
    const void* grad_out, const void* grad_residual_out, const void* input, const void* residual_out,
    const void* post_weight, const void* weight, const void* gate, int64_t rows, int64_t hidden,
    int64_t rows_per_gate, int64_t gate_width, int64_t grad_input_row_stride, int64_t grad_residual_row_stride,
    int64_t grad_gate_row_stride, int64_t grad_out_row_stride, int64_t grad_residual_out_row_stride,
    int64_t input_row_stride, int64_t residual_out_row_stride, int64_t gate_row_stride, double residual_scale,
    double eps, int dtype, void* workspace, int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  int st = check_block_norm(rows, hidden, rows_per_gate, gate_width, gate != nullptr, dtype);
  if (st != HPRN_OK) return st;
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  const int64_t gates = gate ? rows / rows_per_gate : 1;
  if ((rows > 1 && (grad_input_row_stride < hidden || grad_residual_row_stride < hidden ||
                    grad_out_row_stride < hidden || (grad_residual_out && grad_residual_out_row_stride < hidden) ||
                    input_row_stride < hidden || residual_out_row_stride < hidden)) ||
      (gate && gates > 1 && (gate_row_stride < gate_width || grad_gate_row_stride < gate_width)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  BlockGradArgs a{};
  a.dx = static_cast<uint16_t*>(grad_input), a.dr = static_cast<uint16_t*>(grad_residual);
  a.dp = static_cast<uint16_t*>(grad_post_weight), a.dw = static_cast<uint16_t*>(grad_weight);
  a.dg = static_cast<uint16_t*>(grad_gate);
  a.d = static_cast<const uint16_t*>(grad_out), a.e = static_cast<const uint16_t*>(grad_residual_out);
  a.x = static_cast<const uint16_t*>(input), a.t = static_cast<const uint16_t*>(residual_out);
  a.p = static_cast<const uint16_t*>(post_weight), a.w = static_cast<const uint16_t*>(weight);
  a.g = static_cast<const uint16_t*>(gate);
  a.dx_stride = grad_input_row_stride, a.dr_stride = grad_residual_row_stride, a.dg_stride = grad_gate_row_stride;
  a.d_stride = grad_out_row_stride, a.e_stride = grad_residual_out_row_stride, a.x_stride = input_row_stride;
  a.t_stride = residual_out_row_stride, a.g_stride = gate_row_stride;
  a.rows = rows, a.hidden = hidden;
  a.rows_per_gate = gate ? rows_per_gate : 1, a.gates = gates;
  // (With hidden 1 a gate of one value is a row of one.)
  a.gate_row = gate && gate_width == hidden, a.gate_each = a.gate_row && rows_per_gate == 1;
  a.scale = static_cast<float>(residual_scale), a.eps = static_cast<float>(eps);
  const bool shared_row = a.gate_row && !a.gate_each;
  const int64_t share = shared_row ? rows_per_gate : rows;
  a.parts = shared_row ? (64 + gates - 1) / (gates > 0 ? gates : 1) : 64;
  if (a.parts > share) a.parts = share > 0 ? share : 1;
  a.part_rows = (share + a.parts - 1) / a.parts;
  a.parts = a.part_rows > 0 ? (share + a.part_rows - 1) / a.part_rows : 0;
  const BlockGradPlan plan = plan_block_grad(a);
  Workspace ws(workspace, *workspace_bytes);
  a.stats = ws.take<float4>(plan.words > 0 ? 0 : rows);
  a.gate_sums = ws.take<float>(gate && !a.gate_row ? rows : 0);
  if (!gate || a.gate_row) a.gate_sums = nullptr;
  a.parts_ld = round_up(hidden, 8);
  // A run and a gate it meets make one row of sums (for each group of threads that shares
  // it): each step to the next of them goes on by a run, a gate or both, so that run +
  // gate tells them apart.
  const int64_t parts = (shared_row ? gates : 1) * a.parts;
  a.dw_parts = ws.take<float>((plan.words > 0 ? a.ctas : parts) * a.parts_ld);
  a.m_parts = ws.take<float>((plan.words == 0 ? parts : shared_row && gates > 1 ? (a.runs + gates) * (a.own_runs ? 1 : a.row_groups) : a.runs) * a.parts_ld);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (hidden == 0) return ok();
  if (!grad_weight || !weight || (post_weight && !grad_post_weight) ||
      (rows > 0 && (!grad_input || !grad_residual || !grad_out || !input || !residual_out || (gate && !grad_gate))))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!post_weight) a.dp = nullptr;
  for (const void* p : {static_cast<const void*>(grad_input), static_cast<const void*>(grad_residual),
                        static_cast<const void*>(grad_post_weight), static_cast<const void*>(grad_weight),
                        static_cast<const void*>(grad_gate), grad_out, grad_residual_out, input, residual_out,
                        post_weight, weight, gate})
    if (!aligned(p, 2)) return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(grad_input, rows, hidden, grad_input_row_stride),
                         extent16(grad_residual, rows, hidden, grad_residual_row_stride),
                         extent16(a.dp, 1, hidden, hidden), extent16(grad_weight, 1, hidden, hidden),
                         extent16(gate ? grad_gate : nullptr, gates, gate_width, grad_gate_row_stride)};
  const Extent ins[] = {extent16(grad_out, rows, hidden, grad_out_row_stride),
                        extent16(grad_residual_out, rows, hidden, grad_residual_out_row_stride),
                        extent16(input, rows, hidden, input_row_stride),
                        extent16(residual_out, rows, hidden, residual_out_row_stride),
                        extent16(post_weight, 1, hidden, hidden), extent16(weight, 1, hidden, hidden),
                        extent16(gate, gates, gate_width, gate_row_stride)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if ((st = waits_of(dev, &a.waits, "gated_add_rms_norm_backward")) != HPRN_OK) return st;
  return dtype == HPRN_DTYPE_BF16 ? launch_backward<__nv_bfloat16>(a, plan, dev, cs, flags)
                                  : launch_backward<__half>(a, plan, dev, cs, flags);
}

}  // extern "C"

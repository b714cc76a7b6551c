// Log probabilities under the softmax of a linear layer over a vocabulary,
// without keeping the logits: with L = X W^T / T (T the temperature),
//   lse_i = log sum_j exp(L_ij),  log_prob_i = L_{i, t_i} - lse_i,
//   entropy_i = -sum_j p_ij log p_ij,  p_ij = exp(L_ij - lse_i),
// both 0 where the target t_i is `ignore_index`, and the `top` largest log
// probabilities of a row with their indices.
//
// Forward: each tile of X W^T leaves, per row, its largest value m, and relative
// to it s = sum_j e_j and a = sum_j e_j x_j, e_j = 2^x_j, x_j = (l_j - m) log2(e) / T.
// Joined over the tiles (s, a and m the row's), lse = m / T + log s and
// entropy = log s - ln(2) a / s.
//
// The largest ones are found in two steps.  Where they are asked for, the tiles
// also leave the logits of a block of rows and the largest of every 32
// neighbouring ones (LogProbEpilogue<true>); the `top` largest logits lie among the `top`
// groups of 32 with the largest maxima, so that a row's search reads a 32nd of
// its logits' number and a few groups.  Of many rows a first part of the vocabulary
// bounds the largest maxima from below, and only groups that reach the bound leave
// their logits.  A few more than `top` are taken, their logits summed again in 64
// bits, and ordered by those; equal ones go to the lowest index.  So the order does
// not hang on how the tensor cores' sums fall out in their last bits.
//
// Backward, g_i and h_i the gradients of log_prob_i and entropy_i:
//   S_ij = (g_i ([j == t_i] - p_ij) - h_i p_ij (log p_ij + entropy_i)) / T
//   dX = S W,  dW = S^T X
// in pieces of the vocabulary as in linear_cross_entropy.cu, S held in the inputs' 16
// bits, which is what the tensor cores multiply (gradients 2.4e-3 from 64 bits in bf16,
// 1.7e-3 with S in 32), relative to
// the largest finite |g_i| or |h_i| and, in fp16, times 2^14 without and 2^13
// with an entropy gradient: |p (log p + entropy)| is at most 0.7 + ln(vocab) / 4,
// 5.9 for the largest vocabulary, which with 1 for the other term and 2^13 stays
// below 65504.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "few_rows.cuh"
#include "matmul.cuh"
#include "runtime.cuh"
#include "vocabulary.cuh"

namespace hprn {

// max(a, b), NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Exponents below this have powers of 0; -inf itself would make 0 * -inf of them.
constexpr float kLeastExponent = -200.f;

template <bool kTop>
struct LogProbEpilogue {
  static constexpr bool kPaired = false;
  static constexpr int kSegment = kLogitSegment;
  static constexpr bool kUnrolled = true;
  float4* partial = nullptr;  // [rows, parts]: {m, s, a, 0}
  float* target_logit = nullptr;
  const int64_t* target = nullptr;
  int64_t ignore = 0;
  int64_t parts = 0;
  int64_t vocab = 0;  // of these columns, which are those from `first` of `all`
  int64_t first = 0, all = 0;
  float to_log2 = kLog2e;  // log2(e) / T
  float* logits = nullptr;       // [rows, 32 groups]
  float* group_max = nullptr;    // [rows, groups]
  const float* bound = nullptr;  // or: groups with a maximum below it leave no logits
  int64_t groups = 0;

  struct Row {
    float m, s, a, bound;
    int64_t t;
  };
  __device__ __forceinline__ Row begin(const Lane& l, int64_t i) const {
    return Row{-INFINITY, 0.f, 0.f, kTop && bound && l.inside ? bound[i] : -INFINITY,
               l.inside ? target_of(target, i, ignore, all) - first : kIgnored};
  }
  __device__ __forceinline__ void chunk(Row& r, const Lane& l, int64_t i, int64_t j, float (&v)[kChunk]) const {
    if (j + kChunk > vocab) {
      const int left = static_cast<int>(vocab - j);
#pragma unroll
      for (int k = 0; k < kChunk; ++k)
        if (k >= left) v[k] = -INFINITY;
    }
    const int64_t at = r.t - j;
    if (at >= 0 && at < kChunk) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < kChunk; ++k) x = at == k ? v[k] : x;
      target_logit[i] = x;
    }
    float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int k = 4; k < kChunk; ++k) top[k % 4] = fmaxf(top[k % 4], v[k]);
    const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    if constexpr (kTop) {
      if (l.inside) {
        if (!(most < r.bound)) {
          float* q = logits + i * (groups * kChunk) + j;
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            Vec<32> o;
#pragma unroll
            for (int k = 0; k < 8; ++k) o.w[k] = __float_as_uint(v[8 * h + k]);
            st_global<32>(q + 8 * h, o);
          }
        }
        group_max[i * groups + j / kChunk] = most;
      }
    }
    const float m = fmaxf(r.m, most);
    // All so far -inf (or NaN, which fmaxf skips and the sums keep): 2^(-inf) = 0.
    const float ref = m == -INFINITY ? 0.f : m;
    const float x0 = max_nan((r.m - ref) * to_log2, kLeastExponent), f = exp2_fast(x0);
    const float2 minus = make_float2(-ref, -ref), c = make_float2(to_log2, to_log2);
    float2 s[2] = {make_float2(r.s * f, 0.f), make_float2(0.f, 0.f)};
    float2 a[2] = {make_float2(f * fmaf(r.s, x0, r.a), 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < kChunk / 2; ++k) {
      float2 x = __fmul2_rn(__fadd2_rn(make_float2(v[2 * k], v[2 * k + 1]), minus), c);
      x.x = max_nan(x.x, kLeastExponent), x.y = max_nan(x.y, kLeastExponent);
      const float2 e = make_float2(exp2_fast(x.x), exp2_fast(x.y));
      s[k % 2] = __fadd2_rn(s[k % 2], e);
      a[k % 2] = __ffma2_rn(e, x, a[k % 2]);
    }
    r.m = m, r.s = (s[0].x + s[0].y) + (s[1].x + s[1].y), r.a = (a[0].x + a[0].y) + (a[1].x + a[1].y);
  }
  __device__ __forceinline__ void end(Row& r, const Lane& l, int64_t i, int64_t part) const {
    if (l.inside) partial[i * parts + part] = make_float4(r.m, r.s, r.a, 0.f);
  }
};

struct LogProbJoin {
  const float4* partial;
  const float* target_logit;
  const int64_t* target;
  int64_t ignore, rows, vocab, parts;  // parts 0: logits that are sums of no terms
  float inv_t, to_log2;
  float *log_prob, *entropy, *lse;
};

// Threads kThreads of a CTA's that meet at hardware barrier `barrier`.
template <int kThreads>
__device__ __forceinline__ void meet(int barrier) {
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(kThreads) : "memory");
}

// Joins the parts of row i, by kJoinThreads threads `thread`: the largest first, then
// the sums relative to it, so that no term waits for another.  Returns m and log s in
// each of them.
constexpr int kJoinThreads = 128;

__device__ __forceinline__ float2 join_row(const LogProbJoin& q, int64_t i, int thread) {
  constexpr int kThreads = kJoinThreads, kWarps = kThreads / 32;
  __shared__ float most[kWarps], sums[2][kWarps];
  const int lane = thread % 32, warp = thread / 32;
  const float4* parts = q.partial + i * q.parts;
  float m = -INFINITY;
#pragma unroll 4
  for (int64_t k = thread; k < q.parts; k += kThreads) m = fmaxf(m, parts[k].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if (lane == 0) most[warp] = m;
  meet<kThreads>(2);
  m = most[0];
#pragma unroll
  for (int k = 1; k < kWarps; ++k) m = fmaxf(m, most[k]);
  float top = m == -INFINITY ? 0.f : m, s = 0.f, a = 0.f;
#pragma unroll 4
  for (int64_t k = thread; k < q.parts; k += kThreads) {
    const float4 p = parts[k];
    const float x = max_nan((p.x - top) * q.to_log2, kLeastExponent), f = exp2_fast(x);
    s = fmaf(p.y, f, s);
    a = fmaf(f, fmaf(p.y, x, p.z), a);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o), a += __shfl_xor_sync(~0u, a, o);
  if (lane == 0) sums[0][warp] = s, sums[1][warp] = a;
  meet<kThreads>(2);
  s = sums[0][0], a = sums[1][0];
#pragma unroll
  for (int k = 1; k < kWarps; ++k) s += sums[0][k], a += sums[1][k];
  if (q.parts == 0 && q.vocab > 0) top = 0.f, s = static_cast<float>(q.vocab), a = 0.f;
  const float log_s = logf(s), lse = fmaf(top, q.inv_t, log_s);
  if (thread == 0) {
    q.lse[i] = lse;
    const int64_t t = target_of(q.target, i, q.ignore, q.vocab);
    // The two logits first: where the target is the largest one the log probability
    // is -log s, which a sum with a logit of 30 would round to multiples of 2^-19.
    q.log_prob[i] = t == kIgnored   ? 0.f
                    : t == kInvalid ? __int_as_float(0x7fc00000)
                                    : ((q.parts > 0 ? q.target_logit[i] : 0.f) - top) * q.inv_t - log_s;
    q.entropy[i] = t == kIgnored ? 0.f : log_s - 0.693147180559945f * (a / s);
  }
  return make_float2(top, log_s);
}

__global__ void __launch_bounds__(kJoinThreads) log_prob_join(LogProbJoin q) {
  pdl_wait();
  join_row(q, blockIdx.x, threadIdx.x);
}

// Few rows (few_rows.cuh): a CTA computes 32 columns' logits, which are a group and
// a part; a warp each takes a row of them.
struct FewLogits {
  FewOperands in;
  LogProbEpilogue<true> out;  // logits and group_max null where they are not wanted
};

template <typename T, int kTiles>
__global__ void __launch_bounds__(32 * kFewWarps, kTiles == 1 ? 3 : 2) few_logits(FewLogits a) {
  __shared__ FewSums<T, kTiles, 2> sums;
  const int first = blockIdx.x * kChunk;
  few_products<T, kTiles, 2, 16>(a.in, first, sums);
  const int lane = threadIdx.x % 32;
  const LogProbEpilogue<true>& o = a.out;
  for (int i = threadIdx.x / 32; i < a.in.rows; i += kFewWarps) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kFewWarps; ++k) v += sums[k][i][lane];
    const int64_t j = first + lane;
    const bool inside = j < o.vocab;
    if (!inside) v = -INFINITY;
    if (inside && target_of(o.target, i, o.ignore, o.all) == j) o.target_logit[i] = v;
    if (o.logits) o.logits[i * (o.groups * kChunk) + j] = v;
    float m = v;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, s));
    const float x = max_nan((v - (m == -INFINITY ? 0.f : m)) * o.to_log2, kLeastExponent), e = exp2_fast(x);
    float s = e, t = e * x;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(~0u, s, k), t += __shfl_xor_sync(~0u, t, k);
    if (lane > 0) continue;
    o.partial[i * o.parts + blockIdx.x] = make_float4(m, s, t, 0.f);
    if (o.group_max) o.group_max[i * o.groups + blockIdx.x] = m;
  }
}

// ---------------------------------------------------------------------------
// The largest logits of a row.

constexpr int kMostTop = 64;
// Candidates past the ones asked for: so many logits may differ from the last
// one's by no more than the rounding of an fp32 sum before one is missed.
constexpr int kSpareTop = 4;
constexpr int kMostCandidates = kMostTop + kSpareTop;
constexpr int kTopThreads = 256;
constexpr int kHeld = (kMostCandidates * kChunk + kTopThreads - 1) / kTopThreads;

struct TopArgs {
  const float* logits;
  const float* group_max;
  const float* bound;  // as in LogProbEpilogue, or null
  int64_t groups, vocab, hidden;
  const uint16_t* x;
  const uint16_t* w;
  int64_t x_ld, w_ld;
  LogProbJoin join;
  double inv_t;
  int32_t top, candidates;
  float* values;
  int64_t* indices;
};

// Numbers in the order of floats (NaN above all, -0 beside 0), the lower index
// above the higher among equals.  Never 0.
__device__ __forceinline__ uint64_t order_key(float v, uint32_t index) {
  uint32_t u = __float_as_uint(v + 0.f);
  u = v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return static_cast<uint64_t>(u) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - static_cast<uint32_t>(key); }
__device__ __forceinline__ uint64_t order_bits(double v) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return v != v ? ~uint64_t{0} : (u >> 63) ? ~u : u | uint64_t{1} << 63;
}

// The largest key of the searching threads, in each of them.  `part`: one of two buffers that
// calls alternate between.
__device__ __forceinline__ uint64_t block_most(uint64_t key, uint64_t* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor_sync(~0u, key, o);
    key = other > key ? other : key;
  }
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = key;
  meet<kTopThreads>(1);
  key = part[0];
#pragma unroll
  for (int k = 1; k < kTopThreads / 32; ++k) key = part[k] > key ? part[k] : key;
  return key;
}

// sum_k x_k w_k over first <= k < n in 64 bits, by a warp: the product of two 16-bit
// numbers is exact in 32.  Both rows start on 16-byte boundaries, first is a multiple
// of 8.
template <typename T>
__device__ __forceinline__ double exact_dot(const uint16_t* x, const uint16_t* w, int64_t first, int64_t n) {
  const int lane = threadIdx.x % 32;
  // Loads of 1024 elements in flight; four sums a lane.
  constexpr int kAhead = 4;
  double part[4] = {0.0, 0.0, 0.0, 0.0};
  const int64_t whole = n & ~int64_t{7};
  for (int64_t k0 = first; k0 < whole; k0 += kAhead * 256) {
    uint4 a[kAhead], b[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t k = k0 + u * 256 + lane * 8;
      a[u] = b[u] = make_uint4(0, 0, 0, 0);
      if (k < whole) a[u] = *reinterpret_cast<const uint4*>(x + k), b[u] = *reinterpret_cast<const uint4*>(w + k);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float2 p[4] = {mul_pair<T>(a[u].x, b[u].x), mul_pair<T>(a[u].y, b[u].y), mul_pair<T>(a[u].z, b[u].z),
                           mul_pair<T>(a[u].w, b[u].w)};
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e] += static_cast<double>(p[e].x), part[e] += static_cast<double>(p[e].y);
    }
  }
  if (whole >= first && whole + lane < n) part[0] += static_cast<double>(unpack1<T>(x[whole + lane]) * unpack1<T>(w[whole + lane]));
  double s = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return s;
}

// The largest key below `limit` of the thread's share of a row's group maxima.
__device__ __forceinline__ uint64_t best_below(const float* maxima, int groups, uint64_t limit) {
  uint64_t best = 0;
#pragma unroll 4
  for (int k = threadIdx.x; k < groups; k += kTopThreads) {
    const uint64_t key = order_key(maxima[k], static_cast<uint32_t>(k));
    if (key < limit && key > best) best = key;
  }
  return best;
}

// A key that `wanted` of a row's group maxima reach (`groups` of them, as many as wanted
// at least), from the largest one of each of the kTopThreads threads: 4, 2 or 1 lanes
// together hold the largest of theirs, 64, 128 or 256 of them, over twice as many as
// wanted, and those have a wanted-th one.  Each thread by itself where some have none.
__device__ __forceinline__ uint64_t least_wanted(uint64_t mine, int groups, int wanted) {
  __shared__ uint64_t best_of[kTopThreads], least;
  const int tid = threadIdx.x, shift = groups < kTopThreads || wanted > 48 ? 0 : wanted > 24 ? 1 : 2;
  for (int o = 1; o < 1 << shift; o <<= 1) {
    const uint64_t other = __shfl_xor_sync(~0u, mine, o);
    mine = other > mine ? other : mine;
  }
  const int own = tid >> shift, keys = kTopThreads >> shift;
  best_of[own] = mine;
  meet<kTopThreads>(1);
  // The lanes share the keys that theirs is compared with.
  int above = 0;
#pragma unroll 8
  for (int k = tid - (own << shift); k < keys; k += 1 << shift) above += best_of[k] > mine;
  for (int o = 1; o < 1 << shift; o <<= 1) above += __shfl_xor_sync(~0u, above, o);
  if (above == wanted - 1) least = mine;  // keys differ, but for those of threads without groups
  meet<kTopThreads>(1);
  return least;
}

struct BoundArgs {
  float* bound;
  const float* group_max;
  int64_t groups, sample;  // of which so many are there
  int32_t wanted;
};

// Bounds of the rows' largest logits from a sample of their groups.
__global__ void __launch_bounds__(kTopThreads) log_prob_bound(BoundArgs a) {
  pdl_wait();
  const float* maxima = a.group_max + blockIdx.x * a.groups;
  const int groups = static_cast<int>(a.sample);
  const uint64_t least = least_wanted(best_below(maxima, groups, ~uint64_t{0}), groups, a.wanted);
  if (threadIdx.x == 0) a.bound[blockIdx.x] = maxima[key_index(least)];
}

// One CTA per row; four of its warps join the row's parts while eight search.  No
// candidate lies below least_wanted's bound.  Groups that reach it, and then their
// logits that do, are collected (few more than wanted, of logits in no particular
// order) and each one's place is counted.  Where more than kCollect reach it, groups
// and logits are picked one by one.  (7 x 32768
// logits, 5 wanted, hidden 1024: with the product 22.9 us; 27.1 with the join first, in all warps, and 256
// of them whatever was wanted.)
constexpr int kCollect = 512;

template <typename T>
__global__ void __launch_bounds__(kTopThreads + kJoinThreads) log_prob_top(TopArgs a) {
  constexpr int kWarps = kTopThreads / 32, kAllWarps = kWarps + kJoinThreads / 32;
  __shared__ uint64_t part[2][kWarps], collected[kCollect];
  __shared__ uint32_t group_at[kCollect], column[kMostCandidates];
  __shared__ int group_count, count;
  __shared__ double exact[kMostCandidates], off[kMostCandidates], shares[kAllWarps];
  __shared__ float2 joined;
  const int64_t i = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % 32;
  float* values = a.values + i * a.top;
  int64_t* indices = a.indices + i * a.top;
  const uint16_t* x = a.x + i * a.x_ld;
  const int groups = static_cast<int>(a.groups), wanted = min(a.candidates, groups);
  const float* maxima = a.group_max + i * a.groups;
  const float* row = a.logits + i * a.groups * kChunk;
  if (tid == 0) group_count = count = 0;
  if (tid < kMostCandidates) column[tid] = 0;
  auto search = [&] {
    uint64_t mine = best_below(maxima, groups, ~uint64_t{0});
    uint64_t least = least_wanted(mine, groups, wanted);
    if (a.bound) {
      const uint64_t known = order_key(a.bound[i], 0xffffffffu);
      least = known > least ? known : least;
    }
    if (mine >= least) {
      for (int k = tid; k < groups; k += kTopThreads) {
        if (order_key(maxima[k], static_cast<uint32_t>(k)) < least) continue;
        const int at = atomicAdd(&group_count, 1);
        if (at < kCollect) group_at[at] = k;
      }
    }
    meet<kTopThreads>(1);
    // (A logit as large as the least group's maximum counts whatever its index; every
    // logit where the groups are fewer than the candidates.)
    const uint64_t least_logit = wanted < a.candidates ? 0 : least >> 32 << 32;
    for (int g = tid / 32; g < min(group_count, kCollect); g += kWarps) {
      const uint32_t j = group_at[g] * kChunk + lane;
      if (j >= a.vocab) continue;
      const uint64_t key = order_key(row[j], j);
      if (key < least_logit) continue;
      const int at = atomicAdd(&count, 1);
      if (at < kCollect) collected[at] = key;
    }
    meet<kTopThreads>(1);
    if (group_count <= kCollect && count <= kCollect) {
      for (int e = tid; e < count; e += kTopThreads) {
        const uint64_t key = collected[e];
        int place = 0;
#pragma unroll 4
        for (int k = 0; k < count; ++k) place += collected[k] > key;
        if (place < a.candidates) column[place] = key_index(key);
      }
    } else {
      int turn = 0;
      for (int c = 0; c < wanted; ++c) {
        const uint64_t best = block_most(mine, part[turn]);
        turn ^= 1;
        if (mine == best) group_at[c] = key_index(best), mine = best_below(maxima, groups, best);
      }
      meet<kTopThreads>(1);
      uint64_t held[kHeld];
      mine = 0;
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        const int slot = tid + k * kTopThreads;
        held[k] = 0;
        if (slot < wanted * kChunk) {
          const uint32_t j = group_at[slot / kChunk] * kChunk + slot % kChunk;
          if (j < a.vocab) held[k] = order_key(row[j], j);
        }
        mine = held[k] > mine ? held[k] : mine;
      }
      for (int c = 0; c < a.candidates; ++c) {
        const uint64_t best = block_most(mine, part[turn]);
        turn ^= 1;
        if (mine == best) {
          column[c] = key_index(best);
          mine = 0;
#pragma unroll
          for (int k = 0; k < kHeld; ++k) {
            if (held[k] < best) mine = held[k] > mine ? held[k] : mine;
          }
        }
      }
    }
  };
  pdl_wait();
  __syncthreads();
  if (tid >= kTopThreads) {
    const float2 q = join_row(a.join, i, tid - kTopThreads);
    if (tid == kTopThreads) joined = q;
  } else if (a.hidden > 0) {
    search();
  }
  __syncthreads();
  const float most = joined.x, log_s = joined.y;
  if (a.hidden == 0) {  // logits that are sums of no terms
    if (tid < a.top) values[tid] = -log_s, indices[tid] = tid;
    return;
  }
  // The candidates' weights into L2 at once: the warps take them in turn.
  if (tid < a.candidates)
    prefetch_l2(a.w + static_cast<int64_t>(column[tid]) * a.w_ld, static_cast<uint64_t>(a.hidden) * 2);
  // Several warps a candidate where there are more.
  const int parts = max(1, kAllWarps / a.candidates), warp = tid / 32;
  const int64_t length = (a.hidden + 8 * parts - 1) / (8 * parts) * 8;
  for (int task = warp; task < a.candidates * parts; task += kAllWarps) {
    const int c = task / parts;
    const int64_t first = (task - c * parts) * length;
    const double s = exact_dot<T>(x, a.w + static_cast<int64_t>(column[c]) * a.w_ld, first,
                                  min(first + length, a.hidden));
    if (lane == 0) (parts > 1 ? shares[task] : exact[c]) = s;
  }
  // How far the logit that is in s is off, times its share of s.
  const float summed = tid < a.candidates ? row[column[tid]] : 0.f;
  __syncthreads();
  if (tid < a.candidates) {
    double s = exact[tid];
    if (parts > 1) {
      s = 0.0;
      for (int k = 0; k < parts; ++k) s += shares[tid * parts + k];
      exact[tid] = s;
    }
    const float p = expf((summed - most) * a.join.inv_t - log_s);
    off[tid] = p > 0.f ? (s - static_cast<double>(summed)) * static_cast<double>(p) : 0.0;
  }
  __syncthreads();
  if (tid >= a.candidates) return;
  const uint64_t bits = order_bits(exact[tid]);
  int rank = 0;
  double all_off = 0.0;
  for (int c = 0; c < a.candidates; ++c) {
    const uint64_t other = order_bits(exact[c]);
    rank += other > bits || (other == bits && column[c] < column[tid]);
    all_off += off[c];
  }
  if (rank >= a.top) return;
  // lse in 64 bits, moved by what the candidates' logits are off (its derivatives by
  // logits are the shares).  As an fp32 number, near 30 a multiple of 2^-19, it left
  // values above 0 in rows whose largest logit has all the weight, 4e-5 off with logits of
  // 100 where this is 1e-6.
  const double value = (exact[tid] - static_cast<double>(most) - all_off) * a.inv_t - static_cast<double>(log_s);
  values[rank] = value > 0.0 ? 0.f : static_cast<float>(value);
  indices[rank] = column[tid];
}

// ---------------------------------------------------------------------------

template <typename T, bool kEntropy>
struct LogProbGradEpilogue {
  static constexpr bool kPaired = false;
  static constexpr int kSegment = kLogitSegment;
  static constexpr bool kUnrolled = false;
  Out16 s;  // the piece's columns
  const float* lse = nullptr;
  const float* entropy = nullptr;
  const float* grad_log_prob = nullptr;
  const float* grad_entropy = nullptr;
  const float* most = nullptr;  // the largest gradient
  float held = 1.f;             // what S is held times
  float inv_t = 1.f;
  const int64_t* target = nullptr;
  int64_t ignore = 0;
  int64_t vocab = 0;
  int64_t first = 0;  // the piece's first column

  // S_ij = p (c + d (log p + entropy)) - c [j == t], c = -g and d = -h.
  struct Row {
    float c, lse, d, entropy;
    int64_t t;  // within the piece (or outside it)
  };
  __device__ __forceinline__ Row begin(const Lane& l, int64_t i) const {
    const int64_t t = l.inside ? target_of(target, i, ignore, vocab) : kIgnored;
    if (t == kIgnored) return Row{0.f, INFINITY, 0.f, 0.f, kIgnored};
    // A target outside the vocabulary has no log probability: NaN, like itself.
    const float c = t == kInvalid ? __int_as_float(0x7fc00000) : -grad_log_prob[i] / *most * held;
    float d = 0.f, e = 0.f;
    if constexpr (kEntropy) d = -grad_entropy[i] / *most * held, e = entropy[i];
    return Row{c, lse[i], d, e, t >= first ? t - first : kInvalid};
  }
  __device__ __forceinline__ void chunk(Row& r, const Lane& l, int64_t i, int64_t j, float (&v)[kChunk]) const {
    const int64_t at = r.t - j;
    const bool here = at >= 0 && at < kChunk;
    if (r.t == kIgnored) {
#pragma unroll
      for (int k = 0; k < kChunk; ++k) v[k] = 0.f;
    } else {
      const float2 c = make_float2(r.c, r.c), d = make_float2(r.d, r.d), scale = make_float2(inv_t, inv_t);
      const float2 minus = make_float2(-r.lse, -r.lse), base = make_float2(r.entropy, r.entropy);
#pragma unroll
      for (int k = 0; k < kChunk / 2; ++k) {
        const float2 log_p = __ffma2_rn(make_float2(v[2 * k], v[2 * k + 1]), scale, minus);
        float2 by = c;
        if constexpr (kEntropy) by = __ffma2_rn(__fadd2_rn(log_p, base), d, c);
        const float2 p = __fmul2_rn(exp_fast2(log_p), by);
        v[2 * k] = p.x, v[2 * k + 1] = p.y;
      }
      if (here) {
#pragma unroll
        for (int k = 0; k < kChunk; ++k)
          if (at == k) v[k] -= r.c;
      }
    }
    s.template store<T>(l, i, j, v);
  }
  __device__ __forceinline__ void end(Row&, const Lane&, int64_t, int64_t) const {}
};

namespace {

// Temperatures whose inverses fp32 holds with room for log2(e).
constexpr double kLeastTemperature = 1e-30, kMostTemperature = 1e30;

// What a block of rows may take for its logits.
constexpr int64_t kLogitBytes = int64_t{1} << 30;

int32_t candidates_of(int64_t top, int64_t vocab) {
  return static_cast<int32_t>(top + kSpareTop < vocab ? top + kSpareTop : vocab);
}

// Columns whose logits are computed before the others', for a bound below which those
// need not be written (0: none): a wave of tiles (74 pairs of a B200's SMs), and 8 groups for each candidate, of
// which one in 8 others is still written.  Whole and with a sample (us): 131072 x 512
// of 5, 128 rows 54.4 / 56.7, 256 rows 79.4 / 67.0, 512 rows 137 / 100; 131072 x 4096 of
// 20, 128 rows 217 / 217, 256 rows 279 / 263; with a sample of more than a quarter,
// 20000 x 1024 of 1, 300 rows 35.0 / 39.0.
constexpr int64_t kLeastSampled = 256;

int64_t sample_of(int64_t rows, int64_t vocab, int64_t top) {
  if (top == 0 || rows < kLeastSampled) return 0;
  const int64_t wave = 74 / ((rows + 255) / 256) * 256, least = round_up(8 * kChunk * candidates_of(top, vocab), 256);
  const int64_t sample = wave > least ? wave : least;
  return 4 * sample <= vocab ? sample : 0;
}

int64_t rows_of_block(int64_t rows, int64_t groups) {
  int64_t most = kLogitBytes / (groups > 0 ? groups * kChunk * 4 : 1) / 256 * 256;
  if (most < 256) most = 256;
  return rows < most ? rows : most;
}

}  // namespace
}  // namespace hprn

extern "C" {

int hprn_linear_log_probs(float* log_prob, float* entropy, float* lse, float* top_log_probs, int64_t* top_indices,
                          const void* input, const void* weight, const int64_t* target, int64_t ignore_index,
                          double temperature, int64_t top, int64_t rows, int64_t hidden, int64_t vocab,
                          int64_t input_row_stride, int64_t weight_row_stride, int dtype, void* workspace,
                          int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  int st = check_vocabulary(rows, hidden, vocab, dtype, flags, workspace_bytes);
  if (st != HPRN_OK) return st;
  if ((rows > 1 && input_row_stride < hidden) || (vocab > 1 && weight_row_stride < hidden))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  if (!(temperature >= kLeastTemperature) || !(temperature <= kMostTemperature))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "temperature must be between 1e-30 and 1e30");
  if (top < 0 || top > kMostTop || top > vocab)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "top must be between 0 and 64 and at most vocab");
  Workspace ws(workspace, *workspace_bytes);
  const AlignedRows x(ws, input, rows, hidden, input_row_stride, vocab);
  const AlignedRows w(ws, weight, vocab, hidden, weight_row_stride, rows);
  const int64_t groups = top > 0 ? (vocab + kChunk - 1) / kChunk : 0;
  const int64_t block = top > 0 ? rows_of_block(rows, groups) : rows;
  const int64_t sample = sample_of(block, vocab, top);
  const PlannedProduct<false, true, true> of_sample(ws, block, sample > 0 ? sample : vocab, hidden, false),
      product(ws, block, vocab - sample, hidden, false);
  // few_logits, of rows that are read where they are, against the tiles (us, no
  // alternatives): 1 row of 1024 x 32768 17.1 / 18.5, of 2048 x 50000 39.0 / 40.6, of
  // 4096 x 131072 176 / 170; 8 rows 18.5 / 19.3, 40.7 / 40.5; 12 rows 23.3 / 19.3; of 512
  // x 2000 1 row 5.2 / 7.6, 16 rows 5.8 / 7.7.
  const int64_t few_most = rows <= 8 ? int64_t{1} << 27 : rows <= 16 ? int64_t{1} << 22 : 0;
  const bool few = vocab > 0 && hidden > 0 && vocab * hidden <= few_most && hidden % 8 == 0 &&
                   tma_rows(input, rows, input_row_stride) && tma_rows(weight, vocab, weight_row_stride);
  const int64_t sample_parts = of_sample.parts(sample);
  const int64_t parts = few ? (vocab + kChunk - 1) / kChunk : sample_parts + product.parts(vocab - sample);
  float* bound = ws.take<float>(sample > 0 ? block : 0);
  float4* partial = ws.take<float4>(parts * block);
  float* target_logit = ws.take<float>(block);
  float* group_max = ws.take<float>(groups * block);
  float* logits = ws.take<float>(groups * kChunk * block);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (rows == 0) return ok();
  if (!log_prob || !entropy || !lse || !target || (hidden > 0 && (!input || (vocab > 0 && !weight))) ||
      (top > 0 && (!top_log_probs || !top_indices)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(log_prob, 4) || !aligned(entropy, 4) || !aligned(lse, 4) || !aligned(top_log_probs, 4) ||
      !aligned(top_indices, 8) || !aligned(target, 8) || !aligned(input, 2) || !aligned(weight, 2))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent32(log_prob, 1, rows, rows), extent32(entropy, 1, rows, rows),
                         extent32(lse, 1, rows, rows),
                         extent32(top > 0 ? top_log_probs : nullptr, 1, rows * top, rows * top),
                         extent_of(top > 0 ? top_indices : nullptr, 1, rows * top, rows * top, 8)};
  const Extent ins[] = {extent16(input, rows, hidden, input_row_stride),
                        extent16(weight, vocab, hidden, weight_row_stride), extent_of(target, 1, rows, rows, 8)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const char* what = "linear_log_probs";
  const int32_t candidates = candidates_of(top, vocab);
  if (!few && (st = AlignedRows::prepare(x, w, cs, flags)) != HPRN_OK) return st;
  auto all = [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto epilogue, int64_t first, int64_t count) {
      Product q;
      q.a = {x.data() + first * x.ld(), x.ld()};
      q.b = {w.data(), w.ld()};
      q.m = count, q.n = vocab, q.depth = hidden;
      epilogue.partial = partial, epilogue.target_logit = target_logit, epilogue.target = target + first;
      epilogue.ignore = ignore_index, epilogue.parts = parts, epilogue.vocab = epilogue.all = vocab;
      epilogue.to_log2 = static_cast<float>(1.4426950408889634 / temperature);
      epilogue.logits = logits, epilogue.group_max = group_max, epilogue.groups = groups;
      if constexpr (std::is_same<decltype(epilogue), LogProbEpilogue<true>>::value) {
        if (few) {
          FewLogits f{};
          f.out = epilogue;
          if (top == 0) f.out.logits = f.out.group_max = nullptr;
          f.in.x = static_cast<const uint8_t*>(input), f.in.w = static_cast<const uint8_t*>(weight);
          f.in.x_ld = rows > 1 ? input_row_stride * 2 : 0, f.in.w_ld = vocab > 1 ? weight_row_stride * 2 : 0;
          f.in.rows = static_cast<int32_t>(rows), f.in.channels = static_cast<int32_t>(vocab);
          f.in.bytes = static_cast<int32_t>(hidden * 2);
          const auto fn = rows <= 8 ? few_logits<T, 1> : few_logits<T, 2>;
          f.in.first_wave = static_cast<int32_t>(first_wave_ctas(dev, reinterpret_cast<const void*>(fn), 32 * kFewWarps));
          return launch_rows(fn, dim3(static_cast<unsigned>(parts)), dim3(32 * kFewWarps), cs, flags, what, f);
        }
      }
      if (sample == 0) return product.launch_whole<T>(q, epilogue, cs, flags, what);
      q.n = epilogue.vocab = sample;
      int r = of_sample.launch_whole<T>(q, epilogue, cs, flags, what);
      if (r != HPRN_OK) return r;
      BoundArgs b{bound, group_max, groups, sample / kChunk, candidates};
      r = launch_rows(log_prob_bound, dim3(static_cast<unsigned>(count)), dim3(kTopThreads), cs, flags, what, b);
      if (r != HPRN_OK) return r;
      q.b.p = w.data() + sample * w.ld();
      q.n = epilogue.vocab = vocab - sample;
      epilogue.first = sample, epilogue.bound = bound;
      epilogue.partial += sample_parts, epilogue.logits += sample, epilogue.group_max += sample / kChunk;
      return product.launch_whole<T>(q, epilogue, cs, flags, what);
    };
    int r = HPRN_OK;
    for (int64_t first = 0; first < rows; first += block) {
      const int64_t count = rows - first < block ? rows - first : block;
      if (hidden > 0) {
        r = top > 0 || few ? launch(LogProbEpilogue<true>{}, first, count) : launch(LogProbEpilogue<false>{}, first, count);
        if (r != HPRN_OK) return r;
      }
      LogProbJoin q{};
      q.partial = partial, q.target_logit = target_logit, q.target = target + first, q.ignore = ignore_index;
      q.rows = count, q.vocab = vocab, q.parts = hidden > 0 ? parts : 0;
      q.inv_t = static_cast<float>(1.0 / temperature);
      q.to_log2 = static_cast<float>(1.4426950408889634 / temperature);
      q.log_prob = log_prob + first, q.entropy = entropy + first, q.lse = lse + first;
      if (top == 0) {
        r = launch_rows(log_prob_join, dim3(static_cast<unsigned>(count)), dim3(kJoinThreads), cs, flags, what, q);
        if (r != HPRN_OK) return r;
        continue;
      }
      TopArgs a{};
      a.logits = logits, a.group_max = group_max, a.groups = groups, a.vocab = vocab, a.hidden = hidden;
      a.bound = sample > 0 && hidden > 0 ? bound : nullptr;
      a.x = x.data() + first * x.ld(), a.x_ld = x.ld(), a.w = w.data(), a.w_ld = w.ld();
      if (few) a.x = static_cast<const uint16_t*>(input), a.w = static_cast<const uint16_t*>(weight);
      if (few) a.x_ld = rows > 1 ? input_row_stride : hidden, a.w_ld = vocab > 1 ? weight_row_stride : hidden;
      a.join = q, a.inv_t = 1.0 / temperature;
      a.top = static_cast<int32_t>(top);
      a.candidates = candidates;
      a.values = top_log_probs + first * top, a.indices = top_indices + first * top;
      r = launch_rows(log_prob_top<T>, dim3(static_cast<unsigned>(count)), dim3(kTopThreads + kJoinThreads), cs, flags, what, a);
      if (r != HPRN_OK) return r;
    }
    return r;
  };
  return dtype == HPRN_DTYPE_BF16 ? all(__nv_bfloat16{}) : all(__half{});
}

int hprn_linear_log_probs_backward(void* grad_input, void* grad_weight, const float* grad_log_prob,
                                   const float* grad_entropy, const void* input, const void* weight,
                                   const int64_t* target, const float* lse, const float* entropy,
                                   int64_t ignore_index, double temperature, int64_t rows, int64_t hidden,
                                   int64_t vocab, int64_t grad_input_row_stride, int64_t grad_weight_row_stride,
                                   int64_t input_row_stride, int64_t weight_row_stride, int dtype, void* workspace,
                                   int64_t* workspace_bytes, void* stream, unsigned flags) {
  using namespace hprn;
  int st = check_vocabulary(rows, hidden, vocab, dtype, flags, workspace_bytes);
  if (st != HPRN_OK) return st;
  if ((rows > 1 && (input_row_stride < hidden || grad_input_row_stride < hidden)) ||
      (vocab > 1 && (weight_row_stride < hidden || grad_weight_row_stride < hidden)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "row strides must be at least the row lengths");
  if (!(temperature >= kLeastTemperature) || !(temperature <= kMostTemperature))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "temperature must be between 1e-30 and 1e30");
  Workspace ws(workspace, *workspace_bytes);
  const int64_t x_ld = round_up(hidden, 16);
  uint16_t* x = ws.take<uint16_t>(rows * x_ld);  // X without the ignored rows
  const AlignedRows w(ws, weight, vocab, hidden, weight_row_stride, rows);
  const Pieces pieces = pieces_of(rows, vocab);
  uint16_t* s = ws.take<uint16_t>(rows * pieces.cols);
  const int64_t sum_ld = round_up(hidden, kChunk);
  float* sum = pieces.count > 1 ? ws.take<float>(rows * sum_ld) : nullptr;
  float* scale = ws.take<float>(2);
  const float held = dtype != HPRN_DTYPE_FP16 ? 1.f : grad_entropy ? 8192.f : 16384.f;
  const PlannedProduct<false, true, true> logits(ws, rows, pieces.cols, hidden, false);
  const PlannedProduct<false, true, false> to_input(ws, rows, hidden, pieces.cols);
  const PlannedProduct<false, false, false> to_weight(ws, pieces.cols, hidden, rows);
  if (flags & HPRN_WORKSPACE_QUERY) {
    *workspace_bytes = ws.needed();
    return ok();
  }
  if (hidden == 0) return ok();
  if ((rows > 0 && (!grad_input || !grad_log_prob || !input || !target || !lse || (grad_entropy && !entropy))) ||
      (vocab > 0 && (!grad_weight || !weight)))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned(grad_input, 2) || !aligned(grad_weight, 2) || !aligned(grad_log_prob, 4) ||
      !aligned(grad_entropy, 4) || !aligned(input, 2) || !aligned(weight, 2) || !aligned(target, 8) ||
      !aligned(lse, 4) || !aligned(entropy, 4))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "tensor pointers must be aligned to their elements");
  const Extent outs[] = {extent16(grad_input, rows, hidden, grad_input_row_stride),
                         extent16(grad_weight, vocab, hidden, grad_weight_row_stride)};
  const Extent ins[] = {extent32(grad_log_prob, 1, rows, rows), extent32(grad_entropy, 1, rows, rows),
                        extent16(input, rows, hidden, input_row_stride),
                        extent16(weight, vocab, hidden, weight_row_stride), extent_of(target, 1, rows, rows, 8),
                        extent32(lse, 1, rows, rows), extent32(entropy, 1, rows, rows)};
  if (!disjoint(outs, ins)) return fail(HPRN_ERR_INVALID_ARGUMENT, "outputs must not overlap other tensors");
  if (!ws.fits()) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace too small");
  const DeviceInfo* dev = nullptr;
  if ((st = current_device(&dev)) != HPRN_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const char* what = "linear_log_probs_backward";
  if ((st = w.prepare(cs, flags)) != HPRN_OK) return st;
  if (rows > 0) {
    LossPrepareArgs a{};
    a.x = static_cast<const uint16_t*>(input), a.x_ld = input_row_stride;
    a.out = x, a.out_ld = x_ld, a.rows = rows, a.hidden = hidden;
    a.spans = (x_ld + kPrepareSpan - 1) / kPrepareSpan;
    a.vectors = tma_rows(input, rows, input_row_stride);
    a.grad_loss = grad_log_prob, a.grad_entropy = grad_entropy, a.target = target, a.ignore = ignore_index;
    // S is held without the 1 / T of its logits; the sums are multiplied by it.
    a.held = static_cast<float>(held * temperature), a.scale = scale;
    const int64_t ctas = (rows * a.spans + 7) / 8, most = 16 * dev->sm_count;
    st = launch_rows(grad_entropy ? loss_grad_prepare<true> : loss_grad_prepare<false>,
                     dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(256), cs, flags, what, a);
    if (st != HPRN_OK) return st;
  }
  auto all = [&](auto t, auto entropy_too) {
    using T = decltype(t);
    int r = HPRN_OK;
    // Without a vocabulary the input's gradient is an empty sum: zero.
    const int64_t count = pieces.count > 0 ? pieces.count : 1;
    for (int64_t p = 0; p < count && r == HPRN_OK; ++p) {
      const int64_t first = p * pieces.cols;
      const int64_t cols = vocab - first < pieces.cols ? vocab - first : pieces.cols;
      const uint16_t* wp = w.data() + first * w.ld();
      Product q;
      q.a = {x, x_ld};
      q.b = {wp, w.ld()};
      q.m = rows, q.n = cols, q.depth = hidden;
      LogProbGradEpilogue<T, decltype(entropy_too)::value> g;
      g.s = Out16(s, pieces.cols, cols), g.lse = lse, g.entropy = entropy, g.grad_log_prob = grad_log_prob;
      g.grad_entropy = grad_entropy, g.most = scale, g.held = held;
      g.inv_t = static_cast<float>(1.0 / temperature);
      g.target = target, g.ignore = ignore_index, g.vocab = vocab, g.first = first;
      if ((r = logits.launch_whole<T>(q, g, cs, flags, what)) != HPRN_OK) break;

      q.a = {s, pieces.cols};
      q.n = hidden, q.depth = cols;
      StoreEpilogue<T> e;
      e.out = Out16(grad_input, grad_input_row_stride, hidden);
      e.sum = sum, e.sum_ld = sum_ld, e.first = p == 0, e.last = p == count - 1;
      e.scale = rows > 0 ? scale + 1 : nullptr;
      if ((r = to_input.launch<T>(q, e, cs, flags, what)) != HPRN_OK) break;

      q.b = {x, x_ld};
      q.m = cols, q.depth = rows;
      e.out = Out16(static_cast<uint16_t*>(grad_weight) + first * grad_weight_row_stride,
                    grad_weight_row_stride, hidden);
      e.sum = nullptr, e.first = e.last = true;
      r = to_weight.launch<T>(q, e, cs, flags, what);
    }
    return r;
  };
  auto typed = [&](auto t) { return grad_entropy ? all(t, std::true_type{}) : all(t, std::false_type{}); };
  return dtype == HPRN_DTYPE_BF16 ? typed(__nv_bfloat16{}) : typed(__half{});
}

}  // extern "C"

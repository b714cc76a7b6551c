// What the softmax operators over a vocabulary share: targets, exponentials, how
// the logits are summed, and what their backward passes prepare.
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "matmul.cuh"
#include "runtime.cuh"

namespace hprn {

// A row's target: its column, or kIgnored, or kInvalid (outside the vocabulary).
constexpr int64_t kIgnored = -1, kInvalid = -2;
__device__ __forceinline__ int64_t target_of(const int64_t* target, int64_t i, int64_t ignore,
                                             int64_t vocab) {
  const int64_t t = target[i];
  return t == ignore ? kIgnored : (t < 0 || t >= vocab) ? kInvalid : t;
}

constexpr float kLog2e = 1.4426950408889634f;

// exp(x) as 2^(x log2 e), by the hardware's approximation (2 ulp); 1 at 0.
__device__ __forceinline__ float exp_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * kLog2e));
  return y;
}
__device__ __forceinline__ float2 exp_fast2(float2 x) {
  const float2 t = __fmul2_rn(x, make_float2(kLog2e, kLog2e));
  float2 y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(t.y));
  return y;
}

// Stages that the tensor cores sum at once, 512 terms: a loss is a difference
// of logits near the largest ones and would be short throughout.  2048 x 5120 x
// 100003 (fp16): 1.8e-6 of itself with whole sums, 2.0e-7 with these (1.9e-7 in
// fp32 operations), 1685 us instead of 1650; 1670 with 1024 terms.  The backward
// pass takes the same, since its logits have to be the forward pass's.
constexpr int kLogitSegment = 8;

// What the backward products need first.  X with the ignored rows zeroed (on
// aligned rows): a row that is left out leaves dW alone whatever it holds, where
// 0 times its infinities or NaN would not.  And, by the first CTA, c_max and
// what the sums are multiplied by, c_max / held.  A warp takes kPrepareSpan
// elements of a row, all its loads in flight: 16 bytes a lane where X's rows
// start on 16-byte boundaries, else two 2-byte loads a word.
constexpr int kPrepareSpan = 512;

struct LossPrepareArgs {
  const uint16_t* x;
  uint16_t* out;
  int64_t x_ld, out_ld, rows, hidden, spans;  // spans of a row
  bool vectors;
  const float* grad_loss;
  const float* grad_entropy;  // or null
  const int64_t* target;
  int64_t ignore;
  float held;
  float* scale;
};

template <bool kEntropy>
__global__ void __launch_bounds__(256) loss_grad_prepare(LossPrepareArgs a) {
  __shared__ float part[8];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (blockIdx.x == 0) {
    float m = 0.f;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < a.rows; i += 256) {
      // The largest finite one: an infinite or NaN gradient spoils its own row
      // and the weight's, not the scale of the other rows.
      const float c = fabsf(a.grad_loss[i]);
      if (a.target[i] != a.ignore && c < INFINITY) m = fmaxf(m, c);
      if constexpr (kEntropy) {
        const float h = fabsf(a.grad_entropy[i]);
        if (a.target[i] != a.ignore && h < INFINITY) m = fmaxf(m, h);
      }
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (lane == 0) part[warp] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < 8; ++k) m = fmaxf(m, part[k]);
      if (m == 0.f) m = 1.f;
      a.scale[0] = m, a.scale[1] = m / a.held;
    }
  }
  const int64_t all = a.rows * a.spans;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 8 + warp; e < all; e += static_cast<int64_t>(gridDim.x) * 8) {
    const int64_t i = e / a.spans, j0 = (e - i * a.spans) * kPrepareSpan;
    const uint16_t* p = a.x + i * a.x_ld + j0;
    uint16_t* q = a.out + i * a.out_ld + j0;
    const int width = static_cast<int>(min(static_cast<int64_t>(kPrepareSpan), a.out_ld - j0));  // a multiple of 16
    int inside = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(kPrepareSpan), a.hidden - j0)));
    if (a.target[i] == a.ignore) inside = 0;
    if (a.vectors && inside % 8 == 0) {
      uint4 v[kPrepareSpan / 256];
#pragma unroll
      for (int k = 0; k < kPrepareSpan / 256; ++k) {
        const int j = k * 256 + lane * 8;
        v[k] = j < inside ? *reinterpret_cast<const uint4*>(p + j) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < kPrepareSpan / 256; ++k) {
        const int j = k * 256 + lane * 8;
        if (j < width) *reinterpret_cast<uint4*>(q + j) = v[k];
      }
      continue;
    }
    uint32_t w[kPrepareSpan / 64];
#pragma unroll
    for (int k = 0; k < kPrepareSpan / 64; ++k) {
      const int j = k * 64 + lane * 2;
      const uint32_t lo = j < inside ? p[j] : 0, hi = j + 1 < inside ? p[j + 1] : 0;
      w[k] = lo | hi << 16;
    }
#pragma unroll
    for (int k = 0; k < kPrepareSpan / 64; ++k) {
      const int j = k * 64 + lane * 2;
      if (j < width) *reinterpret_cast<uint32_t*>(q + j) = w[k];
    }
  }
}

// S's share of the workspace: pieces of the vocabulary of equal length such
// that a piece's S takes at most this much.
constexpr int64_t kPieceBytes = int64_t{512} << 20;

struct Pieces {
  int64_t count, cols;
};
inline Pieces pieces_of(int64_t rows, int64_t vocab) {
  int64_t most = kPieceBytes / 2 / (rows > 0 ? rows : 1) / 256 * 256;
  if (most < 256) most = 256;
  const int64_t count = vocab > 0 ? (vocab + most - 1) / most : 0;
  const int64_t cols = count > 0 ? round_up((vocab + count - 1) / count, 256) : 0;
  return Pieces{cols > 0 ? (vocab + cols - 1) / cols : 0, cols};
}

inline int check_vocabulary(int64_t rows, int64_t hidden, int64_t vocab, int dtype, unsigned flags,
                            const int64_t* workspace_bytes) {
  if (flags & ~static_cast<unsigned>(HPRN_LAUNCH_PDL | HPRN_WORKSPACE_QUERY))
    return fail(HPRN_ERR_INVALID_ARGUMENT, "unknown launch flags");
  if (dtype != HPRN_DTYPE_BF16 && dtype != HPRN_DTYPE_FP16)
    return fail(HPRN_ERR_UNSUPPORTED_DTYPE, "dtype must be kFloat16 or kBFloat16");
  if (rows < 0 || hidden < 0 || vocab < 0) return fail(HPRN_ERR_INVALID_ARGUMENT, "sizes must be >= 0");
  if (rows > kMaxExtent || hidden > kMaxExtent || vocab > kMaxExtent)
    return fail(HPRN_ERR_INVALID_ARGUMENT, "rows, hidden and vocab must be at most 2^30");
  if (!workspace_bytes) return fail(HPRN_ERR_INVALID_ARGUMENT, "workspace_bytes pointer required");
  return HPRN_OK;
}

}  // namespace hprn

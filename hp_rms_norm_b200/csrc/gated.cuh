// Gated activations on fp32 values, and their derivatives:
//   silu(a)      = a s(a), s(a) = 1 / (1 + exp(-a));  silu'(a) = s (1 + a (1 - s))
//   gelu(a)      = a P(a), P(a) = (1 + erf(a / sqrt 2)) / 2
//                  gelu'(a) = P + a exp(-a^2 / 2) / sqrt(2 pi)
//   gelu_tanh(a) = a (1 + t) / 2, t = tanh(k (a + c a^3)), k = sqrt(2 / pi), c = 0.044715
//                  gelu_tanh'(a) = (1 + t) / 2 + a (1 - t^2) k (1 + 3 c a^2) / 2
#pragma once

#include <math.h>

#include "hp_rms_norm_b200.h"

namespace hprn {

struct ActValue {
  float value, slope;
};

template <int ACT>
__device__ __forceinline__ ActValue activate_with_slope(float a) {
  if constexpr (ACT == HPRN_ACT_SILU) {
    const float s = __fdividef(1.0f, 1.0f + expf(-a));
    return {a * s, fmaf(a * s, 1.0f - s, s)};
  } else if constexpr (ACT == HPRN_ACT_GELU) {
    const float p = 0.5f * (1.0f + erff(a * 0.70710678118654752f));
    return {a * p, fmaf(a, 0.39894228040143268f * expf(-0.5f * a * a), p)};
  } else {
    const float k = 0.79788456080286536f, c = 0.044715f;
    const float t = tanhf(k * (a + c * a * a * a));
    const float h = 0.5f * (1.0f + t), r = 1.0f - t * t;
    // r = 0 where |a| is large, where the other factor may be infinite.
    return {a * h, r == 0.0f ? h : fmaf(0.5f * a * r, k * fmaf(3.0f * c * a, a, 1.0f), h)};
  }
}

}  // namespace hprn

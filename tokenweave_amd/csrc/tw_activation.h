// The activations of a gated block and their slopes, in fp32.
#ifndef TW_ACTIVATION_H
#define TW_ACTIVATION_H

#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/tokenweave_amd.h"

namespace tw {

constexpr float kTanhA = 0.7978845608028654f, kTanhB = 0.044715f;  // sqrt(2 / pi)

// 1 / (1 + e^-x).  e^-x overflows to an infinity below -88.7, whose reciprocal is the zero it should be.
//
// By the exponential instruction on x log2 e, rounded to fp32: |x| 2^-24 of e^-x, where it counts beside 1; the tanh form's
// argument, of x^3, and the exact one's x^2 are rounded likewise.  Against 64 bits, of the value, in units of 2^-24, for x
// in [-1, 20] / [-5, -1] / [-10, -5]: silu 3.7 / 6.4 / 10, exact 4.9 / 24 / 88, tanh 4.9 / 47 / 230.  An exponent in two
// floats would cost four instructions a value more for the first, some ten for the others; every caller rounds the
// product with the up value to 8 bits, 4 or 3 of mantissa, at once, and the gelus below -5 are less than 1e-6 x.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

template <int ACT>
__device__ __forceinline__ float activation(float x) {
  if (ACT == TW_ACT_SILU) return x * sigmoid(x);
  // 0.5 (1 + tanh z) = sigmoid(2 z): no cancellation for large negative z
  if (ACT == TW_ACT_GELU_TANH) return x * sigmoid(2.0f * kTanhA * (x + kTanhB * x * x * x));
  return 0.5f * x * erfcf(-0.70710678118654752f * x);
}

// act(x) and its derivative
template <int ACT>
__device__ __forceinline__ void activation_and_slope(float x, float& f, float& df) {
  if (ACT == TW_ACT_SILU) {
    const float s = sigmoid(x);
    f = x * s;
    df = s * (1.0f + x * (1.0f - s));
  } else if (ACT == TW_ACT_GELU_TANH) {
    const float z = 2.0f * kTanhA * (x + kTanhB * x * x * x), s = sigmoid(z);
    const float c = fminf(fmaxf(x, -16.0f), 16.0f);  // s (1 - s) is zero out there, and must not meet an infinity
    f = x * s;
    df = s + c * s * (1.0f - s) * 2.0f * kTanhA * (1.0f + 3.0f * kTanhB * c * c);
  } else {
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * x);
    f = x * cdf;
    df = cdf + x * 0.3989422804014327f * __expf(-0.5f * x * x);
  }
}

// f(integral_constant<act>): one branch on the activation, outside the loops that apply it.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  if (act == TW_ACT_SILU) f(std::integral_constant<int, TW_ACT_SILU>{});
  else if (act == TW_ACT_GELU) f(std::integral_constant<int, TW_ACT_GELU>{});
  else f(std::integral_constant<int, TW_ACT_GELU_TANH>{});
}

}  // namespace tw

#endif

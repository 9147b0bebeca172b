// Activations of the layer operators and their derivatives, in fp32.
//   gelu       x Phi(x),  Phi the normal distribution function
//   gelu_tanh  x (1 + tanh u) / 2 = x / (1 + exp(-2u)),  u = sqrt(2/pi) (x + 0.044715 x^3)
//   silu       x / (1 + exp(-x))
// exp through the hardware exponential and the division by its reciprocal
// approximation: a few 2^-23 relative for the arguments where the result is
// not negligible, far below the rounding of a bf16 result and within the
// fp32 sums' own error for an fp32 one.
#pragma once
#include "../../include/apk.h"

namespace apk {

__device__ __forceinline__ float sigmoid_f(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

template <int ACT>
__device__ __forceinline__ float act_f(float x) {
  if constexpr (ACT == APK_ACT_RELU) return x <= 0.f ? 0.f : x;  // a NaN stays one
  else if constexpr (ACT == APK_ACT_GELU) return 0.5f * x * (1.f + erff(x * 0.70710678f));
  else if constexpr (ACT == APK_ACT_GELU_TANH) {
    const float u2 = 1.59576912f * (x + 0.044715f * x * x * x);
    return __fdividef(x, 1.f + __expf(-u2));
  } else if constexpr (ACT == APK_ACT_SILU) return __fdividef(x, 1.f + __expf(-x));
  else return x;
}

template <int ACT>
__device__ __forceinline__ float act_grad_f(float x) {
  if constexpr (ACT == APK_ACT_RELU) return x > 0.f ? 1.f : 0.f;
  else if constexpr (ACT == APK_ACT_GELU)
    return 0.5f * (1.f + erff(x * 0.70710678f)) + x * 0.39894228f * __expf(-0.5f * x * x);
  else if constexpr (ACT == APK_ACT_GELU_TANH) {
    // d/dx x s(v) = s + x s (1 - s) v',  v = 2u
    // (where |x| > 100 the second term is 0; unclamped it would be 0 * inf)
    const float s = sigmoid_f(1.59576912f * (x + 0.044715f * x * x * x));
    const float c = fminf(fmaxf(x, -100.f), 100.f);
    return s + c * s * (1.f - s) * 1.59576912f * (1.f + 0.134145f * c * c);
  } else if constexpr (ACT == APK_ACT_SILU) {
    const float s = sigmoid_f(x);
    const float c = fminf(fmaxf(x, -100.f), 100.f);
    return s * (1.f + c * (1.f - s));
  } else return 1.f;
}

template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};
// f(ActTag<act>): one branch outside the element loops.
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case APK_ACT_RELU: f(ActTag<APK_ACT_RELU>()); break;
    case APK_ACT_GELU: f(ActTag<APK_ACT_GELU>()); break;
    case APK_ACT_GELU_TANH: f(ActTag<APK_ACT_GELU_TANH>()); break;
    case APK_ACT_SILU: f(ActTag<APK_ACT_SILU>()); break;
    default: f(ActTag<APK_ACT_NONE>()); break;
  }
}

}  // namespace apk

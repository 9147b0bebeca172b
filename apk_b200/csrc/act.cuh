// Activations of the layer operators and their derivatives, in fp32.
//   gelu       x Phi(x),  Phi the normal distribution function
//   gelu_tanh  x (1 + tanh u) / 2 = x / (1 + exp(-2u)),  u = sqrt(2/pi) (x + 0.044715 x^3)
//   silu       x / (1 + exp(-x))
// The sigmoid 1 / (1 + 2^(-x log2 e)) goes through the hardware's 2^x and
// reciprocal approximations: a few 2^-23 relative where it is not negligible,
// far below the rounding of a bf16 result and within an fp32 sum's own error.
#pragma once
#include "../../include/apk.h"

namespace apk {

// 1 / (1 + 2^t): 0 for t = inf, 1 for t = -inf
__device__ __forceinline__ float rcp_1p_ex2(float t) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}
// min(max(x, -100), 100), a NaN staying one: beyond, every activation's
// derivative is at its limit, and products like inf * 0 do not arise.
__device__ __forceinline__ float clamp100(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(-100.f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(100.f));
  return r;
}

constexpr float LOG2E = 1.44269504f;

// Phi(x), and e = exp(-x^2 / 2): erfc(y) = (a1 t + ... + a5 t^5) exp(-y^2) for
// y >= 0, t = 1 / (1 + p y), Abramowitz and Stegun's 7.1.26, whose error is at
// most 1.5e-7; with fp32 steps Phi is within 3e-7.  Half the operations of
// erff, and the derivative needs the same exponential.
__device__ __forceinline__ float normal_cdf(float x, float& e) {
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f * 0.70710678f, fabsf(x), 1.f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-0.5f * LOG2E * x * x));
  const float a = fmaf(fmaf(fmaf(fmaf(1.061405429f, t, -1.453152027f), t, 1.421413741f), t, -0.284496736f), t,
                       0.254829592f);
  const float h = 0.5f * t * a * e;
  return x >= 0.f ? 1.f - h : h;
}
// 2u = x (GT1 + GT3 x^2)
constexpr float GT1 = 1.59576912f, GT3 = 0.0713548162f;

template <int ACT>
__device__ __forceinline__ float act_f(float x) {
  if constexpr (ACT == APK_ACT_RELU) return x <= 0.f ? 0.f : x;  // a NaN stays one
  else if constexpr (ACT == APK_ACT_GELU) {
    float e;
    return x * normal_cdf(x, e);
  } else if constexpr (ACT == APK_ACT_GELU_TANH)
    return x * rcp_1p_ex2(x * fmaf(-LOG2E * GT3, x * x, -LOG2E * GT1));
  else if constexpr (ACT == APK_ACT_SILU) return x * rcp_1p_ex2(-LOG2E * x);
  else return x;
}

template <int ACT>
__device__ __forceinline__ float act_grad_f(float z) {
  if constexpr (ACT == APK_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  else if constexpr (ACT == APK_ACT_GELU) {
    const float x = clamp100(z);
    float e;
    const float cdf = normal_cdf(x, e);
    return fmaf(x * 0.39894228f, e, cdf);
  } else if constexpr (ACT == APK_ACT_GELU_TANH) {
    // d/dx x s(v) = s (1 + x v' (1 - s)),  v = 2u
    const float x = clamp100(z), x2 = x * x;
    const float s = rcp_1p_ex2(x * fmaf(-LOG2E * GT3, x2, -LOG2E * GT1));
    const float t = x * fmaf(3.f * GT3, x2, GT1);
    return fmaf(s, fmaf(-s, t, t), s);
  } else if constexpr (ACT == APK_ACT_SILU) {
    const float x = clamp100(z), s = rcp_1p_ex2(-LOG2E * x);
    return fmaf(s, fmaf(-s, x, x), s);
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

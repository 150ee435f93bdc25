// The activations of the learned features' layers and their derivatives, on the device.
#pragma once

#include <type_traits>

#include "layers.h"

namespace mgp {

// exp(x + tail) by v_exp_f32.  FAST (the 16-bit types): the exponent's rounding
// makes a relative error of 2^-24 |x|; fp32 takes it out to first order.  A
// library expf and a division made ~40 instructions of each sigmoid, and the
// epilogue of 65536 x 1024 -> 4096 a quarter of the kernel's time.
template <bool FAST>
__device__ __forceinline__ float exp_of(float x, float tail = 0.0f) {
  if constexpr (FAST) return __builtin_amdgcn_exp2f(kLog2e * x);
  constexpr float kLog2eLow = 1.92596299e-8f;  // log2(e) - kLog2e
  x = x < -126.0f ? -126.0f : x;  // beyond, 0 and infinity all the same; NaN stays
  x = x > 126.0f ? 126.0f : x;
  const float t = x * kLog2e;
  const float r = fmaf(x, kLog2e, -t) + fmaf(x, kLog2eLow, tail * kLog2e);
  return __builtin_amdgcn_exp2f(t) * fmaf(r, kLn2, 1.0f);
}

// 1 - Phi(x) over exp(-x^2 / 2) for x = sqrt(2) v, v >= 0: a polynomial in
// 1 / (1 + p v), p and the coefficients fitted by least squares reweighted
// towards the smallest largest relative error over 0 <= v <= 9.5: 5.2e-6 (six
// terms, the 16-bit types), 3.8e-8 (nine; 3.5e-7 as fp32 evaluates it).
template <bool FAST>
__device__ __forceinline__ float normal_tail(float v) {
  if constexpr (FAST) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.44f, v, 1.0f));
    float q = -0.0730530247092247f;
    q = fmaf(q, t, 0.17532674968242645f);
    q = fmaf(q, t, 0.020365050062537193f);
    q = fmaf(q, t, 0.13179342448711395f);
    q = fmaf(q, t, 0.12128471583127975f);
    return fmaf(q, t, 0.12428051233291626f) * t;
  } else {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, v, 1.0f));
    float q = -0.06471703946590424f;
    q = fmaf(q, t, 0.24254822731018066f);
    q = fmaf(q, t, -0.2556132376194f);
    q = fmaf(q, t, 0.2731975317001343f);
    q = fmaf(q, t, -0.04681563004851341f);
    q = fmaf(q, t, 0.10721813887357712f);
    q = fmaf(q, t, 0.07424121350049973f);
    q = fmaf(q, t, 0.08534596860408783f);
    return fmaf(q, t, 0.08459480851888657f) * t;
  }
}

// a = act(g) and its derivative
template <int ACT, bool FAST>
__device__ __forceinline__ void activate(float g, float& a, float& slope) {
  if constexpr (ACT == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + exp_of<FAST>(-g));
    a = g * s;
    slope = s * fmaf(g, 1.0f - s, 1.0f);
  } else if constexpr (ACT == ACT_SIGMOID) {
    a = __builtin_amdgcn_rcpf(1.0f + exp_of<FAST>(-g));
    slope = a * (1.0f - a);
  } else if constexpr (ACT == ACT_RELU) {
    a = g > 0.0f || g != g ? g : 0.0f;
    slope = g > 0.0f ? 1.0f : 0.0f;
  } else {
    // fp32: from |g| = 40 on e is 0, and a square that passes fp32 has no remainder
    const float c = FAST ? g : fminf(fabsf(g), 40.0f);
    const float g2 = c * c;
    const float e = exp_of<FAST>(-0.5f * g2, -0.5f * fmaf(c, c, -g2));
    const float tail = normal_tail<FAST>(fabsf(g) * 0.70710678118654752f) * e;  // 1 - Phi(|g|)
    const float cdf = g > 0.0f ? 1.0f - tail : tail;
    a = g * cdf;
    slope = fmaf(g * 0.39894228040143268f, e, cdf);
  }
}

template <class F>
void dispatch_act(int act, F&& f) {
  switch (act) {
    case ACT_SILU: f(std::integral_constant<int, ACT_SILU>{}); break;
    case ACT_GELU: f(std::integral_constant<int, ACT_GELU>{}); break;
    case ACT_SIGMOID: f(std::integral_constant<int, ACT_SIGMOID>{}); break;
    default: f(std::integral_constant<int, ACT_RELU>{}); break;
  }
}

// The same within a kernel, for an activation that is the same for all threads.
template <class F>
__device__ __forceinline__ void dispatch_act_device(int act, F&& f) {
  if (act == ACT_SILU)
    f(std::integral_constant<int, ACT_SILU>{});
  else if (act == ACT_GELU)
    f(std::integral_constant<int, ACT_GELU>{});
  else if (act == ACT_SIGMOID)
    f(std::integral_constant<int, ACT_SIGMOID>{});
  else
    f(std::integral_constant<int, ACT_RELU>{});
}

}  // namespace mgp

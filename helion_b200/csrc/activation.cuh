// Activations of the gated projection act(g) * u, with the derivative its backward pass needs.
//
//   silu       g s(g), s(g) = 1 / (1 + exp(-g))           derivative s (1 + g (1 - s))
//   gelu       g P(g), P the normal distribution function  derivative P + g exp(-g^2/2) / sqrt(2 pi)
//   gelu_tanh  g p(g), p = (1 + tanh z) / 2 = s(2 z),      derivative p + g p (1 - p) 2 z'
//              z = sqrt(2/pi) (g + 0.044715 g^3)
//
// The logistic form of tanh keeps its relative accuracy where 1 + tanh would cancel.  fp32 throughout, within a few 2^-22 of
// the value (2^-19 in gelu's tail beyond -5, from exp(-g^2/2)), far inside the 2^-12 half step of a 16-bit output.
#pragma once

#include "common.cuh"

namespace hb {

enum Activation : int { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2 };

__device__ __forceinline__ float logistic(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// P(g) from e = exp(-g^2 / 2): for g < 0 it is erfc(z) / 2 with z = |g| / sqrt(2), and exp(z^2) erfc(z) is smooth, here t times
// a polynomial in t = 1 / (1 + 0.33 z) (the form of Abramowitz and Stegun 7.1.26; degree 7, coefficients fitted to least
// relative error over z < 9.5, where e underflows: 8.2e-8).  The derivative shares e.  The math library's normcdff takes four
// times the instructions and made the epilogue the bound of projections with a short K.
__device__ __forceinline__ float normal_cdf(float g, float e) {
  const float t = __fdividef(1.0f, fmaf(0.23334524f, fabsf(g), 1.0f));
  float q = -0.0679644272f;
  q = fmaf(q, t, 0.231344223f);
  q = fmaf(q, t, -0.177719668f);
  q = fmaf(q, t, 0.206270993f);
  q = fmaf(q, t, 0.02250522f);
  q = fmaf(q, t, 0.100961946f);
  q = fmaf(q, t, 0.0914186165f);
  q = fmaf(q, t, 0.0931830555f);
  q *= t * e;
  return g < 0.0f ? q : 1.0f - q;
}

// a = act(g) and, where DERIVATIVE, d = act'(g).
template <int ACT, bool DERIVATIVE>
__device__ __forceinline__ void activate(float g, float& a, float& d) {
  if constexpr (ACT == ACT_SILU) {
    const float s = logistic(g);
    a = g * s;
    if constexpr (DERIVATIVE) d = s * fmaf(g, 1.0f - s, 1.0f);
  } else if constexpr (ACT == ACT_GELU) {
    const float e = __expf(-0.5f * g * g);
    const float p = normal_cdf(g, e);
    a = g * p;
    if constexpr (DERIVATIVE) d = fmaf(g * 0.39894228f, e, p);
  } else {
    const float g2 = g * g;
    const float p = logistic(1.5957691f * fmaf(0.044715f * g2, g, g));
    a = g * p;
    if constexpr (DERIVATIVE) {
      const float q = p * (1.0f - p);  // zero in the tails, where g^2 may be infinite
      d = q == 0.0f ? p : fmaf(g * q, 1.5957691f * fmaf(0.134145f, g2, 1.0f), p);
    }
  }
}

__device__ __forceinline__ float activate_by(int act, float g) {
  float a, d;
  if (act == ACT_SILU) activate<ACT_SILU, false>(g, a, d);
  else if (act == ACT_GELU) activate<ACT_GELU, false>(g, a, d);
  else activate<ACT_GELU_TANH, false>(g, a, d);
  return a;
}

}  // namespace hb

// Activations of the gated projection act(g) * u, with the derivative its backward pass needs.
//
//   silu       g s(g), s(g) = 1 / (1 + exp(-g))           derivative s (1 + g (1 - s))
//   gelu       g P(g), P the normal distribution function  derivative P + g exp(-g^2/2) / sqrt(2 pi)
//   gelu_tanh  g p(g), p = (1 + tanh z) / 2 = s(2 z),      derivative p + g p (1 - p) 2 z'
//              z = sqrt(2/pi) (g + 0.044715 g^3)
//
// The logistic form of tanh keeps its relative accuracy where 1 + tanh would cancel, and s(-v) = e / (1 + e) with e = exp(-v) <= 1 that
// of the far tails (1 / (1 + exp(v)) would be zero from v = 87.3 on, where v s(-v) is 1e-36 and normal).  All of this is fp32;
// relative errors in units of 2^-24, down to where the exponential leaves fp32's normal range:
//   16-bit outputs and what the backward pass keeps: the fast exponential's 4 + 2.4 |v| at its argument v (-g, -g^2/2, -2 z), whose
//     own roundings add up to 2 |v| (gelu) and 6 |v| (gelu_tanh): below 2^-14 at the far end, inside the 2^-12 half step of fp16.
//   FINE, for fp32 outputs: the math library's exponential, a rounded reciprocal and, for gelu, the rounding error of g^2 taken
//     along: 8 (silu), 24 (gelu); gelu_tanh keeps the 6 |2 z| of its argument.
#pragma once

#include "common.cuh"

namespace hb {

enum Activation : int { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2 };

template <bool FINE>
__device__ __forceinline__ float exponential(float v) {
  return FINE ? expf(v) : __expf(v);
}

// 1 / v for v from 1 to 2^126.  FINE: with a Newton step, r + r (1 - v r), which leaves little more than its own rounding (the
// correctly rounded reciprocal branches: 2048 x 128 x 14336 e4m3 to fp32 110 us, with the step 75 us, without it 64 us).
template <bool FINE>
__device__ __forceinline__ float reciprocal(float v) {
  const float r = __fdividef(1.0f, v);
  return FINE ? fmaf(r, fmaf(-v, r, 1.0f), r) : r;
}

template <bool FINE>
__device__ __forceinline__ float logistic(float v) {
  const float e = exponential<FINE>(-fabsf(v));
  const float r = reciprocal<FINE>(1.0f + e);
  return v >= 0.0f ? r : e * r;
}

// exp(-g^2 / 2)
template <bool FINE>
__device__ __forceinline__ float bell(float g) {
  const float g2 = g * g;
  const float e = exponential<FINE>(-0.5f * g2);
  // what g * g lost; nothing is left to correct where e is zero (g^2 may be infinite there)
  return FINE && e > 0.0f ? fmaf(e, -0.5f * fmaf(g, g, -g2), e) : e;
}

// P(g) from e = exp(-g^2 / 2): for g < 0 it is erfc(z) / 2 with z = |g| / sqrt(2), and exp(z^2) erfc(z) is smooth, here t times
// a polynomial in t = 1 / (1 + 0.33 z) (the form of Abramowitz and Stegun 7.1.26; degree 7, coefficients fitted to least
// relative error over z < 9.5, where e underflows: 8.2e-8).  The derivative shares e.  The math library's normcdff takes four
// times the instructions and made the epilogue the bound of projections with a short K.
template <bool FINE>
__device__ __forceinline__ float normal_cdf(float g, float e) {
  const float size = FINE ? fminf(fabsf(g), 64.0f) : fabsf(g);  // e is zero there; an infinite size would make the step a NaN
  const float t = reciprocal<FINE>(fmaf(0.23334524f, size, 1.0f));
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
template <int ACT, bool DERIVATIVE, bool FINE>
__device__ __forceinline__ void activate(float g, float& a, float& d) {
  if constexpr (ACT == ACT_SILU) {
    const float s = logistic<FINE>(g);
    a = g * s;
    if constexpr (DERIVATIVE) d = s * fmaf(g, 1.0f - s, 1.0f);
  } else if constexpr (ACT == ACT_GELU) {
    const float e = bell<FINE>(g);
    const float p = normal_cdf<FINE>(g, e);
    a = g * p;
    if constexpr (DERIVATIVE) d = fmaf(g * 0.39894228f, e, p);
  } else {
    const float g2 = g * g;
    const float p = logistic<FINE>(1.5957691f * fmaf(0.044715f * g2, g, g));
    a = g * p;
    if constexpr (DERIVATIVE) {
      const float q = p * (1.0f - p);  // zero in the tails, where g^2 may be infinite
      d = q == 0.0f ? p : fmaf(g * q, 1.5957691f * fmaf(0.134145f, g2, 1.0f), p);
    }
  }
}

template <bool FINE>
__device__ __forceinline__ float activate_by(int act, float g) {
  float a, d;
  if (act == ACT_SILU) activate<ACT_SILU, false, FINE>(g, a, d);
  else if (act == ACT_GELU) activate<ACT_GELU, false, FINE>(g, a, d);
  else activate<ACT_GELU_TANH, false, FINE>(g, a, d);
  return a;
}

}  // namespace hb

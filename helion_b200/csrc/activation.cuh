// Activations of the gated projection act(g) * u, with the derivative its backward pass needs.
//
//   silu       g s(g), s(g) = 1 / (1 + exp(-g))           derivative s (1 + g (1 - s))
//   gelu       g P(g), P the normal distribution function  derivative P + g exp(-g^2/2) / sqrt(2 pi)
//   gelu_tanh  g p(g), p = (1 + tanh z) / 2 = s(2 z),      derivative p + g p (1 - p) 2 z'
//              z = sqrt(2/pi) (g + 0.044715 g^3)
//
// The logistic form of tanh keeps its relative accuracy where 1 + tanh would cancel.  fp32 throughout; __expf and
// __fdividef are within a few 2^-22 of the value over the range where the result is not zero, far inside the 2^-12
// half step of the finest output type.
#pragma once

#include "common.cuh"

namespace hb {

enum Activation : int { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2 };

__device__ __forceinline__ float logistic(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// a = act(g) and, where DERIVATIVE, d = act'(g).
template <int ACT, bool DERIVATIVE>
__device__ __forceinline__ void activate(float g, float& a, float& d) {
  if constexpr (ACT == ACT_SILU) {
    const float s = logistic(g);
    a = g * s;
    if constexpr (DERIVATIVE) d = s * fmaf(g, 1.0f - s, 1.0f);
  } else if constexpr (ACT == ACT_GELU) {
    const float p = normcdff(g);
    a = g * p;
    if constexpr (DERIVATIVE) d = fmaf(g * 0.39894228f, __expf(-0.5f * g * g), p);
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

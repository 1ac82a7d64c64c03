// Activations of the gated feed-forward block and their derivatives.
#pragma once

#include <stdint.h>

#include "distill_common.cuh"
#include "orda_b200_student.h"

namespace orda {

// erfc(y / sqrt 2) / 2 for y >= 0: with x = y / sqrt 2 and t = 1 / (1 + x / 2), ln(erfc(x) e^{x^2} / t) is smooth
// in t (the ansatz of erfcc in Press et al., Numerical Recipes), and a polynomial of degree 7 fitted to it
// (Chebyshev points over 0 <= x <= 14; the coefficients are this fit's) is off by 8e-7, relatively. In fp32 the
// rounding of the exponent adds to that: 2.5e-6 up to y = 5, 1.5e-5 at y = 13, where the result leaves bf16's
// range. A third of erfcf's instructions, and enough for 16-bit results (half a step of fp16 is 4.9e-4).
__device__ __forceinline__ float half_erfc_of(float y) {
  const float t = __fdividef(1.f, fmaf(0.35355339059327376f, y, 1.f));
  float p = -0.19184046983718872f;
  p = fmaf(p, t, 0.7685127854347229f);
  p = fmaf(p, t, -1.0301551818847656f);
  p = fmaf(p, t, 0.37635737657546997f);
  p = fmaf(p, t, -0.05336221680045128f);
  p = fmaf(p, t, 0.39794403314590454f);
  p = fmaf(p, t, 0.997983455657959f);
  p = fmaf(p, t, -1.265440583229065f);
  return 0.5f * t * fast_exp(fmaf(-0.5f * y, y, p));
}

// act(g) in `a`, act'(g) in `d`. The exponentials use the hardware's approximations (relative error about
// 2^-22), far below the rounding of a 16-bit result; EXACT takes the library functions instead, for
// 32-bit tensors.
template <int ACT, bool EXACT>
__device__ __forceinline__ void glu_act(float g, float& a, float& d) {
  if constexpr (ACT == ORDA_ACT_SILU) {
    const float s = EXACT ? 1.f / (1.f + expf(-g)) : __fdividef(1.f, 1.f + fast_exp(-g));
    a = g * s;
    d = s * (1.f + g * (1.f - s));
  } else if constexpr (ACT == ORDA_ACT_RELU) {
    a = g <= 0.f ? 0.f : g;  // a NaN stays one, in the derivative too (fmaxf would return 0)
    d = g > 0.f ? 1.f : a;
  } else if constexpr (ACT == ORDA_ACT_GELU) {
    float cdf, e;
    if constexpr (EXACT) {
      cdf = 0.5f * erfcf(g * -0.70710678118654752f);
      e = expf(-0.5f * g * g);
    } else {
      const float half_erfc = half_erfc_of(fabsf(g));
      cdf = g > 0.f ? 1.f - half_erfc : half_erfc;
      e = fast_exp(-0.5f * g * g);
    }
    a = g * cdf;
    d = cdf + g * e * 0.39894228040143268f;
  } else {
    // 1/2 (1 + tanh z) = 1 / (1 + e^(-2z)), z = sqrt(2/pi) (g + 0.044715 g^3). Where g^2 is infinite, s is 0 or 1 and
    // d must not be inf * 0
    const float c = 0.79788456080286536f;
    const float z = c * (g + 0.044715f * g * g * g);
    const float s = EXACT ? 1.f / (1.f + expf(-2.f * z)) : __fdividef(1.f, 1.f + fast_exp(-2.f * z));
    a = g * s;
    d = s + g * (2.f * s * (1.f - s)) * c * (1.f + 0.134145f * fminf(g * g, 1e30f));
  }
}

template <int ACT>
struct ActTag {
  static constexpr int kAct = ACT;
};

// f(ActTag<act>): the activation is uniform over the grid, so it is picked once around a loop.
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  if (act == ORDA_ACT_SILU) f(ActTag<ORDA_ACT_SILU>{});
  else if (act == ORDA_ACT_GELU) f(ActTag<ORDA_ACT_GELU>{});
  else if (act == ORDA_ACT_GELU_TANH) f(ActTag<ORDA_ACT_GELU_TANH>{});
  else f(ActTag<ORDA_ACT_RELU>{});
}

}  // namespace orda

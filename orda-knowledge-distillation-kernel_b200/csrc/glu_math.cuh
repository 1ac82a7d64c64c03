// Activations of the gated feed-forward block and their derivatives.
#pragma once

#include <stdint.h>

#include "distill_common.cuh"
#include "orda_b200_student.h"

namespace orda {

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
    a = fmaxf(g, 0.f);
    d = g > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == ORDA_ACT_GELU) {
    const float cdf = 0.5f * erfcf(g * -0.70710678118654752f);
    const float e = EXACT ? expf(-0.5f * g * g) : fast_exp(-0.5f * g * g);
    a = g * cdf;
    d = cdf + g * e * 0.39894228040143268f;
  } else {
    // 1/2 (1 + tanh z) = 1 / (1 + e^(-2z)), z = sqrt(2/pi) (g + 0.044715 g^3)
    const float c = 0.79788456080286536f;
    const float z = c * (g + 0.044715f * g * g * g);
    const float s = EXACT ? 1.f / (1.f + expf(-2.f * z)) : __fdividef(1.f, 1.f + fast_exp(-2.f * z));
    a = g * s;
    d = s + g * (2.f * s * (1.f - s)) * c * (1.f + 0.134145f * g * g);
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

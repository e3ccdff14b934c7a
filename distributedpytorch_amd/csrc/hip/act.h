// Activations that a normalisation or a linear product applies in its epilogue, and their derivatives with respect to the
// value u in front of them.  ids: 0 none, 1 relu, 2 silu (u * sigmoid(u)), 3 gelu (u * Phi(u), Phi the normal distribution).
//
// erf is the rational approximation 7.1.26 of Abramowitz and Stegun (absolute error 1.5e-7, about two roundings of fp32 at
// the sizes that matter here): one reciprocal and one exponential, which the derivative of gelu shares, where the library's
// erff takes some forty instructions - a 256 x 256 output tile spends longer in it than in its matrix instructions.
#pragma once
#include "common.h"

enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

__device__ __forceinline__ float act_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// 1 - Phi(|u|) = erfc(|u| / sqrt 2) / 2, and e = exp(-u^2 / 2)
__device__ __forceinline__ float act_upper_tail(float u, float& e) {
  e = act_exp(-0.5f * u * u);
  const float t = __builtin_amdgcn_rcpf(1.f + 0.23164190f * fabsf(u));          // 0.3275911 / sqrt 2
  const float q = t * (0.127414796f + t * (-0.142248368f + t * (0.710706871f + t * (-0.726576014f + t * 0.530702715f))));      // halves of the a_i
  return q * e;
}

template <int ACT> __device__ __forceinline__ float act_fwd(float u) {
  if (ACT == ACT_RELU) return u > 0.f || u != u ? u : 0.f;          // (NaN stays NaN)
  if (ACT == ACT_SILU) return u * __builtin_amdgcn_rcpf(1.f + act_exp(-u));
  if (ACT == ACT_GELU) {
    float e;
    const float tail = act_upper_tail(u, e);
    return u * (u > 0.f ? 1.f - tail : tail);
  }
  return u;
}

template <int ACT> __device__ __forceinline__ float act_slope(float u) {
  if (ACT == ACT_RELU) return u > 0.f ? 1.f : 0.f;
  if (ACT == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + act_exp(-u));
    return s * (1.f + u * (1.f - s));
  }
  if (ACT == ACT_GELU) {
    float e;
    const float tail = act_upper_tail(u, e);
    return (u > 0.f ? 1.f - tail : tail) + u * 0.39894228040143268f * e;
  }
  return 1.f;
}

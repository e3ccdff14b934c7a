// Activations that a normalisation or a linear product applies in its epilogue, and their derivatives with respect to the
// value u in front of them.  ids: 0 none, 1 relu, 2 silu (u * sigmoid(u)), 3 gelu (u * Phi(u), Phi the normal distribution).
#pragma once
#include "common.h"

enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

template <int ACT> __device__ __forceinline__ float act_fwd(float u) {
  if (ACT == ACT_RELU) return u > 0.f || u != u ? u : 0.f;          // (NaN stays NaN)
  if (ACT == ACT_SILU) return u / (1.f + expf(-u));
  if (ACT == ACT_GELU) return 0.5f * u * (1.f + erff(u * 0.70710678118654752f));
  return u;
}

template <int ACT> __device__ __forceinline__ float act_slope(float u) {
  if (ACT == ACT_RELU) return u > 0.f ? 1.f : 0.f;
  if (ACT == ACT_SILU) { const float s = 1.f / (1.f + expf(-u)); return s * (1.f + u * (1.f - s)); }
  if (ACT == ACT_GELU)
    return 0.5f * (1.f + erff(u * 0.70710678118654752f)) + u * 0.39894228040143268f * expf(-0.5f * u * u);
  return 1.f;
}

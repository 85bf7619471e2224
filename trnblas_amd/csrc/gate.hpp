// The activations of gated projections and their derivatives, in fp32.
#pragma once

#include "common.hpp"

namespace trnblas {

constexpr float kSqrtHalf = 0.70710678f, kInvSqrt2Pi = 0.39894228f, kTanhScale = 1.5957691f;  // 2 sqrt(2 / pi)

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

// act(x). gelu by erfc, gelu_tanh by the sigmoid (0.5 (1 + tanh u) = sigmoid(2 u)): no
// cancellation where x is far below zero.
__device__ __forceinline__ float gate(int act, float x) {
  switch (act) {
    case TRNBLAS_ACT_SILU: return x * sigmoid(x);
    case TRNBLAS_ACT_GELU: return 0.5f * x * erfcf(-kSqrtHalf * x);
    case TRNBLAS_ACT_GELU_TANH: return x * sigmoid(kTanhScale * x * __builtin_fmaf(0.044715f * x, x, 1.0f));
    case TRNBLAS_ACT_RELU: return x < 0.0f ? 0.0f : x;
    default: return sigmoid(x);
  }
}

// act(x) and act'(x). Terms that vanish far from zero are taken at the bound where they
// have done so: an infinite x would make them 0 x infinity.
__device__ __forceinline__ void gate_slope(int act, float x, float& y, float& slope) {
  const float near = x > 60.0f ? 60.0f : x < -120.0f ? -120.0f : x;  // a NaN stays
  switch (act) {
    case TRNBLAS_ACT_SILU: {
      const float s = sigmoid(x);
      y = x * s;
      slope = s * __builtin_fmaf(near, sigmoid(-near), 1.0f);
      return;
    }
    case TRNBLAS_ACT_GELU: {
      const float p = 0.5f * erfcf(-kSqrtHalf * x);
      y = x * p;
      slope = __builtin_fmaf(near * kInvSqrt2Pi, expf(-0.5f * near * near), p);
      return;
    }
    case TRNBLAS_ACT_GELU_TANH: {
      const float s = sigmoid(kTanhScale * x * __builtin_fmaf(0.044715f * x, x, 1.0f));
      const float t = sigmoid(-kTanhScale * near * __builtin_fmaf(0.044715f * near, near, 1.0f));
      y = x * s;
      slope = s * __builtin_fmaf(kTanhScale * near * t, __builtin_fmaf(0.134145f * near, near, 1.0f), 1.0f);
      return;
    }
    case TRNBLAS_ACT_RELU:
      y = x < 0.0f ? 0.0f : x;
      slope = x > 0.0f ? 1.0f : x != x ? x : 0.0f;
      return;
    default:
      y = sigmoid(x);
      slope = y * sigmoid(-x);
  }
}

}  // namespace trnblas

// The activations of gated projections and their derivatives, in fp32.
#pragma once

#include "common.hpp"

namespace trnblas {

constexpr float kLog2e = 1.44269504f, kInvSqrt2Pi = 0.39894228f, kTanhScale = 1.5957691f;  // 2 sqrt(2 / pi)

// exp(x) by the hardware's power of two: the rounding of x log2(e) makes it |x| 2^-24 off, relative,
// which x exp(-|x|) keeps below 2^-24 absolute. In a product's epilogue every wave has a
// hundred of these per lane, and nothing else to do.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(kLog2e * x); }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }

// The normal distribution up to x, and e = exp(-x^2 / 2): with z = |x| / sqrt(2) and t = 1 / (1 +
// 0.3 z), erfc(z) = e t p(t); p is the polynomial of degree 8 with the least relative error
// (1.3e-7 in fp32) for z <= 10, past which e is zero. No cancellation where x is far below zero.
__device__ __forceinline__ float normal(float x, float& e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.21213203f, __builtin_fabsf(x), 1.0f));
  float p = -0.129523143f;
  p = __builtin_fmaf(p, t, 0.485564411f);
  p = __builtin_fmaf(p, t, -0.512280762f);
  p = __builtin_fmaf(p, t, 0.547723293f);
  p = __builtin_fmaf(p, t, -0.0946531370f);
  p = __builtin_fmaf(p, t, 0.214927167f);
  p = __builtin_fmaf(p, t, 0.148338854f);
  p = __builtin_fmaf(p, t, 0.170715272f);
  p = __builtin_fmaf(p, t, 0.169188008f);
  e = exp_fast(-0.5f * x * x);
  const float q = 0.5f * t * p * e;
  return x < 0.0f ? q : 1.0f - q;
}

// act(x); gelu_tanh by the sigmoid: (1 + tanh u) / 2 = sigmoid(2 u).
__device__ __forceinline__ float gate(int act, float x) {
  switch (act) {
    case TRNBLAS_ACT_SILU: return x * sigmoid(x);
    case TRNBLAS_ACT_GELU: {
      float e;
      return x * normal(x, e);
    }
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
      float e;
      const float p = normal(x, e);
      y = x * p;
      slope = __builtin_fmaf(near * kInvSqrt2Pi, e, p);
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

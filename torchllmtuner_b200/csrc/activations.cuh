// Activations of a linear layer's epilogue and their derivatives, fp32.
//   gelu       z Phi(z); Phi(-|z|) = erfc(|z| / sqrt 2) / 2 as one product with the density's exponential (not (1 + erf) / 2, which cancels
//              for z < -3), Phi(|z|) = 1 - Phi(-|z|)
//   gelu_tanh  z s, s = 1 / (1 + exp(-2 u)) = (1 + tanh u) / 2, u = sqrt(2 / pi) (z + 0.044715 z^3)
//   silu       z / (1 + exp(-z))
//   relu       max(z, 0), NaN stays
#pragma once
#include "common.cuh"

namespace llmt {

enum ActKind : int { kActNone = 0, kActGelu = 1, kActGeluTanh = 2, kActSilu = 3, kActRelu = 4, kActKinds = 5 };

constexpr float kSqrtHalf = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f, kSqrt2OverPi = 0.79788456080286536f, kGeluCubic = 0.044715f;

// 2^v and 1 / v in one instruction each (relative error 2^-22 and 2^-23); results below the normal range are zero.
__device__ __forceinline__ float exp2_of(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_of(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid_of(float v) { return rcp_of(1.f + exp2_of(-kLog2e * v)); }   // the power overflows to inf: 0
__device__ __forceinline__ float gelu_sigmoid(float z, float z2) {
  return rcp_of(1.f + exp2_of(z * (-2.f * kLog2e * kSqrt2OverPi - 2.f * kLog2e * kSqrt2OverPi * kGeluCubic * z2)));
}

// Phi(z) and exp(-z^2 / 2). erfc(x) exp(x^2) is a polynomial of degree 7 in t = 1 / (1 + x / 2) without constant term, fitted over 0 <= x <= 10 by
// least squares reweighted towards the largest relative error, which is 2^-19.5 (z^2 / 2 = 100 at the end: the tail is below fp32 beyond).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float t = rcp_of(1.f + 0.5f * kSqrtHalf * fabsf(z));
  e = exp2_of(-0.5f * kLog2e * z * z);
  float q = 0.088204011321067810f;
  q = q * t - 0.35673707723617554f;
  q = q * t + 0.38922297954559326f;
  q = q * t + 0.037891786545515060f;
  q = q * t + 0.28150334954261780f;
  q = q * t + 0.27758222818374634f;
  q = q * t + 0.28233140707015991f;
  const float tail = 0.5f * t * q * e;
  return z < 0.f ? tail : 1.f - tail;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  float e;
  if constexpr (ACT == kActGelu) return z * normal_cdf(z, e);
  if constexpr (ACT == kActGeluTanh) return z * gelu_sigmoid(z, z * z);
  if constexpr (ACT == kActSilu) return z * sigmoid_of(z);
  if constexpr (ACT == kActRelu) return z < 0.f ? 0.f : z;
  return z;
}

// g act'(z)
template <int ACT>
__device__ __forceinline__ float activate_grad(float z, float g) {
  if constexpr (ACT == kActGelu) {
    float e;
    const float cdf = normal_cdf(z, e);
    return g * (cdf + z * kInvSqrt2Pi * e);
  }
  if constexpr (ACT == kActGeluTanh) {
    const float z2 = z * z, s = gelu_sigmoid(z, z2);
    return g * (s + (s - s * s) * (z * (2.f * kSqrt2OverPi + 6.f * kSqrt2OverPi * kGeluCubic * z2)));
  }
  if constexpr (ACT == kActSilu) {
    const float s = sigmoid_of(z);
    return g * (s + (s - s * s) * z);
  }
  if constexpr (ACT == kActRelu) return z <= 0.f ? 0.f : g;
  return g;
}

}  // namespace llmt

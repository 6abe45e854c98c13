// Activations of a linear layer's epilogue and their derivatives, fp32.
//   gelu       z Phi(z); Phi(-|z|) = erfc(|z| / sqrt 2) / 2 as one product with the density's exponential (not (1 + erf) / 2, which cancels
//              for z < -3), Phi(|z|) = 1 - Phi(-|z|)
//   gelu_tanh  z s, s = 1 / (1 + exp(-2 u)) = (1 + tanh u) / 2, u = sqrt(2 / pi) (z + 0.044715 z^3)
//   silu       z / (1 + exp(-z))
//   relu       max(z, 0), NaN stays
#pragma once
#include "vec_io.cuh"

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
// v within [-limit, limit]; NaN stays.
__device__ __forceinline__ float clamp_of(float v, float limit) {
  float r;
  asm("{ .reg .f32 t; min.NaN.f32 t, %1, %2; max.NaN.f32 %0, t, %3; }" : "=f"(r) : "f"(v), "f"(limit), "f"(-limit));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float2 exp2_of(float2 v) { return make_float2(exp2_of(v.x), exp2_of(v.y)); }
__device__ __forceinline__ float2 rcp_of(float2 v) { return make_float2(rcp_of(v.x), rcp_of(v.y)); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Everything on two values at a time: the epilogue that calls this shares its schedulers with nothing but itself, and the instructions per value
// decide whether it stays under the products.
__device__ __forceinline__ float2 sigmoid_of(float2 v) {           // the power overflows to inf: 0
  return rcp_of(add2(both(1.f), exp2_of(mul2(v, both(-kLog2e)))));
}
__device__ __forceinline__ float2 gelu_sigmoid(float2 z, float2 z2) {
  const float a = -2.f * kLog2e * kSqrt2OverPi, b = a * kGeluCubic;
  return rcp_of(add2(both(1.f), exp2_of(mul2(z, fma2(z2, both(b), both(a))))));
}

// Phi(z) and exp(-z^2 / 2). erfc(x) exp(x^2) is a polynomial of degree 7 in t = 1 / (1 + x / 2) without constant term, fitted over 0 <= x <= 10 by
// least squares reweighted towards the largest relative error, which is 2^-19.5 (z^2 / 2 = 100 at the end: the tail is below fp32 beyond).
__device__ __forceinline__ float2 normal_cdf(float2 z, float2& e) {
  const float2 t = rcp_of(fma2(make_float2(fabsf(z.x), fabsf(z.y)), both(0.5f * kSqrtHalf), both(1.f)));
  e = exp2_of(mul2(mul2(z, z), both(-0.5f * kLog2e)));
  float2 q = both(0.5f * 0.088204011321067810f);       // halved: Phi = erfc / 2
  q = fma2(q, t, both(0.5f * -0.35673707723617554f));
  q = fma2(q, t, both(0.5f * 0.38922297954559326f));
  q = fma2(q, t, both(0.5f * 0.037891786545515060f));
  q = fma2(q, t, both(0.5f * 0.28150334954261780f));
  q = fma2(q, t, both(0.5f * 0.27758222818374634f));
  q = fma2(q, t, both(0.5f * 0.28233140707015991f));
  const float2 tail = mul2(mul2(t, q), e);
  return make_float2(z.x < 0.f ? tail.x : 1.f - tail.x, z.y < 0.f ? tail.y : 1.f - tail.y);
}

template <int ACT>
__device__ __forceinline__ float2 activate(float2 z) {
  float2 e;
  if constexpr (ACT == kActGelu) return mul2(z, normal_cdf(z, e));
  if constexpr (ACT == kActGeluTanh) return mul2(z, gelu_sigmoid(z, mul2(z, z)));
  if constexpr (ACT == kActSilu) return mul2(z, sigmoid_of(z));
  if constexpr (ACT == kActRelu) return make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y);
  return z;
}

// g act'(z)
template <int ACT>
__device__ __forceinline__ float2 activate_grad(float2 z, float2 g) {
  if constexpr (ACT == kActGelu) {
    float2 e;
    const float2 cdf = normal_cdf(z, e);
    return mul2(g, fma2(mul2(z, both(kInvSqrt2Pi)), e, cdf));
  }
  if constexpr (ACT == kActGeluTanh) {
    z = make_float2(clamp_of(z.x, 100.f), clamp_of(z.y, 100.f));       // there act' is 0 or 1; u of a z beyond 1e12 would be inf, and 0 inf NaN
    const float2 z2 = mul2(z, z), s = gelu_sigmoid(z, z2), u = mul2(z, fma2(z2, both(6.f * kSqrt2OverPi * kGeluCubic), both(2.f * kSqrt2OverPi)));
    return mul2(g, fma2(fma2(mul2(s, both(-1.f)), s, s), u, s));
  }
  if constexpr (ACT == kActSilu) {
    const float2 s = sigmoid_of(z);
    return mul2(g, fma2(fma2(mul2(s, both(-1.f)), s, s), z, s));
  }
  if constexpr (ACT == kActRelu) return make_float2(z.x <= 0.f ? 0.f : g.x, z.y <= 0.f ? 0.f : g.y);
  return g;
}

}  // namespace llmt

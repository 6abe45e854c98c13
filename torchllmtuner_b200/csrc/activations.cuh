// Activations of a linear layer's epilogue and their derivatives, fp32.
//   gelu       z Phi(z), Phi(z) = erfc(-z / sqrt 2) / 2 (not (1 + erf) / 2, which cancels for z < -3)
//   gelu_tanh  z s, s = 1 / (1 + exp(-2 u)) = (1 + tanh u) / 2, u = sqrt(2 / pi) (z + 0.044715 z^3)
//   silu       z / (1 + exp(-z))
//   relu       max(z, 0), NaN stays
#pragma once
#include "common.cuh"

namespace llmt {

enum ActKind : int { kActNone = 0, kActGelu = 1, kActGeluTanh = 2, kActSilu = 3, kActRelu = 4, kActKinds = 5 };

constexpr float kSqrtHalf = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f, kSqrt2OverPi = 0.79788456080286536f, kGeluCubic = 0.044715f;

__device__ __forceinline__ float sigmoid_of(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }   // exp overflows to inf: 0

template <int V>
__device__ __forceinline__ void activate(int act, float* z) {
  switch (act) {
    case kActGelu:
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] *= 0.5f * erfcf(-kSqrtHalf * z[i]);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] *= sigmoid_of(2.f * kSqrt2OverPi * (z[i] + kGeluCubic * z[i] * z[i] * z[i]));
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] *= sigmoid_of(z[i]);
      break;
    case kActRelu:
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = z[i] < 0.f ? 0.f : z[i];
      break;
    default: break;
  }
}

// g *= act'(z)
template <int V>
__device__ __forceinline__ void activate_grad(int act, const float* z, float* g) {
  switch (act) {
    case kActGelu:
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] *= 0.5f * erfcf(-kSqrtHalf * z[i]) + z[i] * kInvSqrt2Pi * __expf(-0.5f * z[i] * z[i]);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float s = sigmoid_of(2.f * kSqrt2OverPi * (z[i] + kGeluCubic * z[i] * z[i] * z[i]));
        g[i] *= s + z[i] * s * (1.f - s) * 2.f * kSqrt2OverPi * (1.f + 3.f * kGeluCubic * z[i] * z[i]);
      }
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float s = sigmoid_of(z[i]);
        g[i] *= s * (1.f + z[i] * (1.f - s));
      }
      break;
    case kActRelu:
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = z[i] <= 0.f ? 0.f : g[i];
      break;
    default: break;
  }
}

}  // namespace llmt

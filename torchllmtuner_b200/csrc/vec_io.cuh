// Reading and writing V consecutive bf16 or fp32 values as fp32, with the widest accesses their size allows: V * sizeof(T) bytes, at most 16
// per access. The caller guarantees the alignment (min(16, V * sizeof(T)) bytes).
#pragma once
#include "common.cuh"

namespace llmt {

__device__ __forceinline__ void unpack_bf16x2(uint32_t u, float* f) {
  const float2 t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
  f[0] = t.x;
  f[1] = t.y;
}

// Raw registers of V values, so that a load can be issued early and converted where it is used.
template <typename T, int V>
struct Raw {
  static constexpr int kWords = V * (int)sizeof(T) >= 4 ? V * (int)sizeof(T) / 4 : 1;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
    } else if constexpr (V * sizeof(T) == 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x; w[1] = u.y;
    } else if constexpr (V * sizeof(T) == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = __uint_as_float(w[i]);
    } else if constexpr (V == 1) {
      f[0] = __uint_as_float(w[0] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) unpack_bf16x2(w[i], f + 2 * i);
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(f[i]);
    } else if constexpr (V == 1) {
      w[0] = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if constexpr (V * sizeof(T) == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else if constexpr (V * sizeof(T) == 4) {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  Raw<T, V> r;
  r.load(p);
  r.get(f);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  Raw<T, V> r;
  r.set(f);
  r.store(p);
}

// Pairs of fp32 values in one instruction, each rounded as the scalar one.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(*reinterpret_cast<uint64_t*>(&r)) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*reinterpret_cast<uint64_t*>(&r)) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<uint64_t*>(&r))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return r;
}
// Eight values as four pairs.
template <typename T>
__device__ __forceinline__ void get2(const Raw<T, 8>& r, float2* f) {
  float v[8];
  r.get(v);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(v[2 * i], v[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ void store2(T* p, const float2* f) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = f[i].x; v[2 * i + 1] = f[i].y; }
  store_vec<T, 8>(p, v);
}

}  // namespace llmt

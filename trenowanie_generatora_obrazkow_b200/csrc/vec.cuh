// Typed vector access shared by the kernels that take bf16, fp16 and fp32 tensors: V consecutive elements to and from
// fp32 registers, 16 bytes per access where V * sizeof(T) allows it (V = 8 on 16-byte aligned addresses; V = 1 anywhere).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace tgo {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// V elements as they are stored: 16-byte words for V = 8 (one for 2-byte types, two for fp32), one element for V = 1.
template <typename T, int V>
struct Raw {
  static_assert(V == 8, "8 or 1");
  static constexpr int W = sizeof(T) * 8 / 16;
  uint4 u[W];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < W; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(p)[i] = u[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) u[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (sizeof(T) == 4) {
      const float* s = reinterpret_cast<const float*>(u);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = s[i];
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 t;
        if constexpr (sizeof(T) == 2 && __is_same(T, __nv_bfloat16)) {
          t.x = __uint_as_float(w[i] << 16);
          t.y = __uint_as_float(w[i] & 0xffff0000u);
        } else {
          t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        }
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
  }
  __device__ __forceinline__ void put(const float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
      float* d = reinterpret_cast<float*>(u);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = f[i];
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (__is_same(T, __nv_bfloat16)) {
          __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<uint32_t*>(&v);
        } else {
          __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<uint32_t*>(&v);
        }
      }
    }
  }
};
// Pairs of fp32 in one 64-bit register: sm_100 issues one instruction for both (f32x2).
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 x2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ f32x2 x2(float a) { return x2(a, a); }
__device__ __forceinline__ float2 x2_split(f32x2 r) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(r));
  return f;
}
__device__ __forceinline__ f32x2 x2_fma(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 x2_mul(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 x2_add(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float x2_sum(f32x2 r) {
  const float2 f = x2_split(r);
  return f.x + f.y;
}

// 8 stored elements as 4 fp32 pairs, and back
template <typename T>
__device__ __forceinline__ void unpack_x2(const Raw<T, 8>& r, f32x2 (&v)[4]) {
  float f[8];
  r.get(f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = x2(f[2 * i], f[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ void store_x2(T* p, const f32x2 (&v)[4]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = x2_split(v[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
  Raw<T, 8> r;
  r.put(f);
  r.store(p);
}

template <typename T>
struct Raw<T, 1> {
  T e;
  __device__ __forceinline__ void load(const T* p) { e = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = e; }
  __device__ __forceinline__ void zero() { e = from_f<T>(0.f); }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f<T>(e); }
  __device__ __forceinline__ void put(const float (&f)[1]) { e = from_f<T>(f[0]); }
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[V]) {
  Raw<T, V> r;
  r.load(p);
  r.get(f);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
  Raw<T, V> r;
  r.put(f);
  r.store(p);
}

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace tgo

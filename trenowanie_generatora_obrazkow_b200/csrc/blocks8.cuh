// Device helpers of the 8-bit block kernels (blocks8.cu, gemm8.cu): scales, conversions, silu(a) b, an output's place.
#pragma once
#include <cuda_fp8.h>
#include <stdint.h>

namespace tgo {
namespace {

constexpr int TILE = 128;
constexpr int ATOM = 512;

// ---------------------------------------------------------------------------------------------------------- scales
// With u the bits of A: the carry out of the mantissa's top bits is the step from m <= 1.75 to m > 1.75. A block without a finite
// value has A = 0, which maxima that pass over NaN may show as NaN.
__device__ __forceinline__ int scale_byte(float amax) {
  return max(0, (int)((__float_as_uint(fmaxf(amax, 0.f)) + 0x1fffffu) >> 23) - 8);
}
__device__ __forceinline__ float scale_inv(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }  // 2^-e
__device__ __forceinline__ float scale_of(int byte) {                                                          // 2^e
  return __uint_as_float(byte > 0 ? (uint32_t)byte << 23 : 0x00400000u);
}
// 2^e = x y with x = 2^floor(e / 2) or half of it, y = 2 or 4 x. d (x x') (y y') of two scales has no step that leaves fp32's
// range upwards unless the result does (both factors are at least 1, or the first is less), nor downwards unless the result
// is less than 2^-149 (|d| < 2^25 and x x' < 2^-108).
__device__ __forceinline__ float2 scale_halves(int byte) {
  return make_float2(__uint_as_float((uint32_t)((byte >> 1) + 63) << 23), __uint_as_float((uint32_t)((byte + 1 >> 1) + 64) << 23));
}
// offset of the scale byte of row r and block b; quads: atoms of a row tile, ceil(blocks / 4)
__device__ __forceinline__ long long scale_at(int r, int b, int quads) {
  return ((long long)(r >> 7) * quads + (b >> 2)) * ATOM + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ uint32_t codes2(float a, float b) {  // a in the low byte
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t codes4(float2 a, float2 b) { return codes2(a.x, a.y) | (codes2(b.x, b.y) << 16); }
__device__ __forceinline__ float2 values2(uint32_t codes) {  // low two bytes
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ void values8(uint2 c, float k, float2 (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = mul2(values2((i < 2 ? c.x : c.y) >> ((i & 1) * 16)), make_float2(k, k));
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // passes over NaN
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// s = 1 / (1 + exp(-a)) = p q. s leaves fp32's range below a = -87 while products of it may be far inside: there s = exp(a), and p
// = q = 1 / (1 + exp(-a / 2)) = exp(a / 2) (to 2^-62 of it); each operand of a product takes a factor, x s y = (x p) (y q).
// For 16-bit types exp2 and the reciprocal are the hardware's approximations: s is off by (1.25 |a| + 16) 2^-24 of itself at most
// and taken as 0 below a = -174 (s < 2^-251). A result that is rounded to 16 bits hides that; one that goes to 8 bits from
// fp32 takes the neighbouring code where it lies as near as that to a border, one in 2^-4 / 2^-20 = 2^16. Measured in the MLP
// against 64-bit sums and sigmoids, y of 3000 x 1024 x 2048 in fp16 is off by 1.6e-4 (1.2e-4 with the library's; the rest is the
// rounding of [a | b] after sums in another order), in bf16 by the same with either. The library's took 335 us instead of 219
// in swiglu_blocks' backward at 32768 x 5504, 553 instead of 353 in the MLP's. fp32 results take the library's.
template <bool FINE>
__device__ __forceinline__ void sigmoid(float a, float& p, float& q) {
  const bool far = a < -87.f;
  if constexpr (FINE) {
    p = 1.f / (1.f + expf(far ? -0.5f * a : -a));
  } else {
    float t = a * -1.4426950408889634f;
    if (far) t *= 0.5f;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(t));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(1.f + t));
  }
  q = far ? p : 1.f;
}
// silu(a) b
template <bool FINE>
__device__ __forceinline__ float2 swiglu(float2 a, float2 b) {
  float2 p, q;
  sigmoid<FINE>(a.x, p.x, q.x);
  sigmoid<FINE>(a.y, p.y, q.y);
  return mul2(mul2(a, p), mul2(b, q));
}

struct Side {             // one 8-bit output
  uint8_t* codes;
  uint8_t* scales;
  int rows, quads;        // of the codes; atoms of a row tile
  long long width;        // bytes of a row: the blocked axis rounded up to 128
};
inline Side side(uint8_t* codes, uint8_t* scales, int rows, int along) {
  const int nb = (along + TILE - 1) / TILE;
  return Side{codes, scales, rows, (nb + 3) / 4, (long long)nb * TILE};
}

}  // namespace
}  // namespace tgo

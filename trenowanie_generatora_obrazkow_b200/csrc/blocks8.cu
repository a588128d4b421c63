// Packing into 8-bit blocks (blocks8.h) and back, SwiGLU with its input kept in 8 bits, and the product of few rows with a
// packed weight.
//
// A block of 128 values with the largest finite magnitude A has the scale 2^e, the smallest one with A <= 448 2^e: with
// A = 2^a m, 1 <= m < 2, and 448 = 2^8 1.75 that is e = a - 8, one more where m > 1.75 (and -127 at least). Multiplying by
// 2^-e is exact, so the only rounding of a value is the one to e4m3. Values that are not finite become NaN.
//
// All of this reads and writes each byte once: the kernels are bound by memory. A CTA of 256 threads holds a tile of 128 x
// 128 in registers, a thread 8 rows x 8 columns: the row maxima need 16 lanes of a warp, the column maxima the tile's 8
// warps (through shared memory), and eight codes of a column are eight bytes, so the transposed tile is staged in 16 KB
// of shared memory without bank conflicts and leaves as whole lines.
#include <cuda_fp8.h>

#include <algorithm>

#include "block_ops.h"
#include "blocks8.h"
#include "common.cuh"
#include "vec.cuh"

namespace tgo {

namespace {

constexpr int TILE = 128, PACK_THREADS = 256;
constexpr int ATOM = 512;

// ---------------------------------------------------------------------------------------------------------- scales
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  return max(0, (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ float scale_inv(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }  // 2^-e
__device__ __forceinline__ float scale_of(int byte) {                                                          // 2^e
  return __uint_as_float(byte > 0 ? (uint32_t)byte << 23 : 0x00400000u);
}
// offset of the scale byte of row r and block b; quads: atoms of a row tile, ceil(blocks / 4)
__device__ __forceinline__ long long scale_at(int r, int b, int quads) {
  return ((long long)(r >> 7) * quads + (b >> 2)) * ATOM + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}
__device__ __forceinline__ uint32_t codes2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) { return codes2(a, b) | (codes2(c, d) << 16); }
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float k) {
  return make_uint2(codes4(f[0] * k, f[1] * k, f[2] * k, f[3] * k), codes4(f[4] * k, f[5] * k, f[6] * k, f[7] * k));
}
__device__ __forceinline__ float2 values2(uint32_t codes) {  // low two bytes
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ void values8(uint2 c, float k, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = values2((i < 2 ? c.x : c.y) >> ((i & 1) * 16));
    f[2 * i] = t.x * k;
    f[2 * i + 1] = t.y * k;
  }
}

// ------------------------------------------------------------------------------------------------------------ loads
// n (0 to 8) elements of a row; 16-byte loads where vec (the row's start is aligned and n is 0 or 8)
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&f)[8]) {
  Raw<T, 8> r;
  r.zero();
  if (vec) {
    if (n > 0) r.load(p);
    r.get(f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j < n ? to_f(p[j]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&f)[8]) {
  if (vec) {
    if (n <= 0) return;
    Raw<T, 8> r;
    r.put(f);
    r.store(p);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = from_f<T>(f[j]);
  }
}
__device__ __forceinline__ float top8(const float (&f)[8]) {
  float a = fmaxf(fabsf(f[0]), fabsf(f[1])), b = fmaxf(fabsf(f[2]), fabsf(f[3]));
  float c = fmaxf(fabsf(f[4]), fabsf(f[5])), d = fmaxf(fabsf(f[6]), fabsf(f[7]));
  return fmaxf(fmaxf(a, b), fmaxf(c, d));
}
// fmaxf passes over NaN, an infinity shows: it becomes NaN and the largest finite magnitude is taken again
__device__ __forceinline__ float finite_top8(float (&f)[8]) {
  float m = top8(f);
  if (m == INFINITY) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (fabsf(f[j]) == INFINITY) f[j] = NAN;
    m = top8(f);
  }
  return m;
}
__device__ __forceinline__ float max16(float m) {  // over the 16 lanes of a row
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// ------------------------------------------------------------------------------------------------------- tile output
struct Side {             // one 8-bit output
  uint8_t* codes;
  uint8_t* scales;
  int rows, quads;        // of the codes; atoms of a row tile
  long long width;        // bytes of a row: the blocked axis rounded up to 128
};
struct TileShared {
  float part[8][TILE];
  uint4 t[TILE * TILE / 16];  // transposed codes: column c's eight bytes of rows 8 i .. at c * 16 + (i ^ (c / 8 % 16))
};

// rows of the tile: row0 + 8 rg + i, blocks along the columns (block kb of nb)
__device__ __forceinline__ void emit_rows(const Side& o, float (&v)[8][8], int row0, int kb, int nb, int rg, int l16) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = row0 + 8 * rg + i;
    const int byte = scale_byte(max16(finite_top8(v[i])));
    if (r < o.rows) *reinterpret_cast<uint2*>(o.codes + (long long)r * o.width + kb * TILE + 8 * l16) = codes8(v[i], scale_inv(byte));
    if (l16 == 0) {
      uint8_t* s = o.scales + scale_at(r, kb, o.quads);
      s[0] = (uint8_t)byte;
      if (kb == nb - 1)
        for (int b = 1; b < 4 - (kb & 3); ++b) s[b] = 0;
    }
  }
}
// columns col0 + 8 l16 + j as rows of the transposed form, blocks along the tile's rows (block mb of nb)
__device__ __forceinline__ void emit_cols(const Side& o, float (&v)[8][8], int col0, int mb, int nb, int rg, int l16,
                                          TileShared& sh) {
  float m[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) m[j] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    finite_top8(v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = fmaxf(m[j], fabsf(v[i][j]));
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
  __syncthreads();  // the tile before has been read
  if ((rg & 1) == 0) {
    *reinterpret_cast<float4*>(&sh.part[rg >> 1][8 * l16]) = make_float4(m[0], m[1], m[2], m[3]);
    *reinterpret_cast<float4*>(&sh.part[rg >> 1][8 * l16 + 4]) = make_float4(m[4], m[5], m[6], m[7]);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float4 a = *reinterpret_cast<const float4*>(&sh.part[w][8 * l16]);
    const float4 b = *reinterpret_cast<const float4*>(&sh.part[w][8 * l16 + 4]);
    m[0] = fmaxf(m[0], a.x), m[1] = fmaxf(m[1], a.y), m[2] = fmaxf(m[2], a.z), m[3] = fmaxf(m[3], a.w);
    m[4] = fmaxf(m[4], b.x), m[5] = fmaxf(m[5], b.y), m[6] = fmaxf(m[6], b.z), m[7] = fmaxf(m[7], b.w);
  }
  uint2* t = reinterpret_cast<uint2*>(sh.t);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int byte = scale_byte(m[j]);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i][j];
    t[(8 * l16 + j) * 16 + (rg ^ l16)] = codes8(f, scale_inv(byte));
    if (rg == 0) {
      uint8_t* s = o.scales + scale_at(col0 + 8 * l16 + j, mb, o.quads);
      s[0] = (uint8_t)byte;
      if (mb == nb - 1)
        for (int b = 1; b < 4 - (mb & 3); ++b) s[b] = 0;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int at = threadIdx.x + k * PACK_THREADS, c = at >> 3, pair = at & 7, key = (c >> 3) & 15;
    uint4 u = sh.t[c * 8 + (pair ^ (key >> 1))];
    if (key & 1) u = make_uint4(u.z, u.w, u.x, u.y);
    if (col0 + c < o.rows) *reinterpret_cast<uint4*>(o.codes + (long long)(col0 + c) * o.width + mb * TILE + pair * 16) = u;
  }
}

// ------------------------------------------------------------------------------------------------------------- pack
template <typename T, bool ROWS, bool COLS, bool SUMS>
__global__ void __launch_bounds__(PACK_THREADS) pack8_kernel(const T* __restrict__ x, long long ld, int M, int K, bool vec,
                                                            Side rows, Side cols, float* __restrict__ sums) {
  __shared__ __align__(16) TileShared sh;
  const int nkb = (K + TILE - 1) / TILE, nmb = (M + TILE - 1) / TILE;
  const int kb = blockIdx.x % nkb, mb = blockIdx.x / nkb;
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const int row0 = mb * TILE, c = kb * TILE + 8 * l16, n = max(0, min(8, K - c));
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = row0 + 8 * rg + i;
    load8<T>(x + (long long)r * ld + c, r < M ? n : 0, vec, v[i]);
  }
  if constexpr (SUMS) {  // before anything becomes NaN
    float m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = ((v[0][j] + v[1][j]) + (v[2][j] + v[3][j])) + ((v[4][j] + v[5][j]) + (v[6][j] + v[7][j]));
      m[j] += __shfl_xor_sync(0xffffffffu, m[j], 16);
    }
    if ((rg & 1) == 0)
#pragma unroll
      for (int j = 0; j < 8; ++j) sh.part[rg >> 1][8 * l16 + j] = m[j];
    __syncthreads();
    if (threadIdx.x < TILE && kb * TILE + threadIdx.x < K) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) a += sh.part[w][threadIdx.x];
      sums[(long long)mb * K + kb * TILE + threadIdx.x] = a;
    }
  }
  if constexpr (ROWS) emit_rows(rows, v, row0, kb, nkb, rg, l16);
  if constexpr (COLS) emit_cols(cols, v, kb * TILE, mb, nmb, rg, l16, sh);
}

bool aligned16(const void* p, long long stride_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride_bytes & 15) == 0;
}
Side side(uint8_t* codes, uint8_t* scales, int rows, int along) {
  const int nb = (along + TILE - 1) / TILE;
  return Side{codes, scales, rows, (nb + 3) / 4, (long long)nb * TILE};
}

template <typename T>
cudaError_t pack_typed(const Pack8Params& p, cudaStream_t s) {
  const long long tiles = (long long)((p.K + TILE - 1) / TILE) * ((p.M + TILE - 1) / TILE);
  if (tiles >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool vec = p.K % 8 == 0 && aligned16(p.x, p.ld * (long long)sizeof(T));
  const Side r = side(p.codes, p.scales, p.M, p.K), c = side(p.codes_t, p.scales_t, p.K, p.M);
  const T* x = static_cast<const T*>(p.x);
#define PACK(R, C, S) pack8_kernel<T, R, C, S><<<(int)tiles, PACK_THREADS, 0, s>>>(x, p.ld, p.M, p.K, vec, r, c, p.sums)
  if (p.codes != nullptr && p.codes_t != nullptr) {
    if (p.sums != nullptr) PACK(true, true, true);
    else PACK(true, true, false);
  } else if (p.codes != nullptr) {
    PACK(true, false, false);
  } else if (p.sums != nullptr) {
    PACK(false, true, true);
  } else {
    PACK(false, true, false);
  }
#undef PACK
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------------ column sums
// 32 columns x 8 runs of tiles; each run in order, then the runs in order
__global__ void __launch_bounds__(256) colsum_kernel(const float* __restrict__ sums, int T, int K, float* __restrict__ out,
                                                     bool add) {
  __shared__ float part[8][32];
  const int k = blockIdx.x * 32 + threadIdx.x, run = threadIdx.y;
  const int per = (T + 7) / 8, lo = run * per, hi = min(T, lo + per);
  float a = 0.f;
  if (k < K) {
#pragma unroll 8
    for (int t = lo; t < hi; ++t) a += sums[(long long)t * K + k];
  }
  part[run][threadIdx.x] = a;
  __syncthreads();
  if (run == 0 && k < K) {
#pragma unroll
    for (int w = 1; w < 8; ++w) a += part[w][threadIdx.x];
    out[k] = add ? out[k] + a : a;
  }
}

// ----------------------------------------------------------------------------------------------------------- unpack
template <typename T>
__global__ void __launch_bounds__(256) unpack8_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                      int R, int K, long long width, int quads, T* __restrict__ out,
                                                      long long ldo, bool vec) {
  const int per = (int)(width / 8);  // groups of eight codes of a row
  const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (at >= (long long)R * per) return;
  const int r = (int)(at / per), c = (int)(at % per) * 8;
  if (c >= K) return;
  float f[8];
  values8(*reinterpret_cast<const uint2*>(codes + (long long)r * width + c), scale_of(scales[scale_at(r, c >> 7, quads)]), f);
  store8<T>(out + (long long)r * ldo + c, min(8, K - c), vec, f);
}

template <typename T>
cudaError_t unpack_typed(const uint8_t* codes, const uint8_t* scales, int R, int K, void* out, long long ldo, cudaStream_t s) {
  const int nb = (K + TILE - 1) / TILE;
  const long long groups = (long long)R * nb * (TILE / 8), blocks = (groups + 255) / 256;
  if (blocks >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool vec = K % 8 == 0 && aligned16(out, ldo * (long long)sizeof(T));
  unpack8_kernel<T><<<(int)blocks, 256, 0, s>>>(codes, scales, R, K, (long long)nb * TILE, (nb + 3) / 4,
                                               static_cast<T*>(out), ldo, vec);
  return cudaGetLastError();
}

// ----------------------------------------------------------------------------------------------------------- SwiGLU
// g = silu(a) b = a b / (1 + exp(-a)): __expf is within 2 ulp + 2^-21 |a| of exp, which rounding to 16 bits hides; for
// fp32 results expf is used
template <bool FINE>
__device__ __forceinline__ float sigmoid(float a) {
  const float e = FINE ? expf(-a) : __expf(-a);
  return FINE ? 1.f / (1.f + e) : __fdividef(1.f, 1.f + e);
}

// G: g in ab's type; Q: g in 8 bits (Side g8, and g8t where its codes are given). The checkpoint's blocks are those of a
// [M, 2 Hp] matrix: a's first, then b's.
template <typename T, bool G, bool Q>
__global__ void __launch_bounds__(PACK_THREADS) swiglu8_fwd_kernel(const T* __restrict__ ab, long long ld, int M, int H,
                                                                  bool vec, bool vec_g, T* __restrict__ g, Side ck, Side g8,
                                                                  Side g8t) {
  __shared__ __align__(16) TileShared sh;
  const int nhb = (H + TILE - 1) / TILE, nmb = (M + TILE - 1) / TILE;
  const int hb = blockIdx.x % nhb, mb = blockIdx.x / nhb;
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const int row0 = mb * TILE, c = hb * TILE + 8 * l16, n = max(0, min(8, H - c));
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = row0 + 8 * rg + i, nr = r < M ? n : 0;
    float a[8], b[8];
    const T* p = ab + (long long)r * ld + c;
    load8<T>(p, nr, vec, a);
    load8<T>(p + H, nr, vec, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = a[j] * sigmoid<sizeof(T) == 4>(a[j]) * b[j];
    if constexpr (G) store8<T>(g + (long long)r * H + c, nr, vec_g, v[i]);
    if (ck.codes != nullptr) {
      const int ba = scale_byte(max16(finite_top8(a))), bb = scale_byte(max16(finite_top8(b)));
      if (r < M) {
        uint8_t* d = ck.codes + (long long)r * ck.width + c;
        *reinterpret_cast<uint2*>(d) = codes8(a, scale_inv(ba));
        *reinterpret_cast<uint2*>(d + (long long)nhb * TILE) = codes8(b, scale_inv(bb));
      }
      if (l16 == 0) {
        ck.scales[scale_at(r, hb, ck.quads)] = (uint8_t)ba;
        uint8_t* s = ck.scales + scale_at(r, nhb + hb, ck.quads);
        s[0] = (uint8_t)bb;
        if (hb == nhb - 1)
          for (int k = 1; k < 4 - ((nhb + hb) & 3); ++k) s[k] = 0;
      }
    }
  }
  if constexpr (Q) {
    emit_rows(g8, v, row0, hb, nhb, rg, l16);
    if (g8t.codes != nullptr) emit_cols(g8t, v, hb * TILE, mb, nmb, rg, l16, sh);
  }
}

// dg, Q(a), Q(b) -> da = dg b s (1 + a (1 - s)), db = dg a s with s = sigmoid(a). D: in dg's type; Q: in 8 bits, both
// ways. One half after the other, so that a thread holds one tile's values.
template <typename T, bool D, bool Q>
__global__ void __launch_bounds__(PACK_THREADS) swiglu8_bwd_kernel(const T* __restrict__ dg, long long ld, int M, int H,
                                                                  bool vec, bool vec_d, T* __restrict__ dab, Side ck,
                                                                  Side d8, Side d8t) {
  __shared__ __align__(16) TileShared sh;
  const int nhb = (H + TILE - 1) / TILE, nmb = (M + TILE - 1) / TILE;
  const int hb = blockIdx.x % nhb, mb = blockIdx.x / nhb;
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const int row0 = mb * TILE, c = hb * TILE + 8 * l16, n = max(0, min(8, H - c));
  uint2 ca[8], cb[8];
  float dgv[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = row0 + 8 * rg + i;
    load8<T>(dg + (long long)r * ld + c, r < M ? n : 0, vec, dgv[i]);
    ca[i] = cb[i] = make_uint2(0u, 0u);
    if (r < M) {
      const uint8_t* s = ck.codes + (long long)r * ck.width + c;
      ca[i] = *reinterpret_cast<const uint2*>(s);
      cb[i] = *reinterpret_cast<const uint2*>(s + (long long)nhb * TILE);
    }
  }
  float v[8][8];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = row0 + 8 * rg + i;
      float a[8], b[8];
      values8(ca[i], scale_of(ck.scales[scale_at(r, hb, ck.quads)]), a);
      if (half == 0) values8(cb[i], scale_of(ck.scales[scale_at(r, nhb + hb, ck.quads)]), b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float s = sigmoid<sizeof(T) == 4>(a[j]);
        v[i][j] = half == 0 ? dgv[i][j] * b[j] * s * (1.f + a[j] * (1.f - s)) : dgv[i][j] * a[j] * s;
      }
      if constexpr (D) store8<T>(dab + (long long)r * 2 * H + half * H + c, r < M ? n : 0, vec_d, v[i]);
    }
    if constexpr (Q) {
      emit_rows(d8, v, row0, half * nhb + hb, 2 * nhb, rg, l16);
      emit_cols(d8t, v, half * H + hb * TILE, mb, nmb, rg, l16, sh);
    }
  }
}

template <typename T>
cudaError_t swiglu_fwd_typed(const Swiglu8Params& p, cudaStream_t s) {
  const int nhb = (p.H + TILE - 1) / TILE;
  const long long tiles = (long long)nhb * ((p.M + TILE - 1) / TILE);
  if (tiles >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool vec = p.H % 8 == 0 && aligned16(p.ab, p.ld * (long long)sizeof(T));
  const bool vec_g = p.H % 8 == 0 && aligned16(p.g, 0);
  const Side ck = side(p.ck, p.ck_scales, p.M, 2 * nhb * TILE), g8 = side(p.g8, p.g8_scales, p.M, p.H),
             g8t = side(p.g8t, p.g8t_scales, p.H, p.M);
  const T* ab = static_cast<const T*>(p.ab);
  T* g = static_cast<T*>(p.g);
  if (p.g8 != nullptr)
    swiglu8_fwd_kernel<T, false, true><<<(int)tiles, PACK_THREADS, 0, s>>>(ab, p.ld, p.M, p.H, vec, vec_g, g, ck, g8, g8t);
  else
    swiglu8_fwd_kernel<T, true, false><<<(int)tiles, PACK_THREADS, 0, s>>>(ab, p.ld, p.M, p.H, vec, vec_g, g, ck, g8, g8t);
  return cudaGetLastError();
}
template <typename T>
cudaError_t swiglu_bwd_typed(const Swiglu8BwdParams& p, cudaStream_t s) {
  const int nhb = (p.H + TILE - 1) / TILE;
  const long long tiles = (long long)nhb * ((p.M + TILE - 1) / TILE);
  if (tiles >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool vec = p.H % 8 == 0 && aligned16(p.dg, p.ld * (long long)sizeof(T));
  const bool vec_d = p.H % 8 == 0 && aligned16(p.dab, 0);
  const Side ck = side(const_cast<uint8_t*>(p.ck), const_cast<uint8_t*>(p.ck_scales), p.M, 2 * nhb * TILE),
             d8 = side(p.d8, p.d8_scales, p.M, 2 * p.H), d8t = side(p.d8t, p.d8t_scales, 2 * p.H, p.M);
  const T* dg = static_cast<const T*>(p.dg);
  T* dab = static_cast<T*>(p.dab);
  if (p.d8 != nullptr)
    swiglu8_bwd_kernel<T, false, true><<<(int)tiles, PACK_THREADS, 0, s>>>(dg, p.ld, p.M, p.H, vec, vec_d, dab, ck, d8, d8t);
  else
    swiglu8_bwd_kernel<T, true, false><<<(int)tiles, PACK_THREADS, 0, s>>>(dg, p.ld, p.M, p.H, vec, vec_d, dab, ck, d8, d8t);
  return cudaGetLastError();
}

// --------------------------------------------------------------------------------------------------------- few rows
// y [M, N] = Q(x) W^T + bias for at most 16 rows of x (tokens of a serving step). Reading W bounds it (N Kp bytes): one
// launch, x is packed where it is used. A CTA owns 16 rows of W, its warps every eighth block of 128; all of a warp's
// loads of a block are 16 bytes per lane and independent. The products run on mma.m16n8k32 (W rows x tokens); the order
// of k inside a block is free, so a lane's 16 consecutive bytes serve as its operand words of two instructions, for W
// and for x alike. A block's sum is scaled in fp32, the warps' sums are added in order.
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int NT>  // NT: groups of eight rows of x
__global__ void __launch_bounds__(256) few_rows_kernel(const FewRowsParams p, bool vec) {
  __shared__ float part[8][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warps = blockDim.x >> 5;
  const int nb = (p.K + TILE - 1) / TILE, quads = (nb + 3) / 4;
  const long long width = (long long)nb * TILE;
  const int n0 = blockIdx.x * 16;
  const T* x = static_cast<const T*>(p.x);
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  for (int kb = warp; kb < nb; kb += warps) {
    uint4 w[2][2];  // [row g, g + 8][half of the block]
    float ws[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int n = n0 + g + 8 * r;
      w[r][0] = w[r][1] = make_uint4(0u, 0u, 0u, 0u);
      ws[r] = 0.f;
      if (n < p.N) {
        const uint8_t* src = p.codes + n * width + kb * TILE + 16 * t;
        w[r][0] = __ldg(reinterpret_cast<const uint4*>(src));
        w[r][1] = __ldg(reinterpret_cast<const uint4*>(src + 64));
        ws[r] = scale_of(__ldg(p.scales + scale_at(n, kb, quads)));
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int m = 8 * i + g;
      float f[4][8];  // columns 16 t .. + 15 and 64 + 16 t .. + 15 of the block
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int c = kb * TILE + (h >> 1) * 64 + 16 * t + (h & 1) * 8;
        load8<T>(x + m * p.ldx + c, m < p.M ? max(0, min(8, p.K - c)) : 0, vec, f[h]);
      }
      float top = fmaxf(fmaxf(finite_top8(f[0]), finite_top8(f[1])), fmaxf(finite_top8(f[2]), finite_top8(f[3])));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int byte = scale_byte(top);
      const float inv = scale_inv(byte);
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 lo = codes8(f[2 * h], inv), hi = codes8(f[2 * h + 1], inv);
        mma_e4m3(d, w[0][h].x, w[1][h].x, w[0][h].y, w[1][h].y, lo.x, lo.y);
        mma_e4m3(d, w[0][h].z, w[1][h].z, w[0][h].w, w[1][h].w, hi.x, hi.y);
      }
      // d: rows g, g + 8 of W, tokens 2 t, 2 t + 1, whose scales their own lanes hold
      const float s = scale_of(byte);
      const float s0 = __shfl_sync(0xffffffffu, s, 8 * t), s1 = __shfl_sync(0xffffffffu, s, 8 * t + 4);
      acc[i][0] += d[0] * s0 * ws[0];
      acc[i][1] += d[1] * s1 * ws[0];
      acc[i][2] += d[2] * s0 * ws[1];
      acc[i][3] += d[3] * s1 * ws[1];
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    part[warp][g][8 * i + 2 * t] = acc[i][0];
    part[warp][g][8 * i + 2 * t + 1] = acc[i][1];
    part[warp][g + 8][8 * i + 2 * t] = acc[i][2];
    part[warp][g + 8][8 * i + 2 * t + 1] = acc[i][3];
  }
  __syncthreads();
  T* y = static_cast<T*>(p.y);
  for (int at = threadIdx.x; at < 16 * 8 * NT; at += blockDim.x) {
    const int m = at >> 4, r = at & 15, n = n0 + r;
    if (m >= p.M || n >= p.N) continue;
    float v = 0.f;
    for (int w = 0; w < warps; ++w) v += part[w][r][m];
    if (p.bias != nullptr) v += p.bias[n];
    y[(long long)m * p.N + n] = from_f<T>(v);
  }
}

template <typename T>
cudaError_t few_rows_typed(const FewRowsParams& p, cudaStream_t s) {
  const int nb = (p.K + TILE - 1) / TILE, warps = std::min(8, nb);
  const bool vec = p.K % 8 == 0 && aligned16(p.x, p.ldx * (long long)sizeof(T));
  const int grid = (p.N + 15) / 16;
  if (p.M <= 8) few_rows_kernel<T, 1><<<grid, warps * 32, 0, s>>>(p, vec);
  else few_rows_kernel<T, 2><<<grid, warps * 32, 0, s>>>(p, vec);
  return cudaGetLastError();
}

template <typename F>
cudaError_t by_type(int elem, F&& f) {
  switch (elem) {
    case ELEM_BF16: return f(__nv_bfloat16());
    case ELEM_F16: return f(__half());
    case ELEM_F32: return f(float());
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t pack8_launch(const Pack8Params& p, int elem, cudaStream_t s) {
  if (p.M <= 0 || p.K <= 0 || (p.codes == nullptr && p.codes_t == nullptr) || (p.sums != nullptr && p.codes_t == nullptr))
    return cudaErrorInvalidValue;
  return by_type(elem, [&](auto t) { return pack_typed<decltype(t)>(p, s); });
}
cudaError_t colsum_launch(const float* sums, int T, int K, float* out, bool add, cudaStream_t s) {
  if (T <= 0 || K <= 0) return cudaErrorInvalidValue;
  colsum_kernel<<<(K + 31) / 32, dim3(32, 8), 0, s>>>(sums, T, K, out, add);
  return cudaGetLastError();
}
cudaError_t unpack8_launch(const uint8_t* codes, const uint8_t* scales, int R, int K, void* out, long long ldo, int elem,
                           cudaStream_t s) {
  if (R <= 0 || K <= 0) return cudaErrorInvalidValue;
  return by_type(elem, [&](auto t) { return unpack_typed<decltype(t)>(codes, scales, R, K, out, ldo, s); });
}
cudaError_t few_rows_launch(const FewRowsParams& p, int elem, cudaStream_t s) {
  if (p.M <= 0 || p.M > kFewRows || p.N <= 0 || p.K <= 0) return cudaErrorInvalidValue;
  return by_type(elem, [&](auto t) { return few_rows_typed<decltype(t)>(p, s); });
}
cudaError_t swiglu8_fwd_launch(const Swiglu8Params& p, int elem, cudaStream_t s) {
  if (p.M <= 0 || p.H <= 0 || (p.g == nullptr) == (p.g8 == nullptr) || (p.g8t != nullptr && p.g8 == nullptr))
    return cudaErrorInvalidValue;
  return by_type(elem, [&](auto t) { return swiglu_fwd_typed<decltype(t)>(p, s); });
}
cudaError_t swiglu8_bwd_launch(const Swiglu8BwdParams& p, int elem, cudaStream_t s) {
  if (p.M <= 0 || p.H <= 0 || p.ck == nullptr || (p.dab == nullptr) == (p.d8 == nullptr) ||
      (p.d8 != nullptr && (p.d8t == nullptr || p.H % TILE != 0)))
    return cudaErrorInvalidValue;
  return by_type(elem, [&](auto t) { return swiglu_bwd_typed<decltype(t)>(p, s); });
}

}  // namespace tgo

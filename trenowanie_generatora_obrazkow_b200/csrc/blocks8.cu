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
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "block_ops.h"
#include "blocks8.cuh"
#include "blocks8.h"
#include "common.cuh"
#include "vec.cuh"

namespace tgo {

int num_sms();  // gemm.cu

namespace {

constexpr int PACK_THREADS = 256;

// ------------------------------------------------------------------------------------------------------------ loads
// Eight values of a row: fp32 as four pairs; 16-bit types as they are stored, unpacked where they are used (half the
// registers, and maxima of two values at a time).
template <typename T>
struct Eight {
  static constexpr bool WIDE = sizeof(T) == 4;
  using Two = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  uint32_t u[WIDE ? 8 : 4];
  __device__ __forceinline__ float2 pair(int w) const {
    if constexpr (WIDE) return make_float2(__uint_as_float(u[2 * w]), __uint_as_float(u[2 * w + 1]));
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return make_float2(__uint_as_float(u[w] << 16), __uint_as_float(u[w] & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&u[w]));
  }
  __device__ __forceinline__ void set(int w, float2 v) {
    if constexpr (WIDE) {
      u[2 * w] = __float_as_uint(v.x), u[2 * w + 1] = __float_as_uint(v.y);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(v.x, v.y);
      u[w] = *reinterpret_cast<const uint32_t*>(&t);
    } else {
      const __half2 t = __floats2half2_rn(v.x, v.y);
      u[w] = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
  // n (0 to 8) elements of a row; 16-byte loads where vec (the address is aligned and n is 0 or 8)
  __device__ __forceinline__ void load(const T* p, int n, bool vec) {
#pragma unroll
    for (int i = 0; i < (WIDE ? 8 : 4); ++i) u[i] = 0u;
    if (vec) {
      if (n > 0) {
#pragma unroll
        for (int i = 0; i < (WIDE ? 2 : 1); ++i) {
          const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i);
          u[4 * i] = q.x, u[4 * i + 1] = q.y, u[4 * i + 2] = q.z, u[4 * i + 3] = q.w;
        }
      }
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) set(w, make_float2(2 * w < n ? to_f(p[2 * w]) : 0.f, 2 * w + 1 < n ? to_f(p[2 * w + 1]) : 0.f));
    }
  }
  __device__ __forceinline__ void fetch(const T* p) {  // aligned shared memory
#pragma unroll
    for (int i = 0; i < (WIDE ? 2 : 1); ++i) {
      const uint4 q = reinterpret_cast<const uint4*>(p)[i];
      u[4 * i] = q.x, u[4 * i + 1] = q.y, u[4 * i + 2] = q.z, u[4 * i + 3] = q.w;
    }
  }
  __device__ __forceinline__ void store(T* p, int n, bool vec) const {
    if (vec) {
      if (n <= 0) return;
#pragma unroll
      for (int i = 0; i < (WIDE ? 2 : 1); ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) p[j] = from_f<T>((j & 1) ? pair(j >> 1).y : pair(j >> 1).x);
    }
  }
  // magnitudes: NaN passes over, an infinity shows
  static __device__ __forceinline__ uint32_t top2(uint32_t a, uint32_t b) {
    const Two r = __hmax2(__habs2(*reinterpret_cast<const Two*>(&a)), __habs2(*reinterpret_cast<const Two*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float2 widen(uint32_t v) {
    Eight e;
    e.u[0] = v;
    return e.pair(0);
  }
  __device__ __forceinline__ float top() const {
    if constexpr (WIDE) {
      const float2 a = pair(0), b = pair(1), c = pair(2), d = pair(3);
      return fmaxf(max3(max3(fabsf(a.x), fabsf(a.y), fabsf(b.x)), fabsf(b.y), fabsf(c.x)), max3(fabsf(c.y), fabsf(d.x), fabsf(d.y)));
    } else {
      const float2 m = widen(top2(top2(u[0], u[1]), top2(u[2], u[3])));
      return fmaxf(m.x, m.y);
    }
  }
  __device__ __forceinline__ void drop_infinities() {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float2 v = pair(w);
      if (fabsf(v.x) == INFINITY) v.x = NAN;
      if (fabsf(v.y) == INFINITY) v.y = NAN;
      set(w, v);
    }
  }
};

template <typename T>
__device__ __forceinline__ uint2 codes8(const Eight<T>& v, float inv) {
  const float2 k = make_float2(inv, inv);
  return make_uint2(codes4(mul2(v.pair(0), k), mul2(v.pair(1), k)), codes4(mul2(v.pair(2), k), mul2(v.pair(3), k)));
}

// the largest finite magnitude of each row; infinities become NaN (one test for all rows)
template <typename T, int R>
__device__ __forceinline__ void finite_tops(Eight<T> (&v)[R], float (&m)[R]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) top = fmaxf(top, m[i] = v[i].top());
  if (top == INFINITY) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      v[i].drop_infinities();
      m[i] = v[i].top();
    }
  }
}

// ------------------------------------------------------------------------------------------------------- tile output
struct TileShared {
  float part[8][TILE];
  float inv[TILE];
  uint4 t[TILE * TILE / 16];  // transposed codes: column c's eight bytes of rows 8 i .. at c * 16 + (i ^ (c / 8 % 16))
};

// The maxima m of the R rows from r0 on over this thread's columns -> 2^-e of each row over the 16 lanes that share it; the
// scale bytes are written (also of rows past `rows` in their atom). Each exchange halves the rows that a lane still carries:
// 8 shuffles for 8 rows instead of 32.
template <int R>
__device__ __forceinline__ void row_scales(const float (&m)[R], uint8_t* scales, int r0, int kb, int nb, int quads, int rows,
                                           float (&inv)[R]) {
  static_assert(R == 2 || R == 4 || R == 8, "rows of a thread");
  constexpr int KEPT = R == 8 ? 1 : R == 4 ? 2 : 3;  // lane bits below those that choose the row
  const int lane = threadIdx.x & 31;
  float a[R];
#pragma unroll
  for (int i = 0; i < R; ++i) a[i] = m[i];
#pragma unroll
  for (int n = R / 2, bit = 8; bit > 0; n /= 2, bit /= 2) {
    if (n > 0) {
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const float keep = (lane & bit) ? a[n + k] : a[k], send = (lane & bit) ? a[k] : a[n + k];
        a[k] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, bit));
      }
    } else {
      a[0] = fmaxf(a[0], __shfl_xor_sync(0xffffffffu, a[0], bit));
    }
  }
  const int byte = scale_byte(a[0]);
  const float mine = scale_inv(byte);
#pragma unroll
  for (int i = 0; i < R; ++i) inv[i] = __shfl_sync(0xffffffffu, mine, (lane & 16) | (i << KEPT));
  if ((lane & ((1 << KEPT) - 1)) == 0) {
    const int r = r0 + ((lane & 15) >> KEPT);
    if (r < ((rows + TILE - 1) & ~(TILE - 1))) {
      uint8_t* s = scales + scale_at(r, kb, quads);
      s[0] = (uint8_t)byte;
      if (kb == nb - 1)
        for (int k = 1; k < 4 - (kb & 3); ++k) s[k] = 0;
    }
  }
}

// Packs the tile whose rows row0 + 8 rg + i and columns col0 + 8 l16 + j the thread holds in v[i]: blocks along the rows
// (block kb of nkb) and / or along the columns as rows of the transposed form (block mb of nmb).
template <bool ROWS, bool COLS, typename T>
__device__ __forceinline__ void emit(Eight<T> (&v)[8], const Side& r, const Side& c, int row0, int col0, int kb, int nkb, int mb,
                                     int nmb, TileShared& sh) {
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  float m[8];
  finite_tops(v, m);
  if constexpr (COLS) {
    float2 t[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (Eight<T>::WIDE) {
        t[w] = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float2 p = v[i].pair(w), q = v[i + 1].pair(w);
          t[w] = make_float2(max3(t[w].x, fabsf(p.x), fabsf(q.x)), max3(t[w].y, fabsf(p.y), fabsf(q.y)));
        }
      } else {
        uint32_t a = Eight<T>::top2(v[0].u[w], v[1].u[w]);
#pragma unroll
        for (int i = 2; i < 8; ++i) a = Eight<T>::top2(a, v[i].u[w]);
        t[w] = Eight<T>::widen(a);
      }
      t[w].x = fmaxf(t[w].x, __shfl_xor_sync(0xffffffffu, t[w].x, 16));
      t[w].y = fmaxf(t[w].y, __shfl_xor_sync(0xffffffffu, t[w].y, 16));
    }
    if ((rg & 1) == 0) {
      *reinterpret_cast<float4*>(&sh.part[rg >> 1][8 * l16]) = make_float4(t[0].x, t[0].y, t[1].x, t[1].y);
      *reinterpret_cast<float4*>(&sh.part[rg >> 1][8 * l16 + 4]) = make_float4(t[2].x, t[2].y, t[3].x, t[3].y);
    }
    __syncthreads();
    if (threadIdx.x < TILE) {
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) top = fmaxf(top, sh.part[w][threadIdx.x]);
      const int byte = scale_byte(top);
      sh.inv[threadIdx.x] = scale_inv(byte);
      uint8_t* s = c.scales + scale_at(col0 + threadIdx.x, mb, c.quads);
      s[0] = (uint8_t)byte;
      if (mb == nmb - 1)
        for (int k = 1; k < 4 - (mb & 3); ++k) s[k] = 0;
    }
  }
  if constexpr (ROWS) {
    float inv[8];
    row_scales(m, r.scales, row0 + 8 * rg, kb, nkb, r.quads, r.rows, inv);
    uint8_t* d = r.codes + (long long)(row0 + 8 * rg) * r.width + kb * TILE + 8 * l16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint2 q = codes8(v[i], inv[i]);
      if (row0 + 8 * rg + i < r.rows) *reinterpret_cast<uint2*>(d) = q;
      d += r.width;
    }
  }
  if constexpr (COLS) {
    __syncthreads();
    uint2* t = reinterpret_cast<uint2*>(sh.t);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 k = *reinterpret_cast<const float2*>(&sh.inv[8 * l16 + 2 * w]);
      float2 f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = mul2(v[i].pair(w), k);
      t[(8 * l16 + 2 * w) * 16 + (rg ^ l16)] =
          make_uint2(codes2(f[0].x, f[1].x) | codes2(f[2].x, f[3].x) << 16, codes2(f[4].x, f[5].x) | codes2(f[6].x, f[7].x) << 16);
      t[(8 * l16 + 2 * w + 1) * 16 + (rg ^ l16)] =
          make_uint2(codes2(f[0].y, f[1].y) | codes2(f[2].y, f[3].y) << 16, codes2(f[4].y, f[5].y) | codes2(f[6].y, f[7].y) << 16);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = threadIdx.x + k * PACK_THREADS, col = at >> 3, pair = at & 7, key = (col >> 3) & 15;
      uint4 u = sh.t[col * 8 + (pair ^ (key >> 1))];
      if (key & 1) u = make_uint4(u.z, u.w, u.x, u.y);
      if (col0 + col < c.rows) *reinterpret_cast<uint4*>(c.codes + (long long)(col0 + col) * c.width + mb * TILE + pair * 16) = u;
    }
  }
}

// ------------------------------------------------------------------------------------------------------------- pack
template <typename T, bool ROWS, bool COLS, bool SUMS>
__device__ __forceinline__ void pack_tile(const T* __restrict__ x, long long ld, int M, int K, bool vec, const Side& rows,
                                          const Side& cols, float* __restrict__ sums, int tile, TileShared& sh) {
  const int nkb = (K + TILE - 1) / TILE, nmb = (M + TILE - 1) / TILE;
  const int kb = tile % nkb, mb = tile / nkb;
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const int row0 = mb * TILE, c = kb * TILE + 8 * l16, n = max(0, min(8, K - c));
  Eight<T> v[8];
  const T* p = x + (long long)(row0 + 8 * rg) * ld + c;
#pragma unroll
  for (int i = 0; i < 8; ++i, p += ld) v[i].load(p, row0 + 8 * rg + i < M ? n : 0, vec);
  if constexpr (SUMS) {  // before anything becomes NaN
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float2 a = v[0].pair(w);
#pragma unroll
      for (int i = 1; i < 8; ++i) a.x += v[i].pair(w).x, a.y += v[i].pair(w).y;
      a.x += __shfl_xor_sync(0xffffffffu, a.x, 16);
      a.y += __shfl_xor_sync(0xffffffffu, a.y, 16);
      if ((rg & 1) == 0) *reinterpret_cast<float2*>(&sh.part[rg >> 1][8 * l16 + 2 * w]) = a;
    }
    __syncthreads();
    if (threadIdx.x < TILE && kb * TILE + threadIdx.x < K) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) a += sh.part[w][threadIdx.x];
      sums[(long long)mb * K + kb * TILE + threadIdx.x] = a;
    }
    __syncthreads();
  }
  emit<ROWS, COLS, T>(v, rows, cols, row0, kb * TILE, kb, nkb, mb, nmb, sh);
}
template <typename T, bool ROWS, bool COLS, bool SUMS>
__global__ void __launch_bounds__(PACK_THREADS, sizeof(T) == 4 ? 2 : 3)
    pack8_kernel(const T* __restrict__ x, long long ld, int M, int K, bool vec, Side rows, Side cols, float* __restrict__ sums) {
  __shared__ __align__(16) TileShared sh;
  pack_tile<T, ROWS, COLS, SUMS>(x, ld, M, K, vec, rows, cols, sums, blockIdx.x, sh);
}
// tiles of several tensors, of any types
struct PackJobs {
  struct {
    const void* x;
    long long ld;
    int M, K, elem, first;  // first: the tensor's first tile
    bool vec;
    Side rows, cols;
  } job[3];
  int n;
};
__global__ void __launch_bounds__(PACK_THREADS, 2) pack8_jobs_kernel(const __grid_constant__ PackJobs p) {
  __shared__ __align__(16) TileShared sh;
  int k = 0;
  while (k + 1 < p.n && (int)blockIdx.x >= p.job[k + 1].first) ++k;
  const auto& j = p.job[k];
  const int tile = blockIdx.x - j.first;
  auto run = [&](auto t) {
    using T = decltype(t);
    const T* x = static_cast<const T*>(j.x);
    if (j.cols.codes != nullptr) pack_tile<T, true, true, false>(x, j.ld, j.M, j.K, j.vec, j.rows, j.cols, nullptr, tile, sh);
    else pack_tile<T, true, false, false>(x, j.ld, j.M, j.K, j.vec, j.rows, j.cols, nullptr, tile, sh);
  };
  if (j.elem == ELEM_BF16) run(__nv_bfloat16());
  else if (j.elem == ELEM_F16) run(__half());
  else run(float());
}

bool aligned16(const void* p, long long stride_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride_bytes & 15) == 0;
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
// a thread: 16 codes of a row
template <typename T>
__global__ void __launch_bounds__(256) unpack8_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                      int R, int K, int width, int quads, T* __restrict__ out,
                                                      long long ldo, bool vec) {
  const int per = width / 16;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const int r = (int)(at / per), c = (int)(at - (long long)r * per) * 16;
  if (at >= (long long)R * per || c >= K) return;
  const uint4 q = __ldg(reinterpret_cast<const uint4*>(codes + (long long)r * width + c));
  const float k = scale_of(__ldg(scales + scale_at(r, c >> 7, quads)));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float2 f[4];
    values8(h == 0 ? make_uint2(q.x, q.y) : make_uint2(q.z, q.w), k, f);
    Eight<T> e;
#pragma unroll
    for (int w = 0; w < 4; ++w) e.set(w, f[w]);
    e.store(out + (long long)r * ldo + c + 8 * h, max(0, min(8, K - c - 8 * h)), vec);
  }
}

template <typename T>
cudaError_t unpack_typed(const uint8_t* codes, const uint8_t* scales, int R, int K, void* out, long long ldo, cudaStream_t s) {
  const int nb = (K + TILE - 1) / TILE;
  const long long groups = (long long)R * nb * (TILE / 16), blocks = (groups + 255) / 256;
  if (blocks >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool vec = K % 8 == 0 && aligned16(out, ldo * (long long)sizeof(T));
  unpack8_kernel<T><<<(int)blocks, 256, 0, s>>>(codes, scales, R, K, nb * TILE, (nb + 3) / 4, static_cast<T*>(out), ldo, vec);
  return cudaGetLastError();
}

// ----------------------------------------------------------------------------------------------------------- SwiGLU
// g in ab's type, the checkpoint of ab in 8 bits. Rows alone: a thread holds 8 columns of ROW_R rows (two: enough warps to keep
// the memory busy; at 32768 x 5504 the backward took 265 us with four, 212 with two; 219 with sigmoids in two factors). The
// checkpoint's blocks are those of a [M, 2 Hp] matrix: a's first, then b's. Rows past the last are read as the last one and not
// written.
constexpr int ROW_R = 2;
template <typename T, bool VEC, bool CK>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 4)
    swiglu8_fwd_kernel(const T* __restrict__ ab, long long ld, int M, int H, bool vec_g, T* __restrict__ g, Side ck) {
  const int nhb = (H + TILE - 1) / TILE;
  const int hb = blockIdx.x % nhb, l16 = threadIdx.x & 15;
  const int r0 = (blockIdx.x / nhb) * 16 * ROW_R + (threadIdx.x >> 4) * ROW_R;
  const int c = hb * TILE + 8 * l16, n = max(0, min(8, H - c));
  Eight<T> a[ROW_R], b[ROW_R];
#pragma unroll
  for (int i = 0; i < ROW_R; ++i) {
    const T* p = ab + (long long)min(r0 + i, M - 1) * ld + c;
    a[i].load(p, n, VEC);
    b[i].load(p + H, n, VEC);
  }
#pragma unroll
  for (int i = 0; i < ROW_R; ++i) {
    Eight<T> o;
#pragma unroll
    for (int w = 0; w < 4; ++w) o.set(w, swiglu<sizeof(T) == 4>(a[i].pair(w), b[i].pair(w)));
    if (r0 + i < M) o.store(g + (long long)(r0 + i) * H + c, n, vec_g);
  }
  if constexpr (CK) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Eight<T>(&v)[ROW_R] = h == 0 ? a : b;
      float m[ROW_R], inv[ROW_R];
      finite_tops(v, m);
      row_scales(m, ck.scales, r0, h * nhb + hb, 2 * nhb, ck.quads, ck.rows, inv);
      uint8_t* d = ck.codes + (long long)r0 * ck.width + (long long)h * nhb * TILE + c;
#pragma unroll
      for (int i = 0; i < ROW_R; ++i, d += ck.width)
        if (r0 + i < M) *reinterpret_cast<uint2*>(d) = codes8(v[i], inv[i]);
    }
  }
}

// dg, Q(a), Q(b) -> [da | db] in dg's type: da = dg b s (1 + a (1 - s)), db = dg a s with s = sigmoid(a)
template <bool FINE>
__device__ __forceinline__ void swiglu_grad(float2 a, float2 b, float2 dg, float2& da, float2& db) {
  float2 p, q;
  sigmoid<FINE>(a.x, p.x, q.x);
  sigmoid<FINE>(a.y, p.y, q.y);
  const float2 one = make_float2(1.f, 1.f), u = fma2(a, fma2(make_float2(-p.x, -p.y), q, one), one), t = mul2(dg, p);
  da = mul2(mul2(t, mul2(b, q)), u);
  db = mul2(t, mul2(a, q));
}
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) swiglu8_bwd_kernel(const T* __restrict__ dg, long long ld, int M, int H, bool vec_d,
                                                          T* __restrict__ dab, Side ck) {
  const int nhb = (H + TILE - 1) / TILE;
  const int hb = blockIdx.x % nhb, l16 = threadIdx.x & 15;
  const int r0 = (blockIdx.x / nhb) * 16 * ROW_R + (threadIdx.x >> 4) * ROW_R;
  const int c = hb * TILE + 8 * l16, n = max(0, min(8, H - c));
  Eight<T> dv[ROW_R];
  uint2 ca[ROW_R], cb[ROW_R];
  float ka[ROW_R], kb[ROW_R];
#pragma unroll
  for (int i = 0; i < ROW_R; ++i) {
    const int r = min(r0 + i, M - 1);
    dv[i].load(dg + (long long)r * ld + c, n, VEC);
    const uint8_t* q = ck.codes + (long long)r * ck.width + c;
    ca[i] = __ldg(reinterpret_cast<const uint2*>(q));
    cb[i] = __ldg(reinterpret_cast<const uint2*>(q + (long long)nhb * TILE));
    ka[i] = scale_of(__ldg(ck.scales + scale_at(r, hb, ck.quads)));
    kb[i] = scale_of(__ldg(ck.scales + scale_at(r, nhb + hb, ck.quads)));
  }
#pragma unroll
  for (int i = 0; i < ROW_R; ++i) {
    float2 a[4], b[4];
    values8(ca[i], ka[i], a);
    values8(cb[i], kb[i], b);
    Eight<T> oa, ob;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float2 da, db;
      swiglu_grad<sizeof(T) == 4>(a[w], b[w], dv[i].pair(w), da, db);
      oa.set(w, da);
      ob.set(w, db);
    }
    if (r0 + i < M) {
      T* o = dab + (long long)(r0 + i) * 2 * H + c;
      oa.store(o, n, vec_d);
      ob.store(o + H, n, vec_d);
    }
  }
}

// ---- the forms of the MLP: everything that is written is in 8 bits, both ways where a weight's gradient wants it (the
// forward of 16-bit types has them in its product's epilogue but for few rows, which want g along the rows alone). One CTA of
// 512 threads per SM walks over tiles of 128 x 128; the tiles come by TMA, two ahead of the arithmetic (fp32: one), so no
// registers and no address arithmetic go into loads. A thread holds 8 columns of 4 rows; the backward holds da and db at once
// and takes each exponential once. What bounds them is the arithmetic: the backward executes 39 instructions an element
// (352 us at 32768 x 5504, 0.63 of a copy; issue slots 59 % used).
constexpr int QT_THREADS = 512, QT_R = 4;
template <typename T>
struct QtStages {
  static constexpr int N = sizeof(T) == 4 ? 1 : 2;
};
struct QtOut {  // transposed side of one tile: maxima of the 16 warps, 2^-e, codes
  float part[16][TILE];
  float inv[TILE];
  uint4 t[TILE * TILE / 16];  // column c's four bytes of rows 4 i .. at word c * 32 + (i ^ 2 (c / 8 % 16))
};

// rows of the tile into d: blocks along the columns
template <typename T>
__device__ __forceinline__ void qt_rows(Eight<T> (&v)[QT_R], const Side& o, int r0, int kb, int nkb, int l16) {
  float m[QT_R], inv[QT_R];
  finite_tops(v, m);
  row_scales(m, o.scales, r0, kb, nkb, o.quads, o.rows, inv);
  uint8_t* d = o.codes + (long long)r0 * o.width + kb * TILE + 8 * l16;
#pragma unroll
  for (int i = 0; i < QT_R; ++i, d += o.width)
    if (r0 + i < o.rows) *reinterpret_cast<uint2*>(d) = codes8(v[i], inv[i]);
}
__device__ __forceinline__ void qt_cols_part(Eight<float> (&v)[QT_R], QtOut& sh, int l16) {
  float2 t[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 a = v[0].pair(w), b = v[1].pair(w), c = v[2].pair(w), d = v[3].pair(w);
    t[w] = make_float2(fmaxf(max3(fabsf(a.x), fabsf(b.x), fabsf(c.x)), fabsf(d.x)),
                       fmaxf(max3(fabsf(a.y), fabsf(b.y), fabsf(c.y)), fabsf(d.y)));
    t[w].x = fmaxf(t[w].x, __shfl_xor_sync(0xffffffffu, t[w].x, 16));
    t[w].y = fmaxf(t[w].y, __shfl_xor_sync(0xffffffffu, t[w].y, 16));
  }
  if ((threadIdx.x & 16) == 0) {
    float* p = sh.part[threadIdx.x >> 5] + 8 * l16;
    *reinterpret_cast<float4*>(p) = make_float4(t[0].x, t[0].y, t[1].x, t[1].y);
    *reinterpret_cast<float4*>(p + 4) = make_float4(t[2].x, t[2].y, t[3].x, t[3].y);
  }
}
__device__ __forceinline__ void qt_cols_scale(QtOut& sh, int c, const Side& o, int col0, int mb, int nmb) {
  float top = 0.f;
#pragma unroll
  for (int w = 0; w < 16; w += 2) top = max3(top, sh.part[w][c], sh.part[w + 1][c]);
  const int byte = scale_byte(top);
  sh.inv[c] = scale_inv(byte);
  uint8_t* s = o.scales + scale_at(col0 + c, mb, o.quads);
  s[0] = (uint8_t)byte;
  if (mb == nmb - 1)
    for (int k = 1; k < 4 - (mb & 3); ++k) s[k] = 0;
}
__device__ __forceinline__ void qt_cols_codes(Eight<float> (&v)[QT_R], QtOut& sh, int l16) {
  uint32_t* t = reinterpret_cast<uint32_t*>(sh.t) + (8 * l16) * 32 + ((threadIdx.x >> 4) ^ (2 * l16));
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 k = *reinterpret_cast<const float2*>(&sh.inv[8 * l16 + 2 * w]);
    const float2 a = mul2(v[0].pair(w), k), b = mul2(v[1].pair(w), k), c = mul2(v[2].pair(w), k), d = mul2(v[3].pair(w), k);
    t[(2 * w) * 32] = codes2(a.x, b.x) | codes2(c.x, d.x) << 16;
    t[(2 * w + 1) * 32] = codes2(a.y, b.y) | codes2(c.y, d.y) << 16;
  }
}
__device__ __forceinline__ void qt_cols_store(const QtOut& sh, const Side& o, int col0, int mb) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int at = threadIdx.x + k * QT_THREADS, col = at >> 3, quad = at & 7, key = (col >> 3) & 15;
    uint4 u = sh.t[col * 8 + (quad ^ (key >> 1))];
    if (key & 1) u = make_uint4(u.z, u.w, u.x, u.y);
    *reinterpret_cast<uint4*>(o.codes + (long long)(col0 + col) * o.width + mb * TILE + quad * 16) = u;
  }
}

// after a wait that ran out: the loads on their way land (or are given up on) before the CTA ends
template <int N>
__device__ __forceinline__ void drain(uint64_t* full, int it, int tile, int tiles, int* err) {
  for (int k = 0; k < N && tile + k * (int)gridDim.x < tiles; ++k)
    mbar_wait(&full[(it + k) % N], ((it + k) / N) & 1, err, ERR_MBAR_TIMEOUT_EPILOGUE);
}

template <typename T>
struct SwigluFwdShared {
  struct Stage {
    T a[TILE * TILE], b[TILE * TILE];
  } stage[QtStages<T>::N];
  QtOut out;
  uint64_t full[QtStages<T>::N];
};
template <typename T, bool QT, bool CK>
__global__ void __launch_bounds__(QT_THREADS, 1)
    swiglu8_fwd_q_kernel(const __grid_constant__ CUtensorMap tm, int M, int H, Side ck, Side g8, Side g8t, int* err) {
  constexpr int N = QtStages<T>::N;
  extern __shared__ __align__(128) uint8_t raw[];
  SwigluFwdShared<T>& sh = *reinterpret_cast<SwigluFwdShared<T>*>(raw);
  const int nhb = H / TILE, nmb = (M + TILE - 1) / TILE, tiles = nhb * nmb;
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  auto fetch = [&](int tile, int s) {
    const int hb = tile % nhb, mb = tile / nhb;
    mbar_expect_tx(&sh.full[s], sizeof(sh.stage[s]));
    tma_load_3d(sh.stage[s].a, &tm, &sh.full[s], hb * TILE, mb * TILE, 0);
    tma_load_3d(sh.stage[s].b, &tm, &sh.full[s], H + hb * TILE, mb * TILE, 0);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < N; ++s) mbar_init(&sh.full[s], 1);
    fence_barrier_init();
    for (int s = 0; s < N; ++s)
      if ((int)(blockIdx.x + s * gridDim.x) < tiles) fetch(blockIdx.x + s * gridDim.x, s);
  }
  __syncthreads();
  int it = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++it) {
    const int s = it % N, hb = tile % nhb, mb = tile / nhb, r0 = mb * TILE + QT_R * rg;
    const bool got = mbar_wait(&sh.full[s], (it / N) & 1, err, ERR_MBAR_TIMEOUT_EPILOGUE);
    Eight<T> a[QT_R], b[QT_R];
#pragma unroll
    for (int i = 0; i < QT_R; ++i) {
      a[i].fetch(&sh.stage[s].a[(QT_R * rg + i) * TILE + 8 * l16]);
      b[i].fetch(&sh.stage[s].b[(QT_R * rg + i) * TILE + 8 * l16]);
    }
    if (!__syncthreads_and(got)) {  // else the stage has been read
      if (threadIdx.x == 0) drain<N>(sh.full, it, tile, tiles, err);
      break;
    }
    if (threadIdx.x == 0 && tile + N * (int)gridDim.x < tiles) fetch(tile + N * gridDim.x, s);
    Eight<float> v[QT_R];
#pragma unroll
    for (int i = 0; i < QT_R; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) v[i].set(w, swiglu<sizeof(T) == 4>(a[i].pair(w), b[i].pair(w)));
    if constexpr (CK) {
      qt_rows(a, ck, r0, hb, 2 * nhb, l16);
      qt_rows(b, ck, r0, nhb + hb, 2 * nhb, l16);
    }
    qt_rows(v, g8, r0, hb, nhb, l16);
    if constexpr (QT) {
      qt_cols_part(v, sh.out, l16);
      __syncthreads();
      if (threadIdx.x < TILE) qt_cols_scale(sh.out, threadIdx.x, g8t, hb * TILE, mb, nmb);
      __syncthreads();
      qt_cols_codes(v, sh.out, l16);
      __syncthreads();
      qt_cols_store(sh.out, g8t, hb * TILE, mb);
    }
  }
}

template <typename T>
struct SwigluBwdShared {
  struct Stage {
    T dg[TILE * TILE];
    uint8_t a[TILE * TILE], b[TILE * TILE];
    uint8_t sa[ATOM], sb[ATOM];
  } stage[QtStages<T>::N];
  QtOut out[2];
  uint64_t full[QtStages<T>::N];
};
template <typename T>
__global__ void __launch_bounds__(QT_THREADS, 1)
    swiglu8_bwd_q_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tmck, int M, int H, Side ck,
                         Side d8, Side d8t, int* err) {
  constexpr int N = QtStages<T>::N;
  extern __shared__ __align__(128) uint8_t raw[];
  SwigluBwdShared<T>& sh = *reinterpret_cast<SwigluBwdShared<T>*>(raw);
  const int nhb = H / TILE, nmb = (M + TILE - 1) / TILE, tiles = nhb * nmb;
  const int l16 = threadIdx.x & 15, rg = threadIdx.x >> 4;
  auto fetch = [&](int tile, int s) {
    const int hb = tile % nhb, mb = tile / nhb;
    auto& st = sh.stage[s];
    mbar_expect_tx(&sh.full[s], sizeof(st));
    tma_load_3d(st.dg, &tm, &sh.full[s], hb * TILE, mb * TILE, 0);
    tma_load_3d(st.a, &tmck, &sh.full[s], hb * TILE, mb * TILE, 0);
    tma_load_3d(st.b, &tmck, &sh.full[s], H + hb * TILE, mb * TILE, 0);
    bulk_load(st.sa, ck.scales + ((long long)mb * ck.quads + (hb >> 2)) * ATOM, ATOM, &sh.full[s]);
    bulk_load(st.sb, ck.scales + ((long long)mb * ck.quads + ((nhb + hb) >> 2)) * ATOM, ATOM, &sh.full[s]);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < N; ++s) mbar_init(&sh.full[s], 1);
    fence_barrier_init();
    for (int s = 0; s < N; ++s)
      if ((int)(blockIdx.x + s * gridDim.x) < tiles) fetch(blockIdx.x + s * gridDim.x, s);
  }
  __syncthreads();
  int it = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++it) {
    const int s = it % N, hb = tile % nhb, mb = tile / nhb, r0 = mb * TILE + QT_R * rg;
    const auto& st = sh.stage[s];
    const bool got = mbar_wait(&sh.full[s], (it / N) & 1, err, ERR_MBAR_TIMEOUT_EPILOGUE);
    Eight<T> dv[QT_R];
    uint2 ca[QT_R], cb[QT_R];
    uint8_t ba[QT_R], bb[QT_R];
    const int sc = (QT_R * rg & 31) * 16 + (QT_R * rg >> 5) * 4;
#pragma unroll
    for (int i = 0; i < QT_R; ++i) {
      const int at = (QT_R * rg + i) * TILE + 8 * l16;
      dv[i].fetch(&st.dg[at]);
      ca[i] = *reinterpret_cast<const uint2*>(&st.a[at]);
      cb[i] = *reinterpret_cast<const uint2*>(&st.b[at]);
      ba[i] = st.sa[sc + 16 * i + (hb & 3)];
      bb[i] = st.sb[sc + 16 * i + ((nhb + hb) & 3)];
    }
    if (!__syncthreads_and(got)) {  // else the stage has been read
      if (threadIdx.x == 0) drain<N>(sh.full, it, tile, tiles, err);
      break;
    }
    if (threadIdx.x == 0 && tile + N * (int)gridDim.x < tiles) fetch(tile + N * gridDim.x, s);
    Eight<float> va[QT_R], vb[QT_R];
#pragma unroll
    for (int i = 0; i < QT_R; ++i) {
      float2 a[4], b[4];
      values8(ca[i], scale_of(ba[i]), a);
      values8(cb[i], scale_of(bb[i]), b);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float2 da, db;
        swiglu_grad<sizeof(T) == 4>(a[w], b[w], dv[i].pair(w), da, db);
        va[i].set(w, da);
        vb[i].set(w, db);
      }
    }
    qt_rows(va, d8, r0, hb, 2 * nhb, l16);
    qt_rows(vb, d8, r0, nhb + hb, 2 * nhb, l16);
    qt_cols_part(va, sh.out[0], l16);
    qt_cols_part(vb, sh.out[1], l16);
    __syncthreads();
    if (threadIdx.x < TILE) qt_cols_scale(sh.out[0], threadIdx.x, d8t, hb * TILE, mb, nmb);
    else if (threadIdx.x < 2 * TILE) qt_cols_scale(sh.out[1], threadIdx.x - TILE, d8t, H + hb * TILE, mb, nmb);
    __syncthreads();
    qt_cols_codes(va, sh.out[0], l16);
    qt_cols_codes(vb, sh.out[1], l16);
    __syncthreads();
    qt_cols_store(sh.out[0], d8t, hb * TILE, mb);
    qt_cols_store(sh.out[1], d8t, H + hb * TILE, mb);
  }
}

template <typename K>
cudaError_t qt_launch(K kern, size_t shared, std::atomic<uint64_t>& set, int* grid, long long tiles) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !((set.load(std::memory_order_relaxed) >> dev) & 1))) {  // once per device
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
    if (e == cudaSuccess && dev <= 63) set.fetch_or(1ull << dev);
  }
  *grid = (int)std::min<long long>(tiles, num_sms());
  return e;
}
template <typename T, bool QT, bool CK>
cudaError_t swiglu_fwd_q(const CUtensorMap& tm, const Swiglu8Params& p, long long tiles, Side ck, Side g8, Side g8t,
                         cudaStream_t s) {
  static std::atomic<uint64_t> set{0};
  auto kern = swiglu8_fwd_q_kernel<T, QT, CK>;
  static_assert(sizeof(SwigluFwdShared<T>) <= 232448, "shared memory");
  int grid = 0;
  const cudaError_t e = qt_launch(kern, sizeof(SwigluFwdShared<T>), set, &grid, tiles);
  if (e != cudaSuccess) return e;
  kern<<<grid, QT_THREADS, sizeof(SwigluFwdShared<T>), s>>>(tm, p.M, p.H, ck, g8, g8t, p.err);
  return cudaGetLastError();
}

template <typename T>
cudaError_t swiglu_fwd_typed(const Swiglu8Params& p, cudaStream_t s) {
  const int nhb = (p.H + TILE - 1) / TILE;
  const Side ck = side(p.ck, p.ck_scales, p.M, 2 * nhb * TILE), g8 = side(p.g8, p.g8_scales, p.M, p.H),
             g8t = side(p.g8t, p.g8t_scales, p.H, p.M);
  if (p.g8 != nullptr) {
    const long long tiles = (long long)nhb * ((p.M + TILE - 1) / TILE);
    if (tiles >= (1ll << 30) || p.map == nullptr) return cudaErrorInvalidValue;
    if constexpr (sizeof(T) == 4) {
      if (p.g8t != nullptr)
        return p.ck != nullptr ? swiglu_fwd_q<T, true, true>(*p.map, p, tiles, ck, g8, g8t, s)
                               : swiglu_fwd_q<T, true, false>(*p.map, p, tiles, ck, g8, g8t, s);
      if (p.ck != nullptr) return swiglu_fwd_q<T, false, true>(*p.map, p, tiles, ck, g8, g8t, s);
    } else if (p.g8t != nullptr || p.ck != nullptr) {
      return cudaErrorInvalidValue;
    }
    return swiglu_fwd_q<T, false, false>(*p.map, p, tiles, ck, g8, g8t, s);
  }
  const long long blocks = (long long)nhb * ((p.M + 16 * ROW_R - 1) / (16 * ROW_R));
  if (blocks >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool vec = p.H % 8 == 0 && aligned16(p.ab, p.ld * (long long)sizeof(T));
  const bool vec_g = p.H % 8 == 0 && aligned16(p.g, 0);
  const T* ab = static_cast<const T*>(p.ab);
  T* g = static_cast<T*>(p.g);
#define FWD(VEC, CK) swiglu8_fwd_kernel<T, VEC, CK><<<(int)blocks, 256, 0, s>>>(ab, p.ld, p.M, p.H, vec_g, g, ck)
  if (p.ck != nullptr) {
    if (vec) FWD(true, true);
    else FWD(false, true);
  } else {
    if (vec) FWD(true, false);
    else FWD(false, false);
  }
#undef FWD
  return cudaGetLastError();
}
template <typename T>
cudaError_t swiglu_bwd_typed(const Swiglu8BwdParams& p, cudaStream_t s) {
  const int nhb = (p.H + TILE - 1) / TILE;
  const Side ck = side(const_cast<uint8_t*>(p.ck), const_cast<uint8_t*>(p.ck_scales), p.M, 2 * nhb * TILE),
             d8 = side(p.d8, p.d8_scales, p.M, 2 * p.H), d8t = side(p.d8t, p.d8t_scales, 2 * p.H, p.M);
  if (p.d8 != nullptr) {
    const long long tiles = (long long)nhb * ((p.M + TILE - 1) / TILE);
    if (tiles >= (1ll << 30) || p.map == nullptr || p.ck_map == nullptr) return cudaErrorInvalidValue;
    static std::atomic<uint64_t> set{0};
    auto kern = swiglu8_bwd_q_kernel<T>;
    static_assert(sizeof(SwigluBwdShared<T>) <= 232448, "shared memory");
    int grid = 0;
    const cudaError_t e = qt_launch(kern, sizeof(SwigluBwdShared<T>), set, &grid, tiles);
    if (e != cudaSuccess) return e;
    kern<<<grid, QT_THREADS, sizeof(SwigluBwdShared<T>), s>>>(*p.map, *p.ck_map, p.M, p.H, ck, d8, d8t, p.err);
    return cudaGetLastError();
  }
  const long long blocks = (long long)nhb * ((p.M + 16 * ROW_R - 1) / (16 * ROW_R));
  if (blocks >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool vec = p.H % 8 == 0 && aligned16(p.dg, p.ld * (long long)sizeof(T));
  const bool vec_d = p.H % 8 == 0 && aligned16(p.dab, 0);
  const T* dg = static_cast<const T*>(p.dg);
  T* dab = static_cast<T*>(p.dab);
  if (vec) swiglu8_bwd_kernel<T, true><<<(int)blocks, 256, 0, s>>>(dg, p.ld, p.M, p.H, vec_d, dab, ck);
  else swiglu8_bwd_kernel<T, false><<<(int)blocks, 256, 0, s>>>(dg, p.ld, p.M, p.H, vec_d, dab, ck);
  return cudaGetLastError();
}

// --------------------------------------------------------------------------------------------------------- few rows
// y [M, N] = Q(x) W^T + bias for at most 16 rows of x (tokens of a serving step), in one launch: x is packed where it is used.
// Reading W bounds it (N Kp bytes) once it is large. e4m3 values are fp16 values, so the products run on mma.m16n8k16 (W rows x
// tokens) with fp32 sums, after one conversion of two codes each; the order of k inside a block is free, so a lane's 16
// consecutive bytes serve as its operands of four instructions, for W and for x alike. A block's sum d is scaled in fp32, by two
// factors of about half the exponent each (scale_halves): the product of both scales may leave fp32's range where the sum's
// place in y does not, as the largest values of x's and W's blocks need not meet. The warps' sums are added in order.
// W cold in L2: one token 2048 -> 6144 (12.6 MB, 1.9 us at the copy rate) 6.9 us, 2048 -> 11008 8.4, 5504 -> 2048 7.9, 4 tokens
// 5504 -> 11008 18.9, 16 tokens 2048 -> 6144 9.6. A CTA of eight warps for each 32 rows, loads a block at a time: 7.5, 11.1,
// 10.0, 26.0, 14.3 (x packed more often, half-filled second waves).
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four codes as two fp16 pairs
__device__ __forceinline__ void halves(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}

// A CTA owns a few groups of 16 rows of W, each of its warps some of the blocks of 128 along K: the warp packs x's part of a block
// once and multiplies it with that block of each group. A ring in shared memory holds up to FEW_SLOTS - 1 of these pieces on
// their way; each lane reads back what it asked for itself, and adds to sums that it alone keeps there, so no thread waits for
// another before the last product.
constexpr int FEW_SLOTS = 4, FEW_GROUPS = 8;  // groups of a CTA: at most this, half of it for more than eight rows of x
struct FewSlot {
  uint4 w[2][2][32];         // [row g + 8 r][half of the block][lane]
  uint32_t scales[2][32];    // of four blocks, this one among them
};
__device__ __forceinline__ void cp_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
// bytes of shared memory of a warp
__host__ __device__ constexpr int few_ring() { return FEW_SLOTS * (int)sizeof(FewSlot); }
__host__ __device__ constexpr int few_sums(int groups, int nt) { return groups * nt * 32 * 16; }

template <typename T, int NT, int WARPS>  // NT: groups of eight rows of x; WARPS: at most
__global__ void __launch_bounds__(32 * WARPS, WARPS == 8 ? 2 : 1) few_rows_kernel(const FewRowsParams p, int groups, bool vec) {
  extern __shared__ __align__(16) uint8_t raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warps = blockDim.x >> 5;
  FewSlot* const ring = reinterpret_cast<FewSlot*>(raw + warp * few_ring());
  uint8_t* const all_sums = raw + warps * few_ring();
  float4* const sums = reinterpret_cast<float4*>(all_sums + warp * few_sums(groups, NT)) + lane;  // [group][NT][lane]
  const int nb = (p.K + TILE - 1) / TILE, quads = (nb + 3) / 4;
  const long long width = (long long)nb * TILE;
  const int n0 = blockIdx.x * 16 * groups, mine = min(groups, (p.N - n0 + 15) / 16);
  const T* x = static_cast<const T*>(p.x);
  for (int i = 0; i < groups * NT; ++i) sums[i * 32] = make_float4(0.f, 0.f, 0.f, 0.f);
  int next_kb = warp, next = 0;  // the next piece that is asked for
  auto fetch = [&](int slot) {
    if (next_kb < nb) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int n = min(n0 + 16 * next + g + 8 * r, p.N - 1);  // rows past the last: not written
        const uint8_t* src = p.codes + n * width + next_kb * TILE + 16 * t;
        cp_async16(&ring[slot].w[r][0][lane], src);
        cp_async16(&ring[slot].w[r][1][lane], src + 64);
        cp_async4(&ring[slot].scales[r][lane], p.scales + scale_at(n, next_kb & ~3, quads));
      }
      if (++next == mine) {
        next = 0;
        next_kb += warps;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < FEW_SLOTS - 1; ++s) fetch(s);
  int slot = 0;
  for (int kb = warp; kb < nb; kb += warps) {
    uint2 b[NT][2][4];    // x in fp16 values of its codes: [half of the block][instruction]
    float2 s0[NT], s1[NT];  // scales of tokens 2 t and 2 t + 1, as two factors
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      Eight<T> f[4];  // columns 16 t .. + 15 and 64 + 16 t .. + 15 of the block
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int c = kb * TILE + (h >> 1) * 64 + 16 * t + (h & 1) * 8, m = 8 * i + g;
        f[h].load(x + m * p.ldx + c, m < p.M ? max(0, min(8, p.K - c)) : 0, vec);
      }
      float tops[4];
      finite_tops(f, tops);
      float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int byte = scale_byte(top);
      const float inv = scale_inv(byte);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 lo = codes8(f[2 * h], inv), hi = codes8(f[2 * h + 1], inv);
        halves(lo.x, b[i][h][0].x, b[i][h][0].y);
        halves(lo.y, b[i][h][1].x, b[i][h][1].y);
        halves(hi.x, b[i][h][2].x, b[i][h][2].y);
        halves(hi.y, b[i][h][3].x, b[i][h][3].y);
      }
      s0[i] = scale_halves(__shfl_sync(0xffffffffu, byte, 8 * t));
      s1[i] = scale_halves(__shfl_sync(0xffffffffu, byte, 8 * t + 4));
    }
#pragma unroll 1
    for (int r = 0; r < mine; ++r) {
      asm volatile("cp.async.wait_group %0;" ::"n"(FEW_SLOTS - 2) : "memory");
      fetch(slot == 0 ? FEW_SLOTS - 1 : slot - 1);  // into the slot whose values the last products have taken
      const FewSlot& from = ring[slot];
      slot = slot + 1 == FEW_SLOTS ? 0 : slot + 1;
      const float2 w0 = scale_halves((from.scales[0][lane] >> (8 * (kb & 3))) & 0xff);
      const float2 w1 = scale_halves((from.scales[1][lane] >> (8 * (kb & 3))) & 0xff);
      float d[NT][4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 u = from.w[0][h][lane], v = from.w[1][h][lane];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t a0, a1, a2, a3;
          halves(q == 0 ? u.x : q == 1 ? u.y : q == 2 ? u.z : u.w, a0, a2);
          halves(q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w, a1, a3);
#pragma unroll
          for (int i = 0; i < NT; ++i) mma_f16(d[i], a0, a1, a2, a3, b[i][h][q].x, b[i][h][q].y);
        }
      }
      // d: rows g, g + 8 of W, tokens 2 t, 2 t + 1
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float2 x0 = mul2(s0[i], w0), x1 = mul2(s1[i], w0), x2 = mul2(s0[i], w1), x3 = mul2(s1[i], w1);
        float4 a = sums[(r * NT + i) * 32];
        a.x = fmaf(d[i][0] * x0.x, x0.y, a.x);
        a.y = fmaf(d[i][1] * x1.x, x1.y, a.y);
        a.z = fmaf(d[i][2] * x2.x, x2.y, a.z);
        a.w = fmaf(d[i][3] * x3.x, x3.y, a.w);
        sums[(r * NT + i) * 32] = a;
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // the warps' sums in order
  T* y = static_cast<T*>(p.y);
  const float* part = reinterpret_cast<const float*>(all_sums);
  for (int at = threadIdx.x; at < 16 * mine * p.M; at += blockDim.x) {
    const int m = at / (16 * mine), rest = at % (16 * mine), n = n0 + rest;
    if (n >= p.N) continue;
    // row rest % 16 = g or g + 8, token m % 8 = 2 t or 2 t + 1
    const int row = rest & 15, l = (row & 7) * 4 + ((m & 7) >> 1), e = (row >> 3) * 2 + (m & 1);
    const float* q = part + (((rest >> 4) * NT + (m >> 3)) * 32 + l) * 4 + e;
    float v = 0.f;
    for (int k = 0; k < warps; ++k) v += q[k * (few_sums(groups, NT) / 4)];
    if (p.bias != nullptr) v += p.bias[n];
    y[(long long)m * p.N + n] = from_f<T>(v);
  }
}

template <typename T, int NT, int WARPS>
cudaError_t few_rows(const FewRowsParams& p, int groups, bool vec, cudaStream_t s) {
  static std::atomic<uint64_t> set{0};
  auto kern = few_rows_kernel<T, NT, WARPS>;
  const int warps = std::min(WARPS, (p.K + TILE - 1) / TILE);
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !((set.load(std::memory_order_relaxed) >> dev) & 1))) {  // once per device
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WARPS * (few_ring() + few_sums(FEW_GROUPS / NT, NT)));
    if (e == cudaSuccess && dev <= 63) set.fetch_or(1ull << dev);
  }
  if (e != cudaSuccess) return e;
  const int grid = (p.N + 16 * groups - 1) / (16 * groups);
  kern<<<grid, 32 * warps, warps * (few_ring() + few_sums(groups, NT)), s>>>(p, groups, vec);
  return cudaGetLastError();
}
template <typename T, int NT>
cudaError_t few_rows_typed(const FewRowsParams& p, int sms, cudaStream_t s) {
  const bool vec = p.K % 8 == 0 && aligned16(p.x, p.ldx * (long long)sizeof(T));
  const int all = (p.N + 15) / 16;
  // equal waves, one as far as shared memory goes: of CTAs of sixteen warps, one per SM, or, where rows have at most eight blocks,
  // of eight, two per SM
  const int slots = p.K > 8 * TILE ? sms : 2 * sms, waves = (all + slots * (FEW_GROUPS / NT) - 1) / (slots * (FEW_GROUPS / NT));
  const int groups = (all + slots * waves - 1) / (slots * waves);
  return p.K > 8 * TILE ? few_rows<T, NT, 16>(p, groups, vec, s) : few_rows<T, NT, 8>(p, groups, vec, s);
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

cudaError_t pack8_launch(const Pack8Params& p, cudaStream_t s) {
  if (p.M <= 0 || p.K <= 0 || (p.codes == nullptr && p.codes_t == nullptr) || (p.sums != nullptr && p.codes_t == nullptr))
    return cudaErrorInvalidValue;
  return by_type(p.elem, [&](auto t) { return pack_typed<decltype(t)>(p, s); });
}
cudaError_t pack8_jobs_launch(const Pack8Jobs& p, cudaStream_t s) {
  if (p.n < 1 || p.n > 3) return cudaErrorInvalidValue;
  PackJobs q{};
  q.n = p.n;
  long long tiles = 0;
  for (int i = 0; i < p.n; ++i) {
    const Pack8Params& j = p.job[i];
    if (j.M <= 0 || j.K <= 0 || j.codes == nullptr || j.sums != nullptr || j.elem < ELEM_BF16 || j.elem > ELEM_F32)
      return cudaErrorInvalidValue;
    q.job[i].x = j.x;
    q.job[i].ld = j.ld;
    q.job[i].M = j.M;
    q.job[i].K = j.K;
    q.job[i].elem = j.elem;
    q.job[i].first = (int)tiles;
    q.job[i].vec = j.K % 8 == 0 && aligned16(j.x, j.ld * (j.elem == ELEM_F32 ? 4 : 2));
    q.job[i].rows = side(j.codes, j.scales, j.M, j.K);
    q.job[i].cols = side(j.codes_t, j.scales_t, j.K, j.M);
    tiles += (long long)((j.K + TILE - 1) / TILE) * ((j.M + TILE - 1) / TILE);
    if (tiles >= (1ll << 31)) return cudaErrorInvalidValue;
  }
  pack8_jobs_kernel<<<(int)tiles, PACK_THREADS, 0, s>>>(q);
  return cudaGetLastError();
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
  return by_type(elem, [&](auto t) {
    return p.M <= 8 ? few_rows_typed<decltype(t), 1>(p, num_sms(), s) : few_rows_typed<decltype(t), 2>(p, num_sms(), s);
  });
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

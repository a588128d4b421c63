// Norms before and after a block's branch, fused with the branch's gate and residual scale:
//     u = y ry wp                    ry = rsqrt(mean(y^2) + eps)            (u = y without a norm after the branch)
//     x' = x + q u                   q = res_scale gate                     (gate: one row per sample, or 1)
//     h = x' rx w (1 + scale) + shift,   rx = rsqrt(mean(x'^2) + eps)       (no h without w; shift / scale per sample)
// Backward from dx' and dh, with yn = y ry, n = x' rx, cw = w (1 + scale), a = q wp:
//     g = dx' + rx (dh cw - n mean(dh cw n))          dx = g
//     dy = ry (a g - yn mean(a g yn))                 (dy = q g without the norm)
//     per (sample, channel): sum dh, sum dh n, sum g yn -> dshift, dscale = w (.), dgate = res_scale wp (.) and, summed
//     over the samples with (1 + scale) and q, the weights' gradients dw and dwp.
// The backward recomputes x' from x and y (the same bytes as reading a stored x', without its rounding) and rebuilds the
// second mean from sums taken in the same pass as the first: a g = a (dx' + rx (dh cw - n m)), so
//     mean(a g yn) = mean(a yn (dx' + rx dh cw)) - rx m mean(a yn n),    m = mean(dh cw n).
// Statistics and sums are fp32; x' is rounded only when it is stored, so h comes from the unrounded sum.
//
// Column sums: a CTA owns a contiguous span of rows and writes one partial row (three sums per channel) per sample it
// meets. Entry cta + sample is unique (along the spans both only grow), so ctas + samples entries hold them all; two
// small kernels add them in a fixed order.
#include <algorithm>

#include "block_ops.h"
#include "common.cuh"
#include "kernels.h"
#include "vec.cuh"

namespace tgo {

namespace {

constexpr int SW_THREADS = 256;

template <int K>
__device__ __forceinline__ void block_totals(float (&v)[K], float* red) {  // red: [2][32][K], alternating by the caller
#pragma unroll
  for (int i = 0; i < K; ++i) v[i] = warp_total(v[i]);
  if (lane_id() == 0)
#pragma unroll
    for (int i = 0; i < K; ++i) red[warp_id() * K + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < K; ++i) v[i] = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w)
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] += red[w * K + i];
}

__host__ __device__ __forceinline__ int samples_of(const SandwichParams& p) {
  return (p.gate != nullptr || p.scale != nullptr) ? p.M / p.T : 1;
}

}  // namespace

// Any width, stride and alignment: one row at a time, columns strided over the block.
template <typename T>
__global__ void __launch_bounds__(SW_THREADS) sandwich_fwd_any_kernel(SandwichParams p) {
  __shared__ float red[64];
  const T* x = reinterpret_cast<const T*>(p.x);
  const T* y = reinterpret_cast<const T*>(p.y);
  int slot = 0;
  for (int row = blockIdx.x; row < p.M; row += gridDim.x) {
    const long long off = (long long)row * p.D;
    const int b = row / p.T;
    const T* gate = p.gate != nullptr ? reinterpret_cast<const T*>(p.gate) + b * p.gate_bs : nullptr;
    float ry = 1.f;
    if (p.post_w != nullptr) {
      float s[1] = {0.f};
      for (int c = threadIdx.x; c < p.D; c += blockDim.x) {
        const float v = to_f<T>(y[off + c]);
        s[0] = fmaf(v, v, s[0]);
      }
      block_totals<1>(s, red + (slot++ & 1) * 32);
      ry = rsqrtf(s[0] / p.D + p.eps);
      if (threadIdx.x == 0) p.rstd_y[row] = ry;
    }
    auto new_x = [&](int c) {
      float u = to_f<T>(y[off + c]) * ry * p.res_scale;
      if (p.post_w != nullptr) u *= p.post_w[c];
      if (gate != nullptr) u *= to_f<T>(gate[c]);
      return to_f<T>(x[off + c]) + u;
    };
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < p.D; c += blockDim.x) {
      const float v = new_x(c);
      s[0] = fmaf(v, v, s[0]);
      reinterpret_cast<T*>(p.x_new)[off + c] = from_f<T>(v);
    }
    if (p.w == nullptr) continue;
    block_totals<1>(s, red + (slot++ & 1) * 32);
    const float rx = rsqrtf(s[0] / p.D + p.eps);
    if (threadIdx.x == 0) p.rstd_x[row] = rx;
    const T* sc = p.scale != nullptr ? reinterpret_cast<const T*>(p.scale) + b * p.mod_bs : nullptr;
    const T* sh = p.scale != nullptr ? reinterpret_cast<const T*>(p.shift) + b * p.mod_bs : nullptr;
    for (int c = threadIdx.x; c < p.D; c += blockDim.x) {
      float h = new_x(c) * rx * p.w[c];
      if (sc != nullptr) h = fmaf(h, 1.f + to_f<T>(sc[c]), to_f<T>(sh[c]));
      reinterpret_cast<T*>(p.h)[off + c] = from_f<T>(h);
    }
  }
}

// Column sums in dynamic shared memory [3][D]; a thread owns its columns, so no two threads add to one sum.
template <typename T>
__global__ void __launch_bounds__(SW_THREADS) sandwich_bwd_any_kernel(SandwichParams p, SandwichBwdParams q) {
  extern __shared__ float acc[];
  __shared__ float red[2 * 32 * 3];
  const T* x = reinterpret_cast<const T*>(p.x);
  const T* y = reinterpret_cast<const T*>(p.y);
  const T* dxn = reinterpret_cast<const T*>(q.dx_new);
  const T* dh = reinterpret_cast<const T*>(q.dh);
  const bool per_sample = samples_of(p) > 1;
  const int row0 = blockIdx.x * q.rows_per_cta, row1 = min(p.M, row0 + q.rows_per_cta);
  for (int c = threadIdx.x; c < 3 * p.D; c += blockDim.x) acc[c] = 0.f;
  int slot = 0;
  for (int row = row0; row < row1; ++row) {
    const long long off = (long long)row * p.D;
    const int b = row / p.T;
    const T* gate = p.gate != nullptr ? reinterpret_cast<const T*>(p.gate) + b * p.gate_bs : nullptr;
    const T* sc = p.scale != nullptr ? reinterpret_cast<const T*>(p.scale) + b * p.mod_bs : nullptr;
    const float ry = p.post_w != nullptr ? p.rstd_y[row] : 1.f;
    const float rx = p.w != nullptr ? p.rstd_x[row] : 0.f;
    struct El {
      float yn, a, n, dhc, e, dhv;
    };
    auto at = [&](int c) {
      El v;
      v.yn = to_f<T>(y[off + c]) * ry;
      v.a = p.res_scale;
      if (p.post_w != nullptr) v.a *= p.post_w[c];
      if (gate != nullptr) v.a *= to_f<T>(gate[c]);
      v.n = fmaf(v.a, v.yn, to_f<T>(x[off + c])) * rx;
      v.dhv = dh != nullptr ? to_f<T>(dh[off + c]) : 0.f;
      v.dhc = p.w != nullptr ? v.dhv * p.w[c] : 0.f;
      if (sc != nullptr) v.dhc *= 1.f + to_f<T>(sc[c]);
      v.e = dxn != nullptr ? to_f<T>(dxn[off + c]) : 0.f;
      return v;
    };
    float s[3] = {0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < p.D; c += blockDim.x) {
      const El v = at(c);
      s[0] = fmaf(v.dhc, v.n, s[0]);
      s[1] = fmaf(v.a * v.yn, fmaf(rx, v.dhc, v.e), s[1]);
      s[2] = fmaf(v.a * v.yn, v.n, s[2]);
    }
    block_totals<3>(s, red + (slot++ & 1) * 96);
    const float m = s[0] / p.D;
    const float m2 = p.post_w != nullptr ? (s[1] - rx * m * s[2]) / p.D : 0.f;
    for (int c = threadIdx.x; c < p.D; c += blockDim.x) {
      const El v = at(c);
      const float g = v.e + rx * (v.dhc - v.n * m);
      reinterpret_cast<T*>(q.dx)[off + c] = from_f<T>(g);
      reinterpret_cast<T*>(q.dy)[off + c] = from_f<T>(ry * (v.a * g - v.yn * m2));
      acc[c] += v.dhv;
      acc[p.D + c] = fmaf(v.dhv, v.n, acc[p.D + c]);
      acc[2 * p.D + c] = fmaf(g, v.yn, acc[2 * p.D + c]);
    }
    const bool last = row + 1 == row1 || (per_sample && (row + 1) % p.T == 0);
    if (last) {
      float* dst = q.partial + (long long)(blockIdx.x + (per_sample ? b : 0)) * 3 * p.D;
      for (int c = threadIdx.x; c < p.D; c += blockDim.x)
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          dst[i * p.D + c] = acc[i * p.D + c];
          acc[i * p.D + c] = 0.f;
        }
    }
  }
}

// Sums of a sample's partial rows -> its dshift / dscale / dgate rows, and the weights' sums over this block's samples.
constexpr int RED_ROWS = 8;
template <typename T>
__global__ void __launch_bounds__(32 * RED_ROWS) sandwich_reduce_kernel(SandwichParams p, SandwichBwdParams q) {
  __shared__ float part[RED_ROWS][3][32];
  const int samples = samples_of(p);
  const int T_rows = samples > 1 ? p.T : p.M;
  const int c = blockIdx.x * 32 + threadIdx.x;
  const bool ok = c < p.D;
  const int per = (samples + gridDim.y - 1) / gridDim.y;
  const int b0 = blockIdx.y * per, b1 = min(samples, b0 + per);
  const float w = ok && p.w != nullptr ? p.w[c] : 0.f;
  const float pw = ok && p.post_w != nullptr ? p.post_w[c] : 1.f;
  float sum_w = 0.f, sum_p = 0.f;
  for (int b = b0; b < b1; ++b) {
    const int first = (int)((long long)b * T_rows / q.rows_per_cta);
    const int last = (int)(((long long)(b + 1) * T_rows - 1) / q.rows_per_cta);
    float s[3] = {0.f, 0.f, 0.f};
    if (ok)
      for (int k = first + threadIdx.y; k <= last; k += RED_ROWS) {
        const float* src = q.partial + (long long)(k + b) * 3 * p.D + c;
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] += src[(long long)i * p.D];
      }
#pragma unroll
    for (int i = 0; i < 3; ++i) part[threadIdx.y][i][threadIdx.x] = s[i];
    __syncthreads();
    if (threadIdx.y == 0 && ok) {
#pragma unroll
      for (int k = 1; k < RED_ROWS; ++k)
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] += part[k][i][threadIdx.x];
      float sc = 1.f, g = p.res_scale;
      if (p.scale != nullptr) {
        sc += to_f<T>(reinterpret_cast<const T*>(p.scale)[b * p.mod_bs + c]);
        reinterpret_cast<T*>(q.dshift)[(long long)b * p.D + c] = from_f<T>(s[0]);
        reinterpret_cast<T*>(q.dscale)[(long long)b * p.D + c] = from_f<T>(w * s[1]);
      }
      if (p.gate != nullptr) {
        g *= to_f<T>(reinterpret_cast<const T*>(p.gate)[b * p.gate_bs + c]);
        reinterpret_cast<T*>(q.dgate)[(long long)b * p.D + c] = from_f<T>(p.res_scale * pw * s[2]);
      }
      sum_w = fmaf(sc, s[1], sum_w);
      sum_p = fmaf(g, s[2], sum_p);
    }
    __syncthreads();
  }
  if (threadIdx.y == 0 && ok) {
    q.wpart[(long long)blockIdx.y * 2 * p.D + c] = sum_w;
    q.wpart[((long long)blockIdx.y * 2 + 1) * p.D + c] = sum_p;
  }
}

__global__ void sandwich_weights_kernel(SandwichParams p, SandwichBwdParams q) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= p.D) return;
  float a = 0.f, b = 0.f;
  for (int g = 0; g < q.groups; ++g) {
    a += q.wpart[(long long)g * 2 * p.D + c];
    b += q.wpart[((long long)g * 2 + 1) * p.D + c];
  }
  if (q.dw != nullptr) q.dw[c] += a;
  if (q.dpost_w != nullptr) q.dpost_w[c] += b;
}

namespace {

template <typename T>
cudaError_t fwd_run(const SandwichParams& p, cudaStream_t s) {
  sandwich_fwd_any_kernel<T><<<std::min(p.M, num_sms() * 8), SW_THREADS, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t bwd_run(const SandwichParams& p, const SandwichBwdParams& q, cudaStream_t s) {
  const int smem = 3 * p.D * (int)sizeof(float);
  static int allowed = 47 * 1024;  // beside the static shared memory
  if (smem > allowed) {
    cudaError_t e = cudaFuncSetAttribute(sandwich_bwd_any_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    allowed = smem;
  }
  sandwich_bwd_any_kernel<T><<<q.ctas, SW_THREADS, smem, s>>>(p, q);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  sandwich_reduce_kernel<T><<<dim3((p.D + 31) / 32, q.groups), dim3(32, RED_ROWS), 0, s>>>(p, q);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (q.dw != nullptr || q.dpost_w != nullptr)
    sandwich_weights_kernel<<<(p.D + 127) / 128, 128, 0, s>>>(p, q);
  return cudaGetLastError();
}

}  // namespace

cudaError_t sandwich_fwd_launch(const SandwichParams& p, int elem, cudaStream_t s) {
  if (p.M <= 0 || p.D <= 0) return cudaSuccess;
  switch (elem) {
    case ELEM_BF16: return fwd_run<__nv_bfloat16>(p, s);
    case ELEM_F16: return fwd_run<__half>(p, s);
    case ELEM_F32: return fwd_run<float>(p, s);
  }
  return cudaErrorInvalidValue;
}

void sandwich_bwd_plan(const SandwichParams& p, int elem, SandwichBwdParams* q) {
  const int most = num_sms() * 4;
  q->rows_per_cta = std::max(1, (p.M + most - 1) / most);
  q->ctas = (p.M + q->rows_per_cta - 1) / q->rows_per_cta;
  q->groups = std::min(samples_of(p), 64);
}

cudaError_t sandwich_bwd_launch(const SandwichParams& p, const SandwichBwdParams& q, int elem, cudaStream_t s) {
  if (p.M <= 0 || p.D <= 0) return cudaSuccess;
  switch (elem) {
    case ELEM_BF16: return bwd_run<__nv_bfloat16>(p, q, s);
    case ELEM_F16: return bwd_run<__half>(p, q, s);
    case ELEM_F32: return bwd_run<float>(p, q, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tgo

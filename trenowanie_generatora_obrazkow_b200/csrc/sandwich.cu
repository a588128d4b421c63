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
// Column sums: a unit (a CTA, or a group of its threads) owns a contiguous span of rows and writes one partial row (three
// sums per channel) per sample it meets. Entry unit + sample is unique (along the spans both only grow), so
// units + samples entries hold them all; two small kernels add them in a fixed order.
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

// ------------------------------------------------------------------------------------------------------------------
// Vector form: rows of whole 16-byte vectors, up to 4096 channels.
//
// A group of tpg = D / 8 threads (rounded up to warps) owns 8 channels per thread and walks a contiguous span of rows, R
// rows per step; a block holds several groups when rows are short. Rows arrive through untiled bulk copies into a ring of
// SW_STAGES steps: one thread issues them, so the loads of the next steps stay in flight across the block barriers of the
// row reductions, without registers. Modulation, gate and weights of the group's sample stay in registers, and so do the
// backward's column sums.
// ------------------------------------------------------------------------------------------------------------------
namespace {

constexpr int SW_STAGES = 3;
constexpr int SW_MAX_VEC_D = 4096;

struct SwGeom {
  int tpg, groups;      // threads per group, groups per block
  int span;             // rows per group
  int steps;            // of every group (R rows each)
};

// ring slot of (stage, tensor, group): [SW_STAGES][tensors][groups][R][D]
template <typename T, int R, int TENSORS>
struct SwRing {
  uint64_t* full;
  uint8_t* base;
  long long step_bytes, tensor_bytes, group_bytes;  // strides
  __device__ __forceinline__ SwRing(uint8_t* smem, const SwGeom& g, int D) {
    full = reinterpret_cast<uint64_t*>(smem);
    base = smem + 128;
    group_bytes = (long long)R * D * sizeof(T);
    tensor_bytes = group_bytes * g.groups;
    step_bytes = tensor_bytes * TENSORS;
  }
  __device__ __forceinline__ const T* row(int stage, int tensor, int group, int r, int D) const {
    return reinterpret_cast<const T*>(base + stage * step_bytes + tensor * tensor_bytes + group * group_bytes) +
           (long long)r * D;
  }
};

__device__ __forceinline__ int span_rows(int M, long long row0, int span, int done, int R) {
  const long long left = min((long long)M, row0 + span) - (row0 + done);
  return (int)max(0ll, min((long long)R, left));
}

// one thread: the rows of step i of every group of this block, all tensors
template <typename T, int R, int TENSORS>
__device__ __forceinline__ void sw_load(const SwRing<T, R, TENSORS>& ring, const SwGeom& g, int M, int D, int i,
                                        const void* const (&src)[TENSORS]) {
  const int stage = i % SW_STAGES;
  uint32_t bytes = 0;
  for (int k = 0; k < g.groups; ++k) {
    const long long row0 = ((long long)blockIdx.x * g.groups + k) * g.span;
    bytes += (uint32_t)(span_rows(M, row0, g.span, i * R, R) * D * sizeof(T));
  }
  uint32_t present = 0;
#pragma unroll
  for (int t = 0; t < TENSORS; ++t) present += src[t] != nullptr;
  mbar_expect_tx(&ring.full[stage], bytes * present);
  for (int k = 0; k < g.groups; ++k) {
    const long long row0 = ((long long)blockIdx.x * g.groups + k) * g.span;
    const int n = span_rows(M, row0, g.span, i * R, R);
    if (n <= 0) continue;
#pragma unroll
    for (int t = 0; t < TENSORS; ++t)
      if (src[t] != nullptr)
        bulk_load(const_cast<T*>(ring.row(stage, t, k, 0, D)),
                  reinterpret_cast<const T*>(src[t]) + (row0 + (long long)i * R) * D, (uint32_t)(n * D * sizeof(T)),
                  &ring.full[stage]);
  }
}

template <typename T>
__device__ __forceinline__ void load_row8(const void* base, long long off, float (&f)[8]) {
  load_vec<T, 8>(reinterpret_cast<const T*>(base) + off, f);
}

// K per-row values of R rows summed over a group. red: [R * K][warps of the block]; the caller's barrier sits between the
// two halves.
template <int N>
__device__ __forceinline__ void group_put(const float (&v)[N], float* red, int warps) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = warp_total(v[i]);
    if (lane_id() == 0) red[i * warps + warp_id()] = t;
  }
}
template <int N>
__device__ __forceinline__ void group_get(float (&v)[N], const float* red, int warps, int first, int count) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = first; w < first + count; ++w) s += red[i * warps + w];
    v[i] = s;
  }
}

}  // namespace

template <typename T, int R>
__global__ void __launch_bounds__(512) sandwich_fwd_kernel(SandwichParams p, SwGeom g, int* err) {
  extern __shared__ __align__(128) uint8_t sw_smem[];
  __shared__ float red[2][R * 16];
  const int group = threadIdx.x / g.tpg, c0 = (threadIdx.x % g.tpg) * 8;
  const bool on = c0 < p.D;
  const int warps = blockDim.x >> 5, wpg = g.tpg >> 5, w0 = group * wpg;
  const long long row0 = ((long long)blockIdx.x * g.groups + group) * g.span;
  const bool per_sample = samples_of(p) > 1;
  const SwRing<T, R, 2> ring(sw_smem, g, p.D);
  const void* const src[2] = {p.x, p.y};
  if (threadIdx.x == 0) {
    for (int s = 0; s < SW_STAGES; ++s) mbar_init(&ring.full[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < SW_STAGES && i < g.steps; ++i) sw_load<T, R, 2>(ring, g, p.M, p.D, i, src);
  }
  __syncthreads();
  float a[8], cw[8], sh[8];
  int cur = -1;
  auto sample = [&](int b) {  // constants of sample b: a = res_scale gate post_w, cw = w (1 + scale), shift
    if (b == cur || !on) return;
    cur = b;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = p.res_scale, cw[j] = 0.f, sh[j] = 0.f;
    if (p.post_w != nullptr) {
      load_vec<float, 8>(p.post_w + c0, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] *= t[j];
    }
    if (p.gate != nullptr) {
      load_row8<T>(p.gate, b * p.gate_bs + c0, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] *= t[j];
    }
    if (p.w != nullptr) load_vec<float, 8>(p.w + c0, cw);
    if (p.scale != nullptr) {
      load_row8<T>(p.scale, b * p.mod_bs + c0, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) cw[j] = fmaf(cw[j], t[j], cw[j]);
      load_row8<T>(p.shift, b * p.mod_bs + c0, sh);
    }
  };
  for (int i = 0; i < g.steps; ++i) {
    const int stage = i % SW_STAGES;
    const int n = span_rows(p.M, row0, g.span, i * R, R);
    const long long row = row0 + (long long)i * R;
    mbar_wait(&ring.full[stage], (i / SW_STAGES) & 1, err, ERR_MBAR_TIMEOUT_PRODUCER);
    Raw<T, 8> x[R], y[R];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = 0.f;
      if (on && r < n) {
        x[r].load(ring.row(stage, 0, group, r, p.D) + c0);
        y[r].load(ring.row(stage, 1, group, r, p.D) + c0);
        if (p.post_w != nullptr) {
          float f[8];
          y[r].get(f);
#pragma unroll
          for (int j = 0; j < 8; ++j) s[r] = fmaf(f[j], f[j], s[r]);
        }
      } else {
        x[r].zero();
        y[r].zero();
      }
    }
    group_put<R>(s, red[0], warps);
    __syncthreads();  // every thread has taken its rows out of the stage: refill it
    if (threadIdx.x == 0 && i + SW_STAGES < g.steps) sw_load<T, R, 2>(ring, g, p.M, p.D, i + SW_STAGES, src);
    float xn[R][8];
    float ry[R];
    if (p.post_w != nullptr) {
      group_get<R>(ry, red[0], warps, w0, wpg);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ry[r] = rsqrtf(ry[r] / p.D + p.eps);
        if (c0 == 0 && r < n) p.rstd_y[row + r] = ry[r];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = 0.f;
      if (r >= n) continue;
      sample(per_sample ? (int)((row + r) / p.T) : 0);
      if (!on) continue;
      float f[8];
      x[r].get(xn[r]);
      y[r].get(f);
      const float q = p.post_w != nullptr ? ry[r] : 1.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xn[r][j] = fmaf(f[j] * q, a[j], xn[r][j]);
        s[r] = fmaf(xn[r][j], xn[r][j], s[r]);
      }
      store_vec<T, 8>(reinterpret_cast<T*>(p.x_new) + (row + r) * p.D + c0, xn[r]);
    }
    if (p.w != nullptr) {
      group_put<R>(s, red[1], warps);
      __syncthreads();
      float rx[R];
      group_get<R>(rx, red[1], warps, w0, wpg);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= n) continue;
        rx[r] = rsqrtf(rx[r] / p.D + p.eps);
        if (c0 == 0) p.rstd_x[row + r] = rx[r];
        sample(per_sample ? (int)((row + r) / p.T) : 0);
        if (!on) continue;
        float h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = fmaf(xn[r][j] * rx[r], cw[j], sh[j]);
        store_vec<T, 8>(reinterpret_cast<T*>(p.h) + (row + r) * p.D + c0, h);
      }
    } else {
      __syncthreads();  // red[0] is written again
    }
  }
}

template <typename T, int R>
__global__ void __launch_bounds__(512) sandwich_bwd_kernel(SandwichParams p, SandwichBwdParams q, SwGeom g, int* err) {
  extern __shared__ __align__(128) uint8_t sw_smem[];
  __shared__ float red[2][3 * R * 16];
  const int group = threadIdx.x / g.tpg, c0 = (threadIdx.x % g.tpg) * 8;
  const bool on = c0 < p.D;
  const int warps = blockDim.x >> 5, wpg = g.tpg >> 5, w0 = group * wpg;
  const int unit = blockIdx.x * g.groups + group;
  const long long row0 = (long long)unit * g.span;
  const bool per_sample = samples_of(p) > 1;
  const SwRing<T, R, 4> ring(sw_smem, g, p.D);
  const void* const src[4] = {p.x, p.y, q.dh, q.dx_new};
  if (threadIdx.x == 0) {
    for (int s = 0; s < SW_STAGES; ++s) mbar_init(&ring.full[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < SW_STAGES && i < g.steps; ++i) sw_load<T, R, 4>(ring, g, p.M, p.D, i, src);
  }
  __syncthreads();
  float a[8], cw[8], acc[3][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[0][j] = acc[1][j] = acc[2][j] = 0.f;
  int cur = -1, acc_b = -1;
  auto sample = [&](int b) {
    if (b == cur || !on) return;
    cur = b;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = p.res_scale, cw[j] = 0.f;
    if (p.post_w != nullptr) {
      load_vec<float, 8>(p.post_w + c0, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] *= t[j];
    }
    if (p.gate != nullptr) {
      load_row8<T>(p.gate, b * p.gate_bs + c0, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] *= t[j];
    }
    if (p.w != nullptr) load_vec<float, 8>(p.w + c0, cw);
    if (p.scale != nullptr) {
      load_row8<T>(p.scale, b * p.mod_bs + c0, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) cw[j] = fmaf(cw[j], t[j], cw[j]);
    }
  };
  auto flush = [&]() {  // the column sums of sample acc_b
    if (acc_b >= 0 && on) {
      float* dst = q.partial + (long long)(unit + acc_b) * 3 * p.D + c0;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        store_vec<float, 8>(dst + (long long)i * p.D, acc[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
      }
    }
  };
  for (int i = 0; i < g.steps; ++i) {
    const int stage = i % SW_STAGES;
    const int n = span_rows(p.M, row0, g.span, i * R, R);
    const long long row = row0 + (long long)i * R;
    float ry[R], rx[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ry[r] = p.post_w != nullptr && r < n ? p.rstd_y[row + r] : 1.f;
      rx[r] = p.w != nullptr && r < n ? p.rstd_x[row + r] : 0.f;
    }
    mbar_wait(&ring.full[stage], (i / SW_STAGES) & 1, err, ERR_MBAR_TIMEOUT_PRODUCER);
    Raw<T, 8> x[R], y[R], dh[R], e[R];
    float s[3 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[3 * r] = s[3 * r + 1] = s[3 * r + 2] = 0.f;
      dh[r].zero();
      e[r].zero();
      if (r >= n || !on) {
        x[r].zero();
        y[r].zero();
        continue;
      }
      sample(per_sample ? (int)((row + r) / p.T) : 0);
      x[r].load(ring.row(stage, 0, group, r, p.D) + c0);
      y[r].load(ring.row(stage, 1, group, r, p.D) + c0);
      if (q.dh != nullptr) dh[r].load(ring.row(stage, 2, group, r, p.D) + c0);
      if (q.dx_new != nullptr) e[r].load(ring.row(stage, 3, group, r, p.D) + c0);
      float xf[8], yf[8], gf[8], ef[8];
      x[r].get(xf);
      y[r].get(yf);
      dh[r].get(gf);
      e[r].get(ef);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float ay = a[j] * (yf[j] * ry[r]);
        const float nn = (xf[j] + ay) * rx[r];
        const float c = gf[j] * cw[j];
        s[3 * r] = fmaf(c, nn, s[3 * r]);
        s[3 * r + 1] = fmaf(ay, fmaf(rx[r], c, ef[j]), s[3 * r + 1]);
        s[3 * r + 2] = fmaf(ay, nn, s[3 * r + 2]);
      }
    }
    group_put<3 * R>(s, red[i & 1], warps);
    __syncthreads();
    if (threadIdx.x == 0 && i + SW_STAGES < g.steps) sw_load<T, R, 4>(ring, g, p.M, p.D, i + SW_STAGES, src);
    group_get<3 * R>(s, red[i & 1], warps, w0, wpg);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= n || !on) continue;
      const int b = per_sample ? (int)((row + r) / p.T) : 0;
      if (b != acc_b) {
        flush();
        acc_b = b;
      }
      sample(b);
      const float m = s[3 * r] / p.D;
      const float m2 = p.post_w != nullptr ? (s[3 * r + 1] - rx[r] * m * s[3 * r + 2]) / p.D : 0.f;
      float xf[8], yf[8], gf[8], ef[8];
      x[r].get(xf);
      y[r].get(yf);
      dh[r].get(gf);
      e[r].get(ef);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float yn = yf[j] * ry[r];
        const float nn = fmaf(a[j], yn, xf[j]) * rx[r];
        const float gx = fmaf(rx[r], fmaf(gf[j], cw[j], -nn * m), ef[j]);
        acc[0][j] += gf[j];
        acc[1][j] = fmaf(gf[j], nn, acc[1][j]);
        acc[2][j] = fmaf(gx, yn, acc[2][j]);
        xf[j] = gx;
        yf[j] = ry[r] * fmaf(a[j], gx, -yn * m2);
      }
      store_vec<T, 8>(reinterpret_cast<T*>(q.dx) + (row + r) * p.D + c0, xf);
      store_vec<T, 8>(reinterpret_cast<T*>(q.dy) + (row + r) * p.D + c0, yf);
    }
  }
  flush();
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

// rows of the vector form per step and group: two 16-bit rows or one fp32 row
template <typename T>
struct SwRows {
  static constexpr int R = sizeof(T) == 2 ? 2 : 1;
};
int sw_rows(int elem) { return elem == ELEM_F32 ? SwRows<float>::R : SwRows<__half>::R; }

bool sw_vectors(const SandwichParams& p, const SandwichBwdParams* q) {
  if (p.D % 8 != 0 || p.D > SW_MAX_VEC_D || p.gate_bs % 8 != 0 || p.mod_bs % 8 != 0) return false;
  uintptr_t bits = 0;
  for (const void* t : {p.x, p.y, p.gate, p.shift, p.scale, (const void*)p.post_w, (const void*)p.w,
                        (const void*)p.x_new, (const void*)p.h})
    bits |= reinterpret_cast<uintptr_t>(t);
  if (q != nullptr)
    for (const void* t : {q->dx_new, q->dh, (const void*)q->dx, (const void*)q->dy}) bits |= reinterpret_cast<uintptr_t>(t);
  return (bits & 15) == 0;
}

// groups of a block: about 256 threads; spans that fill every SM with the blocks that its shared memory holds (at most 2)
int sw_smem(const SandwichParams& p, const SwGeom& g, int R, int tensors, int es) {
  return 128 + SW_STAGES * tensors * g.groups * R * p.D * es;
}
SwGeom sw_geom(const SandwichParams& p, int R, int tensors, int es) {
  SwGeom g;
  g.tpg = (p.D / 8 + 31) / 32 * 32;
  g.groups = std::max(1, 256 / g.tpg);
  const int fit = 226 * 1024 / (sw_smem(p, g, R, tensors, es) + 2048);
  const int units = num_sms() * std::max(1, std::min(fit, 2)) * g.groups;
  g.span = (p.M + units - 1) / units;
  g.span = (g.span + R - 1) / R * R;
  g.steps = g.span / R;
  return g;
}
int sw_blocks(const SandwichParams& p, const SwGeom& g) {
  const int units = (p.M + g.span - 1) / g.span;
  return (units + g.groups - 1) / g.groups;
}

template <typename K>
cudaError_t sw_smem_limit(K kernel, int smem, int* allowed) {
  if (smem <= *allowed) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) *allowed = smem;
  return e;
}

template <typename T>
cudaError_t fwd_run(const SandwichParams& p, int* err, cudaStream_t s) {
  constexpr int R = SwRows<T>::R;
  if (sw_vectors(p, nullptr)) {
    const SwGeom g = sw_geom(p, R, 2, sizeof(T));
    const int smem = sw_smem(p, g, R, 2, sizeof(T));
    static int allowed = 46 * 1024;
    cudaError_t e = sw_smem_limit(sandwich_fwd_kernel<T, R>, smem, &allowed);
    if (e != cudaSuccess) return e;
    sandwich_fwd_kernel<T, R><<<sw_blocks(p, g), g.tpg * g.groups, smem, s>>>(p, g, err);
  } else {
    sandwich_fwd_any_kernel<T><<<std::min(p.M, num_sms() * 8), SW_THREADS, 0, s>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t bwd_run(const SandwichParams& p, const SandwichBwdParams& q, int* err, cudaStream_t s) {
  cudaError_t e;
  if (sw_vectors(p, &q)) {
    constexpr int R = SwRows<T>::R;
    const SwGeom g = sw_geom(p, R, 4, sizeof(T));
    const int smem = sw_smem(p, g, R, 4, sizeof(T));
    static int allowed = 46 * 1024;
    e = sw_smem_limit(sandwich_bwd_kernel<T, R>, smem, &allowed);
    if (e != cudaSuccess) return e;
    sandwich_bwd_kernel<T, R><<<sw_blocks(p, g), g.tpg * g.groups, smem, s>>>(p, q, g, err);
  } else {
    const int smem = 3 * p.D * (int)sizeof(float);
    static int allowed = 46 * 1024;
    e = sw_smem_limit(sandwich_bwd_any_kernel<T>, smem, &allowed);
    if (e != cudaSuccess) return e;
    sandwich_bwd_any_kernel<T><<<q.ctas, SW_THREADS, smem, s>>>(p, q);
  }
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  sandwich_reduce_kernel<T><<<dim3((p.D + 31) / 32, q.groups), dim3(32, RED_ROWS), 0, s>>>(p, q);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (q.dw != nullptr || q.dpost_w != nullptr)
    sandwich_weights_kernel<<<(p.D + 127) / 128, 128, 0, s>>>(p, q);
  return cudaGetLastError();
}

}  // namespace

cudaError_t sandwich_fwd_launch(const SandwichParams& p, int elem, int* err, cudaStream_t s) {
  if (p.M <= 0 || p.D <= 0) return cudaSuccess;
  switch (elem) {
    case ELEM_BF16: return fwd_run<__nv_bfloat16>(p, err, s);
    case ELEM_F16: return fwd_run<__half>(p, err, s);
    case ELEM_F32: return fwd_run<float>(p, err, s);
  }
  return cudaErrorInvalidValue;
}

void sandwich_bwd_plan(const SandwichParams& p, int elem, SandwichBwdParams* q) {
  if (sw_vectors(p, q)) {
    const SwGeom g = sw_geom(p, sw_rows(elem), 4, elem == ELEM_F32 ? 4 : 2);
    q->rows_per_cta = g.span;
  } else {
    const int most = num_sms() * 4;
    q->rows_per_cta = std::max(1, (p.M + most - 1) / most);
  }
  q->ctas = (p.M + q->rows_per_cta - 1) / q->rows_per_cta;
  q->groups = std::min(samples_of(p), 64);
}

cudaError_t sandwich_bwd_launch(const SandwichParams& p, const SandwichBwdParams& q, int elem, int* err,
                                cudaStream_t s) {
  if (p.M <= 0 || p.D <= 0) return cudaSuccess;
  switch (elem) {
    case ELEM_BF16: return bwd_run<__nv_bfloat16>(p, q, err, s);
    case ELEM_F16: return bwd_run<__half>(p, q, err, s);
    case ELEM_F32: return bwd_run<float>(p, q, err, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tgo

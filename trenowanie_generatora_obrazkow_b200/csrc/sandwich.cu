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

#ifndef STAGES
#define STAGES 3
#endif
constexpr int SW_STAGES = STAGES;
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
__device__ __forceinline__ void load_row8(const void* base, long long off, f32x2 (&v)[4]) {
  Raw<T, 8> r;
  r.load(reinterpret_cast<const T*>(base) + off);
  unpack_x2<T>(r, v);
}
__device__ __forceinline__ void load_w8(const float* p, f32x2 (&v)[4]) {
  Raw<float, 8> r;
  r.load(p);
  unpack_x2<float>(r, v);
}

// N sums over a group's warps. Step 1 (group_put): the lanes' values are summed over the warp while their number is
// halved (a lane pair exchanges the halves that the other keeps), so N values cost about N + 5 shuffles instead of 5 N;
// one lane per value writes it to red[value][group's slot of this warp]. Step 2 (group_get), after the caller's barrier:
// every thread adds the group's slots (padded with zeros to float4s).
constexpr int RED_PITCH = 32;
template <int N>
__device__ __forceinline__ void group_put(float (&v)[N], float* red, int slot) {
  static_assert(N == 1 || N == 2 || N == 4 || N == 8, "a power of two");
  int keep = 0, bit = 16;
#pragma unroll
  for (int h = N / 2; h >= 1; h >>= 1) {
    const bool up = lane_id() & bit;
#pragma unroll
    for (int i = 0; i < h; ++i) {
      const float give = up ? v[i] : v[i + h], mine = up ? v[i + h] : v[i];
      v[i] = mine + __shfl_xor_sync(0xffffffffu, give, bit);
    }
    keep += up ? h : 0;
    bit >>= 1;
  }
  float t = v[0];
#pragma unroll
  for (int o = 16 / N; o >= 1; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if ((lane_id() & (32 / N - 1)) == 0) red[keep * RED_PITCH + slot] = t;
}
template <int N>
__device__ __forceinline__ void group_get(float (&v)[N], const float* red, int first, int quads) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float4* q = reinterpret_cast<const float4*>(red + i * RED_PITCH + first);
    float4 t = q[0];
    for (int k = 1; k < quads; ++k) {
      const float4 u = q[k];
      t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
    }
    v[i] = (t.x + t.y) + (t.z + t.w);
  }
}

// Position of a unit in its samples, advanced step by step (no division in the row loop). R divides T, so a step never
// straddles two samples.
struct SwSample {
  int b, t, T;
  __device__ __forceinline__ SwSample(const SandwichParams& p, bool per_sample, long long row) {
    T = per_sample ? p.T : 0x7fffffff;
    b = per_sample ? (int)(row / p.T) : 0;
    t = per_sample ? (int)(row - (long long)b * p.T) : 0;
  }
  __device__ __forceinline__ bool next(int rows) {  // true: a new sample begins
    t += rows;
    if (t < T) return false;
    t = 0;
    ++b;
    return true;
  }
};

// a = res_scale gate post_w and cw = w (1 + scale) of sample b, channels c0 .. c0 + 7
template <typename T>
__device__ __forceinline__ void sw_constants(const SandwichParams& p, int b, int c0, f32x2 (&a)[4], f32x2 (&cw)[4]) {
  f32x2 t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] = x2(p.res_scale), cw[j] = x2(0.f);
  if (p.post_w != nullptr) {
    load_w8(p.post_w + c0, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = x2_mul(a[j], t[j]);
  }
  if (p.gate != nullptr) {
    load_row8<T>(p.gate, b * p.gate_bs + c0, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = x2_mul(a[j], t[j]);
  }
  if (p.w != nullptr) load_w8(p.w + c0, cw);
  if (p.scale != nullptr) {
    load_row8<T>(p.scale, b * p.mod_bs + c0, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) cw[j] = x2_fma(cw[j], t[j], cw[j]);
  }
}

}  // namespace

// Threads past the last channel of a row (D / 8 not a multiple of 32) work on channel 0's values and keep their sums at 0.
template <typename T, int R, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) sandwich_fwd_kernel(SandwichParams p, SwGeom g, int* err) {
  extern __shared__ __align__(128) uint8_t sw_smem[];
  __shared__ __align__(16) float red[2][R * RED_PITCH];
  const int group = threadIdx.x / g.tpg, tc = (threadIdx.x % g.tpg) * 8;
  const bool on = tc < p.D, lead = tc == 0;
  const int c0 = on ? tc : 0;
  const int wpg = g.tpg >> 5, quads = (wpg + 3) >> 2, first = group * quads * 4, slot = first + warp_id() - group * wpg;
  const long long row0 = ((long long)blockIdx.x * g.groups + group) * g.span;
  const float inv_d = 1.f / p.D;
  const SwRing<T, R, 2> ring(sw_smem, g, p.D);
  const void* const src[2] = {p.x, p.y};
  for (int i = threadIdx.x; i < 2 * R * RED_PITCH; i += blockDim.x) (&red[0][0])[i] = 0.f;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SW_STAGES; ++s) mbar_init(&ring.full[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < SW_STAGES && i < g.steps; ++i) sw_load<T, R, 2>(ring, g, p.M, p.D, i, src);
  }
  __syncthreads();
  const int rows = (int)max(0ll, min((long long)g.span, p.M - row0));
  SwSample at(p, samples_of(p) > 1, row0);
  const bool post = p.post_w != nullptr, pre = p.w != nullptr;
  f32x2 a[4], cw[4], sh[4];
  auto sample = [&]() {
    sw_constants<T>(p, at.b, c0, a, cw);
#pragma unroll
    for (int j = 0; j < 4; ++j) sh[j] = x2(0.f);
    if (p.scale != nullptr) load_row8<T>(p.shift, at.b * p.mod_bs + c0, sh);
  };
  if (rows > 0) sample();
  const T* slots = ring.row(0, 0, group, 0, p.D) + c0;
  const int to_y = (int)(ring.tensor_bytes / sizeof(T)), to_stage = (int)(ring.step_bytes / sizeof(T));
  T* out_x = reinterpret_cast<T*>(p.x_new) + row0 * p.D + c0;
  T* out_h = reinterpret_cast<T*>(p.h) + row0 * p.D + c0;
  float *st_y = p.rstd_y + row0, *st_x = p.rstd_x + row0;
  int stage = 0, phase = 0, left = rows;  // left <= 0: only the barriers
  for (int i = 0; i < g.steps; ++i) {
    mbar_wait(&ring.full[stage], phase, err, ERR_MBAR_TIMEOUT_PRODUCER);
    Raw<T, 8> x[R], y[R];
    float s[R];
    const T* in = slots + stage * to_stage;
#pragma unroll
    for (int r = 0; r < R; ++r) {  // a missing last row reads what its slot held: its results go nowhere
      x[r].load(in + r * p.D);
      y[r].load(in + to_y + r * p.D);
      f32x2 q = x2(0.f), f[4];
      unpack_x2<T>(y[r], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) q = x2_fma(f[j], f[j], q);
      s[r] = on ? x2_sum(q) : 0.f;
    }
    group_put<R>(s, red[0], slot);
    __syncthreads();  // every thread has taken its rows out of the stage: refill it
    if (threadIdx.x == 0 && i + SW_STAGES < g.steps) sw_load<T, R, 2>(ring, g, p.M, p.D, i + SW_STAGES, src);
    if (++stage == SW_STAGES) stage = 0, phase ^= 1;
    group_get<R>(s, red[0], first, quads);
    f32x2 xn[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float ry = post ? rsqrtf(fmaf(s[r], inv_d, p.eps)) : 1.f;
      if (lead && post && r < left) st_y[r] = ry;
      f32x2 f[4], q = x2(0.f);
      const f32x2 ry2 = x2(ry);
      unpack_x2<T>(x[r], xn[r]);
      unpack_x2<T>(y[r], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        xn[r][j] = x2_fma(x2_mul(f[j], ry2), a[j], xn[r][j]);
        q = x2_fma(xn[r][j], xn[r][j], q);
      }
      s[r] = on ? x2_sum(q) : 0.f;
      if (on && r < left) store_x2<T>(out_x + r * p.D, xn[r]);
    }
    group_put<R>(s, red[1], slot);
    __syncthreads();
    if (pre) {
      group_get<R>(s, red[1], first, quads);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float rx = rsqrtf(fmaf(s[r], inv_d, p.eps));
        const f32x2 rx2 = x2(rx);
#pragma unroll
        for (int j = 0; j < 4; ++j) xn[r][j] = x2_fma(x2_mul(xn[r][j], rx2), cw[j], sh[j]);
        if (r < left) {
          if (lead) st_x[r] = rx;
          if (on) store_x2<T>(out_h + r * p.D, xn[r]);
        }
      }
    }
    out_x += R * p.D;
    out_h += R * p.D;
    st_y += R;
    st_x += R;
    left -= R;
    if (at.next(R) && left > 0) sample();
  }
}

// One barrier per step: what the second half needs of a row is kept as fp32 (w1 = dx' + rx dh cw, n, yn).
template <typename T, int R, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) sandwich_bwd_kernel(SandwichParams p, SandwichBwdParams q, SwGeom g,
                                                                  int* err) {
  constexpr int N = R == 1 ? 4 : 8;  // three sums per row
  extern __shared__ __align__(128) uint8_t sw_smem[];
  __shared__ __align__(16) float red[2][N * RED_PITCH];
  const int group = threadIdx.x / g.tpg, tc = (threadIdx.x % g.tpg) * 8;
  const bool on = tc < p.D;
  const int c0 = on ? tc : 0;
  const int wpg = g.tpg >> 5, quads = (wpg + 3) >> 2, first = group * quads * 4, slot = first + warp_id() - group * wpg;
  const int unit = blockIdx.x * g.groups + group;
  const long long row0 = (long long)unit * g.span;
  const float inv_d = 1.f / p.D;
  const SwRing<T, R, 4> ring(sw_smem, g, p.D);
  const void* const src[4] = {p.x, p.y, q.dh, q.dx_new};
  for (int i = threadIdx.x; i < 2 * N * RED_PITCH; i += blockDim.x) (&red[0][0])[i] = 0.f;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SW_STAGES; ++s) mbar_init(&ring.full[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < SW_STAGES && i < g.steps; ++i) sw_load<T, R, 4>(ring, g, p.M, p.D, i, src);
  }
  __syncthreads();
  const int rows = (int)max(0ll, min((long long)g.span, p.M - row0));
  SwSample at(p, samples_of(p) > 1, row0);
  const bool post = p.post_w != nullptr, pre = p.w != nullptr;
  f32x2 a[4], cw[4], acc[3][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[0][j] = acc[1][j] = acc[2][j] = x2(0.f);
  if (rows > 0) sw_constants<T>(p, at.b, c0, a, cw);
  const T* slots = ring.row(0, 0, group, 0, p.D) + c0;
  const int to_next = (int)(ring.tensor_bytes / sizeof(T)), to_stage = (int)(ring.step_bytes / sizeof(T));
  T* out_x = reinterpret_cast<T*>(q.dx) + row0 * p.D + c0;
  T* out_y = reinterpret_cast<T*>(q.dy) + row0 * p.D + c0;
  const float *st_y = p.rstd_y + row0, *st_x = p.rstd_x + row0;
  float ry[R], rx[R];
  int stage = 0, phase = 0, left = rows;
  auto stats = [&](int first_row) {  // the forward's statistics of a step's rows
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ry[r] = post && first_row + r < rows ? st_y[first_row + r] : 1.f;
      rx[r] = pre && first_row + r < rows ? st_x[first_row + r] : 0.f;
    }
  };
  stats(0);
  for (int i = 0; i < g.steps; ++i) {
    mbar_wait(&ring.full[stage], phase, err, ERR_MBAR_TIMEOUT_PRODUCER);
    f32x2 w1[R][4], nn[R][4], yn[R][4];
    float s[N], ky[R];
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ky[r] = ry[r];
      if (r < left && on) {
        const T* in = slots + stage * to_stage + r * p.D;
        Raw<T, 8> x, y, gh, e;
        x.load(in);
        y.load(in + to_next);
        if (q.dh != nullptr) gh.load(in + 2 * to_next);
        else gh.zero();
        if (q.dx_new != nullptr) e.load(in + 3 * to_next);
        else e.zero();
        f32x2 gf[4];
        unpack_x2<T>(x, nn[r]);
        unpack_x2<T>(y, yn[r]);
        unpack_x2<T>(gh, gf);
        unpack_x2<T>(e, w1[r]);
        const f32x2 ry2 = x2(ry[r]), rx2 = x2(rx[r]);
        f32x2 s0 = x2(0.f), s1 = x2(0.f), s2 = x2(0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          yn[r][j] = x2_mul(yn[r][j], ry2);
          const f32x2 ay = x2_mul(a[j], yn[r][j]);
          nn[r][j] = x2_mul(x2_add(nn[r][j], ay), rx2);
          const f32x2 c = x2_mul(gf[j], cw[j]);
          w1[r][j] = x2_fma(rx2, c, w1[r][j]);
          s0 = x2_fma(c, nn[r][j], s0);
          s1 = x2_fma(ay, w1[r][j], s1);
          s2 = x2_fma(ay, nn[r][j], s2);
          acc[0][j] = x2_add(acc[0][j], gf[j]);
          acc[1][j] = x2_fma(gf[j], nn[r][j], acc[1][j]);
        }
        s[3 * r] = x2_sum(s0) * rx[r];  // rx m D
        s[3 * r + 1] = x2_sum(s1);
        s[3 * r + 2] = x2_sum(s2);
      }
    }
    group_put<N>(s, red[i & 1], slot);
    stats((i + 1) * R);  // in flight across the barrier
    __syncthreads();
    if (threadIdx.x == 0 && i + SW_STAGES < g.steps) sw_load<T, R, 4>(ring, g, p.M, p.D, i + SW_STAGES, src);
    if (++stage == SW_STAGES) stage = 0, phase ^= 1;
    float sum[3 * R];
    group_get<3 * R>(sum, red[i & 1], first, quads);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < left && on) {
        const float m = sum[3 * r] * inv_d;
        const float m2 = post ? ky[r] * (sum[3 * r + 1] - m * sum[3 * r + 2]) * inv_d : 0.f;
        const f32x2 ry2 = x2(ky[r]), nm = x2(-m), nm2 = x2(-m2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w1[r][j] = x2_fma(nm, nn[r][j], w1[r][j]);
          acc[2][j] = x2_fma(w1[r][j], yn[r][j], acc[2][j]);
          yn[r][j] = x2_fma(nm2, yn[r][j], x2_mul(ry2, x2_mul(a[j], w1[r][j])));
        }
        store_x2<T>(out_x + r * p.D, w1[r]);
        store_x2<T>(out_y + r * p.D, yn[r]);
      }
    }
    out_x += R * p.D;
    out_y += R * p.D;
    const bool had = left > 0;
    left -= R;
    const int b = at.b;
    const bool turn = at.next(R);
    if (had && on && (turn || left <= 0)) {  // the sample's or the unit's last step: its column sums go out
      float* dst = q.partial + (long long)(unit + b) * 3 * p.D + c0;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        store_x2<float>(dst + (long long)k * p.D, acc[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[k][j] = x2(0.f);
      }
    }
    if (turn && left > 0) sw_constants<T>(p, at.b, c0, a, cw);
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

#ifndef FWD_R
#define FWD_R 2
#define BWD_R 2
#define FWD_B 2
#define BWD_B 2
#endif
// rows per step and group: two rows share a barrier where a sample's rows come in pairs (16-bit types)
int sw_rows(const SandwichParams& p, int es, int most) {
  return es == 2 && most == 2 && (samples_of(p) == 1 || p.T % 2 == 0) ? 2 : 1;
}

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

// groups of a block: about 256 threads; spans that fill every SM with the blocks that its shared memory holds, up to `blocks`
int sw_smem(const SandwichParams& p, const SwGeom& g, int R, int tensors, int es) {
  return 128 + SW_STAGES * tensors * g.groups * R * p.D * es;
}
SwGeom sw_geom(const SandwichParams& p, int R, int tensors, int es, int blocks) {
  SwGeom g;
  g.tpg = (p.D / 8 + 31) / 32 * 32;
  g.groups = std::max(1, 256 / g.tpg);
  const int fit = 226 * 1024 / (sw_smem(p, g, R, tensors, es) + 2048);
  const int units = num_sms() * std::max(1, std::min(fit, blocks)) * g.groups;
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

template <typename T, int R, int MAXT, int MINB>
cudaError_t fwd_vec(const SandwichParams& p, const SwGeom& g, int* err, cudaStream_t s) {
  const int smem = sw_smem(p, g, R, 2, sizeof(T));
  static int allowed = 44 * 1024;
  cudaError_t e = sw_smem_limit(sandwich_fwd_kernel<T, R, MAXT, MINB>, smem, &allowed);
  if (e != cudaSuccess) return e;
  sandwich_fwd_kernel<T, R, MAXT, MINB><<<sw_blocks(p, g), g.tpg * g.groups, smem, s>>>(p, g, err);
  return cudaGetLastError();
}
template <typename T, int R, int MAXT, int MINB>
cudaError_t bwd_vec(const SandwichParams& p, const SandwichBwdParams& q, const SwGeom& g, int* err, cudaStream_t s) {
  const int smem = sw_smem(p, g, R, 4, sizeof(T));
  static int allowed = 44 * 1024;
  cudaError_t e = sw_smem_limit(sandwich_bwd_kernel<T, R, MAXT, MINB>, smem, &allowed);
  if (e != cudaSuccess) return e;
  sandwich_bwd_kernel<T, R, MAXT, MINB><<<sw_blocks(p, g), g.tpg * g.groups, smem, s>>>(p, q, g, err);
  return cudaGetLastError();
}

template <typename T>
cudaError_t fwd_run(const SandwichParams& p, int* err, cudaStream_t s) {
  if (!sw_vectors(p, nullptr)) {
    sandwich_fwd_any_kernel<T><<<std::min(p.M, num_sms() * 8), SW_THREADS, 0, s>>>(p);
    return cudaGetLastError();
  }
  const int R = sw_rows(p, sizeof(T), FWD_R);
  const SwGeom g = sw_geom(p, R, 2, sizeof(T), FWD_B);
  const bool narrow = g.tpg * g.groups <= 256;
  if constexpr (sizeof(T) == 2) {
    if (R == 2) return narrow ? fwd_vec<T, 2, 256, FWD_B>(p, g, err, s) : fwd_vec<T, 2, 512, 1>(p, g, err, s);
  }
  return narrow ? fwd_vec<T, 1, 256, FWD_B>(p, g, err, s) : fwd_vec<T, 1, 512, 1>(p, g, err, s);
}

template <typename T>
cudaError_t bwd_rows(const SandwichParams& p, const SandwichBwdParams& q, int* err, cudaStream_t s) {
  const int R = sw_rows(p, sizeof(T), BWD_R);
  const SwGeom g = sw_geom(p, R, 4, sizeof(T), BWD_B);
  const bool narrow = g.tpg * g.groups <= 256;
#if BWD_R == 2
  if constexpr (sizeof(T) == 2) {
    if (R == 2) return narrow ? bwd_vec<T, 2, 256, BWD_B>(p, q, g, err, s) : bwd_vec<T, 2, 512, 1>(p, q, g, err, s);
  }
#endif
  return narrow ? bwd_vec<T, 1, 256, BWD_B>(p, q, g, err, s) : bwd_vec<T, 1, 512, 1>(p, q, g, err, s);
}

template <typename T>
cudaError_t bwd_run(const SandwichParams& p, const SandwichBwdParams& q, int* err, cudaStream_t s) {
  cudaError_t e;
  if (sw_vectors(p, &q)) {
    e = bwd_rows<T>(p, q, err, s);
    if (e != cudaSuccess) return e;
  } else {
    const int smem = 3 * p.D * (int)sizeof(float);
    static int allowed = 46 * 1024;
    e = sw_smem_limit(sandwich_bwd_any_kernel<T>, smem, &allowed);
    if (e != cudaSuccess) return e;
    sandwich_bwd_any_kernel<T><<<q.ctas, SW_THREADS, smem, s>>>(p, q);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
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
    const int es = elem == ELEM_F32 ? 4 : 2;
    const SwGeom g = sw_geom(p, sw_rows(p, es, BWD_R), 4, es, BWD_B);
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

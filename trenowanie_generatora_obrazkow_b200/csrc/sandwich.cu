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
// Bound by memory (4 rows forward, 6 backward): the kernels of 32 x 1024 x 2048 bf16 take 92 / 161 us, 0.89 / 0.76 of a plain
// copy's rate; below it the row reductions' barriers and, backward, 128 registers (16 warps per SM) are what is left.
//
// Column sums: a unit (a CTA, or a group of its threads) owns a contiguous span of rows and writes one partial row (three
// sums per channel) per sample it meets. Entry unit + sample is unique (along the spans both only grow), so
// units + samples entries hold them all. A second launch adds them in a fixed order, and from 257 samples on a third the
// weights' sums of its groups of samples.
#include <algorithm>
#include <vector>

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

constexpr int SW_STAGES = 2;  // 3 and 4: the backward at 32 x 1024 x 2048 takes 178 and 207 us instead of 170
constexpr int SW_MAX_VEC_D = 4096;
constexpr int SW_MAX_GROUPS = 8;  // 256 threads of 32 each

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

// rows of a step that starts at `row` with `left` rows of its span to go
__device__ __forceinline__ int step_rows(int M, long long row, int left, int R) {
  return max(0, min(min(R, left), (int)min((long long)R, M - row)));
}

// one thread: the rows of step i of every group of this block, all tensors
template <typename T, int R, int TENSORS>
__device__ __forceinline__ void sw_load(const SwRing<T, R, TENSORS>& ring, const SwGeom& g, int M, int D, int i,
                                        int stage, const void* const (&src)[TENSORS]) {
  const int present = TENSORS == 2 ? 2 : 2 + (src[2] != nullptr) + (src[TENSORS - 1] != nullptr);
  const long long row0 = (long long)blockIdx.x * g.groups * g.span + i * R;
  const int row_bytes = D * (int)sizeof(T);
  uint8_t* slot = ring.base + stage * ring.step_bytes;
  int total = 0;
  for (int k = 0; k < g.groups; ++k) total += step_rows(M, row0 + (long long)k * g.span, g.span - i * R, R);
  mbar_expect_tx(&ring.full[stage], (uint32_t)(total * row_bytes * present));
  for (int k = 0; k < g.groups; ++k) {
    const long long row = row0 + (long long)k * g.span;
    const int bytes = step_rows(M, row, g.span - i * R, R) * row_bytes;
    if (bytes <= 0) continue;
#pragma unroll
    for (int t = 0; t < TENSORS; ++t)
      if (t < 2 || src[t] != nullptr)
        bulk_load(slot + t * ring.tensor_bytes + k * ring.group_bytes,
                  reinterpret_cast<const T*>(src[t]) + row * D, (uint32_t)bytes, &ring.full[stage]);
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

// V sums over a group's warps (P slots, wpg <= P of them used, the others hold zeros).
// group_put: the lanes' values are summed over the warp while their number is halved (a lane pair exchanges the halves
// that the other keeps), so V values cost about V + 5 shuffles instead of 5 V; one lane per value writes red[v P + slot].
// group_total, after the caller's barrier: lane l of every warp takes the entries l, l + 32, ... and the P slots of a value,
// which sit in neighbouring lanes, are added by shuffles. Value v is then in every lane of its P, of register v P / 32.
template <int V, int P>
__device__ __forceinline__ void group_put(float (&v)[V], float* red, int slot) {
  static_assert(V == 1 || V == 2 || V == 4 || V == 8, "a power of two");
  int keep = 0, bit = 16;
#pragma unroll
  for (int h = V / 2; h >= 1; h >>= 1) {
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
  for (int o = 16 / V; o >= 1; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if ((lane_id() & (32 / V - 1)) == 0) red[keep * P + slot] = t;
}
template <int V, int P>
struct Totals {
  static constexpr int K = (V * P + 31) / 32;
  float t[K];
  __device__ __forceinline__ explicit Totals(const float* red) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = k * 32 + lane_id();
      t[k] = V * P >= 32 || i < V * P ? red[i] : 0.f;
#pragma unroll
      for (int o = 1; o < P; o <<= 1) t[k] += __shfl_xor_sync(0xffffffffu, t[k], o);
    }
  }
  __device__ __forceinline__ float get(int v) const { return __shfl_sync(0xffffffffu, t[v * P / 32], v * P % 32); }
};

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
template <typename T, int R, int P, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) sandwich_fwd_kernel(SandwichParams p, SwGeom g, int* err) {
  extern __shared__ __align__(128) uint8_t sw_smem[];
  __shared__ float reds[2][SW_MAX_GROUPS * R * P];
  const int group = threadIdx.x / g.tpg, tc = (threadIdx.x % g.tpg) * 8;
  const bool on = tc < p.D;
  const int c0 = on ? tc : 0;
  const int slot = warp_id() - group * (g.tpg >> 5);
  const long long row0 = ((long long)blockIdx.x * g.groups + group) * g.span;
  const float inv_d = 1.f / p.D;
  const SwRing<T, R, 2> ring(sw_smem, g, p.D);
  const void* const src[2] = {p.x, p.y};
  for (int i = threadIdx.x; i < 2 * SW_MAX_GROUPS * R * P; i += blockDim.x) (&reds[0][0])[i] = 0.f;
  float* const red[2] = {reds[0] + group * R * P, reds[1] + group * R * P};
  if (threadIdx.x == 0) {
    for (int s = 0; s < SW_STAGES; ++s) mbar_init(&ring.full[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < SW_STAGES && i < g.steps; ++i) sw_load<T, R, 2>(ring, g, p.M, p.D, i, i, src);
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
    group_put<R, P>(s, red[0], slot);
    __syncthreads();  // every thread has taken its rows out of the stage: refill it
    if (threadIdx.x == 0 && i + SW_STAGES < g.steps) sw_load<T, R, 2>(ring, g, p.M, p.D, i + SW_STAGES, stage, src);
    if (++stage == SW_STAGES) stage = 0, phase ^= 1;
    // the lanes that hold row r's sum turn it into its statistic once
    Totals<R, P> ty(red[0]);
#pragma unroll
    for (int k = 0; k < Totals<R, P>::K; ++k) {
      ty.t[k] = post ? rsqrtf(fmaf(ty.t[k], inv_d, p.eps)) : 1.f;
      const int r = (k * 32 + lane_id()) / P;
      if (post && slot == 0 && lane_id() % P == 0 && r < R && r < left) st_y[r] = ty.t[k];
    }
    f32x2 xn[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float ry = ty.get(r);
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
    group_put<R, P>(s, red[1], slot);
    __syncthreads();
    if (pre) {
      Totals<R, P> tx(red[1]);
#pragma unroll
      for (int k = 0; k < Totals<R, P>::K; ++k) {
        tx.t[k] = rsqrtf(fmaf(tx.t[k], inv_d, p.eps));
        const int r = (k * 32 + lane_id()) / P;
        if (slot == 0 && lane_id() % P == 0 && r < R && r < left) st_x[r] = tx.t[k];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const f32x2 rx2 = x2(tx.get(r));
#pragma unroll
        for (int j = 0; j < 4; ++j) xn[r][j] = x2_fma(x2_mul(xn[r][j], rx2), cw[j], sh[j]);
        if (on && r < left) store_x2<T>(out_h + r * p.D, xn[r]);
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
template <typename T, int R, int P, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) sandwich_bwd_kernel(SandwichParams p, SandwichBwdParams q, SwGeom g,
                                                                  int* err) {
  constexpr int N = R == 1 ? 4 : 8;  // three sums per row
  extern __shared__ __align__(128) uint8_t sw_smem[];
  __shared__ float reds[2][SW_MAX_GROUPS * N * P];
  const int group = threadIdx.x / g.tpg, tc = (threadIdx.x % g.tpg) * 8;
  const bool on = tc < p.D;
  const int c0 = on ? tc : 0;
  const int slot = warp_id() - group * (g.tpg >> 5);
  const int unit = blockIdx.x * g.groups + group;
  const long long row0 = (long long)unit * g.span;
  const float inv_d = 1.f / p.D;
  const SwRing<T, R, 4> ring(sw_smem, g, p.D);
  const void* const src[4] = {p.x, p.y, q.dh, q.dx_new};
  for (int i = threadIdx.x; i < 2 * SW_MAX_GROUPS * N * P; i += blockDim.x) (&reds[0][0])[i] = 0.f;
  float* const red0 = reds[0] + group * N * P;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SW_STAGES; ++s) mbar_init(&ring.full[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    for (int i = 0; i < SW_STAGES && i < g.steps; ++i) sw_load<T, R, 4>(ring, g, p.M, p.D, i, i, src);
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
    group_put<N, P>(s, red0 + (i & 1) * (SW_MAX_GROUPS * N * P), slot);
    stats((i + 1) * R);  // in flight across the barrier
    __syncthreads();
    if (threadIdx.x == 0 && i + SW_STAGES < g.steps) sw_load<T, R, 4>(ring, g, p.M, p.D, i + SW_STAGES, stage, src);
    if (++stage == SW_STAGES) stage = 0, phase ^= 1;
    const Totals<N, P> sums(red0 + (i & 1) * (SW_MAX_GROUPS * N * P));
    float sum[3 * R];
#pragma unroll
    for (int k = 0; k < 3 * R; ++k) sum[k] = sums.get(k) * inv_d;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < left && on) {
        const float m = sum[3 * r];
        const float m2 = post ? ky[r] * (sum[3 * r + 1] - m * sum[3 * r + 2]) : 0.f;
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

// Sums of a sample's partial rows -> its dshift / dscale / dgate rows, and the weights' sums over this block's samples. A
// block owns 32 channels (lane = channel) and 32 warps: `wps` warps share a sample's rows, so few samples with many rows
// (no modulation: one sample) and many samples with few rows both fill the block.
constexpr int RED_WARPS = 32;
template <typename T>
__global__ void __launch_bounds__(32 * RED_WARPS) sandwich_reduce_kernel(SandwichParams p, SandwichBwdParams q,
                                                                         int wps) {
  __shared__ float part[RED_WARPS][3][32];
  const int samples = samples_of(p);
  const int T_rows = samples > 1 ? p.T : p.M;
  const int lane = lane_id(), warp = warp_id(), share = warp % wps;
  const int c = blockIdx.x * 32 + lane;
  const bool ok = c < p.D;
  const int per = (samples + gridDim.y - 1) / gridDim.y, at_once = RED_WARPS / wps;
  const int b0 = blockIdx.y * per, b1 = min(samples, b0 + per);
  const float w = ok && p.w != nullptr ? p.w[c] : 0.f;
  const float pw = ok && p.post_w != nullptr ? p.post_w[c] : 1.f;
  float sum_w = 0.f, sum_p = 0.f;
  for (int bb = b0; bb < b1; bb += at_once) {
    const int b = bb + warp / wps;
    const bool live = b < b1 && ok;
    float s[3] = {0.f, 0.f, 0.f};
    if (live) {
      const int first = b * T_rows / q.rows_per_cta, last = ((b + 1) * T_rows - 1) / q.rows_per_cta;  // rows fit an int
#pragma unroll 8
      for (int k = first + share; k <= last; k += wps) {
        const float* src = q.partial + (long long)(k + b) * 3 * p.D + c;
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] += src[(long long)i * p.D];
      }
    }
    if (wps > 1) {
#pragma unroll
      for (int i = 0; i < 3; ++i) part[warp][i][lane] = s[i];
      __syncthreads();
      if (share == 0)
        for (int k = 1; k < wps; ++k)
#pragma unroll
          for (int i = 0; i < 3; ++i) s[i] += part[warp + k][i][lane];
      __syncthreads();
    }
    if (live && share == 0) {
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
  }
  part[warp][0][lane] = sum_w;
  part[warp][1][lane] = sum_p;
  __syncthreads();
  if (warp < 2 && ok) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < RED_WARPS; ++k) t += part[k][warp][lane];
    float* dst = warp == 0 ? q.dw : q.dpost_w;
    if (gridDim.y > 1) q.wpart[((long long)blockIdx.y * 2 + warp) * p.D + c] = t;
    else if (dst != nullptr) dst[c] = (warp == 0 ? q.add_w : q.add_post_w) ? dst[c] + t : t;
  }
}

// dw / dpost_w from the groups' sums (only with more than one group of samples)
__global__ void __launch_bounds__(256) sandwich_weights_kernel(SandwichParams p, SandwichBwdParams q) {
  __shared__ float part[8][32];
  const int lane = lane_id(), c = blockIdx.x * 32 + lane;
  float* dst = blockIdx.y == 0 ? q.dw : q.dpost_w;
  float s = 0.f;
  if (c < p.D)
    for (int g = warp_id(); g < q.groups; g += 8) s += q.wpart[((long long)g * 2 + blockIdx.y) * p.D + c];
  part[warp_id()][lane] = s;
  __syncthreads();
  if (warp_id() != 0 || c >= p.D || dst == nullptr) return;
  for (int i = 1; i < 8; ++i) s += part[i][lane];
  dst[c] = (blockIdx.y == 0 ? q.add_w : q.add_post_w) ? dst[c] + s : s;
}

namespace {

// Rows per step and group (16-bit and fp32 rows). 32 samples of 2048 bf16 channels, 1023 rows (one per step, as two do not
// divide them) / 1024 rows (two per step): forward 96 / 92 us, backward 159 / 153 us; fp32 32 x 1024 x 1024 backward 2 rows
// spill (165 us against 155 us with one).
template <typename T>
struct SwRows {
  static constexpr int FWD = 2, BWD = sizeof(T) == 2 ? 2 : 1;
};

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

int sw_threads(const SandwichParams& p, SwGeom* g) {  // groups of a block: about 256 threads
  g->tpg = (p.D / 8 + 31) / 32 * 32;
  g->groups = std::max(1, 256 / g->tpg);
  return g->tpg * g->groups;
}
int sw_blocks(const SandwichParams& p, const SwGeom& g) {
  const int units = (p.M + g.span - 1) / g.span;
  return (units + g.groups - 1) / g.groups;
}

// Calls f(kernel, R, tensors, element size) with the variant for p: R rows per step, as many as divide a sample's rows;
// threads up to 256 (8 slots of the group sums) or 512 (16 slots). The backward of 257 to 320 threads (2056 to 2560
// channels) has a variant of its own, two blocks per SM in 96 registers with one row per step; us at 32 x 1024 x 2560 bf16 / fp32:
// that 201 / 341, in 512 threads with two rows 221 (fp32: one row 355), in 320 threads with two rows 356 (spills). 7 x 333 x
// 2560: 24.3, 25.4, 38.4. The forward needs none: 116 / 240 with 320 threads, 116 / 221 with 512.
template <typename T, int R, typename F>
auto sw_fwd_width(const SandwichParams& p, F f) {
  SwGeom g;
  if (sw_threads(p, &g) <= 256) return f(sandwich_fwd_kernel<T, R, 8, 256, 2>, R, 2, (int)sizeof(T));
  return f(sandwich_fwd_kernel<T, R, 16, 512, 1>, R, 2, (int)sizeof(T));
}
bool sw_bwd_narrow(const SandwichParams& p) {
  SwGeom g;
  const int threads = sw_threads(p, &g);
  return threads > 256 && threads <= 320;
}
template <typename T, int R, typename F>
auto sw_bwd_width(const SandwichParams& p, F f) {
  SwGeom g;
  if (sw_threads(p, &g) <= 256) return f(sandwich_bwd_kernel<T, R, 8, 256, 2>, R, 4, (int)sizeof(T));
  if constexpr (R == 1) {
    if (sw_bwd_narrow(p)) return f(sandwich_bwd_kernel<T, R, 16, 320, 2>, R, 4, (int)sizeof(T));
  }
  return f(sandwich_bwd_kernel<T, R, 16, 512, 1>, R, 4, (int)sizeof(T));
}
template <typename T, int R, typename F>
auto sw_fwd_pick(const SandwichParams& p, F f) {
  if constexpr (R > 1) {
    if (samples_of(p) > 1 && p.T % R != 0) return sw_fwd_pick<T, R / 2>(p, f);
  }
  return sw_fwd_width<T, R>(p, f);
}
template <typename T, int R, typename F>
auto sw_bwd_pick(const SandwichParams& p, F f) {
  if constexpr (R > 1) {
    if ((samples_of(p) > 1 && p.T % R != 0) || sw_bwd_narrow(p)) return sw_bwd_pick<T, R / 2>(p, f);
  }
  return sw_bwd_width<T, R>(p, f);
}

// Resident blocks per SM of a kernel with this block and shared memory; the two runtime calls are made once per thread,
// kernel and shape (they cost as much host time as a launch).
template <typename K>
cudaError_t sw_resident(K kernel, int threads, int smem, int* blocks) {
  struct Known {
    const void* kernel;
    int device, threads, smem, blocks;
  };
  thread_local std::vector<Known> known;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const void* id = reinterpret_cast<const void*>(kernel);
  for (const Known& k : known)
    if (k.kernel == id && k.device == dev && k.threads == threads && k.smem == smem) {
      *blocks = k.blocks;
      return cudaSuccess;
    }
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks, kernel, threads, smem);
  if (e == cudaSuccess && *blocks < 1) e = cudaErrorInvalidValue;
  if (e == cudaSuccess) {
    if (known.size() >= 64) known.clear();
    known.push_back({id, dev, threads, smem, *blocks});
  }
  return e;
}

// Spans that fill every SM with the blocks that it holds.
template <typename K>
cudaError_t sw_geom(K kernel, const SandwichParams& p, int R, int tensors, int es, SwGeom* g, int* smem) {
  const int threads = sw_threads(p, g);
  *smem = 128 + SW_STAGES * tensors * g->groups * R * p.D * es;
  int blocks = 0;
  cudaError_t e = sw_resident(kernel, threads, *smem, &blocks);
  if (e != cudaSuccess) return e;
  const int units = num_sms() * blocks * g->groups;
  g->span = ((p.M + units - 1) / units + R - 1) / R * R;
  g->steps = g->span / R;
  return cudaSuccess;
}

template <typename T>
cudaError_t fwd_run(const SandwichParams& p, int* err, cudaStream_t s) {
  if (!sw_vectors(p, nullptr)) {
    sandwich_fwd_any_kernel<T><<<std::min(p.M, num_sms() * 8), SW_THREADS, 0, s>>>(p);
    return cudaGetLastError();
  }
  return sw_fwd_pick<T, SwRows<T>::FWD>(p, [&](auto kernel, int R, int tensors, int es) {
    SwGeom g;
    int smem;
    cudaError_t e = sw_geom(kernel, p, R, tensors, es, &g, &smem);
    if (e != cudaSuccess) return e;
    kernel<<<sw_blocks(p, g), g.tpg * g.groups, smem, s>>>(p, g, err);
    return cudaGetLastError();
  });
}

template <typename T>
cudaError_t bwd_span(const SandwichParams& p, int* span) {
  return sw_bwd_pick<T, SwRows<T>::BWD>(p, [&](auto kernel, int R, int tensors, int es) {
    SwGeom g;
    int smem;
    cudaError_t e = sw_geom(kernel, p, R, tensors, es, &g, &smem);
    *span = g.span;
    return e;
  });
}

template <typename T>
cudaError_t bwd_run(const SandwichParams& p, const SandwichBwdParams& q, int* err, cudaStream_t s) {
  cudaError_t e;
  if (sw_vectors(p, &q)) {
    e = sw_bwd_pick<T, SwRows<T>::BWD>(p, [&](auto kernel, int R, int tensors, int es) {
      SwGeom g;
      int smem;
      cudaError_t e = sw_geom(kernel, p, R, tensors, es, &g, &smem);
      if (e != cudaSuccess) return e;
      if (g.span != q.rows_per_cta) return cudaErrorInvalidValue;  // the partial sums were laid out for this span
      kernel<<<sw_blocks(p, g), g.tpg * g.groups, smem, s>>>(p, q, g, err);
      return cudaGetLastError();
    });
  } else {
    const int smem = 3 * p.D * (int)sizeof(float);
    e = cudaFuncSetAttribute(sandwich_bwd_any_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    sandwich_bwd_any_kernel<T><<<q.ctas, SW_THREADS, smem, s>>>(p, q);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  int wps = 1;
  while (wps < RED_WARPS && wps * samples_of(p) < RED_WARPS) wps *= 2;
  const int tiles = (p.D + 31) / 32;
  sandwich_reduce_kernel<T><<<dim3(tiles, q.groups), 32 * RED_WARPS, 0, s>>>(p, q, wps);
  e = cudaGetLastError();
  if (e != cudaSuccess || q.groups == 1 || (q.dw == nullptr && q.dpost_w == nullptr)) return e;
  sandwich_weights_kernel<<<dim3(tiles, 2), 256, 0, s>>>(p, q);
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

cudaError_t sandwich_bwd_plan(const SandwichParams& p, int elem, SandwichBwdParams* q) {
  if (sw_vectors(p, q)) {
    cudaError_t e = elem == ELEM_F32    ? bwd_span<float>(p, &q->rows_per_cta)
                    : elem == ELEM_BF16 ? bwd_span<__nv_bfloat16>(p, &q->rows_per_cta)
                                        : bwd_span<__half>(p, &q->rows_per_cta);
    if (e != cudaSuccess) return e;
  } else {
    const int most = num_sms() * 4;
    q->rows_per_cta = std::max(1, (p.M + most - 1) / most);
  }
  q->ctas = (p.M + q->rows_per_cta - 1) / q->rows_per_cta;
  q->groups = std::min((samples_of(p) + 255) / 256, 64);  // more than 256 samples: a block would walk them too long
  return cudaSuccess;
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

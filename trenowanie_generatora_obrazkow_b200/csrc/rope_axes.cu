// q / k RMSNorm (optional) and rotary positions with several axes (time, height, width).
//
// The rot rotated channels of a head form rot / 2 pairs: (2 i, 2 i + 1) interleaved, or (i, i + rot / 2) half-split.
// Pair i belongs to position axis axis[i] and turns by phi = pos[axis[i]] 2 pi freq[i] (freq in revolutions per position):
//     (a, b) -> (a cos phi - b sin phi, b cos phi + a sin phi);       channels past rot pass through.
// The angle is reduced before any sine: pos freq as a product of fp32 and a two-part fp32 constant, of which only the
// fraction of a revolution is kept, so positions of a long clip lose nothing that small ones have (|pos| < 2^24).
// Backward: the transposed rotation, then the norm's gradient with x and its rstd recomputed from q / k:
//     n = x r, gn = w g:   dx = r (gn - n mean(gn n)),   dw = sum over tokens and heads of g n.
//
// Bound by memory: one warp per token, LPH lanes of 8 channels per head; the angles and norm weights of a token are
// set up once in registers and used for all of its q and k heads.
#include <algorithm>

#include "block_ops.h"
#include "common.cuh"
#include "kernels.h"
#include "vec.cuh"

namespace tgo {

namespace {

constexpr int ROPE_WARPS = 8;

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float position(const RopeAxesParams& p, long long tok, int axis) {
  const long long i = tok * p.axes + axis;
  return p.pos_f32 ? reinterpret_cast<const float*>(p.pos)[i] : (float)reinterpret_cast<const int*>(p.pos)[i];
}

// cos / sin of the pair of channel c for token tok
__device__ __forceinline__ void turn_of(const RopeAxesParams& p, long long tok, int pair, float& cs, float& sn) {
  const float pos = position(p, tok, p.axis[pair]);
  const float hi = p.freq[pair], lo = p.freq[p.rot / 2 + pair];
  const float whole = pos * hi;
  float rev = whole - rintf(whole);
  rev += fmaf(pos, hi, -whole) + pos * lo;
  sincospif(2.f * rev, &sn, &cs);
}

}  // namespace

// Any head dim, stride and alignment: one warp per (token, head), channels strided over the lanes.
template <typename T>
__global__ void __launch_bounds__(ROPE_WARPS * 32) rope_axes_any_kernel(RopeAxesParams p) {
  const int heads = p.hq + p.hkv, half = p.rot / 2;
  const long long units = (long long)p.M * heads;
  for (long long u = (long long)blockIdx.x * ROPE_WARPS + warp_id(); u < units; u += (long long)gridDim.x * ROPE_WARPS) {
    const long long tok = u / heads;
    const int hh = (int)(u % heads);
    const bool is_q = hh < p.hq;
    const int h = is_q ? hh : hh - p.hq;
    const T* src = reinterpret_cast<const T*>(is_q ? p.q : p.k) + tok * (is_q ? p.q_ts : p.k_ts) + (long long)h * p.hd;
    T* dst = reinterpret_cast<T*>(is_q ? p.q_out : p.k_out) + (tok * (is_q ? p.hq : p.hkv) + h) * p.hd;
    const float* w = is_q ? p.q_w : p.k_w;
    float r = 1.f;
    if (w != nullptr) {
      float ss = 0.f;
      for (int c = lane_id(); c < p.hd; c += 32) {
        const float v = to_f<T>(src[c]);
        ss = fmaf(v, v, ss);
      }
      r = rsqrtf(warp_total(ss) / p.hd + p.eps);
    }
    auto val = [&](int c) { return to_f<T>(src[c]) * r * (w != nullptr ? w[c] : 1.f); };
    for (int i = lane_id(); i < half; i += 32) {
      const int ca = p.interleaved ? 2 * i : i, cb = p.interleaved ? 2 * i + 1 : i + half;
      float cs, sn;
      turn_of(p, tok, i, cs, sn);
      const float a = val(ca), b = val(cb);
      dst[ca] = from_f<T>(a * cs - b * sn);
      dst[cb] = from_f<T>(b * cs + a * sn);
    }
    for (int c = p.rot + lane_id(); c < p.hd; c += 32) dst[c] = from_f<T>(val(c));
  }
}

// Backward of the same, with the weight gradients of a CTA's units in dynamic shared memory: [warps][2][hd] (each warp
// its own sums; a lane owns its channels).
template <typename T>
__global__ void __launch_bounds__(ROPE_WARPS * 32) rope_axes_bwd_any_kernel(RopeAxesParams p, const T* __restrict__ dq,
                                                                            const T* __restrict__ dk,
                                                                            T* __restrict__ dq_in,
                                                                            T* __restrict__ dk_in,
                                                                            float* __restrict__ partial) {
  extern __shared__ float rope_smem[];
  const int heads = p.hq + p.hkv, half = p.rot / 2;
  float* acc = rope_smem + warp_id() * 2 * p.hd;
  for (int c = lane_id(); c < 2 * p.hd; c += 32) acc[c] = 0.f;
  __syncwarp();
  const long long units = (long long)p.M * heads;
  for (long long u = (long long)blockIdx.x * ROPE_WARPS + warp_id(); u < units; u += (long long)gridDim.x * ROPE_WARPS) {
    const long long tok = u / heads;
    const int hh = (int)(u % heads);
    const bool is_q = hh < p.hq;
    const int h = is_q ? hh : hh - p.hq;
    const T* src = reinterpret_cast<const T*>(is_q ? p.q : p.k) + tok * (is_q ? p.q_ts : p.k_ts) + (long long)h * p.hd;
    const long long o = (tok * (is_q ? p.hq : p.hkv) + h) * p.hd;
    const T* g = (is_q ? dq : dk) + o;
    T* dst = (is_q ? dq_in : dk_in) + o;
    const float* w = is_q ? p.q_w : p.k_w;
    auto pair_grad = [&](int i, int& ca, int& cb, float& ga, float& gb) {
      ca = p.interleaved ? 2 * i : i, cb = p.interleaved ? 2 * i + 1 : i + half;
      float cs, sn;
      turn_of(p, tok, i, cs, sn);
      const float a = to_f<T>(g[ca]), b = to_f<T>(g[cb]);
      ga = a * cs + b * sn;
      gb = b * cs - a * sn;
    };
    if (w == nullptr) {
      for (int i = lane_id(); i < half; i += 32) {
        int ca, cb;
        float ga, gb;
        pair_grad(i, ca, cb, ga, gb);
        dst[ca] = from_f<T>(ga);
        dst[cb] = from_f<T>(gb);
      }
      for (int c = p.rot + lane_id(); c < p.hd; c += 32) dst[c] = g[c];
      continue;
    }
    float* aw = acc + (is_q ? 0 : p.hd);
    float ss = 0.f, dot = 0.f;
    auto stat = [&](int c, float gv) {
      const float v = to_f<T>(src[c]);
      ss = fmaf(v, v, ss);
      dot = fmaf(gv * w[c], v, dot);
    };
    for (int i = lane_id(); i < half; i += 32) {
      int ca, cb;
      float ga, gb;
      pair_grad(i, ca, cb, ga, gb);
      stat(ca, ga);
      stat(cb, gb);
    }
    for (int c = p.rot + lane_id(); c < p.hd; c += 32) stat(c, to_f<T>(g[c]));
    const float r = rsqrtf(warp_total(ss) / p.hd + p.eps);
    const float m = warp_total(dot) * r / p.hd;
    auto emit = [&](int c, float gv) {
      const float n = to_f<T>(src[c]) * r;
      dst[c] = from_f<T>(r * (gv * w[c] - n * m));
      aw[c] += gv * n;
    };
    for (int i = lane_id(); i < half; i += 32) {
      int ca, cb;
      float ga, gb;
      pair_grad(i, ca, cb, ga, gb);
      emit(ca, ga);
      emit(cb, gb);
    }
    for (int c = p.rot + lane_id(); c < p.hd; c += 32) emit(c, to_f<T>(g[c]));
  }
  if (partial == nullptr) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.hd; c += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < ROPE_WARPS; ++w) s += rope_smem[w * 2 * p.hd + c];
    partial[(long long)blockIdx.x * 2 * p.hd + c] = s;
  }
}

// dq_w / dk_w += the CTAs' partial sums, in a fixed order
__global__ void rope_weights_kernel(const float* __restrict__ partial, int ctas, int hd, float* __restrict__ dq_w,
                                    float* __restrict__ dk_w) {
  __shared__ float part[8][32];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < 2 * hd)
    for (int b = threadIdx.y; b < ctas; b += 8) s += partial[(long long)b * 2 * hd + c];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y != 0 || c >= 2 * hd) return;
  for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
  if (c < hd) dq_w[c] += s;
  else dk_w[c - hd] += s;
}

namespace {

int rope_grid(const RopeAxesParams& p) {
  const long long units = (long long)p.M * (p.hq + p.hkv);
  return (int)std::min<long long>((units + ROPE_WARPS - 1) / ROPE_WARPS, (long long)num_sms() * 8);
}

template <typename T>
cudaError_t rope_bwd_run(const RopeAxesParams& p, const void* dq, const void* dk, void* dq_in, void* dk_in,
                         float* partial, cudaStream_t s) {
  rope_axes_bwd_any_kernel<T><<<rope_grid(p), ROPE_WARPS * 32, sizeof(float) * ROPE_WARPS * 2 * p.hd, s>>>(
      p, static_cast<const T*>(dq), static_cast<const T*>(dk), static_cast<T*>(dq_in), static_cast<T*>(dk_in), partial);
  return cudaGetLastError();
}

}  // namespace

cudaError_t rope_axes_fwd_launch(const RopeAxesParams& p, int elem, cudaStream_t s) {
  if (p.M <= 0) return cudaSuccess;
  const int grid = rope_grid(p);
  switch (elem) {
    case ELEM_BF16: rope_axes_any_kernel<__nv_bfloat16><<<grid, ROPE_WARPS * 32, 0, s>>>(p); break;
    case ELEM_F16: rope_axes_any_kernel<__half><<<grid, ROPE_WARPS * 32, 0, s>>>(p); break;
    case ELEM_F32: rope_axes_any_kernel<float><<<grid, ROPE_WARPS * 32, 0, s>>>(p); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

int rope_axes_bwd_ctas(const RopeAxesParams& p) { return rope_grid(p); }

cudaError_t rope_axes_bwd_launch(const RopeAxesParams& p, const void* dq, const void* dk, void* dq_in, void* dk_in,
                                 float* partial, float* dq_w, float* dk_w, int elem, cudaStream_t s) {
  if (p.M <= 0) return cudaSuccess;
  cudaError_t e;
  switch (elem) {
    case ELEM_BF16: e = rope_bwd_run<__nv_bfloat16>(p, dq, dk, dq_in, dk_in, partial, s); break;
    case ELEM_F16: e = rope_bwd_run<__half>(p, dq, dk, dq_in, dk_in, partial, s); break;
    case ELEM_F32: e = rope_bwd_run<float>(p, dq, dk, dq_in, dk_in, partial, s); break;
    default: return cudaErrorInvalidValue;
  }
  if (e != cudaSuccess || partial == nullptr) return e;
  rope_weights_kernel<<<(2 * p.hd + 31) / 32, dim3(32, 8), 0, s>>>(partial, rope_grid(p), p.hd, dq_w, dk_w);
  return cudaGetLastError();
}

}  // namespace tgo

// q / k RMSNorm (optional) and rotary positions with several axes (time, height, width).
//
// The rot rotated channels of a head form rot / 2 pairs: (2 i, 2 i + 1) interleaved, or (i, i + rot / 2) half-split.
// Pair i belongs to position axis axis[i] and turns by phi = pos[axis[i]] 2 pi freq[i] (freq in revolutions per position):
//     (a, b) -> (a cos phi - b sin phi, b cos phi + a sin phi);       channels past rot pass through.
// The angle is reduced before any sine: pos freq as a product of fp32 and a two-part fp32 constant, of which only the
// fraction of a revolution is kept, so positions of a long clip lose nothing that small ones have (|pos| < 2^24).
// Backward: the transposed rotation, then the norm's gradient with x and its rstd recomputed from q / k:
//     n = x r, gn = w g:   dx = r (gn - n mean(gn n)),   dw = sum over tokens and heads of g n.
// Bound by memory with many heads per token (32768 tokens x 32 heads of 128 bf16: 99 / 157 us, 0.83 / 0.78 of a plain
// copy's rate), by instruction issue with few (65536 x 12 heads of 64: 79 / 110 us): a token's angles are shared by its
// heads alone.
#include <algorithm>
#include <initializer_list>

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

// cos / sin of an angle of pos (hi + lo) revolutions. The product has to be the rounded one where its whole turns are taken
// off: fused into that subtraction it would bring its rounding error in twice.
__device__ __forceinline__ void turn_at(float pos, float hi, float lo, float& cs, float& sn) {
  const float whole = __fmul_rn(pos, hi);
  float rev = whole - rintf(whole);
  rev += fmaf(pos, hi, -whole) + pos * lo;
  sincospif(2.f * rev, &sn, &cs);
}
__device__ __forceinline__ void turn_of(const RopeAxesParams& p, long long tok, int pair, float& cs, float& sn) {
  turn_at(position(p, tok, p.axis[pair]), p.freq[pair], p.freq[p.rot / 2 + pair], cs, sn);
}

}  // namespace

// ------------------------------------------------------------------------------------------------------------------
// Vector form: head dims of whole 16-byte vectors up to 256 channels. LPH lanes of 8 channels per head (the next power of
// two: a head dim of 96 leaves 4 of 16 lanes idle), 32 / LPH heads per pass, several passes' loads issued together.
// A rotation is out[c] = x[c] A[c] + x[partner(c)] B[c] with A = w cos, B = -+ w sin of the channel's pair: 16 registers
// that a token sets up once for its q heads and once for its k heads. The pairs' cos / sin are computed once per warp
// (rot / 2 of them over 32 lanes) and shared through shared memory. The partner is the neighbour in the lane
// (interleaved) or the same element of the lane rot / 16 further (half-split, rot % 16 == 0): its raw words are shuffled.
// ------------------------------------------------------------------------------------------------------------------
namespace {


constexpr int ROPE_MAX_VEC_HD = 256;

// Table of a warp's token in shared memory: (cos, sin) of pair i at [i], and the identity from rot / 2 on, where the
// lanes of the channels past rot (and idle lanes) look: written once, no token touches it.
template <int SIZE>
__device__ __forceinline__ void identity_turns(const RopeAxesParams& p, float2 (&sh)[SIZE]) {
  for (int i = p.rot / 2 + lane_id(); i < SIZE; i += 32) sh[i] = make_float2(1.f, 0.f);
}

// A warp's share of the pairs (lane, lane + 32, ...): their table entries, kept over the whole kernel, and the next
// token's positions, loaded a token ahead.
template <int PAIRS>
struct Pairs {
  static constexpr int N = (PAIRS + 31) / 32;
  float hi[N], lo[N], pos[N];
  int axis[N];
  __device__ __forceinline__ explicit Pairs(const RopeAxesParams& p) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = lane_id() + 32 * k;
      const bool on = i < p.rot / 2;
      axis[k] = on ? p.axis[i] : -1;
      hi[k] = on ? p.freq[i] : 0.f;
      lo[k] = on ? p.freq[p.rot / 2 + i] : 0.f;
      pos[k] = 0.f;
    }
  }
  __device__ __forceinline__ void fetch(const RopeAxesParams& p, long long tok) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (axis[k] >= 0 && tok < p.M) pos[k] = position(p, tok, axis[k]);
  }
  __device__ __forceinline__ void write(float2* sh) const {
    __syncwarp();  // the last token's readers
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (axis[k] >= 0) {
        float c, s;
        turn_at(pos[k], hi[k], lo[k], c, s);
        sh[lane_id() + 32 * k] = make_float2(c, s);
      }
    __syncwarp();
  }
};

// this lane's cos and signed sin: out[c] = x[c] cs[c] + x[partner] sn[c]
template <bool INTER>
__device__ __forceinline__ void lane_turns(const RopeAxesParams& p, const float2* sh, int e0, float (&cs)[8],
                                           float (&sn)[8]) {
  const int half = p.rot / 2;
  const int at = INTER ? e0 / 2 : (e0 < half ? e0 : e0 - half);
  const float4* t = reinterpret_cast<const float4*>(sh + at);
  if constexpr (INTER) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 v = t[j];
      cs[4 * j] = cs[4 * j + 1] = v.x;
      cs[4 * j + 2] = cs[4 * j + 3] = v.z;
      sn[4 * j] = -v.y, sn[4 * j + 1] = v.y;
      sn[4 * j + 2] = -v.w, sn[4 * j + 3] = v.w;
    }
  } else {
    const float sign = e0 < half ? -1.f : 1.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = t[j];
      cs[2 * j] = v.x, cs[2 * j + 1] = v.z;
      sn[2 * j] = sign * v.y, sn[2 * j + 1] = sign * v.w;
    }
  }
}

template <typename T, bool INTER>
__device__ __forceinline__ void partner_of(const Raw<T, 8>& own, int src_lane, float (&f)[8]) {
  if constexpr (INTER) {
    float o[8];
    own.get(o);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = o[j ^ 1];
  } else {
    Raw<T, 8> r;
    const uint32_t* a = reinterpret_cast<const uint32_t*>(own.u);
    uint32_t* b = reinterpret_cast<uint32_t*>(r.u);
#pragma unroll
    for (int i = 0; i < 4 * Raw<T, 8>::W; ++i) b[i] = __shfl_sync(0xffffffffu, a[i], src_lane);
    r.get(f);
  }
}

// lane (of the warp) that holds the partner channels of this lane's 8 channels, half-split form
__device__ __forceinline__ int partner_lane(const RopeAxesParams& p, int lane, int e0) {
  const int step = p.rot / 16;
  if (e0 < p.rot / 2) return lane + step;
  return e0 < p.rot ? lane - step : lane;
}

}  // namespace

// Loads of the next batch of heads (of the same tensor, the other one, or the next token) are in flight while a batch is
// worked on, and the next token's positions while this token's heads are: a token with few heads is otherwise a chain of
// three memory latencies. 64 registers and 4 blocks per SM with 2 heads in flight per lane beat 3 blocks with 4 (32768
// tokens x 32 heads of 128: 102 and 106 us; 65536 x 12 heads of 64: 82 and 100 us).
template <typename T, int LPH, bool INTER>
__global__ void __launch_bounds__(ROPE_WARPS * 32, sizeof(T) == 4 ? 3 : 4) rope_axes_kernel(RopeAxesParams p) {
  constexpr int HPP = 32 / LPH, U = 2;
  __shared__ __align__(16) float2 turns[ROPE_WARPS][INTER ? LPH * 4 : LPH * 8];
  const int lane = lane_id(), sub = lane / LPH, e0 = (lane % LPH) * 8;
  const bool on = e0 < p.hd;
  const int src = INTER ? lane : partner_lane(p, lane, e0);
  const int ep = INTER ? e0 : (src % LPH) * 8;  // first partner channel
  const bool norm = p.q_w != nullptr;
  const float inv_hd = 1.f / p.hd;
  float2* sh = turns[warp_id()];
  identity_turns(p, turns[warp_id()]);
  const long long stride = (long long)gridDim.x * ROPE_WARPS;
  long long tok = (long long)blockIdx.x * ROPE_WARPS + warp_id();
  Raw<T, 8> x[U];
  auto fetch = [&](const T* in, int h0, int heads) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HPP;
      if (on && h < heads) x[u].load(in + h * p.hd + e0);
      else x[u].zero();
    }
  };
  if (tok < p.M) fetch(reinterpret_cast<const T*>(p.q) + tok * p.q_ts, sub, p.hq);
  Pairs<LPH * 4> pairs(p);
  pairs.fetch(p, tok);
  for (; tok < p.M; tok += stride) {
    pairs.write(sh);
    pairs.fetch(p, tok + stride);
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {  // q heads, then k heads
      const int heads = which == 0 ? p.hq : p.hkv;
      const T* in = which == 0 ? reinterpret_cast<const T*>(p.q) + tok * p.q_ts
                               : reinterpret_cast<const T*>(p.k) + tok * p.k_ts;
      T* out = (which == 0 ? reinterpret_cast<T*>(p.q_out) : reinterpret_cast<T*>(p.k_out)) + tok * heads * p.hd + e0;
      const float* w = which == 0 ? p.q_w : p.k_w;
      float A[8], B[8];
      lane_turns<INTER>(p, sh, e0, A, B);
      if (norm && on) {
        float a[8], b[8];
        load_vec<float, 8>(w + e0, a);
        load_vec<float, 8>(w + ep, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) A[j] *= a[j], B[j] *= b[INTER ? j ^ 1 : j];
      }
#pragma unroll 1
      for (int h0 = sub; h0 - sub < heads; h0 += U * HPP) {
        Raw<T, 8> cur[U];
#pragma unroll
        for (int u = 0; u < U; ++u) cur[u] = x[u];
        if (h0 - sub + U * HPP < heads) fetch(in, h0 + U * HPP, heads);
        else if (which == 0) fetch(reinterpret_cast<const T*>(p.k) + tok * p.k_ts, sub, p.hkv);
        else if (tok + stride < p.M) fetch(reinterpret_cast<const T*>(p.q) + (tok + stride) * p.q_ts, sub, p.hq);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * HPP;
          if (h - sub >= heads) break;  // warp-uniform
          float f[8], g[8];
          cur[u].get(f);
          partner_of<T, INTER>(cur[u], src, g);
          float r = 1.f;
          if (norm) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
            r = rsqrtf(fmaf(head_sum<LPH>(ss), inv_hd, p.eps));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = r * fmaf(f[j], A[j], g[j] * B[j]);
          if (on && h < heads) store_vec<T, 8>(out + h * p.hd, f);
        }
      }
    }
  }
}

// Backward, same layout (4 heads in flight per lane, no look-ahead over batches: with it 227 us, without 158 us at 32768 x 32
// heads of 128). dw partials stay in registers over the whole grid-stride loop: a lane's channels are the same for every
// head and token.
template <typename T, int LPH, bool INTER>
__global__ void __launch_bounds__(ROPE_WARPS * 32, 2) rope_axes_bwd_kernel(RopeAxesParams p, const T* __restrict__ dq,
                                                                        const T* __restrict__ dk,
                                                                        T* __restrict__ dq_in, T* __restrict__ dk_in,
                                                                        float* __restrict__ partial) {
  constexpr int HPP = 32 / LPH, U = sizeof(T) == 4 ? 2 : 4;
  __shared__ __align__(16) float2 turns[ROPE_WARPS][INTER ? LPH * 4 : LPH * 8];
  __shared__ float dw[ROPE_WARPS][2][LPH * 8];
  const int lane = lane_id(), sub = lane / LPH, e0 = (lane % LPH) * 8;
  const bool on = e0 < p.hd;
  const int src = INTER ? lane : partner_lane(p, lane, e0);
  const bool norm = p.q_w != nullptr;
  const float inv_hd = 1.f / p.hd;
  float acc[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[0][j] = acc[1][j] = 0.f;
  float2* sh = turns[warp_id()];
  identity_turns(p, turns[warp_id()]);
  const long long stride = (long long)gridDim.x * ROPE_WARPS;
  long long tok = (long long)blockIdx.x * ROPE_WARPS + warp_id();
  Pairs<LPH * 4> pairs(p);
  pairs.fetch(p, tok);
  for (; tok < p.M; tok += stride) {
    pairs.write(sh);
    pairs.fetch(p, tok + stride);
    float cs[8], sn[8];
    lane_turns<INTER>(p, sh, e0, cs, sn);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int heads = which == 0 ? p.hq : p.hkv;
      const T* in = which == 0 ? reinterpret_cast<const T*>(p.q) + tok * p.q_ts
                               : reinterpret_cast<const T*>(p.k) + tok * p.k_ts;
      const T* grad = (which == 0 ? dq : dk) + tok * heads * p.hd;
      T* out = (which == 0 ? dq_in + tok * p.dq_ts : dk_in + tok * p.dk_ts) + e0;
      float w[8] = {};
      if (norm && on) load_vec<float, 8>((which == 0 ? p.q_w : p.k_w) + e0, w);
#pragma unroll 1
      for (int h0 = sub; h0 - sub < heads; h0 += U * HPP) {
        Raw<T, 8> g[U], x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * HPP;
          const bool ok = on && h < heads;
          if (ok) g[u].load(grad + h * p.hd + e0);
          else g[u].zero();
          if (ok && norm) x[u].load(in + h * p.hd + e0);
          else x[u].zero();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * HPP;
          if (h - sub >= heads) break;
          float gf[8], gp[8];
          g[u].get(gf);
          partner_of<T, INTER>(g[u], src, gp);
#pragma unroll
          for (int j = 0; j < 8; ++j) gf[j] = fmaf(gf[j], cs[j], -gp[j] * sn[j]);
          if (norm) {
            float xf[8], ss = 0.f, dot = 0.f;
            x[u].get(xf);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              ss = fmaf(xf[j], xf[j], ss);
              dot = fmaf(gf[j] * w[j], xf[j], dot);
            }
            ss = head_sum<LPH>(ss);
            dot = head_sum<LPH>(dot);
            const float r = rsqrtf(fmaf(ss, inv_hd, p.eps));
            const float m = dot * r * r * inv_hd;  // n mean(gn n) = x r (r dot / hd)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              acc[which][j] = fmaf(gf[j] * xf[j], r, acc[which][j]);
              gf[j] = r * fmaf(gf[j], w[j], -xf[j] * m);
            }
          }
          if (on && h < heads) store_vec<T, 8>(out + h * p.hd, gf);
        }
      }
    }
  }
  if (partial == nullptr) return;
  // sums over the warp's heads groups, then over the warps, in a fixed order
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = acc[which][j];
#pragma unroll
      for (int o = 16; o >= LPH; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (sub == 0) dw[warp_id()][which][e0 + j] = v;
    }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.hd; c += blockDim.x) {
    const int which = c >= p.hd, e = c - which * p.hd;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < ROPE_WARPS; ++i) s += dw[i][which][e];
    partial[(long long)blockIdx.x * 2 * p.hd + c] = s;
  }
}

// ------------------------------------------------------------------------------------------------------------------
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
  float* acc = rope_smem + warp_id() * 2 * p.hd;  // only with norm weights
  if (p.q_w != nullptr)
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
    T* dst = (is_q ? dq_in + tok * p.dq_ts : dk_in + tok * p.dk_ts) + (long long)h * p.hd;
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

// dq_w / dk_w (+)= the CTAs' partial sums, in a fixed order: lane = channel, the 32 warps share the CTAs
__global__ void __launch_bounds__(1024) rope_weights_kernel(const float* __restrict__ partial, int ctas, int hd,
                                                            float* __restrict__ dq_w, float* __restrict__ dk_w,
                                                            bool add_q, bool add_k) {
  __shared__ float part[32][32];
  const int lane = lane_id(), warp = warp_id(), c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * hd) {
#pragma unroll 8
    for (int b = warp; b < ctas; b += 32) s += partial[(long long)b * 2 * hd + c];
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= 2 * hd) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) s += part[i][lane];
  float* dst = c < hd ? dq_w + c : dk_w + (c - hd);
  *dst = (c < hd ? add_q : add_k) ? *dst + s : s;
}

namespace {

// The vector form needs whole 16-byte vectors at 16-byte addresses, and in the half-split form partners at the same
// element of another lane.
bool rope_vectors(const RopeAxesParams& p, int elem, std::initializer_list<const void*> more = {}) {
  const int per = elem == ELEM_F32 ? 4 : 8;  // elements of a 16-byte word
  if (p.hd % 8 != 0 || p.hd > ROPE_MAX_VEC_HD || p.q_ts % per != 0 || p.k_ts % per != 0 || p.dq_ts % per != 0 ||
      p.dk_ts % per != 0)
    return false;
  if (!p.interleaved && p.rot % 16 != 0) return false;
  uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) |
                   reinterpret_cast<uintptr_t>(p.q_out) | reinterpret_cast<uintptr_t>(p.k_out) |
                   reinterpret_cast<uintptr_t>(p.q_w) | reinterpret_cast<uintptr_t>(p.k_w);
  for (const void* m : more) bits |= reinterpret_cast<uintptr_t>(m);
  return (bits & 15) == 0;
}

// CTAs of the grid-stride kernels: a warp per token (vector form) or per token and head. Backward: the blocks that the SMs
// hold (more would add partial sums: 161 us with 2 per SM, 169 us with 8 at 32768 x 32 heads of 128); forward: a few times
// that, so that the last tokens spread evenly (fp32: 194 us with 3, 179 us with 16).
int rope_grid(const RopeAxesParams& p, bool vectors, int per_sm) {
  const long long units = vectors ? p.M : (long long)p.M * (p.hq + p.hkv);
  return (int)std::min<long long>((units + ROPE_WARPS - 1) / ROPE_WARPS, (long long)num_sms() * per_sm);
}
constexpr int ROPE_FWD_BLOCKS = 16, ROPE_BWD_BLOCKS = 2, ROPE_ANY_BLOCKS = 4;

template <typename T, int LPH>
void rope_fwd_vec(const RopeAxesParams& p, cudaStream_t s) {
  const int grid = rope_grid(p, true, ROPE_FWD_BLOCKS);
  if (p.interleaved) rope_axes_kernel<T, LPH, true><<<grid, ROPE_WARPS * 32, 0, s>>>(p);
  else rope_axes_kernel<T, LPH, false><<<grid, ROPE_WARPS * 32, 0, s>>>(p);
}
template <typename T, int LPH>
void rope_bwd_vec(const RopeAxesParams& p, const T* dq, const T* dk, T* dqi, T* dki, float* partial, int grid,
                  cudaStream_t s) {
  if (p.interleaved)
    rope_axes_bwd_kernel<T, LPH, true><<<grid, ROPE_WARPS * 32, 0, s>>>(p, dq, dk, dqi, dki, partial);
  else
    rope_axes_bwd_kernel<T, LPH, false><<<grid, ROPE_WARPS * 32, 0, s>>>(p, dq, dk, dqi, dki, partial);
}

template <typename T>
cudaError_t rope_fwd_run(const RopeAxesParams& p, int elem, cudaStream_t s) {
  if (!rope_vectors(p, elem)) rope_axes_any_kernel<T><<<rope_grid(p, false, ROPE_ANY_BLOCKS), ROPE_WARPS * 32, 0, s>>>(p);
  else if (p.hd <= 32) rope_fwd_vec<T, 4>(p, s);
  else if (p.hd <= 64) rope_fwd_vec<T, 8>(p, s);
  else if (p.hd <= 128) rope_fwd_vec<T, 16>(p, s);
  else rope_fwd_vec<T, 32>(p, s);
  return cudaGetLastError();
}

template <typename T>
cudaError_t rope_bwd_run(const RopeAxesParams& p, const void* dq, const void* dk, void* dq_in, void* dk_in,
                         float* partial, float* dq_w, float* dk_w, bool add_q_w, bool add_k_w, int elem,
                                 cudaStream_t s) {
  const T *gq = static_cast<const T*>(dq), *gk = static_cast<const T*>(dk);
  T *iq = static_cast<T*>(dq_in), *ik = static_cast<T*>(dk_in);
  const bool vec = rope_vectors(p, elem, {dq, dk, dq_in, dk_in});
  const int grid = rope_grid(p, vec, vec ? ROPE_BWD_BLOCKS : ROPE_ANY_BLOCKS);
  if (!vec) {
    // the weights' sums of every warp: none without weights, more than the default 48 KB above 768 channels
    const int smem = p.q_w != nullptr ? (int)sizeof(float) * ROPE_WARPS * 2 * p.hd : 0;
    if (smem > 48 * 1024) {
      cudaError_t e = cudaFuncSetAttribute(rope_axes_bwd_any_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
    }
    rope_axes_bwd_any_kernel<T><<<grid, ROPE_WARPS * 32, smem, s>>>(p, gq, gk, iq, ik, partial);
  } else if (p.hd <= 32) rope_bwd_vec<T, 4>(p, gq, gk, iq, ik, partial, grid, s);
  else if (p.hd <= 64) rope_bwd_vec<T, 8>(p, gq, gk, iq, ik, partial, grid, s);
  else if (p.hd <= 128) rope_bwd_vec<T, 16>(p, gq, gk, iq, ik, partial, grid, s);
  else rope_bwd_vec<T, 32>(p, gq, gk, iq, ik, partial, grid, s);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || partial == nullptr) return e;
  rope_weights_kernel<<<(2 * p.hd + 31) / 32, 1024, 0, s>>>(partial, grid, p.hd, dq_w, dk_w, add_q_w, add_k_w);
  return cudaGetLastError();
}

}  // namespace

cudaError_t rope_axes_fwd_launch(const RopeAxesParams& p, int elem, cudaStream_t s) {
  if (p.M <= 0) return cudaSuccess;
  switch (elem) {
    case ELEM_BF16: return rope_fwd_run<__nv_bfloat16>(p, elem, s);
    case ELEM_F16: return rope_fwd_run<__half>(p, elem, s);
    case ELEM_F32: return rope_fwd_run<float>(p, elem, s);
  }
  return cudaErrorInvalidValue;
}

int rope_axes_bwd_ctas() { return num_sms() * std::max(ROPE_BWD_BLOCKS, ROPE_ANY_BLOCKS); }

cudaError_t rope_axes_bwd_launch(const RopeAxesParams& p, const void* dq, const void* dk, void* dq_in, void* dk_in,
                                 float* partial, float* dq_w, float* dk_w, bool add_q_w, bool add_k_w, int elem,
                                 cudaStream_t s) {
  if (p.M <= 0) return cudaSuccess;
  switch (elem) {
    case ELEM_BF16: return rope_bwd_run<__nv_bfloat16>(p, dq, dk, dq_in, dk_in, partial, dq_w, dk_w, add_q_w, add_k_w, elem, s);
    case ELEM_F16: return rope_bwd_run<__half>(p, dq, dk, dq_in, dk_in, partial, dq_w, dk_w, add_q_w, add_k_w, elem, s);
    case ELEM_F32: return rope_bwd_run<float>(p, dq, dk, dq_in, dk_in, partial, dq_w, dk_w, add_q_w, add_k_w, elem, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tgo

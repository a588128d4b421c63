// Routing of tokens to experts.
//
// Scores of token n: s = softmax(l) or sigmoid(l) over E experts. Selection scores c = (l for softmax, which orders the
// experts as softmax(l) does; s for sigmoid) + bias. With groups, the E / G experts of a group compete as one first: a
// group's score is its best c (softmax) or the sum of its two best (sigmoid), and only the experts of the top_groups
// best groups stay. The k experts of largest c are chosen, ties to the lowest index; their weights are
//     w_j = scale s_j / (sum of the chosen s + 1e-20)      (renorm)      or      scale s_j.
// Gradient to the logits, with r_j = w_j / scale and m = sum_j r_j dw_j over the chosen:
//     softmax, renorm   dl_j = w_j (dw_j - m)                         sigmoid, renorm   dl_j = scale (dw_j - m) s_j' / S
//     softmax           dl_i = [i chosen] w_i dw_i - scale p_i m      sigmoid           dl_j = scale dw_j s_j'
// s' = s (1 - s), S = sum of the chosen s. The selection and the bias take no gradient.
//
// L lanes hold one token, EPL consecutive experts each, so a row is read once with wide loads and every later step
// works on registers. c is mapped to an unsigned key of the same order (NaN lowest, -0 as +0), and each of the k steps
// is a maximum over the lane's keys and over the L lanes; the lowest lane that holds the maximum wins (its experts have
// the lowest indices) and takes the expert out.
#include "block_ops.h"
#include "common.cuh"
#include "vec.cuh"

namespace tgo {

namespace {

constexpr int ROUTE_WARPS = 4;

__device__ __forceinline__ unsigned order_key(float c) {
  c += 0.f;  // -0 -> +0
  const unsigned u = __float_as_uint(c);
  const unsigned key = (u >> 31) ? ~u : (u | 0x80000000u);
  return c != c ? 1u : key;  // 0 is kept for "not a candidate"
}

template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
  if constexpr (L == 32) {
    return __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}
template <int L>
__device__ __forceinline__ unsigned lanes_or(unsigned v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v |= __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int EPL>
__device__ __forceinline__ void load_logits(const RouteParams& p, long long n, int e0, float (&l)[EPL]) {
  const T* row = reinterpret_cast<const T*>(p.logits) + n * p.ld;
#pragma unroll
  for (int j = 0; j < EPL; ++j) l[j] = e0 + j < p.E ? to_f<T>(row[e0 + j]) : -INFINITY;
}

// sigmoid from e = exp(-|l|) <= 1: no overflow, small scores keep their relative precision
__device__ __forceinline__ float sigmoid_of(float l, float e) { return (l >= 0.f ? 1.f : e) / (1.f + e); }

}  // namespace

template <typename T, int L, int EPL>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) route_fwd_kernel(RouteParams p) {
  constexpr int TOKENS = ROUTE_WARPS * 32 / L;  // per block
  extern __shared__ uint8_t route_smem[];
  // chosen scores and experts [TOKENS][k]; with groups also the selection scores [TOKENS][E] and group scores
  float* sc = reinterpret_cast<float*>(route_smem);
  int* si = reinterpret_cast<int*>(sc + TOKENS * p.k);
  float* cs = reinterpret_cast<float*>(si + TOKENS * p.k);
  float* gsc = cs + TOKENS * p.E;
  const int lane = lane_id(), li = lane % L, tok = threadIdx.x / L;
  const long long n = (long long)blockIdx.x * TOKENS + tok;
  const bool in = n < p.N;
  const int e0 = li * EPL;
  float s[EPL];
  unsigned key[EPL];
  float z = 1.f;
  {
    float l[EPL];
    if (in) {
      load_logits<T, EPL>(p, n, e0, l);
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) l[j] = 0.f;
    }
    if (!p.sigmoid) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < EPL; ++j) mx = fmaxf(mx, l[j]);
      mx = lanes_max<L>(mx);
      if (mx == -INFINITY) mx = 0.f;  // a token with every expert at -inf: all s are 0, and so are its weights
      z = 0.f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        s[j] = e0 + j < p.E ? expf(l[j] - mx) : 0.f;
        z += s[j];
      }
      z = fmaxf(lanes_sum<L>(z), 1e-20f);
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        s[j] = sigmoid_of(l[j], expf(-fabsf(l[j])));
        l[j] = s[j];
      }
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = e0 + j;
      if (p.bias != nullptr && e < p.E) l[j] += p.bias[e];
      key[j] = e < p.E ? order_key(l[j]) : 0u;
      if (p.groups > 1 && e < p.E) cs[tok * p.E + e] = l[j];
    }
  }
  if (p.groups > 1) {
    __syncwarp();
    // lane g scans group g
    for (int g = li; g < p.groups; g += L) {
      const float* c = cs + tok * p.E + g * p.group_size;
      float a = -INFINITY, b = -INFINITY;
      for (int i = 0; i < p.group_size; ++i) {
        const float v = c[i];
        b = fmaxf(b, fminf(a, v));
        a = fmaxf(a, v);
      }
      gsc[tok * kRouteMaxGroups + g] = (p.sigmoid && p.group_size > 1) ? a + b : a;
    }
    __syncwarp();
    unsigned kept = 0;
    for (int g = li; g < p.groups; g += L) {
      const unsigned mine = order_key(gsc[tok * kRouteMaxGroups + g]);
      int above = 0;
      for (int o = 0; o < p.groups; ++o) {
        const unsigned other = order_key(gsc[tok * kRouteMaxGroups + o]);
        above += (other > mine || (other == mine && o < g)) ? 1 : 0;
      }
      if (above < p.top_groups) kept |= 1u << g;
    }
    kept = lanes_or<L>(kept);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const unsigned g = ((unsigned)(e0 + j) * p.group_magic) >> 22;
      if (!((kept >> (g & 31)) & 1u)) key[j] = 0u;
    }
  }
  float chosen = 0.f;
  for (int r = 0; r < p.k; ++r) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) m = max(m, key[j]);
    const unsigned gm = lanes_max<L>(m);
    unsigned who = __ballot_sync(0xffffffffu, m == gm);
    if constexpr (L < 32) who = (who >> (lane - li)) & ((1u << L) - 1u);
    if (__ffs(who) - 1 == li) {
      bool open = true;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        if (open && key[j] == gm) {
          open = false;
          key[j] = 0u;
          chosen += s[j];
          sc[tok * p.k + r] = s[j];
          si[tok * p.k + r] = e0 + j;
        }
      }
    }
  }
  const float total = lanes_sum<L>(chosen);
  __syncwarp();
  if (!in) return;
  const bool ok = p.valid == nullptr || p.valid[n];
  const float den = p.renorm ? total + 1e-20f * z : z;
  for (int r = li; r < p.k; r += L) {
    p.w[n * p.k + r] = ok ? sc[tok * p.k + r] / den * p.scale : 0.f;
    p.idx[n * p.k + r] = ok ? si[tok * p.k + r] : -1;
  }
}

template <typename T, int L, int EPL>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) route_bwd_kernel(RouteParams p, const float* __restrict__ dw,
                                                                     T* __restrict__ dlogits) {
  constexpr int TOKENS = ROUTE_WARPS * 32 / L;
  const int li = lane_id() % L;
  const long long n = (long long)blockIdx.x * TOKENS + threadIdx.x / L;
  const bool in = n < p.N;
  const int e0 = li * EPL;
  const T* row = reinterpret_cast<const T*>(p.logits) + (in ? n : 0) * p.ld;
  const float* w = p.w + (in ? n : 0) * p.k;
  const float* g = dw + (in ? n : 0) * p.k;
  const int* idx = p.idx + (in ? n : 0) * p.k;
  float d[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) d[j] = 0.f;
  const bool live = in && idx[0] >= 0;
  float m = 0.f, total = 1e-20f;
  if (live) {
    for (int r = 0; r < p.k; ++r) {
      m += w[r] * g[r];
      if (p.sigmoid && p.renorm) {
        const float l = to_f<T>(row[idx[r]]);
        total += sigmoid_of(l, expf(-fabsf(l)));
      }
    }
    m /= p.scale;
  }
  if (!p.sigmoid && !p.renorm) {  // dense: every expert's probability is needed (warp-uniform branch)
    float l[EPL];
    float mx = -INFINITY;
    if (live) load_logits<T, EPL>(p, n, e0, l);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      if (!live) l[j] = 0.f;
      mx = fmaxf(mx, l[j]);
    }
    mx = lanes_max<L>(mx);
    if (mx == -INFINITY) mx = 0.f;
    float z = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      l[j] = e0 + j < p.E ? expf(l[j] - mx) : 0.f;
      z += l[j];
    }
    z = fmaxf(lanes_sum<L>(z), 1e-20f);
    if (live) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) d[j] = -p.scale * (l[j] / z) * m;
    }
  }
  if (live) {
    for (int r = 0; r < p.k; ++r) {
      const int e = idx[r];
      float v;
      if (p.sigmoid) {
        const float l = to_f<T>(row[e]);
        const float x = expf(-fabsf(l)), q = 1.f + x;
        const float ds = x / (q * q);
        v = p.renorm ? p.scale * (g[r] - m) / total * ds : p.scale * g[r] * ds;
      } else {
        v = p.renorm ? w[r] * (g[r] - m) : w[r] * g[r];
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (e == e0 + j) d[j] += v;
    }
  }
  if (!in) return;
  T* out = dlogits + n * p.E;
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    if (e0 + j < p.E) out[e0 + j] = from_f<T>(d[j]);
}

namespace {

template <typename T, int L, int EPL>
cudaError_t route_run(const RouteParams& p, const float* dw, void* dlogits, cudaStream_t s) {
  constexpr int TOKENS = ROUTE_WARPS * 32 / L;
  const unsigned grid = (unsigned)((p.N + TOKENS - 1) / TOKENS);
  if (dlogits != nullptr) {
    route_bwd_kernel<T, L, EPL><<<grid, ROUTE_WARPS * 32, 0, s>>>(p, dw, static_cast<T*>(dlogits));
  } else {
    const size_t smem = (size_t)TOKENS * 4 * (2 * p.k + (p.groups > 1 ? p.E + kRouteMaxGroups : 0));
    route_fwd_kernel<T, L, EPL><<<grid, ROUTE_WARPS * 32, smem, s>>>(p);
  }
  return cudaGetLastError();
}

// 8 experts per lane: one token needs as few lanes as its row allows (a warp holds 32 tokens of 8 experts, one token
// of 256), and 16 per lane above 256 experts
template <typename T>
cudaError_t route_any(const RouteParams& p, const float* dw, void* dlogits, cudaStream_t s) {
  if (p.E <= 8) return route_run<T, 1, 8>(p, dw, dlogits, s);
  if (p.E <= 16) return route_run<T, 2, 8>(p, dw, dlogits, s);
  if (p.E <= 32) return route_run<T, 4, 8>(p, dw, dlogits, s);
  if (p.E <= 64) return route_run<T, 8, 8>(p, dw, dlogits, s);
  if (p.E <= 128) return route_run<T, 16, 8>(p, dw, dlogits, s);
  if (p.E <= 256) return route_run<T, 32, 8>(p, dw, dlogits, s);
  if (p.E <= kRouteMaxExperts) return route_run<T, 32, 16>(p, dw, dlogits, s);
  return cudaErrorInvalidValue;
}

cudaError_t route_launch(const RouteParams& p, const float* dw, void* dlogits, int elem, cudaStream_t s) {
  if (p.N <= 0) return cudaSuccess;
  switch (elem) {
    case ELEM_BF16: return route_any<__nv_bfloat16>(p, dw, dlogits, s);
    case ELEM_F16: return route_any<__half>(p, dw, dlogits, s);
    case ELEM_F32: return route_any<float>(p, dw, dlogits, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t route_fwd_launch(const RouteParams& p, int elem, cudaStream_t s) {
  return route_launch(p, nullptr, nullptr, elem, s);
}
cudaError_t route_bwd_launch(const RouteParams& p, const float* dw, void* dlogits, int elem, cudaStream_t s) {
  return dlogits == nullptr ? cudaErrorInvalidValue : route_launch(p, dw, dlogits, elem, s);
}

}  // namespace tgo

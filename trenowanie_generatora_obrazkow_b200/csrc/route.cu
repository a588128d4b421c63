// Routing of tokens to experts.
//
// Scores of token n: s = softmax(l) or sigmoid(l) over E experts. Selection scores c = (l for softmax, which orders the
// experts as softmax(l) does; s for sigmoid) + bias. With groups, the E / G experts of a group compete as one first: a
// group's score is its best c (softmax) or the sum of its two best (sigmoid), and only the experts of the top_groups
// best groups stay. The k experts of largest c are chosen, ties to the lowest index; their weights are
//     w_j = scale s_j / (sum of the chosen s + 1e-20)      (renorm)      or      scale s_j.
// Gradient to the logits, with r_j = w_j / scale and m = sum_j r_j dw_j over the chosen:
//     softmax, renorm   dl_i = [i chosen] w_i (dw_i - m) - scale p_i m 1e-20 / S
//     softmax           dl_i = [i chosen] w_i dw_i - scale p_i m
//     sigmoid, renorm   dl_j = scale (dw_j - m) s_j' / S              sigmoid           dl_j = scale dw_j s_j'
// s' = s (1 - s), S = sum of the chosen s (+ 1e-20). The selection and the bias take no gradient. 1e-20 / S, which is
// 1 - sum of r, matters only where a bias moved the choice to experts of next to no probability: without a bias, and
// where it is below the rounding of the sum, the other experts' logits are not read.
//
// L lanes hold one token, EPL consecutive experts each, so a row is read once with wide loads and every later step works on
// registers. c is mapped to an unsigned key of the same order (NaN lowest, -0 as +0). Each lane keeps its best
// keys at the front (equal keys in index order), then each of the k steps takes the largest head of the L lanes; the
// lowest lane that holds it wins (its experts have the lowest indices) and drops its head. What the weights need beyond
// the choice is computed for the k chosen alone, from logits read again (they are in the cache).
// 65536 x 256 fp32, k 8, 4 of 8 groups: forward 60 us, bound by instruction issue (80 %, about 800 per token: the exact
// sigmoids and the group ranks 10 us each, the lists 20 us; softmax without groups 43 us), 69 us with 2 % of the experts at
// -inf (an overflowed exponential sends its reciprocal down the slow path); backward 26 us; 32768 x 8, 2 chosen: 3.6 / 3.2 us.
#include <algorithm>
#include <cfloat>

#include "block_ops.h"
#include "common.cuh"
#include "kernels.h"
#include "vec.cuh"

namespace tgo {

namespace {

constexpr int ROUTE_WARPS = 4, ROUTE_BWD_BLOCKS = 8;
// Above the rounding of a sum of up to 32 weights divided by their own sum (about 8 units of 2^-24).
constexpr float ROUTE_LOST = 0x1p-20f;
// blocks per SM: 64 registers hold 8 experts per lane (9 blocks spill, 7 take 2 us more), 16 experts want 80
constexpr int route_fwd_blocks(int epl) { return epl > 8 ? 6 : 8; }

// c is no NaN and not -0
__device__ __forceinline__ unsigned number_key(float c) {
  const unsigned u = __float_as_uint(c);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
// NaN comes last; 0 is kept for "not a candidate"
__device__ __forceinline__ unsigned order_key(float c) { return c != c ? 1u : number_key(c); }

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

// shared memory of a forward warp, in bytes (a multiple of 8)
__host__ __device__ __forceinline__ int route_warp_smem(const RouteParams& p, int tokens, int steps) {
  const bool scan = p.groups > 1 && p.group_lanes == 0;
  const int words = steps * tokens * (2 + p.k) + (scan ? tokens * (p.E + kRouteMaxGroups) : 0);
  return (words + 1) / 2 * 8;
}

// EPL logits from expert e0 on; vec: E, the row stride and the base allow 16-byte loads of 8 logits
template <typename T, int EPL>
__device__ __forceinline__ void load_logits(const RouteParams& p, long long n, int e0, float (&l)[EPL]) {
  const T* row = reinterpret_cast<const T*>(p.logits) + n * p.ld;
  if (p.vec) {
#pragma unroll
    for (int v = 0; v < EPL; v += 8) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = -INFINITY;
      if (e0 + v < p.E) load_vec<T, 8>(row + e0 + v, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) l[v + j] = f[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) l[j] = e0 + j < p.E ? to_f<T>(row[e0 + j]) : -INFINITY;
  }
}

// 1 + exp(-l) is rounded once relative to itself, so small scores keep their relative precision, until exp(-l) comes near
// the largest float: below l = -88.7 this is 0. There the score is exp(l) (they differ by exp(l) of it), subnormal
// down to l = -104, and logits are still told apart. Few tokens hold such a logit, and switched-off experts (-inf) are none.
__device__ __forceinline__ float sigmoid_of(float l) { return __frcp_rn(1.f + expf(-l)); }
constexpr float FAR_DOWN = 9.f;
__device__ __forceinline__ bool far_down(float l) { return fabsf(l + 96.f) < FAR_DOWN; }

}  // namespace

// A warp takes a batch of `steps` x 32 / L tokens: each step chooses for its tokens while the next step's logits are in
// flight, and the end computes the weights of the whole batch's choices together, `slots` = the power of two from k on
// lanes per token. At 65536 x 256, k 8, where this took 63 us with its launch, one token per warp (its end in 8 of 32 lanes)
// took 70 us, and a grid of resident warps that walk the batches 68 us, as the last round is not full.
template <typename T, int L, int EPL>
__global__ void __launch_bounds__(ROUTE_WARPS * 32, route_fwd_blocks(EPL)) route_fwd_kernel(RouteParams p, int steps,
                                                                                       int slots) {
  constexpr int TOKENS = 32 / L;  // of a step
  extern __shared__ __align__(16) uint8_t route_smem[];
  const int batch = steps * TOKENS;
  // the warp's: (max, sum) of the whole rows [batch], chosen experts [batch][k]; for groups that do not fall on whole
  // lanes also the step's selection and group scores
  float2* mxz = reinterpret_cast<float2*>(route_smem + warp_id() * route_warp_smem(p, TOKENS, steps));
  int* chosen = reinterpret_cast<int*>(mxz + batch);
  float* cs = reinterpret_cast<float*>(chosen + batch * p.k);
  float* gsc = cs + TOKENS * p.E;
  const int lane = lane_id(), li = lane % L, tok = lane / L;
  const int e0 = li * EPL;
  const unsigned lower = ((1u << li) - 1u) << (lane - li);  // the token's lanes below this one
  const int group_shift = __ffs(p.group_lanes) - 1;
  const bool whole = !p.sigmoid && (p.bias != nullptr || !p.renorm);  // softmax: the sum over all experts matters
  float bias[EPL];  // 0 without one; adding 0 also turns -0 into +0
#pragma unroll
  for (int j = 0; j < EPL; ++j) bias[j] = p.bias != nullptr && e0 + j < p.E ? p.bias[e0 + j] + 0.f : 0.f;
  float next[EPL];
  auto fetch = [&](long long n) {
    if (n < p.N) {
      load_logits<T, EPL>(p, n, e0, next);
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) next[j] = 0.f;
    }
  };
  const long long base = ((long long)blockIdx.x * ROUTE_WARPS + warp_id()) * batch;
  if (base >= p.N) return;
  fetch(base + tok);
  for (int step = 0; step < steps; ++step) {
    if (base + step * TOKENS >= p.N) break;
    const int at = step * TOKENS + tok;  // in the batch
    float l[EPL];
    unsigned key[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) l[j] = next[j];
    if (step + 1 < steps) fetch(base + at + TOKENS);
    if (whole) {
      float mx = -INFINITY, z = 0.f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) mx = fmaxf(mx, l[j]);
      mx = lanes_max<L>(mx);
      if (mx == -INFINITY) mx = 0.f;  // every expert at -inf: all s are 0, and so are the weights
#pragma unroll
      for (int j = 0; j < EPL; ++j) z += e0 + j < p.E ? expf(l[j] - mx) : 0.f;
      z = fmaxf(lanes_sum<L>(z), 1e-20f);
      if (li == 0) mxz[at] = make_float2(mx, z);
    }
    if (p.sigmoid) {
      float far = FAR_DOWN, sc[EPL];
#pragma unroll
      for (int j = 0; j < EPL; j += 2) {
        const float2 t = x2_split(x2_add(x2(l[j], l[j + 1]), x2(96.f)));
        far = fminf(far, fminf(fabsf(t.x), fabsf(t.y)));
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) sc[j] = sigmoid_of(l[j]);
      if (__builtin_expect(far < FAR_DOWN, 0)) {
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          if (far_down(l[j])) sc[j] = expf(l[j]);
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) l[j] = sc[j];
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) l[j] += bias[j];
    // one test finds a lane that may hold NaN (also +inf with -inf) and one a lane past the last expert
    float all = l[0];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      key[j] = number_key(l[j]);
      if (j > 0) all += l[j];
    }
    if (!(fabsf(all) <= FLT_MAX) || e0 + EPL > p.E) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        key[j] = e0 + j < p.E ? order_key(l[j]) : 0u;
        l[j] = fmaxf(l[j], -INFINITY);  // NaN adds nothing to its group's worth (fminf and fmaxf would pass it over)
      }
    }
    if (p.groups > 1 && p.group_lanes > 0) {
      // a group is group_lanes whole lanes (a power of two): its two best scores by shuffles, then its rank
      float a = -INFINITY, b = -INFINITY;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        b = fmaxf(b, fminf(a, l[j]));
        a = fmaxf(a, l[j]);
      }
      for (int o = 1; o < p.group_lanes; o <<= 1) {
        const float a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
        b = fmaxf(fminf(a, a2), fmaxf(b, b2));
        a = fmaxf(a, a2);
      }
      const unsigned mine = number_key(fmaxf(p.sigmoid ? a + b : a, -INFINITY));  // +inf with -inf counts as -inf
      const int g = li >> group_shift;
      int above = 0;  // groups that come before this one; its lanes share the comparisons
      for (int o0 = 0; o0 < p.groups; o0 += p.group_lanes) {
        const int o = o0 + (li & (p.group_lanes - 1));
        const unsigned other = __shfl_sync(0xffffffffu, mine, o << group_shift, L);
        above += o < p.groups && (other > mine || (other == mine && o < g)) ? 1 : 0;
      }
      for (int o = 1; o < p.group_lanes; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
      if (above >= p.top_groups)
#pragma unroll
        for (int j = 0; j < EPL; ++j) key[j] = 0u;
    } else if (p.groups > 1) {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (e0 + j < p.E) cs[tok * p.E + e0 + j] = l[j];
      __syncwarp();
      for (int g = li; g < p.groups; g += L) {  // lane g scans group g
        const float* c = cs + tok * p.E + g * p.group_size;
        float a = -INFINITY, b = -INFINITY;
        for (int i = 0; i < p.group_size; ++i) {
          const float v = c[i];
          b = fmaxf(b, fminf(a, v));
          a = fmaxf(a, v);
        }
        gsc[tok * kRouteMaxGroups + g] = fmaxf((p.sigmoid && p.group_size > 1) ? a + b : a, -INFINITY);
      }
      __syncwarp();
      unsigned kept = 0;
      for (int g = li; g < p.groups; g += L) {
        const unsigned mine = number_key(gsc[tok * kRouteMaxGroups + g]);
        int above = 0;
        for (int o = 0; o < p.groups; ++o) {
          const unsigned other = number_key(gsc[tok * kRouteMaxGroups + o]);
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
    // The lane's two best go to the front by two passes over neighbours, which swap only when the later key is larger
    // (stable). A lane that has given both is rare; then every lane of the warp makes one more pass. (Sorting all
    // eight: 78 us.)
    int id[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) id[j] = e0 + j;
    auto best_to = [&](int front) {
#pragma unroll
      for (int j = EPL - 2; j >= 0; --j) {
        if (j < front) continue;
        const unsigned a = key[j], b = key[j + 1];
        const bool swap = b > a;
        const int ia = id[j], ib = id[j + 1];
        key[j] = max(a, b);
        key[j + 1] = min(a, b);
        id[j] = swap ? ib : ia;
        id[j + 1] = swap ? ia : ib;
      }
    };
    best_to(0);
    best_to(1);
    unsigned won = 0u, spent = 0u;  // lanes that have given one; lanes that have none in front
    for (int r = 0; r < p.k; ++r) {
      if (spent != 0u) best_to(0);
      bool win = true;
      unsigned winners = 0xffffffffu;
      if constexpr (L > 1) {
        const unsigned gm = lanes_max<L>(key[0]);
        const bool top = key[0] == gm;
        const unsigned who = __ballot_sync(0xffffffffu, top);
        if constexpr (L == 32) {
          winners = who & (0u - who);
          win = (winners >> lane) & 1u;
        } else {
          win = top && (who & lower) == 0u;
          winners = __ballot_sync(0xffffffffu, win);
        }
      }
      spent = won & winners;
      won |= winners;
      if (win) {  // the second moves up and leaves a hole, which the next pass carries to the back
        chosen[at * p.k + r] = id[0];
        key[0] = key[1], id[0] = id[1];
        key[1] = 0u;
      }
    }
  }
  __syncwarp();
  const int shift = __ffs(slots) - 1;
  // scores and weights of the batch's choices, `slots` lanes per token (a token's first choice in its first lane)
  for (int i = lane; i - lane < batch * slots; i += 32) {
    const int at = i >> shift, r = i & (slots - 1);
    const long long n = base + at;
    const bool on = at < batch && n < p.N && r < p.k;
    const int e = on ? chosen[at * p.k + r] : 0;
    const float l = on ? to_f<T>(reinterpret_cast<const T*>(p.logits)[n * p.ld + e]) : 0.f;
    float s, z = 1.f;
    if (p.sigmoid) {
      s = far_down(l) ? expf(l) : sigmoid_of(l);
    } else {
      // without the whole row's: the best of all (its group is the best group, and no bias moves the order)
      float mx = __shfl_sync(0xffffffffu, l, lane & ~(slots - 1));
      if (whole && on) {
        const float2 t = mxz[at];
        mx = t.x, z = t.y;
      }
      s = expf(l - (mx == -INFINITY ? 0.f : mx));
    }
    float sum = on ? s : 0.f;
    for (int o = slots / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float div = p.renorm ? sum + 1e-20f * z : z;
    if (whole && p.renorm && __any_sync(0xffffffffu, on && sum < 1e-13f)) {
      // A bias can move the choice far below the row's best. From about 30 on, the rounding of l - mx shows in the scores
      // and they end up subnormal beside 1e-20: such a token's are taken relative to its best choice, 1e-20 z exp(gap)
      // in two factors with the gap's own rounding given back.
      float best = on ? l : -INFINITY;
      for (int o = slots / 2; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
      const float top = on ? mxz[at].x : 0.f;
      if (best == -INFINITY) best = top;  // nothing but switched-off experts: weights of 0
      const float e = on ? expf(l - best) : 0.f;
      float all = e;
      for (int o = slots / 2; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      const float gap = top - best, back = top - gap, lost = (top - (gap + back)) + (back - best);
      const float half_gap = expf(0.5f * gap);
      if (sum < 1e-13f) s = e, div = all + 1e-20f * z * half_gap * half_gap * (1.f + lost);
    }
    if (on) {
      const bool ok = p.valid == nullptr || p.valid[n];
      p.w[n * p.k + r] = ok ? s / div * p.scale : 0.f;
      p.idx[n * p.k + r] = ok ? e : -1;
    }
  }
}

// The chosen experts' values go into a zeroed row in shared memory, from which the lanes write the dense row. A warp walks
// its tokens with a grid stride and, while each lane holds one choice (k <= L), loads two tokens ahead: the choices of the
// token after next, and the next token's logits at its choices (an address that depends on them). Without that, a token
// is a chain of two memory latencies (65536 x 256: 33 us with one token per warp).
template <typename T, int L, int EPL>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) route_bwd_kernel(RouteParams p, const float* __restrict__ dw,
                                                                     T* __restrict__ dlogits) {
  constexpr int TOKENS = ROUTE_WARPS * 32 / L, PITCH = L * EPL;
  __shared__ __align__(16) float rows[TOKENS * PITCH];
  const int li = lane_id() % L, tok = threadIdx.x / L;
  const int e0 = li * EPL;
  float* d = rows + tok * PITCH;
  const bool one = p.k <= L;
  struct Choice {
    int e = -1;  // -1: none (a token past the end, or without experts, or a lane past k)
    float w = 0.f, g = 0.f;
  };
  auto choice = [&](long long n, int r) {
    Choice c;
    if (n < p.N && r < p.k) {
      c.e = p.idx[n * p.k + r];
      c.w = p.w[n * p.k + r];
      c.g = c.e >= 0 ? dw[n * p.k + r] : 0.f;  // whatever reaches a padding row ends here
    }
    return c;
  };
  auto logit = [&](long long n, const Choice& c) {
    return p.sigmoid && c.e >= 0 ? to_f<T>(reinterpret_cast<const T*>(p.logits)[n * p.ld + c.e]) : 0.f;
  };
  auto scores = [&](float l, float& s, float& ds) {  // s and s' = s (1 - s)
    const float x = expf(-fabsf(l)), q = 1.f / (1.f + x);
    s = (l >= 0.f ? 1.f : x) * q;
    ds = x * q * q;
  };
  const long long stride = (long long)gridDim.x * TOKENS;
  long long n = (long long)blockIdx.x * TOKENS + tok;
  const long long rounds = (p.N - (long long)blockIdx.x * TOKENS + stride - 1) / stride;  // the block's, for the barriers
  Choice cur, nxt;
  float lc = 0.f;
  if (one) {
    cur = choice(n, li);
    nxt = choice(n + stride, li);
    lc = logit(n, cur);
  }
  for (long long it = 0; it < rounds; ++it, n += stride) {
    Choice far;
    float ln = 0.f;
    if (one) {
      far = choice(n + 2 * stride, li);
      ln = logit(n + stride, nxt);
    }
    const bool in = n < p.N;
#pragma unroll
    for (int j = 0; j < EPL; j += 4) *reinterpret_cast<float4*>(d + e0 + j) = make_float4(0.f, 0.f, 0.f, 0.f);
    // m = sum of r dw; total = S = sum of the chosen s (sigmoid) or sum of w (softmax)
    float m = 0.f, total = 0.f, se = 0.f, de = 0.f;
    if (one) {
      if (p.sigmoid && cur.e >= 0) scores(lc, se, de);
      m = cur.w * cur.g;
      total = p.sigmoid ? se : cur.w;
    } else {
      for (int r = li; r < p.k; r += L) {
        const Choice c = choice(n, r);
        if (p.sigmoid && c.e >= 0) scores(logit(n, c), se, de);
        m = fmaf(c.w, c.g, m);
        total += p.sigmoid ? (c.e >= 0 ? se : 0.f) : c.w;
      }
    }
    m = lanes_sum<L>(m) / p.scale;
    float others = 1.f;  // share of m that every expert's probability takes part in
    if (p.renorm) {
      others = 0.f;
      if (p.sigmoid) {
        total = lanes_sum<L>(total) + 1e-20f;
      } else if (p.biased) {
        others = 1.f - lanes_sum<L>(total) / p.scale;  // 1e-20 / S
        if (others < ROUTE_LOST) others = 0.f;
      }
    }
    __syncwarp();
    auto put = [&](const Choice& c, float ds) {
      const float up = p.renorm ? c.g - m : c.g;
      if (c.e >= 0) d[c.e] = p.sigmoid ? p.scale * up * ds / (p.renorm ? total : 1.f) : c.w * up;
    };
    if (one) {
      put(cur, de);
    } else {
      for (int r = li; r < p.k; r += L) {
        const Choice c = choice(n, r);
        if (p.sigmoid && c.e >= 0) scores(logit(n, c), se, de);
        put(c, de);
      }
    }
    __syncwarp();
    float v[EPL];
#pragma unroll
    for (int j = 0; j < EPL; j += 4) {
      const float4 t = *reinterpret_cast<const float4*>(d + e0 + j);
      v[j] = t.x, v[j + 1] = t.y, v[j + 2] = t.z, v[j + 3] = t.w;
    }
    // a token without experts has m 0; the lanes of a warp go together
    if (!p.sigmoid && (!p.renorm || (p.biased && __any_sync(0xffffffffu, others * m != 0.f)))) {
      float l[EPL];
      float mx = -INFINITY;
      if (in) load_logits<T, EPL>(p, n, e0, l);
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        if (!in) l[j] = 0.f;
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
      const float f = p.scale * m * others / z;
      if (others * m != 0.f)
#pragma unroll
        for (int j = 0; j < EPL; ++j) v[j] = fmaf(-f, l[j], v[j]);
    }
    if (in) {
      T* out = dlogits + n * p.E;
      if (p.vec) {
#pragma unroll
        for (int j = 0; j < EPL; j += 8)
          if (e0 + j < p.E) store_vec<T, 8>(out + e0 + j, *reinterpret_cast<const float(*)[8]>(&v[j]));
      } else {
#pragma unroll
        for (int j = 0; j < EPL; ++j)
          if (e0 + j < p.E) out[e0 + j] = from_f<T>(v[j]);
      }
    }
    cur = nxt;
    nxt = far;
    lc = ln;
  }
}

namespace {

template <typename T, int L, int EPL>
cudaError_t route_run(RouteParams p, const float* dw, void* dlogits, cudaStream_t s) {
  constexpr int TOKENS = ROUTE_WARPS * 32 / L;
  // whole 16-byte vectors of 8 logits, in rows and outputs; groups of a power of two of whole lanes
  p.vec = p.E % 8 == 0 && p.ld % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.bias) |
                                             reinterpret_cast<uintptr_t>(dlogits)) & 15) == 0;
  const int gl = p.group_size / EPL;
  p.group_lanes = p.group_size % EPL == 0 && (gl & (gl - 1)) == 0 ? gl : 0;
  const unsigned grid = (unsigned)(((long long)p.N + TOKENS - 1) / TOKENS);
  if (dlogits != nullptr) {
    // blocks that the SMs hold, walking the tokens
    route_bwd_kernel<T, L, EPL><<<std::min<unsigned>(grid, num_sms() * ROUTE_BWD_BLOCKS), ROUTE_WARPS * 32, 0, s>>>(
        p, dw, static_cast<T*>(dlogits));
  } else {
    // as many steps per batch as fill the lanes of its end, while every warp that the SMs hold still gets a batch
    int slots = 1;
    while (slots < p.k) slots *= 2;
    const long long warps = (long long)num_sms() * route_fwd_blocks(EPL) * ROUTE_WARPS, per = 32 / L;
    const int steps = (int)std::max(1ll, std::min<long long>(L / slots, p.N / (warps * per)));
    const long long batches = (p.N + steps * per - 1) / (steps * per);
    const unsigned blocks = (unsigned)((batches + ROUTE_WARPS - 1) / ROUTE_WARPS);
    const size_t smem = (size_t)ROUTE_WARPS * route_warp_smem(p, (int)per, steps);
    route_fwd_kernel<T, L, EPL><<<blocks, ROUTE_WARPS * 32, smem, s>>>(p, steps, slots);
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
  return p.N > 0 && dlogits == nullptr ? cudaErrorInvalidValue : route_launch(p, dw, dlogits, elem, s);
}

}  // namespace tgo

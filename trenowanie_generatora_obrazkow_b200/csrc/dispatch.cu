// From routing to the experts' products and back.
//
// plan: assignment a = n k + j (token n, its j-th choice, expert e = idx[a]) gets a row in expert order. Its rank among
// the assignments of e counts those before it in token order (a stable counting sort), and
//     slot[a] = offsets[e] + rank                     packed: expert e owns rows [offsets[e], offsets[e + 1])
//     slot[a] = e C + rank if rank < C, else -1       capacity C: static shapes, overflow dropped
// idx < 0 (a padding token) takes no row. One launch: a cluster of CTAs splits the assignments into contiguous spans,
// each warp counts its own span (lanes with the same expert find one another with match_any, the lowest adds), the
// CTAs exchange their totals through distributed shared memory, and a second walk over the span hands out the rows.
//
// dispatch  xs[slot[n, j]] = x[n]                                backward  dx[n] = sum_j dxs[slot[n, j]]
// combine   out[n] = sum_j w[n, j] y[slot[n, j]]                 backward  dy[slot[n, j]] = w[n, j] dout[n],
//                                                                          dw[n, j] = <dout[n], y[slot[n, j]]>
// All are bound by memory: the kernels walk tokens, not rows, so a token's row is read once for its k copies and a sum
// over its k rows stays in registers (fp32, fixed order: no atomics).
#include <algorithm>

#include "block_ops.h"
#include "common.cuh"
#include "vec.cuh"

namespace tgo {

// ------------------------------------------------------------------------------------------------------------------
// plan
// ------------------------------------------------------------------------------------------------------------------
namespace {

constexpr int PLAN_CTAS = 8;  // cluster size (portable limit)

__device__ __forceinline__ int dsmem_load(const int* p, uint32_t cta) {
  int v;
  const uint32_t addr = mapa_shared(smem_u32(p), cta);
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

}  // namespace

// dynamic shared memory: cnt [warps][E], tot [E] (this CTA's assignments of every expert), pre [E], warp sums [32]
__global__ void plan_kernel(PlanParams p) {
  extern __shared__ int plan_smem[];
  const int warps = blockDim.x >> 5, warp = warp_id(), lane = lane_id();
  int* cnt = plan_smem;
  int* tot = cnt + warps * p.E;
  int* pre = tot + p.E;
  int* wsum = pre + p.E;
  const int ctas = gridDim.x, cta = blockIdx.x;
  // contiguous spans of whole 32-assignment steps
  const int steps = (p.A + 31) / 32, units = ctas * warps;
  const int per = (steps + units - 1) / units;
  const long long a0 = (long long)(cta * warps + warp) * per * 32;
  for (int i = threadIdx.x; i < warps * p.E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  int* mine = cnt + warp * p.E;
  for (int i = 0; i < per; ++i) {
    const long long a = a0 + i * 32 + lane;
    int e = a < p.A ? p.idx[a] : -1;
    if ((unsigned)e >= (unsigned)p.E) e = -1;
    const unsigned peers = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && __ffs(peers) - 1 == lane) mine[e] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int run = 0;
    for (int w = 0; w < warps; ++w) {
      const int t = cnt[w * p.E + e];
      cnt[w * p.E + e] = run;
      run += t;
    }
    tot[e] = run;
  }
  if (ctas > 1) cluster_sync();
  else __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int before = 0, all = 0;
    if (ctas > 1) {
      for (int c = 0; c < ctas; ++c) {
        const int t = dsmem_load(tot + e, c);
        before += c < cta ? t : 0;
        all += t;
      }
    } else {
      all = tot[e];
    }
    for (int w = 0; w < warps; ++w) cnt[w * p.E + e] += before;
    pre[e] = all;
    if (cta == 0) p.counts[e] = all;
  }
  __syncthreads();
  // exclusive prefix of the totals (packed), in steps of the block
  int carry = 0;
  for (int b = 0; b < p.E; b += blockDim.x) {
    const int e = b + threadIdx.x;
    const int v = e < p.E ? pre[e] : 0;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int below = 0, sum = 0;
    for (int w = 0; w < warps; ++w) {
      below += w < warp ? wsum[w] : 0;
      sum += wsum[w];
    }
    if (e < p.E) pre[e] = p.capacity > 0 ? e * p.capacity : carry + below + inc - v;
    carry += sum;
    __syncthreads();
  }
  if (cta == 0) {
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) p.offsets[e] = pre[e];
    if (threadIdx.x == 0) p.offsets[p.E] = p.capacity > 0 ? p.E * p.capacity : carry;
  }
  for (int i = 0; i < per; ++i) {
    const long long a = a0 + i * 32 + lane;
    int e = a < p.A ? p.idx[a] : -1;
    if ((unsigned)e >= (unsigned)p.E) e = -1;
    const unsigned peers = __match_any_sync(0xffffffffu, e);
    const int ahead = __popc(peers & ((1u << lane) - 1u));
    int rank = 0;
    if (e >= 0) rank = mine[e] + ahead;
    __syncwarp();
    if (e >= 0 && ahead == 0) mine[e] += __popc(peers);
    __syncwarp();
    if (a < p.A) p.slot[a] = (e >= 0 && (p.capacity == 0 || rank < p.capacity)) ? pre[e] + rank : -1;
  }
  if (ctas > 1) cluster_sync();  // no CTA leaves while another may still read its totals
}

cudaError_t plan_launch(const PlanParams& p, cudaStream_t s) {
  if (p.A < 0 || p.E <= 0 || p.E > kRouteMaxExperts) return cudaErrorInvalidValue;
  // one CTA while it can keep up with one step of 32 per warp and a few rounds of it, else a cluster of 8
  const bool cluster = p.A > 8192;
  const int threads = cluster ? 1024 : std::min(1024, std::max(128, (p.A + 31) / 32 * 32));
  const size_t smem = sizeof(int) * ((size_t)(threads / 32) * p.E + 2 * p.E + 32);
  static bool set = false;
  if (!set) {
    cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(sizeof(int) * (34 * kRouteMaxExperts + 32)));
    if (e != cudaSuccess) return e;
    set = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(cluster ? PLAN_CTAS : 1);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, plan_kernel, p);
}

// ------------------------------------------------------------------------------------------------------------------
// dispatch / combine
// ------------------------------------------------------------------------------------------------------------------
namespace {

constexpr int ROW_WARPS = 8;   // warps per block, each on its own (token, column part) or rows to clear
constexpr int FILL_ROWS = 8;   // rows that one warp looks over for clearing
template <typename T, int V>
struct RowCfg {  // vectors in flight per lane: 64 bytes of columns per lane and row
  static constexpr int U = V == 8 ? 4 / (sizeof(T) / 2) : 4;
  static constexpr int COLS = U * 32 * V;  // columns of a part
};

// rows [offsets[E], rows) (packed) or the unfilled tail of every expert (capacity)
__device__ __forceinline__ bool row_unused(const ExpertRows& r, long long row) {
  if (r.capacity == 0) return row >= r.offsets[r.E];
  const int e = (int)(row / r.capacity);
  return row - (long long)e * r.capacity >= r.counts[e];
}

template <typename T, int V>
__device__ void clear_rows(const ExpertRows& r, T* out, long long unit) {
  Raw<T, V> z;
  z.zero();
  for (int i = 0; i < FILL_ROWS; ++i) {
    const long long row = unit * FILL_ROWS + i;
    if (row >= r.rows || !row_unused(r, row)) continue;
    for (int c = lane_id() * V; c < r.D; c += 32 * V) z.store(out + row * r.D + c);
  }
}

}  // namespace

template <typename T, int V>
__global__ void __launch_bounds__(ROW_WARPS * 32) dispatch_kernel(ExpertRows r, const T* __restrict__ x, long long ldx,
                                                                  T* __restrict__ xs, int parts) {
  using C = RowCfg<T, V>;
  const long long unit = (long long)blockIdx.x * ROW_WARPS + warp_id();
  if (unit >= (long long)r.N * parts) {
    clear_rows<T, V>(r, xs, unit - (long long)r.N * parts);
    return;
  }
  const int n = (int)(unit / parts), c0 = (int)(unit % parts) * C::COLS + lane_id() * V;
  Raw<T, V> v[C::U];
#pragma unroll
  for (int u = 0; u < C::U; ++u)
    if (c0 + u * 32 * V < r.D) v[u].load(x + (long long)n * ldx + c0 + u * 32 * V);
  for (int j = 0; j < r.k; ++j) {
    const long long slot = r.slot[(long long)n * r.k + j];
    if (slot < 0) continue;
    T* dst = xs + slot * r.D;
#pragma unroll
    for (int u = 0; u < C::U; ++u)
      if (c0 + u * 32 * V < r.D) v[u].store(dst + c0 + u * 32 * V);
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(ROW_WARPS * 32) combine_kernel(ExpertRows r, const T* __restrict__ y,
                                                                 const float* __restrict__ w, T* __restrict__ out,
                                                                 int parts) {
  using C = RowCfg<T, V>;
  const long long unit = (long long)blockIdx.x * ROW_WARPS + warp_id();
  if (unit >= (long long)r.N * parts) return;
  const int n = (int)(unit / parts), c0 = (int)(unit % parts) * C::COLS + lane_id() * V;
  float acc[C::U][V];
#pragma unroll
  for (int u = 0; u < C::U; ++u)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[u][i] = 0.f;
  for (int j = 0; j < r.k; ++j) {
    const long long slot = r.slot[(long long)n * r.k + j];
    if (slot < 0) continue;
    const float wj = w != nullptr ? w[(long long)n * r.k + j] : 1.f;
    const T* src = y + slot * r.D;
    Raw<T, V> v[C::U];
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
      if (c0 + u * 32 * V < r.D) v[u].load(src + c0 + u * 32 * V);
      else v[u].zero();
    }
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
      float f[V];
      v[u].get(f);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[u][i] = fmaf(wj, f[i], acc[u][i]);
    }
  }
#pragma unroll
  for (int u = 0; u < C::U; ++u)
    if (c0 + u * 32 * V < r.D) store_vec<T, V>(out + (long long)n * r.D + c0 + u * 32 * V, acc[u]);
}

// One warp per token: dout's columns are read once per part and used for the k rows; lane j keeps dw of choice j.
template <typename T, int V>
__global__ void __launch_bounds__(ROW_WARPS * 32) combine_bwd_kernel(ExpertRows r, const T* __restrict__ y,
                                                                     const float* __restrict__ w,
                                                                     const T* __restrict__ dout, long long ldo,
                                                                     T* __restrict__ dy, float* __restrict__ dw) {
  using C = RowCfg<T, V>;
  const long long n = (long long)blockIdx.x * ROW_WARPS + warp_id();
  if (n >= r.N) {
    clear_rows<T, V>(r, dy, n - r.N);
    return;
  }
  const int lane = lane_id();
  float mine = 0.f;
  for (int c0 = lane * V; c0 - lane * V < r.D; c0 += C::COLS) {
    Raw<T, V> g[C::U];
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
      if (c0 + u * 32 * V < r.D) g[u].load(dout + n * ldo + c0 + u * 32 * V);
      else g[u].zero();
    }
    for (int j = 0; j < r.k; ++j) {
      const long long slot = r.slot[n * r.k + j];
      if (slot < 0) continue;
      const float wj = w[n * r.k + j];
      Raw<T, V> v[C::U];
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
        if (c0 + u * 32 * V < r.D) v[u].load(y + slot * r.D + c0 + u * 32 * V);
        else v[u].zero();
      }
      float dot = 0.f;
#pragma unroll
      for (int u = 0; u < C::U; ++u) {
        float a[V], b[V], o[V];
        g[u].get(a);
        v[u].get(b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          dot = fmaf(a[i], b[i], dot);
          o[i] = wj * a[i];
        }
        if (c0 + u * 32 * V < r.D) store_vec<T, V>(dy + slot * r.D + c0 + u * 32 * V, o);
      }
      dot = warp_total(dot);
      if (lane == j) mine += dot;
    }
  }
  if (lane < r.k) dw[n * r.k + lane] = mine;
}

namespace {

template <typename T>
bool rows_aligned(const ExpertRows& r, const void* a, const void* b, long long ld) {
  return r.D % 8 == 0 && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(a) & 15) == 0 &&
         (reinterpret_cast<uintptr_t>(b) & 15) == 0;
}
template <typename T, int V>
int row_parts(const ExpertRows& r) {
  return (r.D + RowCfg<T, V>::COLS - 1) / RowCfg<T, V>::COLS;
}
bool row_grid(long long units, unsigned* grid) {
  const long long g = (units + ROW_WARPS - 1) / ROW_WARPS;
  *grid = (unsigned)g;
  return g > 0 && g < (1ll << 31);
}

template <typename T, int V>
cudaError_t dispatch_run(const ExpertRows& r, const T* x, long long ldx, T* xs, cudaStream_t s) {
  const int parts = row_parts<T, V>(r);
  unsigned grid;
  if (!row_grid((long long)r.N * parts + (r.rows + FILL_ROWS - 1) / FILL_ROWS, &grid)) return cudaErrorInvalidValue;
  dispatch_kernel<T, V><<<grid, ROW_WARPS * 32, 0, s>>>(r, x, ldx, xs, parts);
  return cudaGetLastError();
}
template <typename T, int V>
cudaError_t combine_run(const ExpertRows& r, const T* y, const float* w, T* out, cudaStream_t s) {
  const int parts = row_parts<T, V>(r);
  unsigned grid;
  if (!row_grid((long long)r.N * parts, &grid)) return cudaErrorInvalidValue;
  combine_kernel<T, V><<<grid, ROW_WARPS * 32, 0, s>>>(r, y, w, out, parts);
  return cudaGetLastError();
}
template <typename T, int V>
cudaError_t combine_bwd_run(const ExpertRows& r, const T* y, const float* w, const T* dout, long long ldo, T* dy,
                            float* dw, cudaStream_t s) {
  unsigned grid;
  if (!row_grid(r.N + (r.rows + FILL_ROWS - 1) / FILL_ROWS, &grid)) return cudaErrorInvalidValue;
  combine_bwd_kernel<T, V><<<grid, ROW_WARPS * 32, 0, s>>>(r, y, w, dout, ldo, dy, dw);
  return cudaGetLastError();
}

}  // namespace

#define TGO_BY_ELEM(elem, CALL)            \
  switch (elem) {                          \
    case ELEM_BF16: CALL(__nv_bfloat16);   \
    case ELEM_F16: CALL(__half);           \
    case ELEM_F32: CALL(float);            \
  }                                        \
  return cudaErrorInvalidValue

cudaError_t dispatch_launch(const ExpertRows& r, const void* x, long long ldx, void* xs, int elem, cudaStream_t s) {
  if (r.D <= 0 || (r.N <= 0 && r.rows <= 0)) return cudaSuccess;
#define TGO_CALL(T)                                                                                        \
  return rows_aligned<T>(r, x, xs, ldx)                                                                    \
             ? dispatch_run<T, 8>(r, static_cast<const T*>(x), ldx, static_cast<T*>(xs), s)                \
             : dispatch_run<T, 1>(r, static_cast<const T*>(x), ldx, static_cast<T*>(xs), s)
  TGO_BY_ELEM(elem, TGO_CALL);
#undef TGO_CALL
}

cudaError_t combine_launch(const ExpertRows& r, const void* y, const float* w, void* out, int elem, cudaStream_t s) {
  if (r.D <= 0 || r.N <= 0) return cudaSuccess;
#define TGO_CALL(T)                                                                                  \
  return rows_aligned<T>(r, y, out, 8)                                                               \
             ? combine_run<T, 8>(r, static_cast<const T*>(y), w, static_cast<T*>(out), s)            \
             : combine_run<T, 1>(r, static_cast<const T*>(y), w, static_cast<T*>(out), s)
  TGO_BY_ELEM(elem, TGO_CALL);
#undef TGO_CALL
}

cudaError_t combine_bwd_launch(const ExpertRows& r, const void* y, const float* w, const void* dout, long long ldo,
                               void* dy, float* dw, int elem, cudaStream_t s) {
  if (r.N <= 0 && r.rows <= 0) return cudaSuccess;
#define TGO_CALL(T)                                                                                                    \
  return rows_aligned<T>(r, y, dout, ldo) && (reinterpret_cast<uintptr_t>(dy) & 15) == 0                               \
             ? combine_bwd_run<T, 8>(r, static_cast<const T*>(y), w, static_cast<const T*>(dout), ldo,                 \
                                     static_cast<T*>(dy), dw, s)                                                       \
             : combine_bwd_run<T, 1>(r, static_cast<const T*>(y), w, static_cast<const T*>(dout), ldo,                 \
                                     static_cast<T*>(dy), dw, s)
  TGO_BY_ELEM(elem, TGO_CALL);
#undef TGO_CALL
}

}  // namespace tgo

// From routing to the experts' products and back.
//
// plan: assignment a = n k + j (token n, its j-th choice, expert e = idx[a]) gets a row in expert order. Its rank among
// the assignments of e counts those before it in token order (a stable counting sort), and
//     slot[a] = offsets[e] + rank                     packed: expert e owns rows [offsets[e], offsets[e + 1])
//     slot[a] = e C + rank if rank < C, else -1       capacity C: static shapes, overflow dropped
// idx < 0 (a padding token) takes no row. One launch: a cluster of CTAs splits the assignments into contiguous spans,
// each warp counts its own span, the CTAs exchange their totals through distributed shared memory, and a second walk over
// the span hands out the rows (lanes with the same expert find one another by ballots).
//
// dispatch  xs[slot[n, j]] = x[n]                                backward  dx[n] = sum_j dxs[slot[n, j]]
// combine   out[n] = sum_j w[n, j] y[slot[n, j]]                 backward  dy[slot[n, j]] = w[n, j] dout[n],
//                                                                          dw[n, j] = <dout[n], y[slot[n, j]]>
// All are bound by memory: the kernels walk tokens, not rows, so a token's row is read once for its k copies and a sum
// over its k rows stays in registers (fp32, fixed order: no atomics). 32768 x 2048 bf16, 2 choices, with their launches:
// dispatch 84 us, combine 72 us, its backward 125 us (0.85, 0.86, 0.90 of a plain copy's rate); 8191 x 1280, 8 choices: 37,
// 45, 72 us. The plan: 9 us for 65536 assignments to 8 experts, 11 us to 64.
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

// Lanes of the warp with this lane's expert (>= 0), from one ballot per bit of the expert's number: a constant
// log2(E) + 1 ballots, where match_any takes a round per distinct value (8191 x 8 choices of 64: 18.4 us with it).
__device__ __forceinline__ unsigned same_expert(int e, int bits) {
  unsigned peers = __ballot_sync(0xffffffffu, e >= 0);
  for (int b = 0; b < bits; ++b) {
    const bool set = (e >> b) & 1;
    const unsigned m = __ballot_sync(0xffffffffu, set);
    peers &= set ? m : ~m;
  }
  return peers;
}

}  // namespace

// dynamic shared memory: cnt [E][33] (assignments of every expert and warp, one pad against bank conflicts), tot [E] (this
// CTA's assignments of every expert), pre [E], warp sums [32]
constexpr int PLAN_PITCH = 33;
constexpr int PLAN_BATCH = 8;  // steps of 32 assignments whose loads a warp issues together

__global__ void __launch_bounds__(1024) plan_kernel(PlanParams p) {
  extern __shared__ int plan_smem[];
  const int warps = blockDim.x >> 5, warp = warp_id(), lane = lane_id();
  int* cnt = plan_smem;
  int* tot = cnt + PLAN_PITCH * p.E;
  int* pre = tot + p.E;
  int* wsum = pre + p.E;
  const int ctas = gridDim.x, cta = blockIdx.x;
  // contiguous spans of whole 32-assignment steps
  const int steps = (p.A + 31) / 32, units = ctas * warps;
  const int per = (steps + units - 1) / units;
  const long long a0 = (long long)(cta * warps + warp) * per * 32 + lane;
  int e[PLAN_BATCH];
  auto fetch = [&](int i0) {  // experts of the steps i0 .. i0 + PLAN_BATCH - 1, -1: none
#pragma unroll
    for (int i = 0; i < PLAN_BATCH; ++i) {
      const long long a = a0 + (long long)(i0 + i) * 32;
      e[i] = i0 + i < per && a < p.A ? p.idx[a] : -1;
      if ((unsigned)e[i] >= (unsigned)p.E) e[i] = -1;
    }
  };
  fetch(0);
  for (int i = threadIdx.x; i < PLAN_PITCH * p.E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < per; i0 += PLAN_BATCH) {
    if (i0 > 0) fetch(i0);
#pragma unroll
    for (int i = 0; i < PLAN_BATCH; ++i)
      if (e[i] >= 0) atomicAdd(&cnt[e[i] * PLAN_PITCH + warp], 1);
  }
  __syncthreads();
  // a warp per expert: exclusive prefix of its counts over the CTA's warps
  for (int x = warp; x < p.E; x += warps) {
    const int v = lane < warps ? cnt[x * PLAN_PITCH + lane] : 0;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    cnt[x * PLAN_PITCH + lane] = inc - v;
    if (lane == 31) tot[x] = inc;
  }
  if (ctas > 1) cluster_sync();
  else __syncthreads();
  // totals over the CTAs (pre) and what the CTAs before this one hold (tot: read by the others, so kept apart)
  int carry = 0;
  for (int b = 0; b < p.E; b += blockDim.x) {
    const int x = b + threadIdx.x;
    int before = 0, all = 0;
    if (x < p.E) {
      if (ctas > 1) {
        int t[PLAN_CTAS];
#pragma unroll
        for (int c = 0; c < PLAN_CTAS; ++c) t[c] = dsmem_load(tot + x, c);
#pragma unroll
        for (int c = 0; c < PLAN_CTAS; ++c) {
          before += c < cta ? t[c] : 0;
          all += t[c];
        }
      } else {
        all = tot[x];
      }
      if (cta == 0) p.counts[x] = all;
    }
    // exclusive prefix of the totals (packed), in steps of the block
    int inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int w = lane < warps ? wsum[lane] : 0, run = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += t;
    }
    const int below = __shfl_sync(0xffffffffu, run - w, warp), sum = __shfl_sync(0xffffffffu, run, 31);
    if (x < p.E) {
      const int start = p.capacity > 0 ? x * p.capacity : carry + below + inc - all;
      pre[x] = start + before;  // row of this CTA's first assignment of x
      if (cta == 0) p.offsets[x] = start;
    }
    carry += sum;
    __syncthreads();
  }
  if (cta == 0 && threadIdx.x == 0) p.offsets[p.E] = p.capacity > 0 ? p.E * p.capacity : carry;
  int* mine = cnt + warp;
  const int bits = 32 - __clz(p.E - 1);
  for (int i0 = 0; i0 < per; i0 += PLAN_BATCH) {
    if (per > PLAN_BATCH) fetch(i0);
#pragma unroll
    for (int i = 0; i < PLAN_BATCH; ++i) {
      if (i0 + i >= per) break;  // warp-uniform
      const unsigned peers = same_expert(e[i], bits);
      const int ahead = __popc(peers & ((1u << lane) - 1u));
      int row = -1;
      if (e[i] >= 0) row = pre[e[i]] + mine[e[i] * PLAN_PITCH] + ahead;
      __syncwarp();
      if (e[i] >= 0 && ahead == 0) mine[e[i] * PLAN_PITCH] += __popc(peers);
      __syncwarp();
      if (p.capacity > 0 && e[i] >= 0 && row >= (e[i] + 1) * p.capacity) row = -1;
      const long long a = a0 + (long long)(i0 + i) * 32;
      if (a < p.A) p.slot[a] = row;
    }
  }
  if (ctas > 1) cluster_sync();  // no CTA leaves while another may still read its totals
}

cudaError_t plan_launch(const PlanParams& p, cudaStream_t s) {
  if (p.A < 0 || p.E <= 0 || p.E > kRouteMaxExperts) return cudaErrorInvalidValue;
  // One CTA while the cluster's launch and exchange cost more than its 8 times as many warps save. us, one CTA / cluster of 8,
  // 8, 64, 256 experts: 2048 assignments 4.5 / 4.9, 5.3 / 5.6, 6.8 / 7.2; 4096: 5.5 / 5.0, 6.6 / 5.6, 8.2 / 7.2;
  // 65536: 44 / 8.7, 57 / 10.8, 61 / 12.6.
  const bool cluster = p.A > 2048;
  const int threads = cluster ? 1024 : std::min(1024, std::max(128, (p.A + 31) / 32 * 32));
  const size_t smem = sizeof(int) * ((PLAN_PITCH + 2) * p.E + 32);
  if (smem > 48 * 1024) {  // over about 340 experts
    cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
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
  static constexpr int COLS = U * 32 * V;  // the most columns of a part
};

// the slots (and weights) of a token's choices: lane j holds choice j (k <= 32), so no load stands between two rows
struct Choices {
  int slot;
  float w;
  __device__ __forceinline__ Choices(const ExpertRows& r, long long n, const float* weights) {
    const bool on = lane_id() < r.k;
    slot = on ? r.slot[n * r.k + lane_id()] : -1;
    w = on && weights != nullptr ? weights[n * r.k + lane_id()] : 1.f;
  }
  __device__ __forceinline__ long long row(int j) const { return __shfl_sync(0xffffffffu, slot, j); }
  __device__ __forceinline__ float weight(int j) const { return __shfl_sync(0xffffffffu, w, j); }
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

// a part: columns [c0, c1) of a row, at most RowCfg::COLS
template <typename T, int V>
__global__ void __launch_bounds__(ROW_WARPS * 32) dispatch_kernel(ExpertRows r, const T* __restrict__ x, long long ldx,
                                                                  T* __restrict__ xs, int parts, int cols) {
  using C = RowCfg<T, V>;
  const long long unit = (long long)blockIdx.x * ROW_WARPS + warp_id();
  if (unit >= (long long)r.N * parts) {
    clear_rows<T, V>(r, xs, unit - (long long)r.N * parts);
    return;
  }
  const int n = (int)(unit / parts), part = (int)(unit % parts);
  const int c0 = part * cols + lane_id() * V, c1 = min(r.D, (part + 1) * cols);
  Raw<T, V> v[C::U];
#pragma unroll
  for (int u = 0; u < C::U; ++u)
    if (c0 + u * 32 * V < c1) v[u].load(x + (long long)n * ldx + c0 + u * 32 * V);
  const Choices ch(r, n, nullptr);
  for (int j = 0; j < r.k; ++j) {
    const long long slot = ch.row(j);
    if (slot < 0) continue;
    T* dst = xs + slot * r.D;
#pragma unroll
    for (int u = 0; u < C::U; ++u)
      if (c0 + u * 32 * V < c1) v[u].store(dst + c0 + u * 32 * V);
  }
}

// J rows of U vectors per lane in flight, and U vectors of fp32 sums: few choices take wide parts, many take narrow parts
// and more rows (8191 x 1280, 8 choices: U 4, J 2 50.9 us).
template <typename T, int V, int U, int J>
__global__ void __launch_bounds__(ROW_WARPS * 32, 4) combine_kernel(ExpertRows r, const T* __restrict__ y,
                                                                 const float* __restrict__ w, T* __restrict__ out,
                                                                 int parts, int cols) {
  const long long unit = (long long)blockIdx.x * ROW_WARPS + warp_id();
  if (unit >= (long long)r.N * parts) return;
  const int n = (int)(unit / parts), part = (int)(unit % parts);
  const int c0 = part * cols + lane_id() * V, c1 = min(r.D, (part + 1) * cols);
  const Choices ch(r, n, w);
  float acc[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[u][i] = 0.f;
  for (int j0 = 0; j0 < r.k; j0 += J) {
    Raw<T, V> v[J][U];
    float wj[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      // a dropped choice (and a missing one of the last pair) adds nothing: its rows are not read
      const long long slot = ch.row((j0 + j) & 31);
      const bool on = j0 + j < r.k && slot >= 0;
      wj[j] = on ? ch.weight((j0 + j) & 31) : 0.f;  // `on` is the warp's
      const T* src = y + slot * r.D;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (on && c0 + u * 32 * V < c1) v[j][u].load(src + c0 + u * 32 * V);
        else v[j][u].zero();
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[V];
        v[j][u].get(f);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[u][i] = fmaf(wj[j], f[i], acc[u][i]);
      }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c0 + u * 32 * V < c1) store_vec<T, V>(out + (long long)n * r.D + c0 + u * 32 * V, acc[u]);
}

// One warp per token: dout's columns are read once per part of U vectors per lane and used for the k rows; lane j keeps dw
// of choice j. More warps beat more loads per warp here: 8191 x 1280, 8 choices, with two rows in flight and 99 registers
// 90 us, with one row and 64 registers 74 us.
template <typename T, int V>
__global__ void __launch_bounds__(ROW_WARPS * 32, 4) combine_bwd_kernel(ExpertRows r, const T* __restrict__ y,
                                                                     const float* __restrict__ w,
                                                                     const T* __restrict__ dout, long long ldo,
                                                                     T* __restrict__ dy, float* __restrict__ dw) {
  constexpr int U = RowCfg<T, V>::U, COLS = RowCfg<T, V>::COLS;
  const long long n = (long long)blockIdx.x * ROW_WARPS + warp_id();
  if (n >= r.N) {
    clear_rows<T, V>(r, dy, n - r.N);
    return;
  }
  const int lane = lane_id();
  const Choices ch(r, n, w);
  float mine = 0.f;
  for (int c0 = lane * V; c0 - lane * V < r.D; c0 += COLS) {
    Raw<T, V> g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + u * 32 * V < r.D) g[u].load(dout + n * ldo + c0 + u * 32 * V);
      else g[u].zero();
    }
    for (int j = 0; j < r.k; ++j) {
      const long long slot = ch.row(j);
      if (slot < 0) continue;
      const float wj = ch.weight(j);
      Raw<T, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c0 + u * 32 * V < r.D) v[u].load(y + slot * r.D + c0 + u * 32 * V);
        else v[u].zero();
      }
      float dot = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
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
// parts of a row of at most `most` columns, of equal numbers of whole vector columns
int row_parts(const ExpertRows& r, int most, int step, int* cols) {
  const int parts = (r.D + most - 1) / most;
  *cols = ((r.D + parts - 1) / parts + step - 1) / step * step;
  return parts;
}
bool row_grid(long long units, unsigned* grid) {
  const long long g = (units + ROW_WARPS - 1) / ROW_WARPS;
  *grid = (unsigned)g;
  return g > 0 && g < (1ll << 31);
}

template <typename T, int V>
cudaError_t dispatch_run(const ExpertRows& r, const T* x, long long ldx, T* xs, cudaStream_t s) {
  int cols;
  const int parts = row_parts(r, RowCfg<T, V>::COLS, 32 * V, &cols);
  unsigned grid;
  if (!row_grid((long long)r.N * parts + (r.rows + FILL_ROWS - 1) / FILL_ROWS, &grid)) return cudaErrorInvalidValue;
  dispatch_kernel<T, V><<<grid, ROW_WARPS * 32, 0, s>>>(r, x, ldx, xs, parts, cols);
  return cudaGetLastError();
}
template <typename T, int V, int U, int J>
cudaError_t combine_run_with(const ExpertRows& r, const T* y, const float* w, T* out, cudaStream_t s) {
  int cols;
  const int parts = row_parts(r, U * 32 * V, 32 * V, &cols);
  unsigned grid;
  if (!row_grid((long long)r.N * parts, &grid)) return cudaErrorInvalidValue;
  combine_kernel<T, V, U, J><<<grid, ROW_WARPS * 32, 0, s>>>(r, y, w, out, parts, cols);
  return cudaGetLastError();
}
// us, wide parts with 2 rows / narrow parts with 4 rows: 32768 x 2048 bf16 k 1 49.9 / 68.1, k 2 67.9 / 79.6, k 3 88.3 / 90.2,
// k 8 186 / 186; 8191 x 1280 k 2 16.9 / 17.1, k 3 22.3 / 19.7, k 8 43.6 / 41.4; 512 x 2048 k 2 4.8 / 4.2, k 8 9.4 / 7.3.
template <typename T, int V>
cudaError_t combine_run(const ExpertRows& r, const T* y, const float* w, T* out, cudaStream_t s) {
  constexpr int U = RowCfg<T, V>::U;
  return r.k <= 2 ? combine_run_with<T, V, U, 2>(r, y, w, out, s) : combine_run_with<T, V, U / 2, 4>(r, y, w, out, s);
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
  if (r.D <= 0 || r.rows <= 0) return cudaSuccess;
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

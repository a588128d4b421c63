// Launch interfaces of the kernels of a routed transformer block: expert routing, expert dispatch / combine, norms
// before and after a branch with its gate and residual scale, rotary positions with several axes. Plain CUDA types
// only; the torch-facing checks are in block_ops.cpp.
#pragma once
#include <cuda_runtime.h>

namespace tgo {

enum ElemType : int { ELEM_BF16 = 0, ELEM_F16 = 1, ELEM_F32 = 2 };

// ---------------------------------------------------------------- expert routing (route.cu)
constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 32;
struct RouteParams {
  const void* logits;      // [N, E], row stride ld
  long long ld;
  const float* bias;       // [E] or null: added to the selection scores only
  const bool* valid;       // [N] or null
  float* w;                // [N, k]
  int* idx;                // [N, k]
  int N, E, k;
  int groups, top_groups, group_size;
  unsigned group_magic;    // ceil(2^22 / group_size): e / group_size == (e * magic) >> 22 for e < 512
  int sigmoid, renorm;
  int biased;              // backward: the choice was made with a bias
  float scale;
  int vec, group_lanes;    // set by the launchers (route.cu)
};
cudaError_t route_fwd_launch(const RouteParams& p, int elem, cudaStream_t s);
// dlogits [N, E] contiguous, in the logits' type; p.w and p.idx are read
cudaError_t route_bwd_launch(const RouteParams& p, const float* dw, void* dlogits, int elem, cudaStream_t s);

// ---------------------------------------------------------------- expert plan, dispatch, combine (dispatch.cu)
struct PlanParams {
  const int* idx;     // [A]: expert of each assignment (token-major), < 0 or >= E: none
  int A, E;
  int capacity;       // 0: packed by expert
  int* slot;          // [A]
  int* offsets;       // [E + 1]
  int* counts;        // [E]: assignments of each expert, dropped ones included
};
cudaError_t plan_launch(const PlanParams& p, cudaStream_t s);

struct ExpertRows {
  const int* slot;     // [N, k]
  const int* offsets;  // [E + 1]
  const int* counts;   // [E]
  int N, k, D, E, capacity;
  long long rows;      // rows in expert order
};
// xs[slot[n, j]] = x[n] (row stride ldx); rows that no assignment fills are zeroed
cudaError_t dispatch_launch(const ExpertRows& r, const void* x, long long ldx, void* xs, int elem, cudaStream_t s);
// out[n] = sum_j w[n, j] y[slot[n, j]] (w null: 1)
cudaError_t combine_launch(const ExpertRows& r, const void* y, const float* w, void* out, int elem, cudaStream_t s);
// dy[slot[n, j]] = w[n, j] dout[n] (other rows zero), dw[n, j] = <dout[n], y[slot[n, j]]>
cudaError_t combine_bwd_launch(const ExpertRows& r, const void* y, const float* w, const void* dout, long long ldo,
                               void* dy, float* dw, int elem, cudaStream_t s);

// ---------------------------------------------------------------- sandwich norm (sandwich.cu)
struct SandwichParams {
  const void* x;
  const void* y;         // [M, D] contiguous
  const void* gate;      // [B, D] rows (stride gate_bs) or null
  const void* shift;     // [B, D] rows (stride mod_bs) or null, with scale
  const void* scale;
  long long gate_bs, mod_bs;
  const float* post_w;   // [D] or null: no norm of the branch
  const float* w;        // [D] or null: no h
  float res_scale, eps;
  int M, D, T;           // T rows per sample
  void* x_new;           // forward outputs
  void* h;
  float* rstd_y;         // [M], with post_w
  float* rstd_x;         // [M], with w
};
struct SandwichBwdParams {
  const void* dx_new;    // [M, D] or null
  const void* dh;        // [M, D] or null
  void* dx;
  void* dy;
  float* partial;        // [entries][3][D] (see sandwich.cu)
  float* wpart;          // [sample groups][2][D]
  void* dgate;           // [B, D] contiguous, in x's type, or null
  void* dshift;
  void* dscale;
  float* dpost_w;        // [D], added to or written, or null
  float* dw;
  bool add_post_w, add_w;
  int ctas, rows_per_cta, groups;  // units of rows (see sandwich.cu), groups of samples of the reduction
};
// err: device error word of the kernels' bounded waits
cudaError_t sandwich_fwd_launch(const SandwichParams& p, int elem, int* err, cudaStream_t s);
cudaError_t sandwich_bwd_plan(const SandwichParams& p, int elem, SandwichBwdParams* q);  // sets ctas, rows_per_cta, groups
cudaError_t sandwich_bwd_launch(const SandwichParams& p, const SandwichBwdParams& q, int elem, int* err, cudaStream_t s);

// ---------------------------------------------------------------- rotary positions with several axes (rope_axes.cu)
constexpr int kRopeMaxAxes = 4;
struct RopeAxesParams {
  const void* q;
  const void* k;
  long long q_ts, k_ts;    // token strides (heads contiguous: hd elements apart)
  void* q_out;             // [M, hq, hd] contiguous
  void* k_out;             // [M, hkv, hd]
  const void* pos;         // [M, axes] int32 or fp32
  int pos_f32;
  const float* freq;       // [2][rot / 2]: revolutions per position of every rotated pair, high and low parts
  const int* axis;         // [rot / 2]: position axis of every pair
  const float* q_w;        // [hd] or null
  const float* k_w;
  float eps;
  int M, axes, hq, hkv, hd, rot, interleaved;
  long long dq_ts, dk_ts;  // backward: token strides of dq_in / dk_in
};
cudaError_t rope_axes_fwd_launch(const RopeAxesParams& p, int elem, cudaStream_t s);
// dq / dk [M, h, hd] contiguous -> dq_in / dk_in [M, h, hd], a token's heads contiguous; dq_w / dk_w [hd] added to or written through partials
// [rope_axes_bwd_ctas()][2][hd] (the most CTAs of any launch)
int rope_axes_bwd_ctas();
cudaError_t rope_axes_bwd_launch(const RopeAxesParams& p, const void* dq, const void* dk, void* dq_in, void* dk_in,
                                 float* partial, float* dq_w, float* dk_w, bool add_q_w, bool add_k_w, int elem,
                                 cudaStream_t s);

}  // namespace tgo

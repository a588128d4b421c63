// Torch-facing wrappers of the routed block's kernels (block_ops.h): argument checks, outputs, launches on the current
// stream. Registered in the extension module by ops.cpp.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <atomic>
#include <cmath>

#include "block_ops.h"
#include "kernels.h"

namespace tgo {

void count_launches(int n);  // ops.cpp

namespace {

using OptT = c10::optional<at::Tensor>;

#define BLOCK_LAUNCH(expr, n)                                                         \
  do {                                                                                \
    cudaError_t _e = (expr);                                                          \
    TORCH_CHECK(_e == cudaSuccess, "kernel launch failed: ", cudaGetErrorString(_e)); \
    count_launches(n);                                                                \
  } while (0)

int elem_of(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return ELEM_BF16;
    case at::kHalf: return ELEM_F16;
    case at::kFloat: return ELEM_F32;
    default: TORCH_CHECK(false, what, ": bf16, fp16 or fp32 expected, got ", t.scalar_type());
  }
  return -1;
}
// An uninitialised contiguous tensor on as's device, past the dispatcher (half the host time of at::empty; a small step
// makes a dozen of them).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& as) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, as.device(), c10::nullopt));
}
at::Tensor fresh_like(const at::Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }
bool given(const OptT& t) { return t.has_value() && t->defined(); }
void same_device(const at::Tensor& t, const at::Tensor& as, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == as.device(), what, ": a tensor on ", as.device(), " expected");
}
const float* vec_f32(const OptT& t, int64_t n, const at::Tensor& as, const char* what) {
  if (!given(t)) return nullptr;
  same_device(*t, as, what);
  TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == n, what, ": contiguous fp32 [", n,
              "] expected");
  return t->data_ptr<float>();
}
float* acc_f32(const OptT& t, int64_t n, const at::Tensor& as, const char* what) {
  return const_cast<float*>(vec_f32(t, n, as, what));
}

// [N, D] with a row's elements side by side (an empty tensor's strides say nothing: a sum's gradient expands to 0)
bool whole_rows(const at::Tensor& t) { return t.numel() == 0 || t.size(1) == 1 || t.stride(1) == 1; }

int* err_word(const at::Tensor& err, const at::Tensor& as) {
  same_device(err, as, "err");
  TORCH_CHECK(err.scalar_type() == at::kInt && err.numel() >= 1, "err: int32 error word");
  return err.data_ptr<int>();
}

// ---------------------------------------------------------------------------------------------------------- routing
RouteParams route_params(const at::Tensor& logits, int64_t k, bool sigmoid, int64_t groups, int64_t top_groups,
                         bool renorm, double scale) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && whole_rows(logits),
              "route: logits [N, E] with contiguous rows");
  const int64_t N = logits.size(0), E = logits.size(1);
  TORCH_CHECK(N < (1ll << 31) && E >= 1 && E <= kRouteMaxExperts, "route: 1 to ", kRouteMaxExperts, " experts");
  TORCH_CHECK(groups >= 1 && groups <= kRouteMaxGroups && E % groups == 0, "route: groups must divide the experts (at most ",
              kRouteMaxGroups, ")");
  TORCH_CHECK(top_groups >= 1 && top_groups <= groups, "route: 1 <= top_groups <= groups");
  TORCH_CHECK(k >= 1 && k <= kRouteMaxK && k <= top_groups * (E / groups), "route: k between 1 and ", kRouteMaxK,
              " and at most the experts of the kept groups");
  // the backward divides by it
  TORCH_CHECK(std::isnormal((float)scale), "route: scale must be a normal fp32 number and not zero");
  RouteParams p{};
  p.logits = logits.data_ptr();
  p.ld = logits.stride(0);
  p.N = (int)N;
  p.E = (int)E;
  p.k = (int)k;
  p.groups = (int)groups;
  p.top_groups = (int)top_groups;
  p.group_size = (int)(E / groups);
  p.group_magic = (unsigned)(((1u << 22) + p.group_size - 1) / p.group_size);
  p.sigmoid = sigmoid;
  p.renorm = renorm;
  p.scale = (float)scale;
  return p;
}

std::tuple<at::Tensor, at::Tensor> route_fwd(at::Tensor logits, OptT bias, OptT valid, int64_t k, bool sigmoid,
                                             int64_t groups, int64_t top_groups, bool renorm, double scale) {
  RouteParams p = route_params(logits, k, sigmoid, groups, top_groups, renorm, scale);
  const c10::cuda::CUDAGuard guard(logits.device());
  p.bias = vec_f32(bias, p.E, logits, "route: bias");
  if (given(valid)) {
    same_device(*valid, logits, "route: valid");
    TORCH_CHECK(valid->scalar_type() == at::kBool && valid->is_contiguous() && valid->numel() == p.N,
                "route: valid bool [N]");
    p.valid = valid->data_ptr<bool>();
  }
  at::Tensor w = fresh({p.N, k}, at::kFloat, logits);
  at::Tensor idx = fresh({p.N, k}, at::kInt, logits);
  p.w = w.data_ptr<float>();
  p.idx = idx.data_ptr<int>();
  BLOCK_LAUNCH(route_fwd_launch(p, elem_of(logits, "route"), at::cuda::getCurrentCUDAStream()), p.N > 0);
  return {w, idx};
}

at::Tensor route_bwd(at::Tensor logits, at::Tensor w, at::Tensor idx, at::Tensor dw, bool biased, bool sigmoid,
                     bool renorm, double scale) {
  RouteParams p = route_params(logits, w.size(1), sigmoid, 1, 1, renorm, scale);
  p.biased = biased;
  const c10::cuda::CUDAGuard guard(logits.device());
  same_device(idx, logits, "route_bwd: idx");
  TORCH_CHECK(idx.scalar_type() == at::kInt && idx.is_contiguous() && idx.sizes() == w.sizes() && w.size(0) == p.N,
              "route_bwd: idx int32 [N, k]");
  p.w = const_cast<float*>(vec_f32(w, w.numel(), logits, "route_bwd: w"));
  p.idx = idx.data_ptr<int>();
  const float* g = vec_f32(dw, w.numel(), logits, "route_bwd: dw");
  at::Tensor d = fresh({p.N, p.E}, logits.scalar_type(), logits);
  BLOCK_LAUNCH(route_bwd_launch(p, g, d.data_ptr(), elem_of(logits, "route_bwd"), at::cuda::getCurrentCUDAStream()),
               p.N > 0);
  return d;
}

// ------------------------------------------------------------------------------------------ plan, dispatch, combine
std::tuple<at::Tensor, at::Tensor, at::Tensor> expert_plan(at::Tensor idx, int64_t experts, int64_t capacity) {
  TORCH_CHECK(idx.is_cuda() && idx.dim() == 2 && idx.scalar_type() == at::kInt && idx.is_contiguous(),
              "expert_plan: idx int32 [N, k], contiguous");
  TORCH_CHECK(experts >= 1 && experts <= kRouteMaxExperts, "expert_plan: 1 to ", kRouteMaxExperts, " experts");
  // a row number is an int, also before the capacity cuts it off
  TORCH_CHECK(capacity >= 0 && capacity < (1ll << 31) && capacity * experts + idx.numel() < (1ll << 31) - 65536,
              "expert_plan: too many rows");
  const c10::cuda::CUDAGuard guard(idx.device());
  PlanParams p{};
  p.idx = idx.data_ptr<int>();
  p.A = (int)idx.numel();
  p.E = (int)experts;
  p.capacity = (int)capacity;
  at::Tensor slot = fresh_like(idx);
  at::Tensor offsets = fresh({experts + 1}, at::kInt, idx);
  at::Tensor counts = fresh({experts}, at::kInt, idx);
  p.slot = slot.data_ptr<int>();
  p.offsets = offsets.data_ptr<int>();
  p.counts = counts.data_ptr<int>();
  BLOCK_LAUNCH(plan_launch(p, at::cuda::getCurrentCUDAStream()), 1);
  return {slot, offsets, counts};
}

ExpertRows expert_rows(const at::Tensor& slot, const at::Tensor& offsets, const at::Tensor& counts, int64_t capacity,
                       int64_t rows, int64_t D, const at::Tensor& as) {
  same_device(slot, as, "expert rows: slot");
  same_device(offsets, as, "expert rows: offsets");
  same_device(counts, as, "expert rows: counts");
  TORCH_CHECK(slot.scalar_type() == at::kInt && slot.dim() == 2 && slot.is_contiguous() &&
                  offsets.scalar_type() == at::kInt && offsets.is_contiguous() && counts.scalar_type() == at::kInt &&
                  counts.is_contiguous() && offsets.numel() == counts.numel() + 1,
              "expert rows: int32 slot [N, k], offsets [E + 1], counts [E]");
  ExpertRows r{};
  r.slot = slot.data_ptr<int>();
  r.offsets = offsets.data_ptr<int>();
  r.counts = counts.data_ptr<int>();
  r.N = (int)slot.size(0);
  r.k = (int)slot.size(1);
  r.D = (int)D;
  r.E = (int)counts.numel();
  r.capacity = (int)capacity;
  r.rows = rows;
  TORCH_CHECK(r.k <= kRouteMaxK, "expert rows: at most ", kRouteMaxK, " choices per token");
  TORCH_CHECK(rows == (capacity > 0 ? capacity * r.E : slot.numel()), "expert rows: row count");
  return r;
}

at::Tensor expert_dispatch(at::Tensor x, at::Tensor slot, at::Tensor offsets, at::Tensor counts, int64_t capacity,
                           int64_t rows) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(0) == slot.size(0) && whole_rows(x),
              "expert_dispatch: x [N, D] with contiguous rows, one per planned token");
  const c10::cuda::CUDAGuard guard(x.device());
  const ExpertRows r = expert_rows(slot, offsets, counts, capacity, rows, x.size(1), x);
  at::Tensor xs = fresh({rows, x.size(1)}, x.scalar_type(), x);
  BLOCK_LAUNCH(dispatch_launch(r, x.data_ptr(), x.stride(0), xs.data_ptr(), elem_of(x, "expert_dispatch"),
                               at::cuda::getCurrentCUDAStream()), xs.numel() > 0);
  return xs;
}

at::Tensor expert_combine(at::Tensor y, OptT w, at::Tensor slot, at::Tensor offsets, at::Tensor counts,
                          int64_t capacity) {
  TORCH_CHECK(y.is_cuda() && y.dim() == 2 && y.is_contiguous(), "expert_combine: y [rows, D], contiguous");
  const c10::cuda::CUDAGuard guard(y.device());
  const ExpertRows r = expert_rows(slot, offsets, counts, capacity, y.size(0), y.size(1), y);
  const float* wp = vec_f32(w, slot.numel(), y, "expert_combine: w");
  at::Tensor out = fresh({r.N, y.size(1)}, y.scalar_type(), y);
  BLOCK_LAUNCH(combine_launch(r, y.data_ptr(), wp, out.data_ptr(), elem_of(y, "expert_combine"),
                              at::cuda::getCurrentCUDAStream()), out.numel() > 0);
  return out;
}

std::tuple<at::Tensor, at::Tensor> expert_combine_bwd(at::Tensor y, at::Tensor w, at::Tensor dout, at::Tensor slot,
                                                      at::Tensor offsets, at::Tensor counts, int64_t capacity) {
  TORCH_CHECK(y.is_cuda() && y.dim() == 2 && y.is_contiguous(), "expert_combine_bwd: y [rows, D], contiguous");
  TORCH_CHECK(dout.dim() == 2 && dout.size(0) == slot.size(0) && dout.size(1) == y.size(1) &&
                  dout.scalar_type() == y.scalar_type() && whole_rows(dout),
              "expert_combine_bwd: dout [N, D] with contiguous rows, in y's type");
  same_device(dout, y, "expert_combine_bwd: dout");
  const c10::cuda::CUDAGuard guard(y.device());
  const ExpertRows r = expert_rows(slot, offsets, counts, capacity, y.size(0), y.size(1), y);
  const float* wp = vec_f32(w, slot.numel(), y, "expert_combine_bwd: w");
  at::Tensor dy = fresh_like(y), dw = fresh({r.N, r.k}, at::kFloat, y);
  BLOCK_LAUNCH(combine_bwd_launch(r, y.data_ptr(), wp, dout.data_ptr(), dout.stride(0), dy.data_ptr(),
                                  dw.data_ptr<float>(), elem_of(y, "expert_combine_bwd"),
                                  at::cuda::getCurrentCUDAStream()), r.N > 0 || r.rows > 0);
  return {dy, dw};
}

// ---------------------------------------------------------------------------------------------------- sandwich norm
// [B, D] rows of one value per sample and channel, in x's type, channels contiguous
const void* sample_rows(const OptT& t, int64_t B, int64_t D, const at::Tensor& x, long long* stride, const char* what) {
  if (!given(t)) return nullptr;
  same_device(*t, x, what);
  TORCH_CHECK(t->dim() == 2 && t->size(0) == B && t->size(1) == D && t->scalar_type() == x.scalar_type() &&
                  whole_rows(*t),
              what, ": [", B, ", ", D, "] rows in x's type with contiguous channels expected");
  *stride = B > 1 ? t->stride(0) : 0;
  return t->data_ptr();
}

// The row loops count in 32 bits and step past the last row by at most a grid or a span.
void sandwich_limits(const at::Tensor& x) {
  TORCH_CHECK(x.dim() == 3 && x.size(2) >= 1 && x.size(2) <= 16384 && x.size(0) * x.size(1) < (1ll << 31) - (1 << 20),
              "sandwich_norm: x [B, T, D] of at most 16384 channels and 2^31 - 2^20 rows");
}

SandwichParams sandwich_params(const at::Tensor& x, const at::Tensor& y, const OptT& gate, const OptT& post_w,
                               const OptT& w, const OptT& shift, const OptT& scale, double res_scale, double eps) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 3 && x.is_contiguous(), "sandwich_norm: x [B, T, D], contiguous");
  TORCH_CHECK(y.is_contiguous() && y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type(),
              "sandwich_norm: y as x");
  same_device(y, x, "sandwich_norm: y");
  sandwich_limits(x);
  const int64_t B = x.size(0), T = x.size(1), D = x.size(2);
  TORCH_CHECK(given(shift) == given(scale), "sandwich_norm: shift and scale together");
  TORCH_CHECK(given(w) || !given(scale), "sandwich_norm: shift and scale need w (the norm they modulate)");
  SandwichParams p{};
  p.x = x.data_ptr();
  p.y = y.data_ptr();
  p.gate = sample_rows(gate, B, D, x, &p.gate_bs, "sandwich_norm: gate");
  p.scale = sample_rows(scale, B, D, x, &p.mod_bs, "sandwich_norm: scale");
  long long shift_bs = 0;
  p.shift = sample_rows(shift, B, D, x, &shift_bs, "sandwich_norm: shift");
  TORCH_CHECK(shift_bs == p.mod_bs, "sandwich_norm: shift and scale must share a row stride");
  p.post_w = vec_f32(post_w, D, x, "sandwich_norm: post_w");
  p.w = vec_f32(w, D, x, "sandwich_norm: w");
  p.res_scale = (float)res_scale;
  p.eps = (float)eps;
  p.M = (int)(B * T);
  p.D = (int)D;
  p.T = (int)std::max<int64_t>(T, 1);
  return p;
}

std::vector<at::Tensor> sandwich_fwd(at::Tensor x, at::Tensor y, OptT gate, OptT post_w, OptT w, OptT shift, OptT scale,
                                     double res_scale, double eps, at::Tensor err) {
  SandwichParams p = sandwich_params(x, y, gate, post_w, w, shift, scale, res_scale, eps);
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor x_new = fresh_like(x), h, ry, rx;
  p.x_new = x_new.data_ptr();
  if (p.post_w != nullptr) {
    ry = fresh({p.M}, at::kFloat, x);
    p.rstd_y = ry.data_ptr<float>();
  }
  if (p.w != nullptr) {
    h = fresh_like(x);
    rx = fresh({p.M}, at::kFloat, x);
    p.h = h.data_ptr();
    p.rstd_x = rx.data_ptr<float>();
  }
  BLOCK_LAUNCH(sandwich_fwd_launch(p, elem_of(x, "sandwich_norm"), err_word(err, x),
                                   at::cuda::getCurrentCUDAStream()), p.M > 0);
  return {x_new, h, ry, rx};
}

// -> dx, dy, dgate, dshift, dscale; dpost_w and dw are added to (accumulate) or written
std::vector<at::Tensor> sandwich_bwd(OptT dx_new, OptT dh, at::Tensor x, at::Tensor y, OptT gate, OptT post_w, OptT w,
                                     OptT shift, OptT scale, OptT ry, OptT rx, OptT dpost_w, OptT dw, double res_scale,
                                     double eps, at::Tensor err, bool add_post_w, bool add_w) {
  SandwichParams p = sandwich_params(x, y, gate, post_w, w, shift, scale, res_scale, eps);
  const c10::cuda::CUDAGuard guard(x.device());
  p.rstd_y = acc_f32(ry, p.M, x, "sandwich_bwd: ry");
  p.rstd_x = acc_f32(rx, p.M, x, "sandwich_bwd: rx");
  TORCH_CHECK(p.M == 0 || ((p.rstd_y != nullptr || p.post_w == nullptr) && (p.rstd_x != nullptr || p.w == nullptr)),
              "sandwich_bwd: the forward's statistics");
  SandwichBwdParams q{};
  auto grad_in = [&](const OptT& t, const char* what) -> const void* {
    if (!given(t)) return nullptr;
    same_device(*t, x, what);
    TORCH_CHECK(t->is_contiguous() && t->sizes() == x.sizes() && t->scalar_type() == x.scalar_type(), what, ": as x");
    return t->data_ptr();
  };
  q.dx_new = grad_in(dx_new, "sandwich_bwd: dx_new");
  q.dh = grad_in(dh, "sandwich_bwd: dh");
  at::Tensor dx = fresh_like(x), dy = fresh_like(x), dgate, dshift, dscale;
  q.dx = dx.data_ptr();
  q.dy = dy.data_ptr();
  const int64_t B = x.size(0), D = x.size(2);
  if (p.gate != nullptr) {
    dgate = fresh({B, D}, x.scalar_type(), x);
    q.dgate = dgate.data_ptr();
  }
  if (p.scale != nullptr) {
    dshift = fresh({B, D}, x.scalar_type(), x);
    dscale = fresh({B, D}, x.scalar_type(), x);
    q.dshift = dshift.data_ptr();
    q.dscale = dscale.data_ptr();
  }
  q.dpost_w = acc_f32(dpost_w, D, x, "sandwich_bwd: dpost_w");
  q.dw = acc_f32(dw, D, x, "sandwich_bwd: dw");
  q.add_post_w = add_post_w;
  q.add_w = add_w;
  if (p.M == 0) {
    if (q.dpost_w != nullptr && !add_post_w) dpost_w->zero_();
    if (q.dw != nullptr && !add_w) dw->zero_();
    if (dgate.defined()) dgate.zero_();
    if (dshift.defined()) dshift.zero_(), dscale.zero_();
    return {dx, dy, dgate, dshift, dscale};
  }
  const int elem = elem_of(x, "sandwich_bwd");
  BLOCK_LAUNCH(sandwich_bwd_plan(p, elem, &q), 0);
  // one entry per span and per sample that begins in it; without modulation all rows are one sample's
  const int64_t entries = q.ctas + (p.gate != nullptr || p.scale != nullptr ? B : 1), floats = entries * 3 * D + (int64_t)q.groups * 2 * D;
  at::Tensor scratch = fresh({floats}, at::kFloat, x);
  q.partial = scratch.data_ptr<float>();
  q.wpart = q.partial + entries * 3 * D;
  const bool two_steps = q.groups > 1 && (q.dw != nullptr || q.dpost_w != nullptr);  // of the weights' sums
  BLOCK_LAUNCH(sandwich_bwd_launch(p, q, elem, err_word(err, x), at::cuda::getCurrentCUDAStream()), 2 + two_steps);
  return {dx, dy, dgate, dshift, dscale};
}

// -------------------------------------------------------------------------------------------------- multi-axis rotary
// [M, H, d] rows or [B, T, H, d] with evenly strided tokens, the heads of a token contiguous: the token stride; else -1
int64_t token_stride(const at::Tensor& t) {
  if (t.numel() == 0) return 0;
  const int64_t n = t.dim(), d = t.size(n - 1), H = t.size(n - 2), T = t.size(n - 3), B = n == 4 ? t.size(0) : 1;
  if ((d > 1 && t.stride(n - 1) != 1) || (H > 1 && t.stride(n - 2) != d)) return -1;
  if (B > 1 && T > 1 && t.stride(0) != T * t.stride(1)) return -1;
  return T > 1 || B <= 1 ? t.stride(n - 3) : t.stride(0);
}
at::Tensor even_tokens(const at::Tensor& t) {
  return (t.dim() == 3 || t.dim() == 4) && token_stride(t) < 0 ? t.contiguous() : t;
}

RopeAxesParams rope_params(const at::Tensor& q, const at::Tensor& k, const at::Tensor& pos, const at::Tensor& freq,
                           const at::Tensor& axis, const OptT& q_w, const OptT& k_w, bool interleaved, double eps) {
  const int64_t n = q.dim();
  TORCH_CHECK(q.is_cuda() && (n == 3 || n == 4) && k.dim() == n && pos.dim() == n - 1,
              "rope_axes: q [B, T, Hq, d], k [B, T, Hkv, d], pos [B, T, axes] (or all without B)");
  same_device(k, q, "rope_axes: k");
  same_device(pos, q, "rope_axes: pos");
  same_device(freq, q, "rope_axes: freq");
  same_device(axis, q, "rope_axes: axis");
  int64_t M = 1;
  for (int64_t i = 0; i + 2 < n; ++i) {
    M *= q.size(i);
    TORCH_CHECK(k.size(i) == q.size(i) && pos.size(i) == q.size(i), "rope_axes: k and pos for q's tokens");
  }
  const int64_t hd = q.size(n - 1), axes = pos.size(n - 2), hq = q.size(n - 2), hkv = k.size(n - 2);
  TORCH_CHECK(k.size(n - 1) == hd && k.scalar_type() == q.scalar_type(), "rope_axes: k as q");
  const int64_t q_ts = token_stride(q), k_ts = token_stride(k);
  TORCH_CHECK(q_ts >= 0 && k_ts >= 0, "rope_axes: the heads of a token must be contiguous, its tokens evenly strided");
  TORCH_CHECK(hd >= 2 && hd <= 1024 && M < (1ll << 31) && hq >= 1 && hkv >= 1,
              "rope_axes: head dim 2 to 1024, at least one head of each");
  TORCH_CHECK(pos.is_contiguous() && axes >= 1 && axes <= kRopeMaxAxes && (pos.scalar_type() == at::kInt || pos.scalar_type() == at::kFloat),
              "rope_axes: pos int32 or fp32 [M, axes], at most ", kRopeMaxAxes, " axes");
  TORCH_CHECK(freq.scalar_type() == at::kFloat && freq.is_contiguous() && freq.dim() == 2 && freq.size(0) == 2 &&
                  axis.scalar_type() == at::kInt && axis.is_contiguous() && axis.numel() == freq.size(1) &&
                  2 * freq.size(1) <= hd,
              "rope_axes: freq fp32 [2, pairs], axis int32 [pairs], at most d / 2 pairs");
  RopeAxesParams p{};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.q_ts = q_ts;
  p.k_ts = k_ts;
  p.pos = pos.data_ptr();
  p.pos_f32 = pos.scalar_type() == at::kFloat;
  p.freq = freq.data_ptr<float>();
  p.axis = axis.data_ptr<int>();
  p.q_w = vec_f32(q_w, hd, q, "rope_axes: q_w");
  p.k_w = vec_f32(k_w, hd, q, "rope_axes: k_w");
  TORCH_CHECK((p.q_w == nullptr) == (p.k_w == nullptr), "rope_axes: q and k norm weights both or neither");
  p.eps = (float)eps;
  p.M = (int)M;
  p.axes = (int)axes;
  p.hq = (int)hq;
  p.hkv = (int)hkv;
  p.hd = (int)hd;
  p.rot = (int)(2 * freq.size(1));
  p.interleaved = interleaved;
  return p;
}

std::tuple<at::Tensor, at::Tensor> rope_axes_fwd(at::Tensor q, at::Tensor k, at::Tensor pos, at::Tensor freq,
                                                 at::Tensor axis, OptT q_w, OptT k_w, bool interleaved, double eps) {
  RopeAxesParams p = rope_params(q, k, pos, freq, axis, q_w, k_w, interleaved, eps);
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor qo = fresh_like(q), ko = fresh_like(k);
  p.q_out = qo.data_ptr();
  p.k_out = ko.data_ptr();
  BLOCK_LAUNCH(rope_axes_fwd_launch(p, elem_of(q, "rope_axes"), at::cuda::getCurrentCUDAStream()), p.M > 0);
  return {qo, ko};
}

// -> dq_in, dk_in; dq_w and dk_w (both or neither) are added to (accumulate) or written
std::tuple<at::Tensor, at::Tensor> rope_axes_bwd(at::Tensor dq, at::Tensor dk, at::Tensor q, at::Tensor k,
                                                 at::Tensor pos, at::Tensor freq, at::Tensor axis, OptT q_w, OptT k_w,
                                                 OptT dq_w, OptT dk_w, bool interleaved, double eps, bool add_q_w,
                                                 bool add_k_w, OptT dq_out, OptT dk_out) {
  RopeAxesParams p = rope_params(q, k, pos, freq, axis, q_w, k_w, interleaved, eps);
  const c10::cuda::CUDAGuard guard(q.device());
  auto grad_ok = [&](const at::Tensor& g, const at::Tensor& t) {
    return g.is_contiguous() && g.sizes() == t.sizes() && g.scalar_type() == t.scalar_type() &&
           g.device() == t.device();
  };
  TORCH_CHECK(grad_ok(dq, q) && grad_ok(dk, k), "rope_axes_bwd: dq / dk contiguous, as q / k");
  auto out_ok = [&](const at::Tensor& o, const at::Tensor& t) {
    return o.sizes() == t.sizes() && o.scalar_type() == t.scalar_type() && o.device() == t.device() &&
           token_stride(o) >= 0;
  };
  TORCH_CHECK((!given(dq_out) || out_ok(*dq_out, q)) && (!given(dk_out) || out_ok(*dk_out, k)),
              "rope_axes_bwd: dq_out / dk_out as q / k, a token's heads contiguous");
  at::Tensor dqi = given(dq_out) ? *dq_out : fresh_like(dq), dki = given(dk_out) ? *dk_out : fresh_like(dk);
  at::Tensor partial;
  p.dq_ts = token_stride(dqi);
  p.dk_ts = token_stride(dki);
  float* gq = acc_f32(dq_w, p.hd, q, "rope_axes_bwd: dq_w");
  float* gk = acc_f32(dk_w, p.hd, q, "rope_axes_bwd: dk_w");
  TORCH_CHECK((gq == nullptr) == (gk == nullptr) && (gq == nullptr || p.q_w != nullptr),
              "rope_axes_bwd: dq_w and dk_w both or neither, with the norm weights");
  if (p.M == 0) {
    if (gq != nullptr && !add_q_w) dq_w->zero_();
    if (gk != nullptr && !add_k_w) dk_w->zero_();
    return {dqi, dki};
  }
  if (gq != nullptr)
    partial = fresh({rope_axes_bwd_ctas(), 2, p.hd}, at::kFloat, q);
  BLOCK_LAUNCH(rope_axes_bwd_launch(p, dq.data_ptr(), dk.data_ptr(), dqi.data_ptr(), dki.data_ptr(),
                                    gq != nullptr ? partial.data_ptr<float>() : nullptr, gq, gk, add_q_w, add_k_w,
                                    elem_of(q, "rope_axes_bwd"), at::cuda::getCurrentCUDAStream()),
               gq != nullptr ? 2 : 1);
  return {dqi, dki};
}

// ------------------------------------------------------------------------------------------------------ autograd
// The differentiable forms are C++ autograd functions: a small training step is bound by the host, and a Python
// autograd.Function costs more than the kernels it launches (forward + backward of 32768 x 8 routing: 79 us with it).
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// The backward kernels record nothing: a second derivative would silently miss their part.
void first_order_only() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "routed block operators are differentiable once (create_graph=True is not "
              "supported)");
}
// Nor have they a forward-mode form: a dual tensor would lose its tangent on the way.
bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (const at::Tensor* t : ts)
      TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "routed block operators have no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
at::Tensor or_undefined(const OptT& t) { return given(t) ? *t : at::Tensor(); }
OptT opt(const at::Tensor& t) { return t.defined() ? OptT(t) : OptT(); }

// Python's grad-ready hooks (ops/fused.py): called with the parameter after its gradient was accumulated in place
// (never freed: the callback must not outlive the interpreter that would have to release it)
struct GradReady {
  std::atomic<bool> on{false};
  py::object notify;
};
GradReady& grad_ready() {
  static GradReady* r = new GradReady;
  return *r;
}
void set_grad_ready(bool on, py::object notify) {
  grad_ready().notify = std::move(notify);
  grad_ready().on = on;
}

// Where a backward with two norm weights puts their gradients: in place into a leaf's .grad (no temporary, no accumulation
// kernel), or a temporary that autograd takes. A leaf without a .grad gets the buffer that the kernel writes, once it is
// launched (a refusal before that leaves no .grad behind). The parameter itself is kept beside the saved tensors: under
// saved-tensor hooks a saved leaf comes back as another tensor, whose .grad nobody reads.
// The kernels write the two gradients without regard to each other, so they never share memory: one leaf in both places
// (tied weights), or two with one .grad, has its second gradient written to a temporary and added after the launch.
struct WeightGrad {
  at::Tensor w, g;
  bool direct = false, add = false;
  WeightGrad(AutogradContext* ctx, const char* name) {
    const auto it = ctx->saved_data.find(name);
    if (it == ctx->saved_data.end()) return;
    w = it->second.toTensor();
    if (!w.requires_grad()) return;
    if (w.is_leaf() && w.scalar_type() == at::kFloat) {
      const at::Tensor& have = w.grad();
      if (!have.defined()) {
        direct = true;
      } else if (have.scalar_type() == at::kFloat && have.is_contiguous() && have.device() == w.device()) {
        direct = add = true;
        g = have.detach();
      }
    }
    if (!add) g = fresh_like(w);
  }
  // after the launch: what autograd still has to add
  at::Tensor put() const {
    if (!direct) return g;
    at::Tensor& have = w.mutable_grad();
    if (!have.defined()) have = g;
    else if (!add) have.add_(g);
    return at::Tensor();
  }
};
struct WeightGrads {
  WeightGrad a, b;
  static void keep(AutogradContext* ctx, const char* name, const OptT& weight) {
    if (given(weight)) ctx->saved_data[name] = *weight;
  }
  WeightGrads(AutogradContext* ctx, const char* first, const char* second) : a(ctx, first), b(ctx, second) {
    if (a.add && b.add) {
      const float *p = a.g.data_ptr<float>(), *q = b.g.data_ptr<float>();
      if (p < q + b.g.numel() && q < p + a.g.numel()) {
        b.g = fresh_like(b.w);
        b.add = false;
      }
    }
  }
  void done(at::Tensor& first, at::Tensor& second) const {
    first = a.put();
    second = b.put();
    if (!grad_ready().on) return;
    py::gil_scoped_acquire gil;  // each parameter once, when all of its gradient is there
    if (a.direct) grad_ready().notify(a.w);
    if (b.direct && !(a.direct && b.w.is_same(a.w))) grad_ready().notify(b.w);
  }
};

struct RouteFn : public torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, at::Tensor logits, OptT bias, OptT valid, int64_t k,
                               bool sigmoid, int64_t groups, int64_t top_groups, bool renorm, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [w, idx] = route_fwd(logits, bias, valid, k, sigmoid, groups, top_groups, renorm, scale);
    ctx->save_for_backward({logits, w, idx});
    ctx->saved_data["biased"] = given(bias);
    ctx->saved_data["sigmoid"] = sigmoid;
    ctx->saved_data["renorm"] = renorm;
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({idx});
    return {w, idx};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const auto saved = ctx->get_saved_variables();
    at::Tensor d = route_bwd(saved[0], saved[1], saved[2], grads[0].contiguous(), ctx->saved_data["biased"].toBool(),
                             ctx->saved_data["sigmoid"].toBool(), ctx->saved_data["renorm"].toBool(),
                             ctx->saved_data["scale"].toDouble());
    variable_list out(9);
    out[0] = d;
    return out;
  }
};
std::tuple<at::Tensor, at::Tensor> route_experts(at::Tensor logits, OptT bias, OptT valid, int64_t k, bool sigmoid,
                                                 int64_t groups, int64_t top_groups, bool renorm, double scale) {
  if (logits.dim() == 2 && !whole_rows(logits)) logits = logits.contiguous();
  if (!wants_grad({&logits})) return route_fwd(logits, bias, valid, k, sigmoid, groups, top_groups, renorm, scale);
  auto out = RouteFn::apply(logits, bias, valid, k, sigmoid, groups, top_groups, renorm, scale);
  return {out[0], out[1]};
}

struct DispatchFn : public torch::autograd::Function<DispatchFn> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor x, at::Tensor slot, at::Tensor offsets, at::Tensor counts,
                            int64_t capacity, int64_t rows) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({slot, offsets, counts});
    ctx->saved_data["capacity"] = capacity;
    return expert_dispatch(x, slot, offsets, counts, capacity, rows);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const auto s = ctx->get_saved_variables();
    variable_list out(6);
    out[0] = expert_combine(grads[0].contiguous(), OptT(), s[0], s[1], s[2], ctx->saved_data["capacity"].toInt());
    return out;
  }
};
at::Tensor dispatch_rows(at::Tensor x, at::Tensor slot, at::Tensor offsets, at::Tensor counts, int64_t capacity,
                         int64_t rows) {
  if (x.dim() == 2 && !whole_rows(x)) x = x.contiguous();
  if (!wants_grad({&x})) return expert_dispatch(x, slot, offsets, counts, capacity, rows);
  return DispatchFn::apply(x, slot, offsets, counts, capacity, rows);
}

struct CombineFn : public torch::autograd::Function<CombineFn> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor y, at::Tensor w, at::Tensor slot, at::Tensor offsets,
                            at::Tensor counts, int64_t capacity) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({y, w, slot, offsets, counts});
    ctx->saved_data["capacity"] = capacity;
    return expert_combine(y, w, slot, offsets, counts, capacity);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const auto s = ctx->get_saved_variables();
    at::Tensor g = grads[0];
    if (!whole_rows(g)) g = g.contiguous();
    auto [dy, dw] = expert_combine_bwd(s[0], s[1], g, s[2], s[3], s[4], ctx->saved_data["capacity"].toInt());
    variable_list out(6);
    out[0] = dy;
    out[1] = dw;
    return out;
  }
};
at::Tensor combine_rows(at::Tensor y, at::Tensor w, at::Tensor slot, at::Tensor offsets, at::Tensor counts,
                        int64_t capacity) {
  y = y.contiguous();
  w = w.to(at::kFloat).contiguous();
  if (!wants_grad({&y, &w})) return expert_combine(y, w, slot, offsets, counts, capacity);
  return CombineFn::apply(y, w, slot, offsets, counts, capacity);
}

struct SandwichFn : public torch::autograd::Function<SandwichFn> {
  static variable_list forward(AutogradContext* ctx, at::Tensor x, at::Tensor y, OptT gate, OptT post_w, OptT w,
                               OptT shift, OptT scale, double res_scale, double eps, at::Tensor err) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = sandwich_fwd(x, y, gate, post_w, w, shift, scale, res_scale, eps, err);
    ctx->save_for_backward({x, y, or_undefined(gate), or_undefined(post_w), or_undefined(w), or_undefined(shift),
                            or_undefined(scale), r[2], r[3]});
    WeightGrads::keep(ctx, "post_w", post_w);
    WeightGrads::keep(ctx, "w", w);
    ctx->saved_data["err"] = err;
    ctx->saved_data["res_scale"] = res_scale;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    if (!r[1].defined()) return {r[0]};
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const auto s = ctx->get_saved_variables();
    const at::Tensor dx_new = grads[0].defined() ? grads[0].contiguous() : at::Tensor();
    const at::Tensor dh = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : at::Tensor();
    const WeightGrads gw(ctx, "post_w", "w");
    auto r = sandwich_bwd(opt(dx_new), opt(dh), s[0], s[1], opt(s[2]), opt(s[3]), opt(s[4]), opt(s[5]), opt(s[6]),
                          opt(s[7]), opt(s[8]), opt(gw.a.g), opt(gw.b.g), ctx->saved_data["res_scale"].toDouble(),
                          ctx->saved_data["eps"].toDouble(), ctx->saved_data["err"].toTensor(), gw.a.add, gw.b.add);
    variable_list out(10);
    out[0] = r[0];
    out[1] = r[1];
    out[2] = r[2];
    gw.done(out[3], out[4]);
    out[5] = r[3];
    out[6] = r[4];
    return out;
  }
};
std::tuple<at::Tensor, OptT> sandwich_norm(at::Tensor x, at::Tensor y, OptT gate, OptT post_w, OptT w, OptT shift,
                                           OptT scale, double res_scale, double eps, at::Tensor err) {
  sandwich_limits(x);  // before anything is copied
  x = x.contiguous();
  y = y.contiguous();
  if (given(shift) && given(scale) && shift->strides() != scale->strides()) {
    shift = shift->contiguous();
    scale = scale->contiguous();
  }
  const at::Tensor g = or_undefined(gate), p = or_undefined(post_w), ww = or_undefined(w), sh = or_undefined(shift),
                   sc = or_undefined(scale);
  if (!wants_grad({&x, &y, &g, &p, &ww, &sh, &sc})) {
    auto r = sandwich_fwd(x, y, gate, post_w, w, shift, scale, res_scale, eps, err);
    return {r[0], opt(r[1])};
  }
  auto out = SandwichFn::apply(x, y, gate, post_w, w, shift, scale, res_scale, eps, err);
  return {out[0], out.size() > 1 ? OptT(out[1]) : OptT()};
}

struct RopeAxesFn : public torch::autograd::Function<RopeAxesFn> {
  static variable_list forward(AutogradContext* ctx, at::Tensor q, at::Tensor k, at::Tensor pos, at::Tensor freq,
                               at::Tensor axis, OptT q_w, OptT k_w, bool interleaved, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [qo, ko] = rope_axes_fwd(q, k, pos, freq, axis, q_w, k_w, interleaved, eps);
    ctx->save_for_backward({q, k, pos, freq, axis, or_undefined(q_w), or_undefined(k_w)});
    WeightGrads::keep(ctx, "q_w", q_w);
    WeightGrads::keep(ctx, "k_w", k_w);
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["eps"] = eps;
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const auto s = ctx->get_saved_variables();
    const WeightGrads gw(ctx, "q_w", "k_w");
    // the two weights' sums come together: one that needs no gradient gets a scratch row
    at::Tensor wq = gw.a.g, wk = gw.b.g;
    if (wq.defined() != wk.defined()) (wq.defined() ? wk : wq) = fresh_like(wq.defined() ? wq : wk);
    auto [dq, dk] = rope_axes_bwd(grads[0].contiguous(), grads[1].contiguous(), s[0], s[1], s[2], s[3], s[4], opt(s[5]),
                                  opt(s[6]), opt(wq), opt(wk), ctx->saved_data["interleaved"].toBool(),
                                  ctx->saved_data["eps"].toDouble(), gw.a.add, gw.b.add, OptT(), OptT());
    variable_list out(9);
    out[0] = dq;
    out[1] = dk;
    gw.done(out[5], out[6]);
    return out;
  }
};
std::tuple<at::Tensor, at::Tensor> rope_axes(at::Tensor q, at::Tensor k, at::Tensor pos, at::Tensor freq,
                                             at::Tensor axis, OptT q_w, OptT k_w, bool interleaved, double eps) {
  q = even_tokens(q);
  k = even_tokens(k);
  pos = pos.to(pos.is_floating_point() ? at::kFloat : at::kInt).contiguous();
  const at::Tensor wq = or_undefined(q_w), wk = or_undefined(k_w);
  if (!wants_grad({&q, &k, &wq, &wk})) return rope_axes_fwd(q, k, pos, freq, axis, q_w, k_w, interleaved, eps);
  auto out = RopeAxesFn::apply(q, k, pos, freq, axis, q_w, k_w, interleaved, eps);
  return {out[0], out[1]};
}

}  // namespace

void bind_block_ops(pybind11::module_& m) {
  m.def("route_experts", &route_experts, "expert scores, group-limited top-k and weights of every token");
  m.def("expert_plan", &expert_plan, "stable row of every assignment in expert order, offsets and counts");
  m.def("dispatch_rows", &dispatch_rows, "token rows into expert order");
  m.def("combine_rows", &combine_rows, "weighted sum of a token's rows from expert order");
  m.def("sandwich_norm", &sandwich_norm, "x + r gate rmsnorm(y) post_w, then rmsnorm, w, scale and shift");
  m.def("rope_axes", &rope_axes, "q/k RMSNorm and rotary positions with several axes");
  m.def("rope_axes_fwd", &rope_axes_fwd, "rope_axes of token rows without autograd");
  m.def("rope_axes_bwd", &rope_axes_bwd, "backward of rope_axes_fwd", py::arg("dq"), py::arg("dk"), py::arg("q"),
        py::arg("k"), py::arg("pos"), py::arg("freq"), py::arg("axis"), py::arg("q_w"), py::arg("k_w"),
        py::arg("dq_w"), py::arg("dk_w"), py::arg("interleaved"), py::arg("eps"), py::arg("add_q_w") = true,
        py::arg("add_k_w") = true, py::arg("dq_out") = OptT(), py::arg("dk_out") = OptT());
  m.def("set_grad_ready", &set_grad_ready, "callback for gradients that a backward accumulated in place");
}

}  // namespace tgo

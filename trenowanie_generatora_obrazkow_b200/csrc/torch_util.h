// Helpers of the torch-facing operators with a C++ autograd node (block_ops.cpp, blocks8_ops.cpp): checks of arguments,
// allocation past the dispatcher, refusals of higher derivatives, gradients written in place.
#pragma once
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <torch/extension.h>

#include <atomic>

#include "block_ops.h"

namespace tgo {

void count_launches(int n);  // ops.cpp

using OptT = c10::optional<at::Tensor>;

#define BLOCK_LAUNCH(expr, n)                                                         \
  do {                                                                                \
    cudaError_t _e = (expr);                                                          \
    TORCH_CHECK(_e == cudaSuccess, "kernel launch failed: ", cudaGetErrorString(_e)); \
    count_launches(n);                                                                \
  } while (0)

inline int elem_of(const at::Tensor& t, const char* what) {
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
inline at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& as) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, as.device(), c10::nullopt));
}
inline at::Tensor fresh_like(const at::Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }
inline bool given(const OptT& t) { return t.has_value() && t->defined(); }
inline void same_device(const at::Tensor& t, const at::Tensor& as, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == as.device(), what, ": a tensor on ", as.device(), " expected");
}
inline const float* vec_f32(const OptT& t, int64_t n, const at::Tensor& as, const char* what) {
  if (!given(t)) return nullptr;
  same_device(*t, as, what);
  TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == n, what, ": contiguous fp32 [", n,
              "] expected");
  return t->data_ptr<float>();
}
inline float* acc_f32(const OptT& t, int64_t n, const at::Tensor& as, const char* what) {
  return const_cast<float*>(vec_f32(t, n, as, what));
}

// [N, D] with a row's elements side by side (an empty tensor's strides say nothing: a sum's gradient expands to 0)
inline bool whole_rows(const at::Tensor& t) { return t.numel() == 0 || t.size(1) == 1 || t.stride(1) == 1; }

inline int* err_word(const at::Tensor& err, const at::Tensor& as) {
  same_device(err, as, "err");
  TORCH_CHECK(err.scalar_type() == at::kInt && err.numel() >= 1, "err: int32 error word");
  return err.data_ptr<int>();
}

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// The backward kernels record nothing: a second derivative would silently miss their part.
inline void first_order_only(const char* what = "routed block operators") {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " are differentiable once (create_graph=True is not supported)");
}
// Nor have they a forward-mode form: a dual tensor would lose its tangent on the way.
inline bool wants_grad(std::initializer_list<const at::Tensor*> ts, const char* what = "routed block operators") {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (const at::Tensor* t : ts)
      TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, " have no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
inline at::Tensor or_undefined(const OptT& t) { return given(t) ? *t : at::Tensor(); }
inline OptT opt(const at::Tensor& t) { return t.defined() ? OptT(t) : OptT(); }

// Python's grad-ready hooks (ops/fused.py): called with the parameter after its gradient was accumulated in place
// (never freed: the callback must not outlive the interpreter that would have to release it)
struct GradReady {
  std::atomic<bool> on{false};
  py::object notify;
};
inline GradReady& grad_ready() {
  static GradReady* r = new GradReady;
  return *r;
}
// Where a backward puts a weight's gradient: in place into a leaf's .grad (no temporary, no accumulation
// kernel), or a temporary that autograd takes. A leaf without a .grad gets the buffer that the kernel writes, once it is
// launched (a refusal before that leaves no .grad behind). The parameter itself is kept beside the saved tensors: under
// saved-tensor hooks a saved leaf comes back as another tensor, whose .grad nobody reads.
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

}  // namespace tgo

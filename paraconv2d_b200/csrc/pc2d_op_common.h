// Shared pieces of the torch ops of torch.ops.paraconv2d_b200: the checks of
// arguments, and what their Autograd kernels need.
#pragma once

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <climits>
#include <vector>

#include "paraconv2d.h"

namespace pc2d_ops {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

inline int seq_dtype_code(const Tensor &t, const char *what, bool with_double = false) {
  if (t.scalar_type() == at::kFloat) return PC2D_DTYPE_F32;
  if (t.scalar_type() == at::kHalf) return PC2D_DTYPE_F16;
  if (t.scalar_type() == at::kBFloat16) return PC2D_DTYPE_BF16;
  if (with_double && t.scalar_type() == at::kDouble) return PC2D_DTYPE_F64;
  TORCH_CHECK_NOT_IMPLEMENTED(false, what, ": not implemented for '", t.scalar_type(), "' (float32, float16, bfloat16",
                              with_double ? " and float64)" : ")");
  return -1;
}

inline void check_status(int st, const char *what) {
  TORCH_CHECK(st == PC2D_OK, what, ": ", pc2d_status_string(st), ": ", pc2d_last_error());
}

// Contiguous and on a 16-byte boundary.
inline Tensor dense(const Tensor &t) {
  Tensor c = t.contiguous();
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) c = c.clone(at::MemoryFormat::Contiguous);
  return c;
}

// The checked arguments of one call: its name, its device, and the tensors
// made dense.
struct Call {
  const char *what;
  c10::Device device;

  Tensor need(const Tensor &t, const char *name, at::ScalarType type, at::IntArrayRef shape) const {
    TORCH_CHECK(t.device() == device, what, ": ", name, " must be on ", device, ", got ", t.device());
    TORCH_CHECK(t.scalar_type() == type, what, ": ", name, " must be of type ", type, ", got ", t.scalar_type());
    TORCH_CHECK(t.sizes() == shape, what, ": ", name, " must be ", shape, ", got ", t.sizes());
    return dense(t);
  }
  Tensor maybe(const OptTensor &t, const char *name, at::ScalarType type, at::IntArrayRef shape) const {
    return t.has_value() && t->defined() ? need(*t, name, type, shape) : Tensor();
  }
  // in place: neither copied nor moved
  void in_place_any(const Tensor &t, const char *name, at::ScalarType type, at::IntArrayRef shape) const {
    TORCH_CHECK(t.device() == device, what, ": ", name, " must be on ", device, ", got ", t.device());
    TORCH_CHECK(t.scalar_type() == type, what, ": ", name, " must be of type ", type, ", got ", t.scalar_type());
    TORCH_CHECK(t.sizes() == shape, what, ": ", name, " must be ", shape, ", got ", t.sizes());
    TORCH_CHECK(t.is_contiguous(), what, ": ", name, " is updated in place and must be contiguous");
  }
  void in_place(const Tensor &t, const char *name, at::ScalarType type, at::IntArrayRef shape) const {
    in_place_any(t, name, type, shape);
    TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, what, ": ", name,
                " is updated in place and must start on a 16-byte boundary");
  }
  // What a step reads may not lie within the state that it moves on: one row's
  // place may be written before another row has read its input.
  void apart(const Tensor &state, std::initializer_list<const Tensor *> inputs) const {
    const auto first = reinterpret_cast<uintptr_t>(state.data_ptr()), last = first + state.nbytes();
    for (const Tensor *t : inputs) {
      if (!t->defined()) continue;
      const auto at = reinterpret_cast<uintptr_t>(t->data_ptr());
      TORCH_CHECK(at >= last || at + t->nbytes() <= first || !t->numel() || !state.numel(), what,
                  ": an input shares memory with the state, which is updated in place");
    }
  }
};

template <typename T = void>
T *ptr(const Tensor &t) {
  return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}
inline void *stream_now() { return (void *)c10::cuda::getCurrentCUDAStream().stream(); }

inline int as_int(int64_t v, const char *what, const char *name) {
  TORCH_CHECK(v >= 0 && v <= INT_MAX, what, ": ", name, " = ", v, " is out of range");
  return (int)v;
}

inline Tensor workspace(size_t bytes, const Tensor &like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// What a call changes in place, autograd must know to be no longer what it may
// have saved.  (Here, and not in an Autograd kernel, which inference mode and
// redispatched calls pass by.)
inline void changed(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ------------------------------------------------------------------ autograd

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline bool needs_grad(std::initializer_list<const Tensor *> tensors, std::initializer_list<const OptTensor *> optional) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : tensors)
    if (t->requires_grad()) return true;
  for (const OptTensor *t : optional)
    if (t->has_value() && (*t)->defined() && (*t)->requires_grad()) return true;
  return false;
}

// A derivative that comes with an input (forward mode) would be lost without a
// word in the kernels' outputs.  (What autograd has nothing to say about has
// none: steps, which the host bounds, mostly end there.)
inline bool has_tangent(const Tensor &t) {
  return t.defined() && t.unsafeGetTensorImpl()->autograd_meta() && t._fw_grad(0).defined();
}
inline void no_forward_mode(const char *what, std::initializer_list<const Tensor *> tensors,
                     std::initializer_list<const OptTensor *> optional) {
  bool any = false;
  for (const Tensor *t : tensors) any = any || has_tangent(*t);
  for (const OptTensor *t : optional) any = any || (t->has_value() && has_tangent(**t));
  TORCH_CHECK_NOT_IMPLEMENTED(!any, "paraconv2d_b200.", what, ": forward-mode derivatives are not implemented");
}

inline void check_cuda(const Tensor &t, const char *what) {
  TORCH_CHECK_NOT_IMPLEMENTED(t.is_cuda(), "paraconv2d_b200.", what, ": CUDA tensors only, got one on ", t.device());
}

// The op's kernel below Autograd, through the dispatcher: modes and tracers that
// stand in between (fake tensors among them) see the call.  Signature: that of
// the CUDA function.
template <typename Signature>
auto below_autograd(const char *name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}
#define PC2D_BELOW(op)                                                                                 \
  ([]() -> const auto & {                                                                              \
    static const auto handle = below_autograd<decltype(op##_cuda)>("paraconv2d_b200::" #op);          \
    return handle;                                                                                     \
  }())

// A step changes its state in place: there is no gradient.
inline void no_step_grad(const char *what, bool needs) {
  TORCH_CHECK(!needs, "paraconv2d_b200.", what, " moves its state on in place and has no backward pass: call it under "
              "torch.no_grad(), or use the operator over whole sequences");
}

inline OptTensor optional_of(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// Runs a backward pass without recording it; where the caller asked for a graph
// of it (create_graph), the gradients raise when they are differentiated.
template <typename F>
variable_list once(const char *what, F &&run) {
  variable_list grads;
  {
    at::AutoGradMode off(false);
    at::AutoDispatchBelowADInplaceOrView below;
    grads = run();
  }
  if (at::GradMode::is_enabled()) {
    variable_list defined;
    for (const Tensor &t : grads)
      if (t.defined()) defined.push_back(t);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("paraconv2d_b200.") + what + " is differentiable once only", (int)defined.size());
    // (a gradient that needs none would not lead to the error)
    for (Tensor &t : defined) t = t.detach().requires_grad_(true);
    defined = (*error)(std::move(defined));
    size_t k = 0;
    for (Tensor &t : grads)
      if (t.defined()) t = defined[k++];
  }
  return grads;
}

}  // namespace pc2d_ops

// What the native autograd functions share: errors as RuntimeError, checks,
// allocations and the stream.
#pragma once
#include <torch/extension.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <vector>

#include "cpab_hip.h"

namespace cpab_torch {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

[[noreturn]] inline void fail(const std::string& msg) { throw std::runtime_error(msg); }

inline void check(int rc, const char* what) {
  if (rc != 0) fail(std::string(what) + " failed: " + cpab_last_error_string());
}

inline std::string shape_of(const Tensor& t) {   // as str(tuple(t.shape))
  std::ostringstream s;
  s << "(";
  for (int64_t k = 0; k < t.dim(); ++k) s << (k ? ", " : "") << t.size(k);
  s << (t.dim() == 1 ? ",)" : ")");
  return s.str();
}

inline std::string dtype_of(const Tensor& t) {
  return std::string("torch.") + c10::getDtypeNames(t.scalar_type()).first;
}

inline const float* in(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
inline float* out(Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

inline Tensor empty(at::IntArrayRef size, const Tensor& like) {
  return at::empty(size, at::TensorOptions().device(like.device()).dtype(at::kFloat));
}

// Device memory used by this call alone: back in torch's caching allocator,
// for work queued behind it on the current stream, when the call returns.
inline at::DataPtr scratch(int64_t bytes) {
  return c10::hip::HIPCachingAllocator::get()->allocate((size_t)(bytes > 0 ? bytes : 1));
}

inline void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// torch.autograd.function.once_differentiable: the gradients cannot be
// differentiated again.
inline variable_list once(variable_list grads, const Tensor& grad_out) {
  if (!at::GradMode::is_enabled() || !grad_out.requires_grad()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  torch::autograd::DelayedError err(
      "trying to differentiate twice a function that was marked with @once_differentiable",
      (int64_t)grads.size());
  return err.apply(std::move(grads));
}

inline Tensor plain(const Tensor& t) { return t.detach().contiguous(); }

typedef std::optional<Tensor> Maybe;

inline int type_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? CPAB_F32 : CPAB_BF16; }
inline bool has_type(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
}
inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline Tensor of(const Maybe& t) { return t.has_value() ? *t : Tensor(); }

// A gradient of type `type`, or none.
inline Tensor grad_of(const Tensor& g, at::ScalarType type) {
  return !g.defined() || g.scalar_type() == type ? g : g.to(type);
}

// Whether a gradient came at all: a function behind an output may have none to give.
inline bool any_defined(const variable_list& grads) {
  for (const Tensor& g : grads)
    if (g.defined()) return true;
  return false;
}

inline bool any_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// The gradients, which cannot be differentiated again (create_graph): not through the
// upstream gradient, and not through the inputs.
inline variable_list once_any(variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  for (const Tensor& g : out)
    if (g.defined()) {
      Tensor asks = at::empty({0}, g.options()).set_requires_grad(true);
      return once(std::move(out), asks);
    }
  return out;
}

}  // namespace cpab_torch

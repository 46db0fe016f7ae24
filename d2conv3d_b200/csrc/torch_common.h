// What the sources of the PyTorch front-end share: error checks, allocations and autograd helpers over the C ABI.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <initializer_list>
#include <optional>

#include "d2conv3d.h"

// TORCH_CHECK(expr) of the reference reads "Expected <expr> to be true ..."
#define D2C_REQUIRE(cond, text) TORCH_CHECK(cond, "Expected " text " to be true, but got false.")

namespace d2c_torch {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

inline void check(int status, const char* what) {
  TORCH_CHECK(status == 0, what, ": ", d2c_status_string(status), status > 0 ? ": " : "",
              status > 0 ? d2c_last_cuda_error() : "", " (status ", status, ")");
}

inline Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
inline Tensor like(const Tensor& t) { return t.defined() ? at::empty_like(t, at::MemoryFormat::Contiguous) : t; }
inline Tensor bytes_on(size_t n, const Tensor& t) {
  return n ? at::empty({(int64_t)n}, t.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}
inline void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The operators have no forward-mode derivative, and they pass the dispatcher by, which would say so: a tangent must not get lost.
inline void refuse_tangents(const char* op, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), op, ": forward-mode derivatives are not implemented");
}

// A tensor that a node keeps for its backward.  Saved-tensor hooks decide what comes back: another layout is for the caller to deal with
// (contiguous(), or fresh strides), another size, type or device is refused here, since the kernels go by the forward's sizes.
class Saved {
 public:
  Saved() = default;
  Saved(const Tensor& t, bool is_output)
      : variable_(t, is_output), sizes_(t.sizes().begin(), t.sizes().end()), type_(t.scalar_type()), device_(t.device()) {}
  Tensor unpack(std::shared_ptr<Node> owner = nullptr) const {
    Tensor t = variable_.unpack(std::move(owner));
    if (t.defined())
      TORCH_CHECK(t.sizes() == at::IntArrayRef(sizes_) && t.scalar_type() == type_ && t.device() == device_ && t.layout() == at::kStrided,
                  "a saved tensor came back from its hooks as ", t.scalar_type(), " ", t.sizes(), " on ", t.device(),
                  ": it was saved as ", type_, " ", at::IntArrayRef(sizes_), " on ", device_);
    return t;
  }
  void reset() { variable_.reset_data(); }

 private:
  SavedVariable variable_;
  at::DimVector sizes_;
  at::ScalarType type_ = at::kFloat;
  at::Device device_ = at::kCUDA;
};

// Results of a backward node: gradients are computed outside the graph, so a second derivative has to fail loudly.
inline variable_list once_differentiable(variable_list&& grads) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)grads.size());
  error->set_next_edges(torch::autograd::edge_list(1));
  for (Tensor& t : grads)
    if (t.defined()) t.set_requires_grad(true);
  return (*error)(std::move(grads));
}

void bind_token_ops(py::module_& m);      // torch_tokens.cpp

}  // namespace d2c_torch

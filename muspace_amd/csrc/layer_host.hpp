// What the autograd nodes of the layer's dense operators share (layer_host.cpp,
// layer_host_block.cpp): the library's entry points, checks of a call's tensors.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/muspace_layer.h"

namespace layer_host {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// The library's entry points, bound by the Python loader.
struct Api {
  decltype(&::muspace_last_error) last_error = nullptr;
  decltype(&::linear_forward) linear_forward = nullptr;
  decltype(&::linear_checkpoint) linear_checkpoint = nullptr;
  decltype(&::linear_backward_workspace_size_for) linear_workspace = nullptr;
  decltype(&::linear_backward) linear_backward = nullptr;
  decltype(&::layer_norm_forward) norm_forward = nullptr;
  decltype(&::layer_norm_backward_workspace_size) norm_workspace = nullptr;
  decltype(&::layer_norm_backward) norm_backward = nullptr;
  decltype(&::gated_linear_forward) gated_forward = nullptr;
  decltype(&::gated_linear_backward_workspace_size) gated_workspace = nullptr;
  decltype(&::gated_linear_backward) gated_backward = nullptr;
  decltype(&::quantize_int8) quantize = nullptr;
  decltype(&::linear_int8_workspace_size) int8_workspace = nullptr;
  decltype(&::linear_int8_forward) int8_forward = nullptr;
  decltype(&::dropout_forward) dropout_forward = nullptr;
  decltype(&::residual_norm_forward) residual_forward = nullptr;
  decltype(&::residual_norm_backward_workspace_size) residual_workspace = nullptr;
  decltype(&::residual_norm_backward) residual_backward = nullptr;
};

inline Api api;

inline void check(int rc, const char *name) {
  if (rc == 0) return;
  const char *text = api.last_error();
  throw std::runtime_error(text != nullptr && text[0] != '\0'
                               ? std::string(text)
                               : std::string(name) + " failed with code " + std::to_string(rc));
}

inline int code_of(at::ScalarType type, const char *name) {
  switch (type) {
    case at::kFloat:
      return 0;
    case at::kHalf:
      return 1;
    case at::kBFloat16:
      return 2;
    default:
      throw std::runtime_error(std::string(name) + " must be float32, float16 or bfloat16");
  }
}

inline void *stream_of(const Tensor &t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

inline int64_t rows_of(const Tensor &t) {
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
  return rows;
}

// `t` with its values in memory as they are, row by row: a view may also be one that
// is read with its sign changed (the imaginary part of a conjugate), which a
// contiguous tensor keeps.
inline Tensor dense(const Tensor &t) {
  const Tensor c = t.contiguous();
  return c.is_neg() ? c.resolve_neg() : c;
}

// `t` on the input's device and dense; undefined where absent
inline Tensor prepared(const OptTensor &t, const Tensor &input, const char *name) {
  if (!t.has_value() || !t->defined()) return Tensor();
  if (t->device() != input.device()) {
    throw std::runtime_error(std::string(name) + " must be a ROCm device tensor on " +
                             input.device().str() + " like the input, got device " +
                             t->device().str());
  }
  return dense(*t);
}

inline bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

inline OptTensor opt(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

inline Tensor scratch(size_t bytes, const Tensor &like) {
  if (bytes == 0) return Tensor();
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// Under create_graph the results stand for functions whose derivatives are not
// there: differentiating them again raises.
inline variable_list once(variable_list grads, const char *name) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate ") + name + " twice; its HIP gradients are computed once",
      static_cast<int64_t>(grads.size()));
  variable_list marked;
  for (auto &g : grads) {
    marked.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
  }
  return (*error)(std::move(marked));
}

inline bool supported(at::ScalarType type) {
  return type == at::kFloat || type == at::kHalf || type == at::kBFloat16;
}

// a given `t` is one row of `size` values of `type`
inline bool row_of(const OptTensor &t, int64_t size, at::ScalarType type) {
  return !t.has_value() || !t->defined() ||
         (t->dim() == 1 && t->size(0) == size && t->scalar_type() == type);
}

// Kernels fill tensors that torch has only seen allocated. A tracer would record the
// allocation alone, and a module traced so would answer with uninitialised memory.
inline void refuse_tracing(const char *name) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing() || Modes::get_mode(Key::PROXY).has_value() ||
      Modes::get_mode(Key::FUNCTIONAL).has_value() || Modes::get_mode(Key::FAKE).has_value()) {
    throw std::runtime_error(std::string(name) +
                             ": HIP kernels cannot be traced (the PyTorch path can)");
  }
}

// Forward-mode derivatives are not there, and must not be dropped.
inline void refuse_tangents(const char *name, std::initializer_list<const Tensor *> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor *t : tensors) {
    if (t->defined() && t->_fw_grad(/*level=*/0).defined()) {
      throw std::runtime_error(std::string(name) + ": the HIP path has no forward-mode "
                               "derivatives (the PyTorch path has)");
    }
  }
}

}  // namespace layer_host

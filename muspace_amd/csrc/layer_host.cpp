// Host side of the layer's dense operators: their autograd nodes.
//
// The nodes call the C-ABI (include/muspace_layer.h) of libmuspace_msda.so, whose
// addresses the Python loader hands over (bind), so this module links torch only and
// holds no kernel. It is C++ because a backward runs in the autograd engine's own
// thread: a Python node there waits for the interpreter and pays two to three times
// for every line, and with these operators' few launches that was most of a call
// (layer norm of 300 x 256, forward and backward: 51 us on one thread, 107 on two).
//
// Contract with the callers in muspace_amd/ops: tensors whose types or shapes do not
// belong together give no result, and the caller says which one it is; devices,
// strides and whether a graph is recorded are seen to here. A C-ABI error becomes
// std::runtime_error (RuntimeError in Python) with the library's text.
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include "layer_host.hpp"

namespace layer_host {

void define_block(pybind11::module_ &m);  // layer_host_block.cpp

}  // namespace layer_host

namespace {

using namespace layer_host;

template <typename F>
void bind_one(F &to, const std::map<std::string, std::uintptr_t> &addresses, const char *name) {
  to = reinterpret_cast<F>(addresses.at(name));
}

void bind(const std::map<std::string, std::uintptr_t> &addresses) {
  bind_one(api.last_error, addresses, "muspace_last_error");
  bind_one(api.linear_forward, addresses, "linear_forward");
  bind_one(api.linear_checkpoint, addresses, "linear_checkpoint");
  bind_one(api.linear_workspace, addresses, "linear_backward_workspace_size_for");
  bind_one(api.linear_backward, addresses, "linear_backward");
  bind_one(api.norm_forward, addresses, "layer_norm_forward");
  bind_one(api.norm_workspace, addresses, "layer_norm_backward_workspace_size");
  bind_one(api.norm_backward, addresses, "layer_norm_backward");
  bind_one(api.gated_forward, addresses, "gated_linear_forward");
  bind_one(api.gated_workspace, addresses, "gated_linear_backward_workspace_size");
  bind_one(api.gated_backward, addresses, "gated_linear_backward");
  bind_one(api.quantize, addresses, "quantize_int8");
  bind_one(api.int8_workspace, addresses, "linear_int8_workspace_size");
  bind_one(api.int8_forward, addresses, "linear_int8_forward");
  bind_one(api.dropout_forward, addresses, "dropout_forward");
  bind_one(api.residual_forward, addresses, "residual_norm_forward");
  bind_one(api.residual_workspace, addresses, "residual_norm_backward_workspace_size");
  bind_one(api.residual_backward, addresses, "residual_norm_backward");
}

// ------------------------------------------------------------------ linear ---

// room for the 8-bit checkpoint of `input`: codes and scales
std::pair<Tensor, Tensor> checkpoint_like(const Tensor &input) {
  const int64_t rows = rows_of(input), padded = (input.size(-1) + 31) / 32 * 32;
  return {at::empty({rows, padded}, input.options().dtype(at::kChar)),
          at::empty({rows, padded / 32}, input.options().dtype(at::kByte))};
}

struct Kept {
  Tensor activation;     // relu's bits or gelu's derivatives
  Tensor codes, scales;  // the input's checkpoint
};

// The output; with `keep`, what the gradients need besides tensors that are there.
Tensor linear_run(const Tensor &input, const Tensor &weight, const Tensor &bias,
                  const Tensor &residual, int64_t activation, bool keep, bool checkpoint,
                  Kept *kept) {
  const int64_t rows = rows_of(input), cols = weight.size(1), out = weight.size(0);
  auto shape = input.sizes().vec();
  shape.back() = out;
  Tensor output = at::empty(shape, input.options());
  Tensor aside, codes, scales;
  if (keep && activation == 1) {
    aside = at::empty({(out + 63) / 64, rows, 8}, input.options().dtype(at::kByte));
  } else if (keep && activation == 2) {
    aside = at::empty({rows, out}, input.options());
  }
  if (checkpoint) std::tie(codes, scales) = checkpoint_like(input);
  check(api.linear_forward(
            input.data_ptr(), code_of(input.scalar_type(), "input"), weight.data_ptr(),
            pointer(bias), pointer(residual), output.data_ptr(),
            activation == 1 ? static_cast<uint8_t *>(pointer(aside)) : nullptr,
            activation == 2 ? pointer(aside) : nullptr, static_cast<int8_t *>(pointer(codes)),
            static_cast<uint8_t *>(pointer(scales)), rows, cols, out,
            static_cast<int>(activation), stream_of(input)),
        "linear_forward");
  if (kept != nullptr) *kept = {aside, codes, scales};
  return output;
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &input, const Tensor &weight,
                        const OptTensor &bias, const OptTensor &residual, int64_t activation,
                        bool checkpoint) {
    const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    const bool need_input = input.requires_grad(), need_weight = weight.requires_grad();
    Kept kept;
    Tensor output = linear_run(input, weight, b, r, activation,
                               need_input || need_weight || wants_grad(b),
                               need_weight && checkpoint, &kept);
    ctx->save_for_backward({need_weight && !checkpoint ? input : Tensor(), kept.codes, kept.scales,
                            need_input ? weight : Tensor(), kept.activation});
    ctx->saved_data["input"] = input.sizes();
    ctx->saved_data["weight"] = weight.sizes();
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["has_bias"] = b.defined();
    ctx->saved_data["has_residual"] = r.defined();
    return output;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    // edges are counted over the tensors that were given
    const bool has_bias = ctx->saved_data["has_bias"].toBool();
    const bool need_input = ctx->needs_input_grad(0), need_weight = ctx->needs_input_grad(1);
    const bool need_bias = has_bias && ctx->needs_input_grad(2);
    const bool need_residual = ctx->saved_data["has_residual"].toBool() &&
                               ctx->needs_input_grad(has_bias ? 3 : 2);
    Tensor grad_input, grad_weight, grad_bias;
    if (need_input || need_weight || need_bias) {
      const variable_list saved = ctx->get_saved_variables();
      const Tensor &x = saved[0], &codes = saved[1], &scales = saved[2], &weight = saved[3],
                   &kept = saved[4];
      const auto shape = ctx->saved_data["input"].toIntVector();
      const auto wshape = ctx->saved_data["weight"].toIntVector();
      const int activation = static_cast<int>(ctx->saved_data["activation"].toInt());
      const Tensor g = dense(grads[0]);
      const c10::DeviceGuard guard(g.device());
      const int64_t cols = wshape[1], out = wshape[0];
      int64_t rows = 1;
      for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
      if (need_input) grad_input = at::empty(shape, g.options());
      if (need_weight) grad_weight = at::empty(wshape, g.options());
      if (need_bias) grad_bias = at::empty({out}, g.options());
      const int code = code_of(g.scalar_type(), "grad_output");
      const size_t bytes = api.linear_workspace(code, rows, cols, out, activation, need_input,
                                                 need_weight, need_bias);
      const Tensor workspace = scratch(bytes, g);
      check(api.linear_backward(
                g.data_ptr(), code, pointer(x), static_cast<const int8_t *>(pointer(codes)),
                static_cast<const uint8_t *>(pointer(scales)), pointer(weight),
                activation == 1 ? static_cast<const uint8_t *>(pointer(kept)) : nullptr,
                activation == 2 ? pointer(kept) : nullptr, pointer(grad_input),
                pointer(grad_weight), pointer(grad_bias), rows, cols, out, activation,
                pointer(workspace), bytes, stream_of(g)),
            "linear_backward");
    }
    return once({grad_input, grad_weight, grad_bias, need_residual ? grads[0] : Tensor(), Tensor(),
                 Tensor()},
                "linear");
  }
};

bool linear_fits(const Tensor &input, const Tensor &weight, const OptTensor &bias,
                 const OptTensor &residual) {
  const at::ScalarType type = input.scalar_type();
  if (!supported(type) || input.dim() == 0 || weight.dim() != 2 ||
      weight.size(1) != input.size(-1) || weight.scalar_type() != type ||
      !row_of(bias, weight.size(0), type)) {
    return false;
  }
  if (!residual.has_value() || !residual->defined()) return true;
  const Tensor &r = *residual;
  return r.scalar_type() == type && r.dim() == input.dim() && r.size(-1) == weight.size(0) &&
         r.sizes().slice(0, r.dim() - 1) == input.sizes().slice(0, input.dim() - 1);
}

OptTensor linear(const Tensor &input, const Tensor &weight, const OptTensor &bias,
                 const OptTensor &residual, int64_t activation, bool checkpoint) {
  if (!linear_fits(input, weight, bias, residual)) return OptTensor();
  refuse_tracing("linear");
  const c10::DeviceGuard guard(input.device());
  const Tensor x = dense(input);
  const Tensor w = prepared(weight, x, "weight"), b = prepared(bias, x, "bias"),
               r = prepared(residual, x, "residual");
  refuse_tangents("linear", {&x, &w, &b, &r});
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(w) || wants_grad(b) || wants_grad(r))) {
    return LinearFunction::apply(x, w, opt(b), opt(r), activation, checkpoint);
  }
  return linear_run(x, w, b, r, activation, false, false, nullptr);
}

std::pair<Tensor, Tensor> checkpoint(const Tensor &input) {
  refuse_tracing("checkpoint_int8");
  const c10::DeviceGuard guard(input.device());
  const Tensor x = dense(input);
  auto kept = checkpoint_like(x);
  check(api.linear_checkpoint(x.data_ptr(), code_of(x.scalar_type(), "input"),
                              static_cast<int8_t *>(kept.first.data_ptr()),
                              static_cast<uint8_t *>(kept.second.data_ptr()), rows_of(x),
                              x.size(-1), stream_of(x)),
        "linear_checkpoint");
  return kept;
}

// -------------------------------------------------------------- layer norm ---

Tensor norm_run(const Tensor &input, const Tensor &weight, const Tensor &bias,
                at::ScalarType weight_type, const Tensor &stats, double eps) {
  Tensor output = at::empty(input.sizes(), input.options());
  check(api.norm_forward(input.data_ptr(), code_of(input.scalar_type(), "input"), pointer(weight),
                         pointer(bias), code_of(weight_type, "weight"), output.data_ptr(),
                         static_cast<float *>(pointer(stats)), rows_of(input), input.size(-1),
                         static_cast<float>(eps), stream_of(input)),
        "layer_norm_forward");
  return output;
}

at::ScalarType norm_type(const Tensor &input, const Tensor &weight, const Tensor &bias) {
  return (weight.defined() ? weight : bias.defined() ? bias : input).scalar_type();
}

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &input, const OptTensor &weight,
                        const OptTensor &bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    const at::ScalarType type = norm_type(input, w, b);
    Tensor stats = at::empty({rows_of(input), 2}, input.options().dtype(at::kFloat));
    Tensor output = norm_run(input, w, b, type, stats, eps);
    ctx->save_for_backward({input, w, stats});
    ctx->saved_data["type"] = static_cast<int64_t>(type);
    ctx->saved_data["has_bias"] = b.defined();
    return output;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
    const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
    const Tensor g = dense(grads[0]);
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = rows_of(x), cols = x.size(-1);
    Tensor grad_input, grad_weight, grad_bias;
    if (ctx->needs_input_grad(0)) grad_input = at::empty(x.sizes(), x.options());
    if (weight.defined() && ctx->needs_input_grad(1)) {
      grad_weight = at::empty({cols}, x.options().dtype(type));
    }
    if (ctx->saved_data["has_bias"].toBool() && ctx->needs_input_grad(weight.defined() ? 2 : 1)) {
      grad_bias = at::empty({cols}, x.options().dtype(type));
    }
    const int code = code_of(x.scalar_type(), "input");
    size_t bytes = 0;
    if (grad_weight.defined() || grad_bias.defined()) bytes = api.norm_workspace(code, rows, cols);
    const Tensor workspace = scratch(bytes, x);
    check(api.norm_backward(g.data_ptr(), code, x.data_ptr(), pointer(weight),
                            code_of(type, "weight"), static_cast<const float *>(stats.data_ptr()),
                            pointer(grad_input), pointer(grad_weight), pointer(grad_bias), rows,
                            cols, pointer(workspace), bytes, stream_of(x)),
          "layer_norm_backward");
    return once({grad_input, grad_weight, grad_bias, Tensor()}, "layer_norm");
  }
};

bool norm_fits(const Tensor &input, const OptTensor &weight, const OptTensor &bias, double eps) {
  if (!supported(input.scalar_type()) || input.dim() == 0 || !(eps >= 0.0)) return false;
  const at::ScalarType type =
      norm_type(input, weight.value_or(Tensor()), bias.value_or(Tensor()));
  return (type == at::kFloat || type == input.scalar_type()) &&
         row_of(weight, input.size(-1), type) && row_of(bias, input.size(-1), type);
}

OptTensor layer_norm(const Tensor &input, const OptTensor &weight, const OptTensor &bias,
                     double eps) {
  if (!norm_fits(input, weight, bias, eps)) return OptTensor();
  refuse_tracing("layer_norm");
  const c10::DeviceGuard guard(input.device());
  const Tensor x = dense(input);
  const Tensor w = prepared(weight, x, "weight"), b = prepared(bias, x, "bias");
  refuse_tangents("layer_norm", {&x, &w, &b});
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) {
    return LayerNormFunction::apply(x, opt(w), opt(b), eps);
  }
  return norm_run(x, w, b, norm_type(x, w, b), Tensor(), eps);
}

}  // namespace

PYBIND11_MODULE(muspace_layer_host, m) {
  namespace py = pybind11;
  // of the headers that this module's calls are compiled from
  m.attr("abi_version") = MUSPACE_MSDA_ABI_VERSION;
  m.def("bind", &bind);
  m.def("linear", &linear, py::call_guard<py::gil_scoped_release>());
  m.def("checkpoint", &checkpoint, py::call_guard<py::gil_scoped_release>());
  m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
  layer_host::define_block(m);
}

// Autograd nodes of a layer's blocks besides linear and layer norm: the gated layer,
// dropout and the residual norm; and linear on 8-bit integers, which has no gradients. The
// contract is that of layer_host.cpp.
#include <pybind11/stl.h>

#include <cmath>
#include <vector>

#include "layer_host.hpp"

namespace {

using namespace layer_host;

// ------------------------------------------------------------ gated linear ---

Tensor gated_run(const Tensor &input, const Tensor &weight, const Tensor &bias,
                 int64_t activation) {
  auto shape = input.sizes().vec();
  shape.back() = weight.size(0) / 2;
  Tensor output = at::empty(shape, input.options());
  check(api.gated_forward(input.data_ptr(), code_of(input.scalar_type(), "input"),
                          weight.data_ptr(), pointer(bias), output.data_ptr(), rows_of(input),
                          weight.size(1), weight.size(0) / 2, static_cast<int>(activation),
                          stream_of(input)),
        "gated_linear_forward");
  return output;
}

struct GatedFunction : torch::autograd::Function<GatedFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &input, const Tensor &weight,
                        const OptTensor &bias, int64_t activation) {
    // every gradient needs both halves of the product, which are computed again
    ctx->save_for_backward({input, weight, bias.value_or(Tensor())});
    ctx->saved_data["activation"] = activation;
    return gated_run(input, weight, bias.value_or(Tensor()), activation);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2];
    const Tensor g = dense(grads[0]);
    const c10::DeviceGuard guard(g.device());
    const int64_t rows = rows_of(x), cols = weight.size(1), hidden = weight.size(0) / 2;
    Tensor grad_input, grad_weight, grad_bias;
    if (ctx->needs_input_grad(0)) grad_input = at::empty(x.sizes(), x.options());
    if (ctx->needs_input_grad(1)) grad_weight = at::empty(weight.sizes(), x.options());
    if (bias.defined() && ctx->needs_input_grad(2)) {
      grad_bias = at::empty(bias.sizes(), x.options());
    }
    const int code = code_of(x.scalar_type(), "input");
    const size_t bytes = api.gated_workspace(code, rows, cols, hidden, grad_input.defined(),
                                             grad_weight.defined(), grad_bias.defined());
    const Tensor workspace = scratch(bytes, x);
    check(api.gated_backward(g.data_ptr(), code, x.data_ptr(), weight.data_ptr(), pointer(bias),
                             pointer(grad_input), pointer(grad_weight), pointer(grad_bias), rows,
                             cols, hidden, static_cast<int>(ctx->saved_data["activation"].toInt()),
                             pointer(workspace), bytes, stream_of(x)),
          "gated_linear_backward");
    return once({grad_input, grad_weight, grad_bias, Tensor()}, "gated_linear");
  }
};

OptTensor gated_linear(const Tensor &input, const Tensor &weight, const OptTensor &bias,
                       int64_t activation) {
  const at::ScalarType type = input.scalar_type();
  if (!supported(type) || input.dim() == 0 || weight.dim() != 2 || weight.size(0) % 2 != 0 ||
      weight.size(1) != input.size(-1) || weight.scalar_type() != type ||
      !row_of(bias, weight.size(0), type)) {
    return OptTensor();
  }
  refuse_tracing("gated_linear");
  const c10::DeviceGuard guard(input.device());
  const Tensor x = dense(input), w = prepared(weight, x, "weight"), b = prepared(bias, x, "bias");
  refuse_tangents("gated_linear", {&x, &w, &b});
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) {
    return GatedFunction::apply(x, w, opt(b), activation);
  }
  return gated_run(x, w, b, activation);
}

// ---------------------------------------------------------- 8-bit integers ---

std::pair<Tensor, Tensor> quantize(const Tensor &input) {
  refuse_tracing("quantize_int8");
  const c10::DeviceGuard guard(input.device());
  const Tensor x = dense(input);
  std::pair<Tensor, Tensor> made{
      at::empty(x.sizes(), x.options().dtype(at::kChar)),
      at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat))};
  check(api.quantize(x.data_ptr(), code_of(x.scalar_type(), "input"),
                     static_cast<int8_t *>(made.first.data_ptr()),
                     static_cast<float *>(made.second.data_ptr()), rows_of(x), x.size(-1),
                     stream_of(x)),
        "quantize_int8");
  return made;
}

OptTensor linear_int8(const Tensor &input, const Tensor &weight, const Tensor &weight_scale,
                      const OptTensor &bias, const OptTensor &residual, int64_t activation) {
  const at::ScalarType type = input.scalar_type();
  if (!supported(type) || input.dim() == 0 || weight.dim() != 2 ||
      weight.size(1) != input.size(-1) || weight.scalar_type() != at::kChar ||
      !row_of(weight_scale, weight.size(0), at::kFloat) || !row_of(bias, weight.size(0), type)) {
    return OptTensor();
  }
  auto shape = input.sizes().vec();
  shape.back() = weight.size(0);
  if (residual.has_value() &&
      (residual->scalar_type() != type || residual->sizes() != at::IntArrayRef(shape))) {
    return OptTensor();
  }
  refuse_tracing("linear_int8");
  const c10::DeviceGuard guard(input.device());
  const Tensor x = dense(input);
  const Tensor w = prepared(weight, x, "weight"), s = prepared(weight_scale, x, "weight_scale"),
               b = prepared(bias, x, "bias"), r = prepared(residual, x, "residual");
  refuse_tangents("linear_int8", {&x, &s, &b, &r});
  if (at::GradMode::is_enabled()) {
    for (const Tensor *t : {&x, &s, &b, &r}) {
      if (wants_grad(*t)) {
        throw std::runtime_error("linear_int8 has no gradients: call it under torch.no_grad() or "
                                 "on tensors that require none");
      }
    }
  }
  Tensor output = at::empty(shape, x.options());
  const int code = code_of(type, "input");
  const int64_t rows = rows_of(x), cols = w.size(1), out = w.size(0);
  const size_t bytes = api.int8_workspace(code, rows, cols, out);
  const Tensor workspace = scratch(bytes, x);
  check(api.int8_forward(x.data_ptr(), code, static_cast<const int8_t *>(w.data_ptr()),
                         static_cast<const float *>(s.data_ptr()), pointer(b), pointer(r),
                         output.data_ptr(), rows, cols, out, static_cast<int>(activation),
                         pointer(workspace), bytes, stream_of(x)),
        "linear_int8_forward");
  return output;
}

// ----------------------------------------------------------------- dropout ---

// The dropout of a call: its seed is a number or one int64 element on the device.
struct Drop {
  double p = 0.0;
  Tensor device_seed;
  uint64_t seed = 0, offset = 0;

  const int64_t *seed_pointer() const {
    return device_seed.defined() ? static_cast<const int64_t *>(device_seed.data_ptr()) : nullptr;
  }
  // (numbers go through the node's saved data; the tensor is saved with the others)
  void keep(AutogradContext *ctx) const {
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = static_cast<int64_t>(seed);
    ctx->saved_data["offset"] = static_cast<int64_t>(offset);
  }
  static Drop kept(AutogradContext *ctx, const Tensor &device_seed) {
    return Drop{ctx->saved_data["p"].toDouble(), device_seed,
                static_cast<uint64_t>(ctx->saved_data["seed"].toInt()),
                static_cast<uint64_t>(ctx->saved_data["offset"].toInt())};
  }
};

bool drop_fits(double p, const OptTensor &seed) {
  return p >= 0.0 && p <= 1.0 &&
         (!seed.has_value() || (seed->scalar_type() == at::kLong && seed->numel() == 1));
}

Tensor dropout_run(const Tensor &input, const Tensor &residual, const Drop &drop) {
  Tensor output = at::empty(input.sizes(), input.options());
  check(api.dropout_forward(input.data_ptr(), code_of(input.scalar_type(), "input"),
                            pointer(residual), output.data_ptr(), input.numel(), drop.p, drop.seed,
                            drop.seed_pointer(), drop.offset, stream_of(input)),
        "dropout_forward");
  return output;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &input, const OptTensor &residual,
                        const Drop &drop) {
    drop.keep(ctx);
    ctx->saved_data["has_residual"] = residual.has_value();
    ctx->save_for_backward({drop.device_seed});
    return dropout_run(input, residual.value_or(Tensor()), drop);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const bool has_residual = ctx->saved_data["has_residual"].toBool();
    Tensor grad_input;
    if (ctx->needs_input_grad(0)) {
      const Tensor g = dense(grads[0]);
      const c10::DeviceGuard guard(g.device());
      grad_input = dropout_run(g, Tensor(), Drop::kept(ctx, ctx->get_saved_variables()[0]));
    }
    const bool need_residual = has_residual && ctx->needs_input_grad(1);
    return once({grad_input, need_residual ? grads[0] : Tensor(), Tensor()}, "dropout");
  }
};

OptTensor dropout(const Tensor &input, const OptTensor &residual, double p, const OptTensor &seed,
                  uint64_t seed_value, uint64_t offset) {
  if (!supported(input.scalar_type()) || !drop_fits(p, seed) ||
      (residual.has_value() && (residual->scalar_type() != input.scalar_type() ||
                                residual->sizes() != input.sizes()))) {
    return OptTensor();
  }
  refuse_tracing("dropout");
  const c10::DeviceGuard guard(input.device());
  const Tensor x = dense(input), r = prepared(residual, x, "residual");
  const Drop drop{p, prepared(seed, x, "seed"), seed_value, offset};
  refuse_tangents("dropout", {&x, &r});
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(r))) {
    return DropoutFunction::apply(x, opt(r), drop);
  }
  return dropout_run(x, r, drop);
}

// ----------------------------------------------------------- residual norm ---

// A call's vectors over the columns, absent ones undefined.
struct Vectors {
  Tensor weight, bias, gate, post_weight, post_bias;

  at::ScalarType type(const Tensor &input) const {
    for (const Tensor *t : {&weight, &bias, &gate, &post_weight, &post_bias}) {
      if (t->defined()) return t->scalar_type();
    }
    return input.scalar_type();
  }
};

struct Norms {
  int64_t norm = 0, post = -1;
  double eps = 0.0, scale = 1.0;
};

struct NormKept {
  Tensor stream, stats, post_stats;
};

Tensor residual_run(const Tensor &block, const Tensor &residual, const Vectors &v, const Norms &n,
                    const Drop &drop, const NormKept &kept) {
  Tensor output = at::empty(block.sizes(), block.options());
  check(api.residual_forward(
            block.data_ptr(), code_of(block.scalar_type(), "block"), residual.data_ptr(),
            pointer(v.weight), pointer(v.bias), pointer(v.gate), pointer(v.post_weight),
            pointer(v.post_bias), code_of(v.type(block), "weight"), output.data_ptr(),
            pointer(kept.stream), static_cast<float *>(pointer(kept.stats)),
            static_cast<float *>(pointer(kept.post_stats)), rows_of(block), block.size(-1),
            static_cast<int>(n.norm), static_cast<int>(n.post), static_cast<float>(n.eps),
            static_cast<float>(n.scale), drop.p, drop.seed, drop.seed_pointer(), drop.offset,
            stream_of(block)),
        "residual_norm_forward");
  return output;
}

struct ResidualFunction : torch::autograd::Function<ResidualFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &block, const Tensor &residual,
                               const OptTensor &weight, const OptTensor &bias,
                               const OptTensor &gate, const OptTensor &post_weight,
                               const OptTensor &post_bias, const Norms &n, const Drop &drop,
                               bool want_stream) {
    const Vectors v{weight.value_or(Tensor()), bias.value_or(Tensor()), gate.value_or(Tensor()),
                    post_weight.value_or(Tensor()), post_bias.value_or(Tensor())};
    const auto stats = [&] {
      return at::empty({rows_of(block), 4}, block.options().dtype(at::kFloat));
    };
    // what the backward reads (muspace_layer.h)
    const bool sums = block.scalar_type() != at::kFloat;
    const NormKept kept{
        sums && !want_stream ? Tensor() : at::empty(block.sizes(), block.options()), stats(),
        n.post >= 0 ? stats() : Tensor()};
    Tensor output = residual_run(block, residual, v, n, drop, kept);
    const bool block_kept = sums || n.post >= 0 || wants_grad(v.gate);
    ctx->save_for_backward({block_kept ? block : Tensor(), sums ? residual : kept.stream,
                            kept.stats, kept.post_stats, v.weight, v.gate, v.post_weight,
                            v.post_bias, drop.device_seed});
    drop.keep(ctx);
    ctx->saved_data["norm"] = n.norm;
    ctx->saved_data["post"] = n.post;
    ctx->saved_data["scale"] = n.scale;
    ctx->saved_data["type"] = static_cast<int64_t>(v.type(block));
    int64_t given = 0;
    for (const OptTensor *t : {&weight, &bias, &gate, &post_weight, &post_bias}) {
      given = given << 1 | (t->has_value() ? 1 : 0);
    }
    ctx->saved_data["given"] = given;
    ctx->set_materialize_grads(false);
    if (want_stream) return {output, kept.stream};
    return {output};
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    // (the stream, or the residual that it is summed from)
    const Tensor &block = saved[0], &stream = saved[1], &stats = saved[2], &post_stats = saved[3];
    const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
    const int64_t given = ctx->saved_data["given"].toInt();
    const int post = static_cast<int>(ctx->saved_data["post"].toInt());
    const double scale = ctx->saved_data["scale"].toDouble();
    const Drop drop = Drop::kept(ctx, saved[8]);
    const c10::DeviceGuard guard(stream.device());
    const Tensor g = grads[0].defined() ? dense(grads[0]) : Tensor();
    const Tensor gs = grads.size() > 1 && grads[1].defined() ? dense(grads[1]) : Tensor();
    const int64_t rows = rows_of(stream), cols = stream.size(-1);
    // block, residual, then the vectors: edges are counted over the tensors that were given
    Tensor out[7];
    if (g.defined() || gs.defined()) {
      int edge = 2, sums = 0;
      for (int i = 0; i < 5; ++i) {
        if (!(given >> (4 - i) & 1)) continue;
        // (the norm's own vectors do not reach the stream)
        if (ctx->needs_input_grad(edge++) && (i >= 2 || g.defined())) {
          out[2 + i] = at::empty({cols}, stream.options().dtype(type));
          ++sums;
        }
      }
      const bool need_block = ctx->needs_input_grad(0), need_residual = ctx->needs_input_grad(1);
      const bool gated = (given & 4) != 0;
      const bool same = post < 0 && !gated && drop.p == 0.0 && scale == 1.0;
      if (need_block || (same && need_residual)) out[0] = at::empty_like(stream);
      if (need_residual && !same) out[1] = at::empty_like(stream);
      const int code = code_of(stream.scalar_type(), "block");
      const size_t bytes = sums > 0 ? api.residual_workspace(code, rows, cols, sums) : 0;
      const Tensor workspace = scratch(bytes, stream);
      check(api.residual_backward(
                pointer(g), pointer(gs), code, pointer(block),
                code != 0 ? stream.data_ptr() : nullptr, code == 0 ? stream.data_ptr() : nullptr,
                pointer(saved[4]), pointer(saved[5]), pointer(saved[6]), pointer(saved[7]),
                code_of(type, "weight"),
                static_cast<const float *>(stats.data_ptr()),
                static_cast<const float *>(pointer(post_stats)), pointer(out[0]), pointer(out[1]),
                pointer(out[2]), pointer(out[3]), pointer(out[4]), pointer(out[5]),
                pointer(out[6]), rows, cols, static_cast<int>(ctx->saved_data["norm"].toInt()),
                post, static_cast<float>(scale), drop.p, drop.seed, drop.seed_pointer(),
                drop.offset, pointer(workspace), bytes, stream_of(stream)),
            "residual_norm_backward");
      if (same) {
        out[1] = need_residual ? out[0] : Tensor();
        if (!need_block) out[0] = Tensor();
      }
    }
    return once({out[0], out[1], out[2], out[3], out[4], out[5], out[6], Tensor(), Tensor(),
                 Tensor()},
                "residual_norm");
  }
};

bool residual_fits(const Tensor &block, const Tensor &residual,
                   std::initializer_list<const OptTensor *> vectors, const Norms &n, double p,
                   const OptTensor &seed) {
  const at::ScalarType type = block.scalar_type();
  if (!supported(type) || block.dim() == 0 || residual.scalar_type() != type ||
      residual.sizes() != block.sizes() || !(n.eps >= 0.0) ||
      !std::isfinite(static_cast<float>(n.scale)) || !drop_fits(p, seed)) {
    return false;
  }
  OptTensor first;
  for (const OptTensor *t : vectors) {
    if (!t->has_value()) continue;
    if (!first.has_value()) first = *t;
    if (!row_of(*t, block.size(-1), first->scalar_type())) return false;
  }
  return !first.has_value() || first->scalar_type() == type || first->scalar_type() == at::kFloat;
}

// The output and, with want_stream, the stream; nothing where the tensors do not fit.
std::optional<std::vector<Tensor>> residual_norm(
    const Tensor &block, const Tensor &residual, const OptTensor &weight, const OptTensor &bias,
    const OptTensor &gate, const OptTensor &post_weight, const OptTensor &post_bias, int64_t norm,
    int64_t post, double eps, double scale, double p, const OptTensor &seed, uint64_t seed_value,
    uint64_t offset, bool want_stream) {
  const Norms n{norm, post, eps, scale};
  if (!residual_fits(block, residual, {&weight, &bias, &gate, &post_weight, &post_bias}, n, p,
                     seed) ||
      (post < 0 && (post_weight.has_value() || post_bias.has_value()))) {
    return std::nullopt;
  }
  refuse_tracing("residual_norm");
  const c10::DeviceGuard guard(block.device());
  const Tensor x = dense(block), r = prepared(residual, x, "residual");
  const Vectors v{prepared(weight, x, "weight"), prepared(bias, x, "bias"),
                  prepared(gate, x, "gate"), prepared(post_weight, x, "post_weight"),
                  prepared(post_bias, x, "post_bias")};
  const Drop drop{p, prepared(seed, x, "seed"), seed_value, offset};
  refuse_tangents("residual_norm",
                  {&x, &r, &v.weight, &v.bias, &v.gate, &v.post_weight, &v.post_bias});
  bool graph = false;
  for (const Tensor *t : {&x, &r, &v.weight, &v.bias, &v.gate, &v.post_weight, &v.post_bias}) {
    graph = graph || wants_grad(*t);
  }
  if (at::GradMode::is_enabled() && graph) {
    return ResidualFunction::apply(x, r, opt(v.weight), opt(v.bias), opt(v.gate),
                                   opt(v.post_weight), opt(v.post_bias), n, drop, want_stream);
  }
  const NormKept kept{want_stream ? at::empty(x.sizes(), x.options()) : Tensor(), Tensor(),
                      Tensor()};
  Tensor output = residual_run(x, r, v, n, drop, kept);
  if (want_stream) return std::vector<Tensor>{output, kept.stream};
  return std::vector<Tensor>{output};
}

}  // namespace

namespace layer_host {

void define_block(pybind11::module_ &m) {
  namespace py = pybind11;
  m.def("gated_linear", &gated_linear, py::call_guard<py::gil_scoped_release>());
  m.def("quantize", &quantize, py::call_guard<py::gil_scoped_release>());
  m.def("linear_int8", &linear_int8, py::call_guard<py::gil_scoped_release>());
  m.def("dropout", &dropout, py::call_guard<py::gil_scoped_release>());
  m.def("residual_norm", &residual_norm, py::call_guard<py::gil_scoped_release>());
}

}  // namespace layer_host

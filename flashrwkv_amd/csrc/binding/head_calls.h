// Whole calls of the training head, in the pattern of the decode chain's: the
// checks of the Python wrappers' tables, the outputs, the launches and, for
// training, the autograd node in native code. A call that these checks do not
// pass, or whose arguments are not plain, returns None; the wrapper then runs
// its tables (which raise their errors) and its own autograd function. Part of
// torch_ops.cpp. Host time of a call: norm of one row 9.7 -> 5.4 us; norm of one
// row with its gradients 109 -> 45 us, a small cross entropy with its gradients
// 133 -> 68 us (a Python node costs the engine about 60 us).
#pragma once

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// What a backward returns. Where it is itself recorded, its outputs have no
// gradient of their own: differentiating them raises. always: also where the
// upstream gradients are constants.
variable_list first_order(variable_list grads, const variable_list& upstream, const char* name,
                          bool always = false) {
  bool recorded = always;
  for (const Tensor& g : upstream) recorded = recorded || (g.defined() && g.requires_grad());
  if (!recorded || !at::GradMode::is_enabled()) return grads;
  std::vector<size_t> at;
  variable_list given;
  for (size_t i = 0; i < grads.size(); ++i) {
    if (!grads[i].defined()) continue;
    at.push_back(i);
    given.push_back(grads[i].detach().requires_grad_(true));
  }
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice ") + name +
          ", whose backward is not differentiable",
      static_cast<int64_t>(given.size()));
  variable_list marked = (*error)(std::move(given));
  for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = marked[i];
  return grads;
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const std::optional<Tensor>& residual, const Tensor& weight,
                               const Tensor& bias, double eps) {
    ctx->set_materialize_grads(false);
    std::vector<Tensor> out = layer_norm_forward(x, residual, weight, bias, eps, true);
    const Tensor rstd = out.back();
    out.pop_back();
    const Tensor mean = out.back();
    out.pop_back();
    ctx->save_for_backward({residual.has_value() ? out[1] : x, weight, mean, rstd});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& upstream) {
    const bool residual = upstream.size() > 1;
    const Tensor grad_y = upstream[0];
    const Tensor grad_stream = residual ? upstream[1] : Tensor();
    variable_list out(5);
    // The context counts the tensors among the inputs, which a residual that is
    // not there is none of.
    const auto give = [&](int i, const Tensor& g) {
      if (ctx->needs_input_grad(i > 0 && !residual ? i - 1 : i)) out[i] = g;
    };
    if (!grad_y.defined()) {
      give(0, grad_stream);
      if (residual) give(1, grad_stream);
      return out;
    }
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<Tensor> grads = layer_norm_backward(
        grad_y.contiguous(), saved[0],
        grad_stream.defined() ? std::optional<Tensor>(grad_stream.contiguous()) : std::nullopt,
        saved[1], saved[2], saved[3]);
    give(0, grads[0]);
    if (residual) give(1, grads[0]);
    give(2, grads[1]);
    give(3, grads[2]);
    return first_order(std::move(out), upstream, "pretrain_layer_norm");
  }
};

// teacher_logits: undefined for cross entropy, whose targets are `indices`.
struct LinearLossNode : torch::autograd::Function<LinearLossNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                        const Tensor& indices, const std::optional<Tensor>& teacher_logits,
                        int64_t ignore_index, double temperature, int64_t reduction,
                        bool backward_follows) {
    const auto [loss, saved] =
        teacher_logits.has_value()
            ? linear_topk_distillation_forward(hidden, weight, *teacher_logits, indices,
                                               temperature, reduction)
            : linear_cross_entropy_forward(hidden, weight, indices, ignore_index, reduction,
                                           backward_follows);
    ctx->save_for_backward({weight, saved});
    ctx->saved_data["shape"] = hidden.sizes().vec();
    ctx->saved_data["top"] = teacher_logits.has_value() ? indices.size(-1) : int64_t{1};
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& upstream) {
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const bool want_hidden = ctx->needs_input_grad(0), want_weight = ctx->needs_input_grad(1);
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
    const std::vector<Tensor> grads = linear_loss_backward(
        upstream[0].contiguous(), saved[0], saved[1], rows, ctx->saved_data["top"].toInt(),
        ctx->saved_data["temperature"].toDouble(), ctx->saved_data["reduction"].toInt(),
        want_hidden, want_weight);
    variable_list out(8);
    if (want_hidden) out[0] = grads.front().view(shape);
    if (want_weight) out[1] = grads.back();
    return first_order(std::move(out), upstream, "a head loss");
  }
};

struct HeadArgs : PlainArgs {
  bool plain_cuda(const Tensor& t) const {
    return ok && t.is_cuda() && t.is_contiguous() && t.numel() > 0;
  }
  bool like(const Tensor& t, const Tensor& x) const {
    return plain_cuda(t) && t.scalar_type() == x.scalar_type() && t.device() == x.device();
  }
};

struct LayerNormArgs : HeadArgs {
  Tensor x, weight, bias;
  std::optional<Tensor> residual;
  double eps = 0.0;
  LayerNormArgs(const pybind11::object& x_, const pybind11::object& residual_,
                const pybind11::object& weight_, const pybind11::object& bias_,
                const pybind11::object& eps_) {
    x = tensor(x_);
    require(ok && plain_cuda(x) && x.dim() >= 1 && x.size(-1) <= 16384 &&
            (x.scalar_type() == at::kFloat || x.scalar_type() == at::kHalf ||
             x.scalar_type() == at::kBFloat16));
    weight = tensor(weight_);
    require(ok && like(weight, x) && weight.dim() == 1 && weight.size(0) == x.size(-1));
    bias = tensor(bias_);
    require(ok && like(bias, x) && bias.dim() == 1 && bias.size(0) == x.size(-1));
    residual = optional_tensor(residual_);
    require(ok && (!residual.has_value() ||
                   (like(*residual, x) && residual->sizes() == x.sizes())));
    eps = number(eps_);
    require(ok && std::isfinite(eps) && eps >= 0.0);
  }
};

pybind11::object layer_norm_infer_call(const pybind11::object& x, const pybind11::object& residual,
                                       const pybind11::object& weight,
                                       const pybind11::object& bias, const pybind11::object& eps) {
  const LayerNormArgs args(x, residual, weight, bias, eps);
  if (!args.ok || args.x.dim() != 2) return pybind11::none();
  std::vector<Tensor> out =
      layer_norm_forward(args.x, args.residual, args.weight, args.bias, args.eps, false);
  if (!args.residual.has_value()) return pybind11::cast(std::move(out[0]));
  return pybind11::make_tuple(std::move(out[0]), std::move(out[1]));
}

pybind11::object layer_norm_train_call(const pybind11::object& x, const pybind11::object& residual,
                                       const pybind11::object& weight,
                                       const pybind11::object& bias, const pybind11::object& eps) {
  const LayerNormArgs args(x, residual, weight, bias, eps);
  if (!args.ok || stream_is_capturing(args.x)) return pybind11::none();
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    out = LayerNormNode::apply(args.x, args.residual, args.weight, args.bias, args.eps);
  }
  if (!args.residual.has_value()) return pybind11::cast(std::move(out[0]));
  return pybind11::make_tuple(std::move(out[0]), std::move(out[1]));
}

// teacher_logits None: cross entropy of targets `indices`.
pybind11::object linear_loss_call(const pybind11::object& hidden_, const pybind11::object& weight_,
                                  const pybind11::object& indices_,
                                  const pybind11::object& teacher_logits_,
                                  const pybind11::object& ignore_index_,
                                  const pybind11::object& temperature_, int64_t reduction) {
  HeadArgs args;
  const Tensor hidden = args.tensor(hidden_);
  args.require(args.ok && args.plain_cuda(hidden) && hidden.dim() >= 1 &&
               hidden.size(-1) % 64 == 0 && hidden.size(-1) <= 65536 &&
               (hidden.scalar_type() == at::kHalf || hidden.scalar_type() == at::kBFloat16));
  const Tensor weight = args.tensor(weight_);
  args.require(args.ok && args.like(weight, hidden) && weight.dim() == 2 &&
               weight.size(1) == hidden.size(-1));
  const Tensor indices = args.tensor(indices_);
  args.require(args.ok && args.plain_cuda(indices) && indices.device() == hidden.device() &&
               (indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong));
  const std::optional<Tensor> teacher = args.optional_tensor(teacher_logits_);
  const double temperature = args.number(temperature_);
  const int64_t ignore_index = args.integer(ignore_index_, false);
  args.require(!ignore_index_.is_none());
  if (!args.ok) return pybind11::none();
  const auto lead = hidden.sizes().slice(0, hidden.dim() - 1);
  if (teacher.has_value()) {
    const Tensor& t = *teacher;
    args.require(args.plain_cuda(t) && t.device() == hidden.device() &&
                 (t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf ||
                  t.scalar_type() == at::kBFloat16) &&
                 t.dim() == hidden.dim() && t.sizes().slice(0, t.dim() - 1) == lead &&
                 t.size(-1) <= 1024 && indices.sizes() == t.sizes() && temperature > 1e-30 &&
                 temperature < 1e30);
  } else {
    args.require(indices.sizes() == lead);
  }
  if (!args.ok || stream_is_capturing(hidden)) return pybind11::none();
  Tensor loss;
  {
    pybind11::gil_scoped_release release;
    loss = LinearLossNode::apply(hidden, weight, indices, teacher, ignore_index, temperature,
                                 reduction,
                                 torch::autograd::compute_requires_grad(hidden, weight));
  }
  return pybind11::cast(std::move(loss));
}

}  // namespace

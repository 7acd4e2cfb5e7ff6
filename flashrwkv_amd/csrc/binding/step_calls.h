// Whole calls of step_ops.h's operators, in the pattern of head_calls.h: the
// checks of the Python wrappers' tables, the outputs, the launches and the autograd
// nodes in native code; None for a call that these checks do not pass. Part of
// torch_ops.cpp, behind head_calls.h.
#pragma once

namespace {

std::optional<Tensor> defined_or_none(const Tensor& t) {
  return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
}

std::optional<Tensor> contiguous_or_none(const Tensor& t) {
  return t.defined() ? std::optional<Tensor>(t.contiguous()) : std::nullopt;
}

struct LinearLogProbsNode : torch::autograd::Function<LinearLogProbsNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                               const Tensor& targets, int64_t ignore_index, double temperature,
                               bool entropy) {
    ctx->set_materialize_grads(false);
    std::vector<Tensor> out = linear_log_probs_forward(hidden, weight, targets, ignore_index,
                                                       temperature, entropy);
    const Tensor saved = out.back();
    out.pop_back();
    ctx->save_for_backward({weight, saved});
    ctx->saved_data["shape"] = hidden.sizes().vec();
    ctx->saved_data["temperature"] = temperature;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& upstream) {
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const bool want_hidden = ctx->needs_input_grad(0), want_weight = ctx->needs_input_grad(1);
    variable_list out(6);
    const Tensor grad_entropy = upstream.size() > 1 ? upstream[1] : Tensor();
    if (!upstream[0].defined() && !grad_entropy.defined()) return out;
    refuse_capture(saved[0], "pretrain_linear_log_probs's backward");
    const int64_t rows = c10::multiply_integers(shape.begin(), shape.end() - 1);
    const std::vector<Tensor> grads = linear_log_probs_backward(
        contiguous_or_none(upstream[0]), contiguous_or_none(grad_entropy), saved[0], saved[1],
        rows, ctx->saved_data["temperature"].toDouble(), want_hidden, want_weight);
    if (want_hidden) out[0] = grads.front().view(shape);
    if (want_weight) out[1] = grads.back();
    return first_order(std::move(out), upstream, "pretrain_linear_log_probs", true);
  }
};

struct PolicyOptions {
  double clip_low, clip_high, dual_clip, kl_weight, entropy_weight;
  int64_t reduction;
  bool metrics, slopes;
};

// {loss} or {loss, metrics}.
struct PolicyLossNode : torch::autograd::Function<PolicyLossNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& log_probs,
                               const std::optional<Tensor>& entropy, const Tensor& old_log_probs,
                               const Tensor& advantages,
                               const std::optional<Tensor>& reference_log_probs,
                               const std::optional<Tensor>& mask,
                               const std::optional<Tensor>& cu_seqlens,
                               const PolicyOptions& options) {
    std::vector<Tensor> out = policy_loss_forward(
        log_probs, old_log_probs, advantages, reference_log_probs, entropy, mask, cu_seqlens,
        options.clip_low, options.clip_high, options.dual_clip, options.kl_weight,
        options.entropy_weight, options.reduction, options.metrics, options.slopes);
    ctx->save_for_backward({out[1], mask.value_or(Tensor()), cu_seqlens.value_or(Tensor())});
    ctx->saved_data["shape"] = log_probs.sizes().vec();
    ctx->saved_data["dtype"] = log_probs.scalar_type();
    ctx->saved_data["entropy_dtype"] =
        entropy.has_value() ? entropy->scalar_type() : at::kFloat;
    ctx->saved_data["entropy"] = entropy.has_value();
    ctx->saved_data["entropy_weight"] = options.entropy_weight;
    ctx->saved_data["reduction"] = options.reduction;
    out.erase(out.begin() + 1);
    if (options.metrics) ctx->mark_non_differentiable({out[1]});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& upstream) {
    variable_list out(8);
    if (!upstream[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const bool want_log_probs = ctx->needs_input_grad(0);
    const bool want_entropy = ctx->saved_data["entropy"].toBool() && ctx->needs_input_grad(1);
    const std::vector<Tensor> grads = policy_loss_backward(
        upstream[0].contiguous(), saved[0], defined_or_none(saved[1]), defined_or_none(saved[2]),
        ctx->saved_data["shape"].toIntVector(), ctx->saved_data["dtype"].toScalarType(),
        ctx->saved_data["entropy_dtype"].toScalarType(),
        ctx->saved_data["entropy_weight"].toDouble(), ctx->saved_data["reduction"].toInt(),
        want_log_probs, want_entropy);
    if (want_log_probs) out[0] = grads.front();
    if (want_entropy) out[1] = grads.back();
    return first_order(std::move(out), upstream, "pretrain_policy_loss", true);
  }
};

// {loss, rewards}.
struct PreferenceLossNode : torch::autograd::Function<PreferenceLossNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& log_probs,
                               const Tensor& cu_seqlens,
                               const std::optional<Tensor>& reference_log_probs,
                               const std::optional<Tensor>& mask, double beta, double margin,
                               double label_smoothing, int64_t kind, bool normalize,
                               int64_t reduction) {
    const auto [loss, rewards, saved] =
        preference_loss_forward(log_probs, cu_seqlens, reference_log_probs, mask, beta, margin,
                                label_smoothing, kind, normalize, reduction);
    ctx->save_for_backward({saved, cu_seqlens, mask.value_or(Tensor())});
    ctx->saved_data["shape"] = log_probs.sizes().vec();
    ctx->saved_data["dtype"] = log_probs.scalar_type();
    ctx->saved_data["reduction"] = reduction;
    ctx->mark_non_differentiable({rewards});
    return {loss, rewards};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& upstream) {
    variable_list out(10);
    if (!upstream[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    out[0] = preference_loss_backward(
        upstream[0].contiguous(), saved[0], saved[1], defined_or_none(saved[2]),
        ctx->saved_data["shape"].toIntVector(), ctx->saved_data["dtype"].toScalarType(),
        ctx->saved_data["reduction"].toInt());
    return first_order(std::move(out), upstream, "pretrain_preference_loss", true);
  }
};

// None, or the outputs as a tuple.
pybind11::object outputs(variable_list out) {
  pybind11::tuple got(out.size());
  for (size_t i = 0; i < out.size(); ++i) got[i] = pybind11::cast(std::move(out[i]));
  return std::move(got);
}

pybind11::object linear_log_probs_call(const pybind11::object& hidden_,
                                       const pybind11::object& weight_,
                                       const pybind11::object& targets_,
                                       const pybind11::object& ignore_index_,
                                       const pybind11::object& temperature_, bool entropy) {
  HeadArgs args;
  const Tensor hidden = args.tensor(hidden_);
  args.require(args.ok && args.plain_cuda(hidden) && hidden.dim() >= 1 &&
               hidden.size(-1) % 64 == 0 && hidden.size(-1) <= 65536 &&
               (hidden.scalar_type() == at::kHalf || hidden.scalar_type() == at::kBFloat16));
  const Tensor weight = args.tensor(weight_);
  args.require(args.ok && args.like(weight, hidden) && weight.dim() == 2 &&
               weight.size(1) == hidden.size(-1));
  const Tensor targets = args.tensor(targets_);
  args.require(args.ok && args.plain_cuda(targets) && targets.device() == hidden.device() &&
               (targets.scalar_type() == at::kInt || targets.scalar_type() == at::kLong) &&
               targets.sizes() == hidden.sizes().slice(0, hidden.dim() - 1));
  const double temperature = args.number(temperature_);
  const int64_t ignore_index = args.integer(ignore_index_, false);
  args.require(!ignore_index_.is_none() && temperature > 1e-30 && temperature < 1e30);
  if (!args.ok || stream_is_capturing(hidden)) return pybind11::none();
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    out = LinearLogProbsNode::apply(hidden, weight, targets, ignore_index, temperature, entropy);
  }
  return outputs(std::move(out));
}

struct SequenceArgs : HeadArgs {
  Tensor log_probs;
  bool wants_grad(const Tensor& t) const {
    return t.requires_grad() && at::GradMode::is_enabled();
  }
  bool is_column(const Tensor& t) const {
    return ok && plain_cuda(t) && gradient_dtype(t) && t.device() == log_probs.device();
  }
  // Beside log_probs: constant, and a token each.
  std::optional<Tensor> column(const pybind11::object& x, bool constant) {
    const std::optional<Tensor> t = optional_tensor(x);
    require(ok && (!t.has_value() || (is_column(*t) && t->sizes() == log_probs.sizes() &&
                                      !(constant && wants_grad(*t)))));
    return t;
  }
  std::optional<Tensor> mask(const pybind11::object& x) {
    const std::optional<Tensor> t = optional_tensor(x);
    require(ok && (!t.has_value() ||
                   (plain_cuda(*t) && t->device() == log_probs.device() &&
                    t->sizes() == log_probs.sizes() &&
                    (t->scalar_type() == at::kBool || t->scalar_type() == at::kByte))));
    return t;
  }
  std::optional<Tensor> offsets(const pybind11::object& x) {
    const std::optional<Tensor> t = optional_tensor(x);
    require(ok && (!t.has_value() || (plain_cuda(*t) && t->device() == log_probs.device() &&
                                      t->scalar_type() == at::kInt && t->dim() == 1 &&
                                      t->numel() >= 2)));
    return t;
  }
};

// (loss,) or (loss, metrics). dual_clip: 0 for none.
pybind11::object policy_loss_call(
    const pybind11::object& log_probs_, const pybind11::object& old_,
    const pybind11::object& advantages_, const pybind11::object& reference_,
    const pybind11::object& entropy_, const pybind11::object& mask_,
    const pybind11::object& cu_seqlens_, const pybind11::object& clip_low,
    const pybind11::object& clip_high, const pybind11::object& dual_clip,
    const pybind11::object& kl_weight, const pybind11::object& entropy_weight, int64_t reduction,
    bool metrics) {
  SequenceArgs args;
  args.log_probs = args.tensor(log_probs_);
  args.require(args.ok && args.plain_cuda(args.log_probs) && gradient_dtype(args.log_probs));
  const std::optional<Tensor> old = args.ok ? args.column(old_, true) : std::nullopt;
  args.require(old.has_value());
  const std::optional<Tensor> reference = args.column(reference_, true);
  const std::optional<Tensor> entropy = args.column(entropy_, false);
  const std::optional<Tensor> mask = args.mask(mask_);
  const std::optional<Tensor> cu = args.offsets(cu_seqlens_);
  const Tensor advantages = args.tensor(advantages_);
  args.require(args.ok && args.is_column(advantages) && !args.wants_grad(advantages) &&
               (advantages.sizes() == args.log_probs.sizes() ||
                (cu.has_value() && advantages.dim() == 1 &&
                 advantages.size(0) == cu->size(0) - 1)));
  PolicyOptions o{args.number(clip_low),  args.number(clip_high),
                  args.number(dual_clip), args.number(kl_weight),
                  args.number(entropy_weight), reduction, metrics, false};
  args.require(o.clip_low >= 0.0 && o.clip_low <= 1.0 && o.clip_high >= 0.0 &&
               o.clip_high <= 1e30 &&
               (o.dual_clip == 0.0 || (o.dual_clip > 1.0 && o.dual_clip <= 1e30)) &&
               std::fabs(o.kl_weight) <= 1e30 && std::fabs(o.entropy_weight) <= 1e30 &&
               (o.kl_weight == 0.0 || reference.has_value()) &&
               (o.entropy_weight == 0.0 || entropy.has_value()) &&
               (cu.has_value() || reduction != FRWKV_REDUCE_SEQUENCE_MEAN));
  if (!args.ok || stream_is_capturing(args.log_probs)) return pybind11::none();
  o.slopes = args.wants_grad(args.log_probs);
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    out = PolicyLossNode::apply(args.log_probs, entropy, *old, advantages, reference, mask, cu, o);
  }
  return outputs(std::move(out));
}

// (loss, rewards).
pybind11::object preference_loss_call(const pybind11::object& log_probs_,
                                      const pybind11::object& cu_seqlens_,
                                      const pybind11::object& reference_,
                                      const pybind11::object& mask_,
                                      const pybind11::object& beta_,
                                      const pybind11::object& margin_,
                                      const pybind11::object& label_smoothing_, int64_t kind,
                                      bool normalize, int64_t reduction) {
  SequenceArgs args;
  args.log_probs = args.tensor(log_probs_);
  args.require(args.ok && args.plain_cuda(args.log_probs) && gradient_dtype(args.log_probs));
  if (!args.ok) return pybind11::none();
  const std::optional<Tensor> reference = args.column(reference_, true);
  const std::optional<Tensor> mask = args.mask(mask_);
  const std::optional<Tensor> cu = args.offsets(cu_seqlens_);
  args.require(cu.has_value() && cu->numel() % 2 == 1);
  const double beta = args.number(beta_), margin = args.number(margin_);
  const double smoothing = args.number(label_smoothing_);
  args.require(beta >= 1e-30 && beta <= 1e30 && std::fabs(margin) <= 1e30 && smoothing >= 0.0 &&
               smoothing <= 0.5);
  if (!args.ok || stream_is_capturing(args.log_probs)) return pybind11::none();
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    out = PreferenceLossNode::apply(args.log_probs, *cu, reference, mask, beta, margin, smoothing,
                                    kind, normalize, reduction);
  }
  return outputs(std::move(out));
}

// Plain tensors of a list or tuple; ok says whether all are.
std::vector<Tensor> plain_list(PlainArgs& args, const pybind11::object& x) {
  std::vector<Tensor> out;
  args.require(PyList_CheckExact(x.ptr()) || PyTuple_CheckExact(x.ptr()));
  if (!args.ok) return out;
  const pybind11::sequence items = pybind11::reinterpret_borrow<pybind11::sequence>(x);
  const size_t count = items.size();
  out.reserve(count);
  for (size_t i = 0; i < count && args.ok; ++i) {
    out.push_back(args.tensor(pybind11::reinterpret_borrow<pybind11::object>(
        PySequence_Fast_GET_ITEM(x.ptr(), static_cast<Py_ssize_t>(i)))));
  }
  return out;
}

pybind11::object grad_norm_call(const pybind11::object& tensors_) {
  PlainArgs args;
  const std::vector<Tensor> tensors = plain_list(args, tensors_);
  args.require(!tensors.empty());
  for (size_t i = 0; i < tensors.size() && args.ok; ++i) {
    args.require(is_gradient(tensors[i], tensors[0]));
  }
  if (!args.ok) return pybind11::none();
  return pybind11::cast(grad_norm(tensors));
}

// out None: in place.
pybind11::object clip_grad_norm_call(const pybind11::object& tensors_,
                                     const pybind11::object& out_,
                                     const pybind11::object& max_norm_,
                                     const pybind11::object& eps_) {
  PlainArgs args;
  const std::vector<Tensor> tensors = plain_list(args, tensors_);
  const std::vector<Tensor> out =
      out_.is_none() || !args.ok ? tensors : plain_list(args, out_);
  const double max_norm = args.number(max_norm_), eps = args.number(eps_);
  args.require(std::isfinite(max_norm) && max_norm >= 0.0 && std::isfinite(eps) && eps >= 0.0);
  if (!args.ok || !may_clip(tensors, out)) return pybind11::none();
  const std::vector<frwkv_gradient> list = gradient_list(tensors, &out);
  if (!apart(list)) return pybind11::none();
  return pybind11::cast(clip_gradients(tensors, out, list, max_norm, eps));
}

}  // namespace

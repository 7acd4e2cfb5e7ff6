// Whole calls of step_ops.h's operators, in the pattern of head_calls.h: the
// checks of the Python wrappers' tables, the outputs, the launches and the autograd
// nodes in native code; None for a call that these checks do not pass. Part of
// torch_ops.cpp, behind head_calls.h.
#pragma once

#include <torch/csrc/autograd/saved_variable.h>

namespace {

std::optional<Tensor> contiguous_or_none(const Tensor& t) {
  return t.defined() ? std::optional<Tensor>(t.contiguous()) : std::nullopt;
}

// The autograd nodes hold what they need as members. A node made from
// torch::autograd::Function keeps it in a map from names to boxed values, which the
// forward fills and the backward reads: a policy loss of 300 tokens with its
// gradient takes 61 us of host time so, and 49 with these.
struct StepNode : torch::autograd::Node {
  std::vector<torch::autograd::SavedVariable> saved;
  bool released = false;

  // Kept for the backward; a caller's tensors with their versions.
  void save(const std::optional<Tensor>& t) {
    saved.emplace_back(t.has_value() ? *t : Tensor(), false);
  }
  std::optional<Tensor> unpack(size_t i) const {
    Tensor t = saved[i].unpack();
    return t.defined() ? std::optional<Tensor>(std::move(t)) : std::nullopt;
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    saved.clear();
    released = true;
  }
  void check_held() const { TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE); }
};

// f(node) where one of the inputs needs a gradient: a new node with their edges,
// which becomes the outputs' history.
template <typename N, typename F, typename... Inputs>
void record(const variable_list& outputs, F&& fill, const Inputs&... inputs) {
  if (!torch::autograd::compute_requires_grad(inputs...)) return;
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  fill(*node);
  for (const Tensor& t : outputs) torch::autograd::set_history(t, node);
}

struct LinearLogProbsNode : StepNode {  // saved: weight, the forward's buffer
  std::vector<int64_t> shape;
  double temperature = 1.0;

  std::string name() const override { return "LinearLogProbsBackward"; }
  variable_list apply(variable_list&& upstream) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    check_held();
    const bool want_hidden = task_should_compute_output(0);
    const bool want_weight = task_should_compute_output(1);
    variable_list out(2);
    const Tensor grad_entropy = upstream.size() > 1 ? upstream[1] : Tensor();
    if (!upstream[0].defined() && !grad_entropy.defined()) return out;
    const Tensor weight = *unpack(0);
    refuse_capture(weight, "pretrain_linear_log_probs's backward");
    const int64_t rows = c10::multiply_integers(shape.begin(), shape.end() - 1);
    const std::vector<Tensor> grads = linear_log_probs_backward(
        contiguous_or_none(upstream[0]), contiguous_or_none(grad_entropy), weight, *unpack(1),
        rows, temperature, want_hidden, want_weight);
    if (want_hidden) out[0] = grads.front().view(shape);
    if (want_weight) out[1] = grads.back();
    return first_order(std::move(out), upstream, "pretrain_linear_log_probs", true);
  }
};

struct PolicyLossNode : StepNode {  // saved: the forward's buffer, mask, offsets
  std::vector<int64_t> shape;
  at::ScalarType dtype = at::kFloat, entropy_dtype = at::kFloat;
  double entropy_weight = 0.0;
  int64_t reduction = 0;

  std::string name() const override { return "PolicyLossBackward"; }
  variable_list apply(variable_list&& upstream) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    check_held();
    variable_list out(num_outputs());
    if (!upstream[0].defined()) return out;
    const bool want_log_probs = task_should_compute_output(0);
    const bool want_entropy = num_outputs() > 1 && task_should_compute_output(1);
    const std::vector<Tensor> grads = policy_loss_backward(
        upstream[0].contiguous(), *unpack(0), unpack(1), unpack(2), shape, dtype, entropy_dtype,
        entropy_weight, reduction, want_log_probs, want_entropy);
    if (want_log_probs) out[0] = grads.front();
    if (want_entropy) out[1] = grads.back();
    return first_order(std::move(out), upstream, "pretrain_policy_loss", true);
  }
};

struct PreferenceLossNode : StepNode {  // saved: the forward's buffer, mask, offsets
  std::vector<int64_t> shape;
  at::ScalarType dtype = at::kFloat;
  int64_t reduction = 0;

  std::string name() const override { return "PreferenceLossBackward"; }
  variable_list apply(variable_list&& upstream) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    check_held();
    variable_list out(1);
    if (!upstream[0].defined()) return out;
    out[0] = preference_loss_backward(upstream[0].contiguous(), *unpack(0), *unpack(2), unpack(1),
                                      shape, dtype, reduction);
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
  args.require(args.ok && !has_tangent(hidden) && !has_tangent(weight));
  if (!args.ok || stream_is_capturing(hidden)) return pybind11::none();
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    out = linear_log_probs_forward(hidden, weight, targets, ignore_index, temperature, entropy,
                                   torch::autograd::compute_requires_grad(hidden, weight));
    const Tensor saved = std::move(out.back());
    out.pop_back();
    record<LinearLogProbsNode>(
        out,
        [&](LinearLogProbsNode& node) {
          node.save(weight);
          node.save(saved);
          node.shape = hidden.sizes().vec();
          node.temperature = temperature;
        },
        hidden, weight);
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
                                      !has_tangent(*t) && !(constant && wants_grad(*t)))));
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
               !has_tangent(advantages) &&
               (advantages.sizes() == args.log_probs.sizes() ||
                (cu.has_value() && advantages.dim() == 1 &&
                 advantages.size(0) == cu->size(0) - 1)));
  const double low = args.number(clip_low), high = args.number(clip_high);
  const double dual = args.number(dual_clip), kl = args.number(kl_weight);
  const double ew = args.number(entropy_weight);
  args.require(low >= 0.0 && low <= 1.0 && high >= 0.0 && high <= 1e30 &&
               (dual == 0.0 || (dual > 1.0 && dual <= 1e30)) && std::fabs(kl) <= 1e30 &&
               std::fabs(ew) <= 1e30 && (kl == 0.0 || reference.has_value()) &&
               (ew == 0.0 || entropy.has_value()) &&
               (cu.has_value() || reduction != FRWKV_REDUCE_SEQUENCE_MEAN));
  const Tensor& x = args.log_probs;
  args.require(args.ok && !has_tangent(x));
  if (!args.ok || stream_is_capturing(x)) return pybind11::none();
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    out = policy_loss_forward(x, *old, advantages, reference, entropy, mask, cu, low, high, dual,
                              kl, ew, reduction, metrics, args.wants_grad(x));
    const Tensor saved = std::move(out[1]);
    out.erase(out.begin() + 1);
    const auto fill = [&](PolicyLossNode& node) {
      node.save(saved);
      node.save(mask);
      node.save(cu);
      node.shape = x.sizes().vec();
      node.dtype = x.scalar_type();
      node.entropy_dtype = entropy.has_value() ? entropy->scalar_type() : at::kFloat;
      node.entropy_weight = ew;
      node.reduction = reduction;
    };
    if (entropy.has_value()) {
      record<PolicyLossNode>({out[0]}, fill, x, *entropy);
    } else {
      record<PolicyLossNode>({out[0]}, fill, x);
    }
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
  const Tensor& x = args.log_probs;
  args.require(args.ok && !has_tangent(x));
  if (!args.ok || stream_is_capturing(x)) return pybind11::none();
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    auto [loss, rewards, saved] = preference_loss_forward(
        x, *cu, reference, mask, beta, margin, smoothing, kind, normalize, reduction);
    record<PreferenceLossNode>(
        {loss},
        [&, &kept = saved](PreferenceLossNode& node) {
          node.save(kept);
          node.save(mask);
          node.save(cu);
          node.shape = x.sizes().vec();
          node.dtype = x.scalar_type();
          node.reduction = reduction;
        },
        x);
    out = {std::move(loss), std::move(rewards)};
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
    args.require(is_gradient(tensors[i], tensors[0]) && is_constant(tensors[i]));
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

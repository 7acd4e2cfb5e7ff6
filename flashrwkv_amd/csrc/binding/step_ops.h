// Ops of a policy or preference training step: log probabilities and entropies
// from the hidden rows, the losses over packed sequences of them, and the norm of
// gradients (no counterpart in the reference's binding). Part of torch_ops.cpp,
// behind head_ops.h, whose helpers it uses.
#pragma once

namespace {

// {log_probs}, {log_probs, entropy}, and what the backward reads after them.
std::vector<Tensor> linear_log_probs_forward(Tensor hidden, Tensor weight, Tensor targets,
                                             int64_t ignore_index, double temperature,
                                             bool entropy, bool backward_follows) {
  const int64_t rows = check_head(hidden, weight, FRWKV_REDUCE_NONE);
  check_device_contiguous(targets, "targets");
  const int bytes = index_bytes(targets, "targets");
  TORCH_CHECK(targets.numel() == rows && targets.device() == hidden.device(),
              "targets must have one entry a row of hidden, on its device");
  c10::DeviceGuard guard(hidden.device());
  const int64_t c = hidden.size(-1), vocab = weight.size(0);
  const auto fp32 = hidden.options().dtype(at::kFloat);
  std::vector<Tensor> out;
  for (int i = 0; i < 1 + entropy; ++i) out.push_back(at::empty(targets.sizes(), fp32));
  // Sizes that the call refuses have no bytes; its error says why.
  const size_t saved_bytes = frwkv_linear_loss_saved_bytes(rows, c, 1);
  const size_t work_bytes = frwkv_linear_log_probs_forward_workspace_bytes(rows, vocab, entropy);
  Tensor saved = workspace_like(hidden, saved_bytes), work = workspace_like(hidden, work_bytes);
  check_rc(frwkv_linear_log_probs_forward(
      io_code(hidden.scalar_type()), rows, c, vocab, hidden.const_data_ptr(),
      weight.const_data_ptr(), bytes, targets.const_data_ptr(), ignore_index,
      static_cast<float>(temperature), backward_follows, out[0].data_ptr<float>(),
      entropy ? out[1].data_ptr<float>() : nullptr, scratch_ptr(saved), saved_bytes,
      scratch_ptr(work), work_bytes, current_stream(hidden)));
  out.push_back(saved);
  return out;
}

const float* check_upstream(const std::optional<Tensor>& grad, int64_t count, const Tensor& like,
                            const char* name) {
  if (!grad.has_value()) return nullptr;
  check_device_contiguous(*grad, name);
  TORCH_CHECK(grad->scalar_type() == at::kFloat && grad->numel() == count &&
                  grad->device() == like.device(),
              name, " must be float32 with one entry an output, on the outputs' device");
  return grad->const_data_ptr<float>();
}

// {grad_hidden [rows, C]} and / or {grad_weight}, those asked for in that order.
std::vector<Tensor> linear_log_probs_backward(std::optional<Tensor> grad_log_probs,
                                              std::optional<Tensor> grad_entropy, Tensor weight,
                                              Tensor saved, int64_t rows, double temperature,
                                              bool want_hidden, bool want_weight) {
  check_device_contiguous(weight, "weight");
  check_device_contiguous(saved, "saved");
  TORCH_CHECK(weight.dim() == 2 && weight.numel() > 0, "weight must have shape [V, C]");
  TORCH_CHECK(saved.device() == weight.device(), "saved must share weight's device");
  const float* gx = check_upstream(grad_log_probs, rows, weight, "grad_log_probs");
  const float* ge = check_upstream(grad_entropy, rows, weight, "grad_entropy");
  c10::DeviceGuard guard(weight.device());
  const int64_t vocab = weight.size(0), c = weight.size(1);
  std::vector<Tensor> out;
  void *gh = nullptr, *gw = nullptr;
  if (want_hidden) {
    out.push_back(at::empty({rows, c}, weight.options()));
    gh = out.back().data_ptr();
  }
  if (want_weight) {
    out.push_back(at::empty_like(weight));
    gw = out.back().data_ptr();
  }
  const size_t bytes = frwkv_linear_log_probs_backward_workspace_bytes(
      rows, c, vocab, want_hidden, ge != nullptr);
  Tensor work = workspace_like(weight, bytes);
  check_rc(frwkv_linear_log_probs_backward(
      io_code(weight.scalar_type()), rows, c, vocab, weight.const_data_ptr(),
      static_cast<float>(temperature), gx, ge, saved.const_data_ptr(),
      static_cast<size_t>(saved.numel()), gh, gw, scratch_ptr(work), bytes,
      current_stream(weight)));
  return out;
}

// A vector of token values beside log_probs: its dtype code and its data.
struct TokenColumn {
  int dtype = FRWKV_DTYPE_F32;
  const void* data = nullptr;
};

TokenColumn token_column(const std::optional<Tensor>& t, const Tensor& log_probs,
                         const char* name) {
  if (!t.has_value()) return {};
  check_device_contiguous(*t, name);
  TORCH_CHECK(t->numel() == log_probs.numel() && t->device() == log_probs.device(), name,
              " must have one entry a token, on log_probs' device");
  return {io_code(t->scalar_type()), t->const_data_ptr()};
}

const uint8_t* check_mask(const std::optional<Tensor>& mask, int64_t tokens, const Tensor& like) {
  if (!mask.has_value()) return nullptr;
  check_device_contiguous(*mask, "mask");
  TORCH_CHECK((mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte) &&
                  mask->numel() == tokens && mask->device() == like.device(),
              "mask must be bool or uint8 with one entry a token, on log_probs' device");
  return static_cast<const uint8_t*>(mask->const_data_ptr());
}

// Offsets and how many sequences they make; none without them.
const int32_t* check_offsets(const std::optional<Tensor>& cu, const Tensor& like,
                             int64_t* sequences) {
  *sequences = 0;
  if (!cu.has_value()) return nullptr;
  check_device_contiguous(*cu, "cu_seqlens");
  TORCH_CHECK(cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->numel() >= 2 &&
                  cu->device() == like.device(),
              "cu_seqlens must be int32 of shape [sequences + 1], on log_probs' device");
  *sequences = cu->numel() - 1;
  return cu->const_data_ptr<int32_t>();
}

// One of the codes up to `last`: shapes are chosen by it before it is narrowed.
int reduction_code(int64_t reduction, int last) {
  TORCH_CHECK(reduction >= FRWKV_REDUCE_NONE && reduction <= last, "unknown reduction ", reduction);
  return static_cast<int>(reduction);
}

// What the backward reads and the call's scratch, small beside it, as one allocation:
// one takes 1.3 us of a call's 8.
struct Buffers {
  Tensor all;
  size_t saved_bytes, work_bytes;
  Buffers(const Tensor& like, size_t saved, size_t work)
      : all(workspace_like(like, saved + work)), saved_bytes(saved), work_bytes(work) {}
  void* saved() const { return scratch_ptr(all); }
  // Both sizes are multiples of 256.
  void* work() const { return all.defined() ? all.data_ptr<uint8_t>() + saved_bytes : nullptr; }
};

// {loss, saved}, and the metrics after them where they are asked for.
std::vector<Tensor> policy_loss_forward(Tensor log_probs, Tensor old_log_probs, Tensor advantages,
                                        std::optional<Tensor> reference_log_probs,
                                        std::optional<Tensor> entropy, std::optional<Tensor> mask,
                                        std::optional<Tensor> cu_seqlens, double clip_low,
                                        double clip_high, double dual_clip, double kl_weight,
                                        double entropy_weight, int64_t reduction, bool metrics,
                                        bool slopes) {
  const int64_t tokens = log_probs.numel();
  TORCH_CHECK(tokens > 0, "log_probs must hold at least one token");
  const int reduce = reduction_code(reduction, FRWKV_REDUCE_SEQUENCE_MEAN);
  const TokenColumn x = token_column(log_probs, log_probs, "log_probs");
  const TokenColumn old = token_column(old_log_probs, log_probs, "old_log_probs");
  const TokenColumn reference =
      token_column(reference_log_probs, log_probs, "reference_log_probs");
  const TokenColumn h = token_column(entropy, log_probs, "entropy");
  const uint8_t* m = check_mask(mask, tokens, log_probs);
  int64_t sequences;
  const int32_t* cu = check_offsets(cu_seqlens, log_probs, &sequences);
  const bool per_sequence = advantages.sizes() != log_probs.sizes();
  check_device_contiguous(advantages, "advantages");
  TORCH_CHECK(advantages.device() == log_probs.device() &&
                  (!per_sequence || (sequences > 0 && advantages.dim() == 1 &&
                                     advantages.size(0) == sequences)),
              "advantages must have log_probs' shape, or one entry a sequence of cu_seqlens");
  c10::DeviceGuard guard(log_probs.device());
  const auto fp32 = log_probs.options().dtype(at::kFloat);
  Tensor loss = reduce == FRWKV_REDUCE_NONE ? at::empty(log_probs.sizes(), fp32)
                                            : at::empty({}, fp32);
  Tensor found;
  if (metrics) found = at::empty({4}, fp32);
  const Buffers buffers(log_probs, frwkv_policy_loss_saved_bytes(tokens, sequences),
                        frwkv_sequence_loss_workspace_bytes(tokens, sequences));
  check_rc(frwkv_policy_loss_forward(
      tokens, sequences, cu, m, x.dtype, x.data, old.dtype, old.data,
      io_code(advantages.scalar_type()), advantages.const_data_ptr(), per_sequence,
      reference.dtype, reference.data, h.dtype, h.data, clip_low, clip_high, dual_clip,
      static_cast<float>(kl_weight), static_cast<float>(entropy_weight), reduce,
      loss.data_ptr<float>(), metrics ? found.data_ptr<float>() : nullptr, slopes, buffers.saved(), buffers.saved_bytes,
      buffers.work(), buffers.work_bytes, current_stream(log_probs)));
  if (metrics) return {loss, buffers.all, found};
  return {loss, buffers.all};
}

// {grad_log_probs} and / or {grad_entropy}, those asked for in that order.
std::vector<Tensor> policy_loss_backward(Tensor grad_loss, Tensor saved,
                                         std::optional<Tensor> mask,
                                         std::optional<Tensor> cu_seqlens,
                                         std::vector<int64_t> shape,
                                         at::ScalarType log_probs_dtype,
                                         at::ScalarType entropy_dtype, double entropy_weight,
                                         int64_t reduction, bool want_log_probs,
                                         bool want_entropy) {
  check_device_contiguous(saved, "saved");
  refuse_capture(saved, "the policy loss's backward");
  const int reduce = reduction_code(reduction, FRWKV_REDUCE_SEQUENCE_MEAN);
  const int64_t tokens = c10::multiply_integers(shape);
  const float* up = check_upstream(
      grad_loss, reduce == FRWKV_REDUCE_NONE ? tokens : 1, saved, "grad_loss");
  const uint8_t* m = check_mask(mask, tokens, saved);
  int64_t sequences;
  const int32_t* cu = check_offsets(cu_seqlens, saved, &sequences);
  c10::DeviceGuard guard(saved.device());
  std::vector<Tensor> out;
  void *gx = nullptr, *gh = nullptr;
  if (want_log_probs) {
    out.push_back(at::empty(shape, saved.options().dtype(log_probs_dtype)));
    gx = out.back().data_ptr();
  }
  if (want_entropy) {
    out.push_back(at::empty(shape, saved.options().dtype(entropy_dtype)));
    gh = out.back().data_ptr();
  }
  check_rc(frwkv_policy_loss_backward(
      tokens, sequences, cu, m, static_cast<float>(entropy_weight), reduce, up,
      saved.const_data_ptr(), static_cast<size_t>(saved.numel()), io_code(log_probs_dtype), gx,
      io_code(entropy_dtype), gh, current_stream(saved)));
  return out;
}

// (loss, rewards, saved).
std::tuple<Tensor, Tensor, Tensor> preference_loss_forward(
    Tensor log_probs, Tensor cu_seqlens, std::optional<Tensor> reference_log_probs,
    std::optional<Tensor> mask, double beta, double margin, double label_smoothing, int64_t kind,
    bool normalize, int64_t reduction) {
  const int64_t tokens = log_probs.numel();
  TORCH_CHECK(tokens > 0, "log_probs must hold at least one token");
  const int reduce = reduction_code(reduction, FRWKV_REDUCE_SUM);
  const TokenColumn x = token_column(log_probs, log_probs, "log_probs");
  const TokenColumn reference =
      token_column(reference_log_probs, log_probs, "reference_log_probs");
  const uint8_t* m = check_mask(mask, tokens, log_probs);
  int64_t sequences;
  const int32_t* cu = check_offsets(cu_seqlens, log_probs, &sequences);
  TORCH_CHECK(sequences % 2 == 0, "cu_seqlens must have shape [2 * pairs + 1]");
  const int64_t pairs = sequences / 2;
  c10::DeviceGuard guard(log_probs.device());
  const auto fp32 = log_probs.options().dtype(at::kFloat);
  Tensor loss =
      reduce == FRWKV_REDUCE_NONE ? at::empty({pairs}, fp32) : at::empty({}, fp32);
  Tensor rewards = at::empty({pairs, 2}, fp32);
  const Buffers buffers(log_probs, frwkv_preference_loss_saved_bytes(pairs),
                        frwkv_sequence_loss_workspace_bytes(tokens, sequences));
  check_rc(frwkv_preference_loss_forward(
      tokens, pairs, cu, m, x.dtype, x.data, reference.dtype, reference.data, beta, margin,
      label_smoothing, static_cast<int>(kind), normalize, reduce,
      loss.data_ptr<float>(), rewards.data_ptr<float>(), buffers.saved(), buffers.saved_bytes,
      buffers.work(), buffers.work_bytes, current_stream(log_probs)));
  return {loss, rewards, buffers.all};
}

Tensor preference_loss_backward(Tensor grad_loss, Tensor saved, Tensor cu_seqlens,
                                std::optional<Tensor> mask, std::vector<int64_t> shape,
                                at::ScalarType log_probs_dtype, int64_t reduction) {
  check_device_contiguous(saved, "saved");
  refuse_capture(saved, "the preference loss's backward");
  const int reduce = reduction_code(reduction, FRWKV_REDUCE_SUM);
  const int64_t tokens = c10::multiply_integers(shape);
  int64_t sequences;
  const int32_t* cu = check_offsets(cu_seqlens, saved, &sequences);
  const float* up = check_upstream(
      grad_loss, reduce == FRWKV_REDUCE_NONE ? sequences / 2 : 1, saved, "grad_loss");
  const uint8_t* m = check_mask(mask, tokens, saved);
  c10::DeviceGuard guard(saved.device());
  Tensor out = at::empty(shape, saved.options().dtype(log_probs_dtype));
  check_rc(frwkv_preference_loss_backward(
      tokens, sequences / 2, cu, m, reduce, up, saved.const_data_ptr(),
      static_cast<size_t>(saved.numel()), io_code(log_probs_dtype), out.data_ptr(),
      current_stream(saved)));
  return out;
}

// ------------------------------------------------------------------ gradients
// Without a node of torch::autograd::Function nothing refuses forward-mode
// derivatives: calls with tangents are declined.
bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }

// Whether nothing is to be differentiated by it: norms and clipped tensors have no history.
bool is_constant(const Tensor& t) {
  return !(t.requires_grad() && at::GradMode::is_enabled()) && !has_tangent(t);
}

bool gradient_dtype(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf ||
         t.scalar_type() == at::kBFloat16;
}

// Whether a tensor's elements fill one range of memory, in any order.
bool is_gradient(const Tensor& t, const Tensor& first) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided &&
         t.device() == first.device() && gradient_dtype(t) &&
         t.is_non_overlapping_and_dense();
}

// Whether no written range of memory meets another tensor's. Ranges that are
// their own output's count once.
bool apart(const std::vector<frwkv_gradient>& list) {
  struct Range {
    uintptr_t from, to;
    bool written;
  };
  std::vector<Range> ranges;
  ranges.reserve(2 * list.size());
  const auto add = [&](const void* p, int64_t numel, int32_t dtype, bool written) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const int64_t bytes = dtype == FRWKV_DTYPE_F32 ? 4 : 2;
    if (numel > 0) ranges.push_back({at, at + static_cast<uintptr_t>(numel * bytes), written});
  };
  for (const frwkv_gradient& x : list) {
    add(x.out, x.numel, x.out_dtype, true);
    if (x.data != x.out) add(x.data, x.numel, x.dtype, false);
  }
  std::sort(ranges.begin(), ranges.end(),
            [](const Range& a, const Range& b) { return a.from < b.from; });
  uintptr_t written = 0, any = 0;  // ends of the ranges so far
  for (const Range& x : ranges) {
    if (x.from < written || (x.written && x.from < any)) return false;
    any = std::max(any, x.to);
    if (x.written) written = std::max(written, x.to);
  }
  return true;
}

// out null: nothing is written. A tensor that is written and shares its memory until
// then gets memory of its own, before any address is taken.
std::vector<frwkv_gradient> gradient_list(const std::vector<Tensor>& tensors,
                                          const std::vector<Tensor>* out) {
  std::vector<frwkv_gradient> list(tensors.size());
  for (size_t i = 0; out != nullptr && i < tensors.size(); ++i) {
    list[i].out = (*out)[i].mutable_data_ptr();
  }
  for (size_t i = 0; i < tensors.size(); ++i) {
    const Tensor& x = tensors[i];
    list[i].data = x.const_data_ptr();
    list[i].numel = x.numel();
    list[i].dtype = io_code(x.scalar_type());
    list[i].out_dtype = io_code((out != nullptr ? (*out)[i] : x).scalar_type());
  }
  return list;
}

Tensor grad_norm(const std::vector<Tensor>& tensors) {
  TORCH_CHECK(!tensors.empty(), "tensors must hold at least one tensor");
  for (const Tensor& t : tensors) {
    TORCH_CHECK(is_gradient(t, tensors[0]),
                "tensors must be CUDA float32, float16 or bfloat16 without gaps, on one device");
  }
  c10::DeviceGuard guard(tensors[0].device());
  const std::vector<frwkv_gradient> list = gradient_list(tensors, nullptr);
  const int64_t count = static_cast<int64_t>(list.size());
  Tensor norm = at::empty({}, tensors[0].options().dtype(at::kFloat));
  const size_t bytes = frwkv_grad_norm_workspace_bytes(count, list.data());
  Tensor work = workspace_like(tensors[0], bytes);
  check_rc(frwkv_grad_norm(count, list.data(), norm.data_ptr<float>(), scratch_ptr(work), bytes,
                           current_stream(tensors[0])));
  return norm;
}

bool may_clip(const std::vector<Tensor>& tensors, const std::vector<Tensor>& out) {
  if (tensors.empty() || out.size() != tensors.size()) return false;
  for (size_t i = 0; i < tensors.size(); ++i) {
    const Tensor &x = tensors[i], &y = out[i];
    if (!is_gradient(x, tensors[0]) || !is_gradient(y, tensors[0]) || !is_constant(x) ||
        !is_constant(y) || y.sizes() != x.sizes() || y.strides() != x.strides()) {
      return false;
    }
  }
  return true;
}

// Clips into out (tensors themselves: in place). list: gradient_list of both.
Tensor clip_gradients(const std::vector<Tensor>& tensors, const std::vector<Tensor>& out,
                      const std::vector<frwkv_gradient>& list, double max_norm, double eps) {
  c10::DeviceGuard guard(tensors[0].device());
  const int64_t count = static_cast<int64_t>(list.size());
  Tensor norm = at::empty({}, tensors[0].options().dtype(at::kFloat));
  const size_t bytes = frwkv_grad_norm_workspace_bytes(count, list.data());
  Tensor work = workspace_like(tensors[0], bytes);
  check_rc(frwkv_grad_clip(count, list.data(), max_norm, eps, norm.data_ptr<float>(),
                           scratch_ptr(work), bytes, current_stream(tensors[0])));
  for (const Tensor& t : out) {
    if (!t.unsafeGetTensorImpl()->is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  return norm;
}

Tensor clip_grad_norm_op(std::vector<Tensor> tensors, std::vector<Tensor> out, double max_norm,
                         double eps) {
  TORCH_CHECK(may_clip(tensors, out),
              "tensors and out must be CUDA float32, float16 or bfloat16 without gaps, on one "
              "device, pairwise of one layout, and must not require gradients");
  const std::vector<frwkv_gradient> list = gradient_list(tensors, &out);
  TORCH_CHECK(apart(list), "tensors that are written must not overlap others");
  return clip_gradients(tensors, out, list, max_norm, eps);
}

Tensor grad_norm_op(std::vector<Tensor> tensors) { return grad_norm(tensors); }

}  // namespace

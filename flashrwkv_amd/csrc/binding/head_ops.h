// Ops of the training head: layer norm with the residual add, and the losses
// from the hidden rows (no counterpart in the reference's binding). Part of
// torch_ops.cpp, whose helpers it uses.
#pragma once

namespace {

void check_like(const Tensor& t, const Tensor& x, const char* name) {
  check_device_contiguous(t, name);
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have x's dtype");
  TORCH_CHECK(t.device() == x.device(), name, " must share x's device");
}

void check_channels(const Tensor& t, const Tensor& x, const char* name) {
  check_like(t, x, name);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(-1), name, " must have shape [C]");
}

const void* data_or_null(const std::optional<Tensor>& t) {
  return t.has_value() ? t->const_data_ptr() : nullptr;
}

// {y}, {y, stream}, and mean and rstd after them where statistics are asked for.
std::vector<Tensor> layer_norm_forward(Tensor x, std::optional<Tensor> residual, Tensor weight,
                                       Tensor bias, double eps, bool statistics) {
  check_device_contiguous(x, "x");
  TORCH_CHECK(x.dim() >= 1 && x.numel() > 0, "x must have non-empty shape [..., C]");
  check_channels(weight, x, "weight");
  check_channels(bias, x, "bias");
  if (residual.has_value()) {
    check_like(*residual, x, "residual");
    TORCH_CHECK(residual->sizes() == x.sizes(), "residual must match x");
  }
  c10::DeviceGuard guard(x.device());
  const int64_t c = x.size(-1), rows = x.numel() / c;
  std::vector<Tensor> out = {at::empty_like(x)};
  void* stream_out = nullptr;
  if (residual.has_value()) {
    out.push_back(at::empty_like(x));
    stream_out = out.back().data_ptr();
  }
  float *mean = nullptr, *rstd = nullptr;
  if (statistics) {
    const auto fp32 = x.options().dtype(at::kFloat);
    out.push_back(at::empty({rows}, fp32));
    mean = out.back().data_ptr<float>();
    out.push_back(at::empty({rows}, fp32));
    rstd = out.back().data_ptr<float>();
  }
  check_rc(frwkv_layer_norm_forward(io_code(x.scalar_type()), rows, c, x.const_data_ptr(),
                                    data_or_null(residual), weight.const_data_ptr(),
                                    bias.const_data_ptr(), static_cast<float>(eps),
                                    out[0].data_ptr(), stream_out, mean, rstd,
                                    current_stream(x)));
  return out;
}

// {grad_x, grad_weight, grad_bias}.
std::vector<Tensor> layer_norm_backward(Tensor grad_y, Tensor normed,
                                        std::optional<Tensor> grad_stream, Tensor weight,
                                        Tensor mean, Tensor rstd) {
  check_device_contiguous(normed, "normed");
  TORCH_CHECK(normed.dim() >= 1 && normed.numel() > 0, "normed must have non-empty shape [..., C]");
  check_channels(weight, normed, "weight");
  const int64_t c = normed.size(-1), rows = normed.numel() / c;
  check_like(grad_y, normed, "grad_y");
  TORCH_CHECK(grad_y.sizes() == normed.sizes(), "grad_y must match normed");
  if (grad_stream.has_value()) {
    check_like(*grad_stream, normed, "grad_stream");
    TORCH_CHECK(grad_stream->sizes() == normed.sizes(), "grad_stream must match normed");
  }
  for (const Tensor* t : {&mean, &rstd}) {
    TORCH_CHECK(t->is_cuda() && t->is_contiguous() && t->scalar_type() == at::kFloat &&
                    t->numel() == rows && t->device() == normed.device(),
                "mean and rstd must be float32 [rows]");
  }
  c10::DeviceGuard guard(normed.device());
  Tensor gx = at::empty_like(normed), gw = at::empty_like(weight), gb = at::empty_like(weight);
  const size_t bytes = frwkv_layer_norm_backward_workspace_bytes(rows, c);
  Tensor work = workspace_like(normed, bytes);
  check_rc(frwkv_layer_norm_backward(
      io_code(normed.scalar_type()), rows, c, grad_y.const_data_ptr(), normed.const_data_ptr(),
      data_or_null(grad_stream), weight.const_data_ptr(), mean.const_data_ptr<float>(),
      rstd.const_data_ptr<float>(), gx.data_ptr(), gw.data_ptr(), gb.data_ptr(),
      work.data_ptr(), bytes, current_stream(normed)));
  return {gx, gw, gb};
}

// Rows of [..., C] hidden and what has to fit [V, C] weight.
int64_t check_head(const Tensor& hidden, const Tensor& weight, int64_t reduction) {
  check_device_contiguous(hidden, "hidden");
  check_device_contiguous(weight, "weight");
  TORCH_CHECK(hidden.dim() >= 1 && hidden.numel() > 0, "hidden must have non-empty shape [..., C]");
  TORCH_CHECK(weight.dim() == 2 && weight.numel() > 0 && weight.size(1) == hidden.size(-1),
              "weight must have shape [V, C]");
  TORCH_CHECK(weight.scalar_type() == hidden.scalar_type() && weight.device() == hidden.device(),
              "weight must have hidden's dtype and device");
  TORCH_CHECK(reduction >= FRWKV_REDUCE_NONE && reduction <= FRWKV_REDUCE_SUM,
              "reduction must be 0 (none), 1 (mean) or 2 (sum)");
  return hidden.numel() / hidden.size(-1);
}

int index_bytes(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name,
              " must be int32 or int64");
  return t.scalar_type() == at::kInt ? 4 : 8;
}

std::tuple<Tensor, Tensor> linear_cross_entropy_forward(Tensor hidden, Tensor weight,
                                                        Tensor targets, int64_t ignore_index,
                                                        int64_t reduction) {
  const int64_t rows = check_head(hidden, weight, reduction);
  check_device_contiguous(targets, "targets");
  const int bytes = index_bytes(targets, "targets");
  TORCH_CHECK(targets.numel() == rows && targets.device() == hidden.device(),
              "targets must have one entry a row of hidden, on its device");
  c10::DeviceGuard guard(hidden.device());
  const int64_t c = hidden.size(-1), vocab = weight.size(0);
  const auto fp32 = hidden.options().dtype(at::kFloat);
  Tensor loss = reduction == FRWKV_REDUCE_NONE ? at::empty(targets.sizes(), fp32)
                                               : at::empty({}, fp32);
  // Sizes that the call refuses have no bytes; its error says why.
  const size_t saved_bytes = frwkv_linear_loss_saved_bytes(rows, c, 1);
  const size_t work_bytes = frwkv_linear_loss_forward_workspace_bytes(rows, vocab);
  Tensor saved = workspace_like(hidden, saved_bytes), work = workspace_like(hidden, work_bytes);
  check_rc(frwkv_linear_cross_entropy_forward(
      io_code(hidden.scalar_type()), rows, c, vocab, hidden.const_data_ptr(),
      weight.const_data_ptr(), bytes, targets.const_data_ptr(), ignore_index,
      static_cast<int>(reduction), loss.data_ptr<float>(), scratch_ptr(saved), saved_bytes,
      scratch_ptr(work), work_bytes, current_stream(hidden)));
  return {loss, saved};
}

std::tuple<Tensor, Tensor> linear_topk_distillation_forward(Tensor hidden, Tensor weight,
                                                            Tensor teacher_logits,
                                                            Tensor teacher_indices,
                                                            double temperature,
                                                            int64_t reduction) {
  const int64_t rows = check_head(hidden, weight, reduction);
  check_device_contiguous(teacher_logits, "teacher_logits");
  check_device_contiguous(teacher_indices, "teacher_indices");
  const int bytes = index_bytes(teacher_indices, "teacher_indices");
  TORCH_CHECK(teacher_logits.dim() >= 1 && teacher_logits.sizes() == teacher_indices.sizes() &&
                  teacher_logits.size(-1) > 0 &&
                  teacher_logits.numel() == rows * teacher_logits.size(-1),
              "teacher_logits and teacher_indices must have shape [..., K], a row each of hidden");
  TORCH_CHECK(teacher_logits.device() == hidden.device() &&
                  teacher_indices.device() == hidden.device(),
              "teacher tensors must share hidden's device");
  c10::DeviceGuard guard(hidden.device());
  const int64_t c = hidden.size(-1), vocab = weight.size(0), top = teacher_logits.size(-1);
  const auto fp32 = hidden.options().dtype(at::kFloat);
  const auto lead = teacher_logits.sizes().slice(0, teacher_logits.dim() - 1);
  Tensor loss = reduction == FRWKV_REDUCE_NONE ? at::empty(lead, fp32) : at::empty({}, fp32);
  const size_t saved_bytes = frwkv_linear_loss_saved_bytes(rows, c, top);
  const size_t work_bytes = frwkv_linear_loss_forward_workspace_bytes(rows, vocab);
  Tensor saved = workspace_like(hidden, saved_bytes), work = workspace_like(hidden, work_bytes);
  check_rc(frwkv_linear_topk_distillation_forward(
      io_code(hidden.scalar_type()), rows, c, vocab, top, hidden.const_data_ptr(),
      weight.const_data_ptr(), io_code(teacher_logits.scalar_type()),
      teacher_logits.const_data_ptr(), bytes, teacher_indices.const_data_ptr(),
      static_cast<float>(temperature), static_cast<int>(reduction), loss.data_ptr<float>(),
      scratch_ptr(saved), saved_bytes, scratch_ptr(work), work_bytes, current_stream(hidden)));
  return {loss, saved};
}

// {grad_hidden [rows, C]} and / or {grad_weight}, those asked for in that order.
std::vector<Tensor> linear_loss_backward(Tensor grad_loss, Tensor weight, Tensor saved,
                                         int64_t rows, int64_t top, double temperature,
                                         int64_t reduction, bool want_hidden, bool want_weight) {
  check_device_contiguous(weight, "weight");
  check_device_contiguous(grad_loss, "grad_loss");
  check_device_contiguous(saved, "saved");
  TORCH_CHECK(weight.dim() == 2 && weight.numel() > 0, "weight must have shape [V, C]");
  const int64_t expected = reduction == FRWKV_REDUCE_NONE ? rows : 1;
  TORCH_CHECK(grad_loss.scalar_type() == at::kFloat && grad_loss.numel() == expected &&
                  grad_loss.device() == weight.device() && saved.device() == weight.device(),
              "grad_loss must be float32 with one entry a loss, on weight's device");
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
  const size_t bytes = frwkv_linear_loss_backward_workspace_bytes(rows, c, vocab, want_hidden);
  Tensor work = workspace_like(weight, bytes);
  check_rc(frwkv_linear_loss_backward(
      io_code(weight.scalar_type()), rows, c, vocab, top, weight.const_data_ptr(),
      static_cast<float>(temperature), static_cast<int>(reduction),
      grad_loss.const_data_ptr<float>(), saved.const_data_ptr(),
      static_cast<size_t>(saved.numel()), gh, gw, scratch_ptr(work), bytes,
      current_stream(weight)));
  return out;
}

}  // namespace

"""Losses of a language model's head, from its hidden rows, and of its tokens.

The first three take the hidden rows ``[..., C]`` (after the last norm) and the head's
weight ``[V, C]`` instead of logits: the product, the softmax over the
vocabulary and the loss run piece by piece, and the ``[rows, V]`` logits never
exist in memory, forward or backward.

* :func:`pretrain_linear_cross_entropy`: softmax cross entropy against one
  token a row. Without gradients, ``reduction="none"`` is the scoring form
  (minus the log probability of each token).
* :func:`pretrain_linear_topk_distillation`: the divergence from a teacher that
  is known by its K largest logits a row.
* :func:`pretrain_linear_log_probs`: the log probability of one token a row at a
  sampling temperature, and the entropy beside it; not a loss, but what the two
  below are taken from.
* :func:`pretrain_policy_loss`, :func:`pretrain_preference_loss`: losses over
  packed sequences of such log probabilities (:mod:`.sequences`).

The head's are of float16 and bfloat16, fp32 sums, ``C`` a multiple of 64, any ``V`` and row
count. Rows that take no part (``ignore_index``; no teacher entry) are left out
before the products, so they cost nothing there and what they hold, NaN
included, reaches neither the loss nor a gradient. Only what needs a gradient
gets one: with a frozen head the weight's product is not computed. Nothing
synchronises with the host, so a token out of range cannot be raised as an
error: it makes its row's loss, and with it the gradients, NaN.

Sums are in a fixed order: the same call gives the same bits. The kernels are
in ``csrc/linear_loss.hip`` and ``csrc/sequence_loss.hip``; the reference's loss operators are not part of
this package, and these do not take their names.
"""

from __future__ import annotations

import torch

from .. import _contract as C
from .._contract import check, is_tensor
from .sequences import pretrain_policy_loss, pretrain_preference_loss

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
MAX_TOP = 1024
MAX_CHANNELS = 65536
_INDEX = (torch.int32, torch.int64)

HEAD = (
    is_tensor("hidden"),
    check("hidden", C.dtype_is(torch.float16, torch.bfloat16), TypeError,
          "hidden must be float16 or bfloat16"),
    check("hidden", C.cuda_contiguous, ValueError, "hidden must be CUDA and contiguous"),
    check("hidden", lambda x, ns: x.ndim >= 1 and x.shape[-1] > 0 and x.shape[-1] % 64 == 0
          and x.shape[-1] <= MAX_CHANNELS, ValueError,
          f"hidden must have shape [...,C] with C a multiple of 64, at most {MAX_CHANNELS}"),
    is_tensor("weight"),
    check("weight", lambda x, ns: x.dtype == ns["hidden"].dtype, TypeError,
          "weight must have hidden's dtype"),
    check("weight", C.cuda_contiguous, ValueError, "weight must be CUDA and contiguous"),
    check("weight", C.same_device_as("hidden"), ValueError, "weight must share hidden's device"),
    check("weight", lambda x, ns: x.ndim == 2 and x.shape[0] > 0
          and x.shape[1] == ns["hidden"].shape[-1], ValueError, "weight must have shape [V,C]"),
)

_TARGETS = (
    is_tensor("targets"),
    check("targets", C.dtype_is(*_INDEX), TypeError, "targets must be int32 or int64"),
    check("targets", C.cuda_contiguous, ValueError, "targets must be CUDA and contiguous"),
    check("targets", C.same_device_as("hidden"), ValueError,
          "targets must share hidden's device"),
    check("targets", lambda x, ns: x.shape == ns["hidden"].shape[:-1], ValueError,
          "targets must have hidden's shape without the channels"),
    check("ignore_index", C.plain_int, TypeError, "ignore_index must be an int"),
)

_TEMPERATURE = (
    check("temperature", lambda x, ns: C.finite_number(x, ns) and not isinstance(x, bool)
          and 1e-30 < x < 1e30, ValueError, "temperature must be positive and finite"),
)

_REDUCTION = (
    check("reduction", C.one_of(tuple(REDUCTIONS)), ValueError,
          "reduction must be one of 'none', 'mean' or 'sum'"),
)

CROSS_ENTROPY = (*HEAD, *_REDUCTION, *_TARGETS)

LOG_PROBS = (*HEAD, *_TARGETS, *_TEMPERATURE)

DISTILLATION = (
    *HEAD,
    *_REDUCTION,
    is_tensor("teacher_logits"),
    check("teacher_logits", C.dtype_is(torch.float32, torch.float16, torch.bfloat16), TypeError,
          "teacher_logits must be float32, float16 or bfloat16"),
    check("teacher_logits", C.cuda_contiguous, ValueError,
          "teacher_logits must be CUDA and contiguous"),
    check("teacher_logits", C.same_device_as("hidden"), ValueError,
          "teacher_logits must share hidden's device"),
    check("teacher_logits", lambda x, ns: x.ndim == ns["hidden"].ndim
          and x.shape[:-1] == ns["hidden"].shape[:-1] and 0 < x.shape[-1] <= MAX_TOP, ValueError,
          f"teacher_logits must have shape [...,K] with hidden's leading shape and K at most "
          f"{MAX_TOP}"),
    is_tensor("teacher_indices"),
    check("teacher_indices", C.dtype_is(*_INDEX), TypeError,
          "teacher_indices must be int32 or int64"),
    check("teacher_indices", C.cuda_contiguous, ValueError,
          "teacher_indices must be CUDA and contiguous"),
    check("teacher_indices", C.same_device_as("hidden"), ValueError,
          "teacher_indices must share hidden's device"),
    check("teacher_indices", C.same_shape_as("teacher_logits"), ValueError,
          "teacher_indices must match teacher_logits"),
    *_TEMPERATURE,
)


class _LinearLoss(torch.autograd.Function):
    """Calls that the native whole call declines (tensor subclasses, modes, no
    rows). Forward keeps the rows that take part, their log sums and target
    logits (one buffer) and the weight; backward makes the logits again, piece
    by piece."""

    @staticmethod
    def forward(ctx, hidden, weight, launch, top, temperature, reduction):
        ctx.shape, ctx.top = hidden.shape, top
        ctx.temperature, ctx.reduction = temperature, reduction
        ctx.rows = hidden.numel() // hidden.shape[-1]
        if ctx.rows == 0:
            shape = hidden.shape[:-1] if reduction == 0 else ()
            ctx.save_for_backward(weight)
            return torch.zeros(shape, device=hidden.device, dtype=torch.float32)
        loss, saved = launch(hidden, weight, any(ctx.needs_input_grad))
        ctx.save_for_backward(weight, saved)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        weight, *saved = ctx.saved_tensors
        want = ctx.needs_input_grad[:2]
        grads = [None, None]
        if ctx.rows == 0:
            made = [weight.new_empty(ctx.shape), torch.zeros_like(weight)]
            grads = [g if w else None for g, w in zip(made, want)]
        else:
            made = C.native().linear_loss_backward(
                grad_loss.contiguous(), weight, *saved, ctx.rows, ctx.top, ctx.temperature,
                ctx.reduction, *want)
            if want[0]:
                grads[0] = made[0].view(ctx.shape)
            if want[1]:
                grads[1] = made[-1]
        return (*grads, None, None, None, None)


class _LinearLogProbs(torch.autograd.Function):
    """The same for log probabilities and entropies."""

    @staticmethod
    def forward(ctx, hidden, weight, launch, temperature, entropy):
        ctx.set_materialize_grads(False)
        ctx.shape, ctx.temperature = hidden.shape, temperature
        ctx.rows = hidden.numel() // hidden.shape[-1]
        if ctx.rows == 0:
            ctx.save_for_backward(weight)
            return tuple(torch.zeros(hidden.shape[:-1], device=hidden.device,
                                     dtype=torch.float32) for _ in range(1 + entropy))
        *out, saved = launch(hidden, weight, any(ctx.needs_input_grad))
        ctx.save_for_backward(weight, saved)
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *upstream):
        weight, *saved = ctx.saved_tensors
        want = ctx.needs_input_grad[:2]
        grads = [None, None]
        upstream = [None if g is None else g.contiguous() for g in (*upstream, None)][:2]
        if ctx.rows == 0:
            made = [weight.new_empty(ctx.shape), torch.zeros_like(weight)]
            grads = [g if w else None for g, w in zip(made, want)]
        elif any(g is not None for g in upstream):
            made = C.native().linear_log_probs_backward(*upstream, weight, *saved, ctx.rows,
                                                        ctx.temperature, *want)
            if want[0]:
                grads[0] = made[0].view(ctx.shape)
            if want[1]:
                grads[1] = made[-1]
        return (*grads, None, None, None)


def _refuse_capture(name):
    C.native()
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name} does not run under HIP graph capture: training steps are "
                           "not validated inside a captured graph")


def _run(name, hidden, weight, launch, top, temperature, reduction):
    _refuse_capture(name)
    return _LinearLoss.apply(hidden, weight, launch, top, float(temperature),
                             REDUCTIONS[reduction])


def pretrain_linear_cross_entropy(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    *,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """Softmax cross entropy of ``hidden weight^T`` against ``targets``.

    ``hidden`` ``[..., C]``, ``weight`` ``[V, C]``, ``targets`` ``[...]`` (int32
    or int64; rows with ``ignore_index`` take no part). Returns the fp32 loss:
    per row (0 for rows that take no part), their mean over the rows that take
    part (0 if none does) or their sum. Gradients for hidden and weight.
    """
    call = C.whole_call("linear_loss_call")
    if call and isinstance(reduction, str) and reduction in REDUCTIONS:
        loss = call(hidden, weight, targets, None, ignore_index, 1.0, REDUCTIONS[reduction])
        if loss is not None:
            return loss
    C.enforce(CROSS_ENTROPY, {"hidden": hidden, "weight": weight, "targets": targets,
                              "ignore_index": ignore_index, "reduction": reduction})

    def launch(h, w, backward_follows):
        return C.native().linear_cross_entropy_forward(h, w, targets, ignore_index,
                                                       REDUCTIONS[reduction], backward_follows)

    return _run("pretrain_linear_cross_entropy", hidden, weight, launch, 1, 1.0, reduction)


def pretrain_linear_topk_distillation(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_indices: torch.Tensor,
    *,
    temperature: float = 1.0,
    reduction: str = "mean",
) -> torch.Tensor:
    """Divergence of the head's distribution from a teacher's top logits.

    ``teacher_logits`` / ``teacher_indices`` ``[..., K]``: the teacher's K
    largest logits a row and their tokens; an entry with a negative index or a
    logit of -inf is absent, a row without entries takes no part. With p =
    softmax(teacher_logits / T) over a row's entries and q = softmax(hidden
    weight^T / T) over the whole vocabulary the loss is
    ``T^2 sum p (log p - log q)`` over the entries, reduced as in
    :func:`pretrain_linear_cross_entropy`. A token listed twice pulls with the sum
    of its p, so the gradients are those of the joined entries; the loss has both
    entries as they stand, which is less than the joined ones' divergence by
    ``T^2 sum p log(P / p)`` (P: the token's sum of p) and can be negative.
    Gradients for hidden and weight; none for the teacher.
    """
    call = C.whole_call("linear_loss_call") if teacher_logits is not None else None
    if call and isinstance(reduction, str) and reduction in REDUCTIONS:
        loss = call(hidden, weight, teacher_indices, teacher_logits, 0, temperature,
                    REDUCTIONS[reduction])
        if loss is not None:
            return loss
    C.enforce(DISTILLATION, {"hidden": hidden, "weight": weight,
                             "teacher_logits": teacher_logits,
                             "teacher_indices": teacher_indices, "temperature": temperature,
                             "reduction": reduction})

    def launch(h, w, _):
        return C.native().linear_topk_distillation_forward(
            h, w, teacher_logits, teacher_indices, temperature, REDUCTIONS[reduction])

    return _run("pretrain_linear_topk_distillation", hidden, weight, launch,
                teacher_logits.shape[-1], temperature, reduction)


def pretrain_linear_log_probs(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    *,
    temperature: float = 1.0,
    ignore_index: int = -100,
    entropy: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Log probability of each row's token under ``q = softmax(hidden weight^T /
    temperature)``, and with ``entropy=True`` (log_probs, entropy), ``-sum q log q``
    of each row beside it.

    ``targets`` as in :func:`pretrain_linear_cross_entropy`, whose loss at
    temperature 1 is minus the first. fp32 in ``targets``' shape; both are 0 for rows
    with ``ignore_index`` and NaN for a token out of range. Gradients for hidden and weight from
    either or both.
    """
    call = C.whole_call("linear_log_probs_call")
    if call:
        got = call(hidden, weight, targets, ignore_index, temperature, bool(entropy))
        if got is not None:
            return got if entropy else got[0]
    C.enforce(LOG_PROBS, {"hidden": hidden, "weight": weight, "targets": targets,
                          "temperature": temperature, "ignore_index": ignore_index})
    _refuse_capture("pretrain_linear_log_probs")

    def launch(h, w, backward_follows):
        return C.native().linear_log_probs_forward(h, w, targets, ignore_index, temperature,
                                                   entropy, backward_follows)

    got = _LinearLogProbs.apply(hidden, weight, launch, float(temperature), bool(entropy))
    return got if entropy else got[0]


__all__ = [
    "pretrain_linear_cross_entropy",
    "pretrain_linear_log_probs",
    "pretrain_linear_topk_distillation",
    "pretrain_policy_loss",
    "pretrain_preference_loss",
]

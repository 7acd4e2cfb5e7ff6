"""Losses over packed sequences of token log probabilities.

* :func:`pretrain_policy_loss`: the clipped policy loss with a KL term, from the
  log probabilities of sampled tokens.
* :func:`pretrain_preference_loss`: the preference loss of paired sequences.

Both take log probabilities of any shape, read in memory order: what
:func:`..pretrain_linear_log_probs` returns, or any others. ``cu_seqlens`` int32
``[sequences + 1]`` says which tokens are a sequence (offsets that start at 0 and
do not fall; tokens behind the last one take no part, as a padded batch has
them); ``mask`` (bool or uint8, one entry a token) leaves tokens out. What stands in tokens that
take no part, NaN included, reaches nothing, and their gradients are 0. Each
vector is float32, float16 or bfloat16 by itself. A policy's ratios, and with them a
token's loss, are in 32 bits from log ratios that are rounded once (on which side of
a clip border one is, is decided as in 64); sums over tokens, and all of a
preference pair, are in 64 bits and in a fixed order.

Nothing synchronises with the host: offsets that may not be cannot be raised as
an error, they make a reduced loss and the gradients of all tokens NaN.
"""

from __future__ import annotations

import torch

from .. import _contract as C
from .._contract import check, is_tensor, when

POLICY_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2, "sequence_mean": 3}
PAIR_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
KINDS = {"sigmoid": 0, "hinge": 1, "squared": 2}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _number(x, low, high):
    return C.finite_number(x, None) and not isinstance(x, bool) and low <= x <= high


def _given(name):
    return lambda ns: ns[name] is not None


def _vector(name, *, constant, shaped=True):
    rules = [
        is_tensor(name),
        check(name, C.dtype_is(*_FLOATS), TypeError,
              f"{name} must be float32, float16 or bfloat16"),
        check(name, C.cuda_contiguous, ValueError, f"{name} must be CUDA and contiguous"),
    ]
    if name != "log_probs":
        rules.append(check(name, C.same_device_as("log_probs"), ValueError,
                           f"{name} must share log_probs' device"))
        if shaped:
            rules.append(check(name, C.same_shape_as("log_probs"), ValueError,
                               f"{name} must match log_probs"))
    if constant:
        rules.append(check(name, C.constant, ValueError,
                           f"{name} must not require gradients: it has none here (detach it)"))
    return rules


def _optional(name, rules):
    return [when(_given(name), rule) for rule in rules]


_MASK = _optional("mask", [
    is_tensor("mask"),
    check("mask", C.dtype_is(torch.bool, torch.uint8), TypeError, "mask must be bool or uint8"),
    check("mask", C.cuda_contiguous, ValueError, "mask must be CUDA and contiguous"),
    check("mask", C.same_device_as("log_probs"), ValueError,
          "mask must share log_probs' device"),
    check("mask", C.same_shape_as("log_probs"), ValueError, "mask must match log_probs"),
])

_OFFSETS = [
    is_tensor("cu_seqlens"),
    check("cu_seqlens", C.dtype_is(torch.int32), TypeError, "cu_seqlens must be int32"),
    check("cu_seqlens", C.cuda_contiguous, ValueError, "cu_seqlens must be CUDA and contiguous"),
    check("cu_seqlens", C.same_device_as("log_probs"), ValueError,
          "cu_seqlens must share log_probs' device"),
    check("cu_seqlens", lambda x, ns: x.ndim == 1 and x.numel() >= 2, ValueError,
          "cu_seqlens must have shape [sequences + 1]"),
]


def _advantages_fit(x, ns):
    if x.shape == ns["log_probs"].shape:
        return True
    cu = ns["cu_seqlens"]
    return cu is not None and x.shape == (cu.numel() - 1,)


POLICY = (
    *_vector("log_probs", constant=False),
    *_vector("old_log_probs", constant=True),
    *_optional("cu_seqlens", _OFFSETS),
    *_vector("advantages", constant=True, shaped=False),
    check("advantages", _advantages_fit, ValueError,
          "advantages must match log_probs, or have one entry a sequence of cu_seqlens"),
    *_optional("reference_log_probs", _vector("reference_log_probs", constant=True)),
    *_optional("entropy", _vector("entropy", constant=False)),
    *_MASK,
    check("clip_low", lambda x, ns: _number(x, 0.0, 1.0), ValueError,
          "clip_low must be a number in [0, 1]"),
    check("clip_high", lambda x, ns: _number(x, 0.0, 1e30), ValueError,
          "clip_high must be a finite number, not negative"),
    when(_given("dual_clip"),
         check("dual_clip", lambda x, ns: _number(x, 1.0, 1e30) and x > 1.0, ValueError,
               "dual_clip must be None or a finite number above 1")),
    check("kl_weight", lambda x, ns: _number(x, -1e30, 1e30), ValueError,
          "kl_weight must be a finite number"),
    check("kl_weight", lambda x, ns: x == 0 or ns["reference_log_probs"] is not None, ValueError,
          "kl_weight needs reference_log_probs"),
    check("entropy_weight", lambda x, ns: _number(x, -1e30, 1e30), ValueError,
          "entropy_weight must be a finite number"),
    check("entropy_weight", lambda x, ns: x == 0 or ns["entropy"] is not None, ValueError,
          "entropy_weight needs entropy"),
    check("reduction", C.one_of(tuple(POLICY_REDUCTIONS)), ValueError,
          "reduction must be one of 'none', 'mean', 'sum' or 'sequence_mean'"),
    check("reduction", lambda x, ns: x != "sequence_mean" or ns["cu_seqlens"] is not None,
          ValueError, "reduction 'sequence_mean' needs cu_seqlens"),
)

PREFERENCE = (
    *_vector("log_probs", constant=False),
    *_OFFSETS,
    check("cu_seqlens", lambda x, ns: x.numel() % 2 == 1, ValueError,
          "cu_seqlens must have shape [2 * pairs + 1]"),
    *_optional("reference_log_probs", _vector("reference_log_probs", constant=True)),
    *_MASK,
    check("beta", lambda x, ns: _number(x, 1e-30, 1e30), ValueError,
          "beta must be positive and finite"),
    check("margin", lambda x, ns: _number(x, -1e30, 1e30), ValueError,
          "margin must be a finite number"),
    check("label_smoothing", lambda x, ns: _number(x, 0.0, 0.5), ValueError,
          "label_smoothing must be a number in [0, 0.5]"),
    check("kind", C.one_of(tuple(KINDS)), ValueError,
          "kind must be one of 'sigmoid', 'hinge' or 'squared'"),
    check("label_smoothing", lambda x, ns: x == 0 or ns["kind"] == "sigmoid", ValueError,
          "label_smoothing is of kind 'sigmoid' only"),
    check("reduction", C.one_of(tuple(PAIR_REDUCTIONS)), ValueError,
          "reduction must be one of 'none', 'mean' or 'sum'"),
)


class _PolicyLoss(torch.autograd.Function):
    """Calls that the native whole call declines (tensor subclasses, modes)."""

    @staticmethod
    def forward(ctx, log_probs, entropy, mask, cu_seqlens, entropy_weight, reduction, launch):
        loss, saved, *metrics = launch(log_probs, entropy, ctx.needs_input_grad[0])
        ctx.save_for_backward(saved, mask, cu_seqlens)
        ctx.shape, ctx.dtype = list(log_probs.shape), log_probs.dtype
        ctx.entropy_dtype = torch.float32 if entropy is None else entropy.dtype
        ctx.entropy_weight, ctx.reduction = entropy_weight, reduction
        ctx.mark_non_differentiable(*metrics)
        return (loss, *metrics)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss, *_):
        saved, mask, cu_seqlens = ctx.saved_tensors
        want = ctx.needs_input_grad[:2]
        made = C.native().policy_loss_backward(
            grad_loss.contiguous(), saved, mask, cu_seqlens, ctx.shape, ctx.dtype,
            ctx.entropy_dtype, ctx.entropy_weight, ctx.reduction, *want)
        return (made[0] if want[0] else None, made[-1] if want[1] else None, *[None] * 5)


class _PreferenceLoss(torch.autograd.Function):
    """Calls that the native whole call declines."""

    @staticmethod
    def forward(ctx, log_probs, mask, cu_seqlens, reduction, launch):
        loss, rewards, saved = launch(log_probs)
        ctx.save_for_backward(saved, mask, cu_seqlens)
        ctx.shape, ctx.dtype = list(log_probs.shape), log_probs.dtype
        ctx.reduction = reduction
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss, _):
        saved, mask, cu_seqlens = ctx.saved_tensors
        grad = C.native().preference_loss_backward(
            grad_loss.contiguous(), saved, cu_seqlens, mask, ctx.shape, ctx.dtype, ctx.reduction)
        return (grad, *[None] * 4)


def _begin(name):
    C.native()
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name} does not run under HIP graph capture: training steps are "
                           "not validated inside a captured graph")


def _nothing(log_probs, shape, *others):
    """The loss of no tokens, with gradients that have no elements."""
    loss = sum(t.float().sum() for t in (log_probs, *others) if t is not None)
    return loss.expand(shape) if shape != () else loss


def pretrain_policy_loss(
    log_probs: torch.Tensor,
    old_log_probs: torch.Tensor,
    advantages: torch.Tensor,
    *,
    reference_log_probs: torch.Tensor | None = None,
    entropy: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    dual_clip: float | None = None,
    kl_weight: float = 0.0,
    entropy_weight: float = 0.0,
    reduction: str = "mean",
    metrics: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Clipped policy loss of sampled tokens, with a KL term.

    With ``d = log_probs - old_log_probs`` (of the policy that sampled), ``r =
    exp(d)`` and the advantage A (``log_probs``' shape, or ``[sequences]`` with
    ``cu_seqlens``; one a token where both fit) a token's loss is

        -min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A)
        + kl_weight k3(reference_log_probs - log_probs) - entropy_weight entropy

    with ``k3(x) = exp(x) - 1 - x``; with ``dual_clip`` the first term is at most
    ``-dual_clip A`` where A < 0. A term whose weight is 0 is not there, whatever it would
    be. ``reduction``: the mean or sum over the tokens that
    take part, the mean over sequences of each one's mean (``"sequence_mean"``;
    sequences without such tokens do not count), 0 without any, or ``"none"``: a
    loss a token in ``log_probs``' shape.

    ``metrics=True`` returns (loss, metrics): fp32 ``[4]`` without gradients, the means
    over those tokens of r, of whether a token's gradient is clipped away, of k3(d)
    (the KL from the old policy) and of the reference's k3 (0 without one).
    Gradients for log_probs and entropy, none for the others, which must not
    require any.
    """
    dual = 0.0 if dual_clip is None else dual_clip
    call = C.whole_call("policy_loss_call")
    if (call and isinstance(reduction, str) and reduction in POLICY_REDUCTIONS
            and (dual_clip is None or dual_clip != 0)):
        got = call(log_probs, old_log_probs, advantages, reference_log_probs, entropy, mask,
                   cu_seqlens, clip_low, clip_high, dual, kl_weight, entropy_weight,
                   POLICY_REDUCTIONS[reduction], bool(metrics))
        if got is not None:
            return got if metrics else got[0]
    C.enforce(POLICY, {
        "log_probs": log_probs, "old_log_probs": old_log_probs, "advantages": advantages,
        "reference_log_probs": reference_log_probs, "entropy": entropy, "mask": mask,
        "cu_seqlens": cu_seqlens, "clip_low": clip_low, "clip_high": clip_high,
        "dual_clip": dual_clip, "kl_weight": kl_weight, "entropy_weight": entropy_weight,
        "reduction": reduction})
    _begin("pretrain_policy_loss")
    if log_probs.numel() == 0:
        loss = _nothing(log_probs, log_probs.shape if reduction == "none" else (), entropy)
        return (loss, torch.zeros(4, device=log_probs.device)) if metrics else loss

    def launch(x, h, slopes):
        return C.native().policy_loss_forward(
            x, old_log_probs, advantages, reference_log_probs, h, mask, cu_seqlens, clip_low,
            clip_high, dual, kl_weight, entropy_weight, POLICY_REDUCTIONS[reduction], bool(metrics),
            slopes)

    got = _PolicyLoss.apply(log_probs, entropy, mask, cu_seqlens, float(entropy_weight),
                            POLICY_REDUCTIONS[reduction], launch)
    return got if metrics else got[0]


def pretrain_preference_loss(
    log_probs: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    reference_log_probs: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    beta: float = 0.1,
    margin: float = 0.0,
    label_smoothing: float = 0.0,
    kind: str = "sigmoid",
    normalize: bool = False,
    reduction: str = "mean",
) -> tuple[torch.Tensor, torch.Tensor]:
    """Preference loss of pairs of answers from their tokens' log probabilities.

    ``cu_seqlens`` ``[2 pairs + 1]``: sequence 2p is the chosen answer of pair p,
    2p + 1 the rejected one. With s the sum over a sequence's tokens of ``log_probs -
    reference_log_probs`` (0 without a reference; their mean with ``normalize``) and
    ``m = beta (s_chosen - s_rejected) - margin`` a pair's loss is, by ``kind``,

        "sigmoid"  -(1 - label_smoothing) log sigmoid(m) - label_smoothing log sigmoid(-m)
        "hinge"    max(0, 1 - m)
        "squared"  ((m - 1/2) / beta)^2

    Pairs of which one side has no token that takes part do not count (loss 0).
    Returns the fp32 loss (their mean, 0 without any; their sum; or ``[pairs]``) and the
    rewards ``beta s`` ``[pairs, 2]`` without gradients. Gradients for log_probs; the
    reference must not require any.
    """
    call = C.whole_call("preference_loss_call")
    if (call and isinstance(reduction, str) and reduction in PAIR_REDUCTIONS
            and isinstance(kind, str) and kind in KINDS
            and (kind == "sigmoid" or label_smoothing == 0)):
        got = call(log_probs, cu_seqlens, reference_log_probs, mask, beta, margin,
                   label_smoothing, KINDS[kind], bool(normalize), PAIR_REDUCTIONS[reduction])
        if got is not None:
            return got
    C.enforce(PREFERENCE, {
        "log_probs": log_probs, "cu_seqlens": cu_seqlens,
        "reference_log_probs": reference_log_probs, "mask": mask, "beta": beta,
        "margin": margin, "label_smoothing": label_smoothing, "kind": kind,
        "reduction": reduction})
    _begin("pretrain_preference_loss")
    if log_probs.numel() == 0:
        pairs = cu_seqlens.numel() // 2
        loss = _nothing(log_probs, (pairs,) if reduction == "none" else ())
        return loss, torch.zeros(pairs, 2, device=log_probs.device)

    def launch(x):
        return C.native().preference_loss_forward(
            x, cu_seqlens, reference_log_probs, mask, beta, margin, label_smoothing, KINDS[kind],
            bool(normalize), PAIR_REDUCTIONS[reduction])

    return _PreferenceLoss.apply(log_probs, mask, cu_seqlens, PAIR_REDUCTIONS[reduction], launch)


__all__ = ["pretrain_policy_loss", "pretrain_preference_loss"]

"""Layer norm over the channels, with the residual add in front of it.

A block's norm reads the residual stream after the last branch was added to
it; here both are one pass: ``s = x + residual`` (rounded to the io dtype, the
stream as the model keeps it), ``y = (s - mean) / sqrt(var + eps) weight +
bias`` with the biased variance over the channels, all inside in fp32.

* :func:`infer_layer_norm_forward_varlen`: packed rows ``[total_tokens, C]``,
  no gradient, runs under HIP graph capture (decode).
* :func:`pretrain_layer_norm`: any leading shape, with autograd.

float32, float16 and bfloat16; any ``C`` up to 16384. ``C`` a multiple of 8 with
16-byte aligned tensors is the fastest; any other works. The weight's and bias'
gradients are summed over rows in a fixed order. The kernels are in
``csrc/layer_norm.hip``; the reference's normalization operators are not part
of this package, and these do not take their names.
"""

from __future__ import annotations

import torch

from .. import _contract as C
from .._contract import Each, check, is_tensor

MAX_CHANNELS = 16384
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _like_x(x, ns) -> bool:
    return x.dtype == ns["x"].dtype


_X = (
    is_tensor("x"),
    check("x", C.dtype_is(*_DTYPES), TypeError, "x must be float32, float16 or bfloat16"),
    check("x", C.cuda_contiguous, ValueError, "x must be CUDA and contiguous"),
)
_OTHERS = (
    check("x", lambda x, ns: x.shape[-1] <= MAX_CHANNELS, ValueError,
          f"x must have at most {MAX_CHANNELS} channels"),
    Each(("weight", "bias"), (
        is_tensor(),
        check(None, _like_x, TypeError, "{name} must have x's dtype"),
        check(None, C.cuda_contiguous, ValueError, "{name} must be CUDA and contiguous"),
        check(None, C.same_device_as("x"), ValueError, "{name} must share x's device"),
        check(None, lambda x, ns: x.shape == (ns["x"].shape[-1],), ValueError,
              "{name} must have shape [C]"),
    )),
    check("eps", lambda x, ns: C.finite_number(x, ns) and not isinstance(x, bool) and x >= 0,
          ValueError, "eps must be a finite number, not negative"),
)
_RESIDUAL = (
    is_tensor("residual"),
    check("residual", _like_x, TypeError, "residual must have x's dtype"),
    check("residual", C.cuda_contiguous, ValueError, "residual must be CUDA and contiguous"),
    check("residual", C.same_device_as("x"), ValueError, "residual must share x's device"),
    check("residual", C.same_shape_as("x"), ValueError, "residual must match x's shape"),
)

INFER = (*_X, check("x", C.packed_rows, ValueError, "x must have packed shape [total_tokens,C]"),
         *_OTHERS)
PRETRAIN = (*_X, check("x", lambda x, ns: x.ndim >= 1 and x.shape[-1] > 0, ValueError,
                       "x must have shape [...,C] with at least one channel"), *_OTHERS)


def _enforce(table, ns: dict) -> None:
    C.enforce(table, ns)
    if ns["residual"] is not None:
        C.enforce(_RESIDUAL, ns)


def infer_layer_norm_forward_varlen(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    *,
    residual: torch.Tensor | None = None,
    eps: float = 1e-5,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Layer norm of packed rows ``[total_tokens, C]``; with ``residual`` the
    norm of ``x + residual``. Returns ``y``, or ``(y, stream)`` with a residual."""
    if call := C.whole_call("layer_norm_infer_call"):
        out = call(x, residual, weight, bias, eps)
        if out is not None:
            return out
    ns = {"x": x, "weight": weight, "bias": bias, "residual": residual, "eps": eps}
    _enforce(INFER, ns)
    out = C.native().layer_norm_forward(x, residual, weight, bias, eps)
    return out[0] if residual is None else (out[0], out[1])


class _LayerNorm(torch.autograd.Function):
    """Calls that the native whole call declines (tensor subclasses, modes, empty
    rows). Forward keeps the rows that were normed (x itself without a residual)
    and their mean and rstd; backward is one pass over them and the ordered sum
    of the weight's and bias' gradients."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        ctx.set_materialize_grads(False)
        ctx.has_residual = residual is not None
        if x.numel() == 0:
            ctx.save_for_backward(x, weight)
            return (torch.empty_like(x), torch.empty_like(x)) if ctx.has_residual \
                else torch.empty_like(x)
        *out, mean, rstd = C.native().layer_norm_forward(x, residual, weight, bias, eps, True)
        ctx.save_for_backward(out[1] if ctx.has_residual else x, weight, mean, rstd)
        return tuple(out) if ctx.has_residual else out[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_stream=None):
        rows, weight, *statistics = ctx.saved_tensors
        if grad_y is None:
            # Nothing came back through y: the stream's gradient passes, the
            # parameters have none.
            return grad_stream, grad_stream if ctx.has_residual else None, None, None, None
        if rows.numel() == 0:
            grad_x, grad_weight, grad_bias = (torch.zeros_like(t) for t in (rows, weight, weight))
        else:
            grad_x, grad_weight, grad_bias = C.native().layer_norm_backward(
                grad_y.contiguous(), rows,
                None if grad_stream is None else grad_stream.contiguous(), weight, *statistics)
        need = ctx.needs_input_grad
        return (grad_x if need[0] else None, grad_x if ctx.has_residual and need[1] else None,
                grad_weight if need[2] else None, grad_bias if need[3] else None, None)


def pretrain_layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    *,
    residual: torch.Tensor | None = None,
    eps: float = 1e-5,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Layer norm over the last axis of ``x`` ``[..., C]`` with autograd. With
    ``residual`` it is the norm of ``stream = x + residual``, returned as
    ``(y, stream)``: the stream goes on to the next block, and its gradient
    joins the norm's in one pass. ``x`` and ``residual`` have the same gradient."""
    if call := C.whole_call("layer_norm_train_call"):
        out = call(x, residual, weight, bias, eps)
        if out is not None:
            return out
    ns = {"x": x, "weight": weight, "bias": bias, "residual": residual, "eps": eps}
    _enforce(PRETRAIN, ns)
    C.native()
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("pretrain_layer_norm does not run under HIP graph capture: training "
                           "steps are not validated inside a captured graph")
    return _LayerNorm.apply(x, residual, weight, bias, float(eps))


__all__ = ["infer_layer_norm_forward_varlen", "pretrain_layer_norm"]

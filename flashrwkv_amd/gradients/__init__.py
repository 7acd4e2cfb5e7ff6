"""The norm of all gradients of a step, and clipping by it.

* :func:`pretrain_grad_norm`: the norm of many tensors together.
* :func:`pretrain_clip_grad_norm`: the same, and the tensors scaled down to a
  largest norm, in place or into other tensors (bfloat16 gradients into the
  float32 ones that an optimizer with master weights takes).

float32, float16 and bfloat16 tensors in one list, of any shapes, of any order of
their dimensions in memory as long as they leave no gaps. Squares and their sums
are in 64 bits and in a fixed order. Nothing synchronises with the host, and both
run under HIP graph capture. The kernels are in ``csrc/grad_norm.hip``; the
reference has no counterpart.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from .. import _contract as C
from .._contract import check

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _dense(t):
    return torch.ops.aten.is_non_overlapping_and_dense(t)


def _each(ok):
    return lambda x, ns: all(ok(t, ns) for t in x)


def _list_of(name):
    return (
        check(name, lambda x, ns: isinstance(x, (list, tuple)) and len(x) > 0
              and all(isinstance(t, torch.Tensor) for t in x), TypeError,
              f"{name} must be a list or tuple of at least one torch.Tensor"),
        check(name, _each(lambda t, ns: t.dtype in _FLOATS), TypeError,
              f"{name} must be float32, float16 or bfloat16"),
        check(name, _each(lambda t, ns: t.is_cuda and t.layout == torch.strided), ValueError,
              f"{name} must be CUDA and strided"),
        check(name, _each(lambda t, ns: t.device == ns["tensors"][0].device), ValueError,
              f"{name} must share the first tensor's device"),
        check(name, _each(lambda t, ns: not t.is_neg()), ValueError,
              f"{name} must hold their values, not be negated views"),
        check(name, _each(lambda t, ns: _dense(t)), ValueError,
              f"{name} must leave no gaps in memory"),
        check(name, _each(C.constant), ValueError,
              f"{name} must not require gradients: the norm has none (detach them)"),
    )


def _pairwise(ok):
    return lambda x, ns: all(ok(a, b) for a, b in zip(x, ns["tensors"]))


def _apart(x, ns):
    """Whether no tensor that is written meets another one in memory."""
    ranges = [(t.data_ptr(), t.numel() * t.element_size(), True) for t in x]
    ranges += [(t.data_ptr(), t.numel() * t.element_size(), False)
               for t, y in zip(ns["tensors"], x) if t.data_ptr() != y.data_ptr()]
    written = seen = 0
    for start, size, writes in sorted(r for r in ranges if r[1] > 0):
        if start < written or (writes and start < seen):
            return False
        seen = max(seen, start + size)
        written = max(written, start + size) if writes else written
    return True


def _amount(x, ns):
    return C.finite_number(x, ns) and not isinstance(x, bool) and x >= 0


NORM = _list_of("tensors")

CLIP = (
    *NORM,
    *_list_of("out"),
    check("out", lambda x, ns: len(x) == len(ns["tensors"]), ValueError,
          "out must have one tensor for each of tensors"),
    check("out", _pairwise(lambda a, b: a.shape == b.shape and a.stride() == b.stride()),
          ValueError, "out must match tensors in shape and strides"),
    check("out", _pairwise(lambda a, b: a.data_ptr() != b.data_ptr() or a.dtype == b.dtype
                           or a.numel() == 0), ValueError,
          "a tensor that is written in place must keep its dtype"),
    check("out", _apart, ValueError, "tensors that are written must not overlap others"),
    check("max_norm", _amount, ValueError, "max_norm must be a finite number, not negative"),
    check("eps", _amount, ValueError, "eps must be a finite number, not negative"),
)


def pretrain_grad_norm(tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    """``sqrt(sum x^2)`` over all elements of all tensors, an fp32 scalar on their
    device, without gradients: the tensors must not require any. A tensor that is listed
    twice counts twice."""
    call = C.whole_call("grad_norm_call")
    norm = call(tensors) if call else None
    if norm is not None:
        return norm
    C.enforce(NORM, {"tensors": tensors})
    return C.native().grad_norm(tensors)


def pretrain_clip_grad_norm(
    tensors: Sequence[torch.Tensor],
    max_norm: float,
    *,
    out: Sequence[torch.Tensor] | None = None,
    eps: float = 1e-6,
) -> torch.Tensor:
    """Scales the tensors by ``min(1, max_norm / (norm + eps))``; returns their norm
    from before, an fp32 scalar on their device.

    In place, or with ``out`` into other tensors of the same shapes and strides
    and of dtypes of their own. The factor is rounded to 32 bits (below their normal
    numbers it keeps 64), its product with an element to 32 bits and then to the
    output's type. Where the norm is not finite nothing is scaled (``out`` takes the
    tensors as they are), so that a caller who looks at the norm can skip the step. A tensor that is written may be its own source but must not overlap
    any other tensor of the call, so none is scaled twice.
    """
    call = C.whole_call("clip_grad_norm_call")
    norm = call(tensors, out, max_norm, eps) if call else None
    if norm is not None:
        return norm
    targets = tensors if out is None else out
    C.enforce(CLIP, {"tensors": tensors, "out": targets, "max_norm": max_norm, "eps": eps})
    return C.native().clip_grad_norm(tensors, targets, max_norm, eps)


__all__ = ["pretrain_clip_grad_norm", "pretrain_grad_norm"]

"""CPU tests of the public layer of a policy or preference step's operators: names,
refusals before any launch, and the C ABI's argument errors."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import flashrwkv_amd
from flashrwkv_amd import capi
from flashrwkv_amd.gradients import pretrain_clip_grad_norm, pretrain_grad_norm
from flashrwkv_amd.loss import (
    pretrain_linear_log_probs,
    pretrain_policy_loss,
    pretrain_preference_loss,
)


def test_names_are_exported():
    for name in ("pretrain_linear_log_probs", "pretrain_policy_loss", "pretrain_preference_loss",
                 "pretrain_grad_norm", "pretrain_clip_grad_norm"):
        assert name in flashrwkv_amd.__all__ and callable(getattr(flashrwkv_amd, name))


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on the GPU: reaches the checks behind that one."""

    @property
    def is_cuda(self):
        return True


def _fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def test_log_probs_refusals():
    h, w = _fake(3, 64, dtype=torch.bfloat16), _fake(9, 64, dtype=torch.bfloat16)
    t = _fake(3, dtype=torch.int64)
    with pytest.raises(TypeError, match="hidden must be float16 or bfloat16"):
        pretrain_linear_log_probs(_fake(3, 64), w, t)
    with pytest.raises(ValueError, match="hidden must be CUDA and contiguous"):
        pretrain_linear_log_probs(torch.zeros(3, 64, dtype=torch.bfloat16), w, t)
    with pytest.raises(ValueError, match=r"weight must have shape \[V,C\]"):
        pretrain_linear_log_probs(h, _fake(9, 128, dtype=torch.bfloat16), t)
    with pytest.raises(TypeError, match="targets must be int32 or int64"):
        pretrain_linear_log_probs(h, w, _fake(3))
    with pytest.raises(ValueError, match="targets must have hidden's shape"):
        pretrain_linear_log_probs(h, w, _fake(4, dtype=torch.int64))
    for bad in (0.0, -1.0, math.nan, math.inf, "1", True):
        with pytest.raises(ValueError, match="temperature must be positive and finite"):
            pretrain_linear_log_probs(h, w, t, temperature=bad)
    with pytest.raises(TypeError, match="ignore_index must be an int"):
        pretrain_linear_log_probs(h, w, t, ignore_index=1.0)


def test_policy_refusals():
    x, cu = _fake(6), torch.tensor([0, 2, 6], dtype=torch.int32).as_subclass(_Cuda)

    def call(log_probs=x, old=x, advantages=x, **more):
        return pretrain_policy_loss(log_probs, old, advantages, **more)

    with pytest.raises(TypeError, match="log_probs must be a torch.Tensor"):
        call(log_probs=None)
    with pytest.raises(TypeError, match="log_probs must be float32, float16 or bfloat16"):
        call(log_probs=_fake(6, dtype=torch.float64))
    with pytest.raises(ValueError, match="old_log_probs must be CUDA and contiguous"):
        call(old=torch.zeros(6))
    with pytest.raises(ValueError, match="old_log_probs must match log_probs"):
        call(old=_fake(5))
    with pytest.raises(ValueError, match="old_log_probs must not require gradients"):
        call(old=_fake(6).requires_grad_())
    with pytest.raises(ValueError, match="advantages must match log_probs, or have one entry"):
        call(advantages=_fake(2))
    with pytest.raises(ValueError, match="advantages must match log_probs, or have one entry"):
        call(advantages=_fake(3), cu_seqlens=cu)
    with pytest.raises(ValueError, match="advantages must not require gradients"):
        call(advantages=_fake(6).requires_grad_())
    with pytest.raises(ValueError, match="reference_log_probs must not require gradients"):
        call(reference_log_probs=_fake(6).requires_grad_())
    with pytest.raises(ValueError, match="entropy must match log_probs"):
        call(entropy=_fake(6, 1))
    with pytest.raises(TypeError, match="mask must be bool or uint8"):
        call(mask=_fake(6, dtype=torch.int32))
    with pytest.raises(ValueError, match="mask must match log_probs"):
        call(mask=_fake(1, 6, dtype=torch.bool))
    with pytest.raises(TypeError, match="cu_seqlens must be int32"):
        call(cu_seqlens=cu.long())
    with pytest.raises(ValueError, match=r"cu_seqlens must have shape \[sequences \+ 1\]"):
        call(cu_seqlens=cu[:1])
    for bad in (-0.1, 1.1, math.nan, "0", True):
        with pytest.raises(ValueError, match="clip_low must be a number in"):
            call(clip_low=bad)
    for bad in (-0.1, math.inf, None):
        with pytest.raises(ValueError, match="clip_high must be a finite number"):
            call(clip_high=bad)
    for bad in (0, 0.0, 1.0, 0.5, math.nan, math.inf, "3"):
        with pytest.raises(ValueError, match="dual_clip must be None or a finite number above 1"):
            call(dual_clip=bad)
    with pytest.raises(ValueError, match="kl_weight must be a finite number"):
        call(kl_weight=math.inf)
    with pytest.raises(ValueError, match="kl_weight needs reference_log_probs"):
        call(kl_weight=0.1)
    with pytest.raises(ValueError, match="entropy_weight needs entropy"):
        call(entropy_weight=0.1)
    for bad in ("mean ", 1, None):
        with pytest.raises(ValueError, match="reduction must be one of"):
            call(reduction=bad)
    with pytest.raises(ValueError, match="'sequence_mean' needs cu_seqlens"):
        call(reduction="sequence_mean")


def test_preference_refusals():
    x, cu = _fake(6), torch.tensor([0, 2, 6], dtype=torch.int32).as_subclass(_Cuda)

    def call(log_probs=x, offsets=cu, **more):
        return pretrain_preference_loss(log_probs, offsets, **more)

    with pytest.raises(TypeError, match="cu_seqlens must be a torch.Tensor"):
        call(offsets=None)
    with pytest.raises(ValueError, match=r"cu_seqlens must have shape \[2 \* pairs \+ 1\]"):
        call(offsets=cu[:2])
    with pytest.raises(ValueError, match="reference_log_probs must match log_probs"):
        call(reference_log_probs=_fake(5))
    with pytest.raises(ValueError, match="reference_log_probs must not require gradients"):
        call(reference_log_probs=_fake(6).requires_grad_())
    for bad in (0.0, -0.1, math.nan, math.inf, True):
        with pytest.raises(ValueError, match="beta must be positive and finite"):
            call(beta=bad)
    with pytest.raises(ValueError, match="margin must be a finite number"):
        call(margin=math.nan)
    for bad in (-0.1, 0.6, "0"):
        with pytest.raises(ValueError, match="label_smoothing must be a number in"):
            call(label_smoothing=bad)
    with pytest.raises(ValueError, match="label_smoothing is of kind 'sigmoid' only"):
        call(label_smoothing=0.1, kind="hinge")
    with pytest.raises(ValueError, match="kind must be one of"):
        call(kind="logistic")
    with pytest.raises(ValueError, match="reduction must be one of"):
        call(reduction="sequence_mean")


def test_gradient_refusals():
    a = _fake(4)
    for bad in (None, [], a, [None], (a, 1)):
        with pytest.raises(TypeError, match="tensors must be a list or tuple"):
            pretrain_grad_norm(bad)
    with pytest.raises(TypeError, match="tensors must be float32, float16 or bfloat16"):
        pretrain_grad_norm([a, _fake(4, dtype=torch.int32)])
    with pytest.raises(ValueError, match="tensors must be CUDA and strided"):
        pretrain_grad_norm([torch.zeros(4)])
    with pytest.raises(ValueError, match="tensors must leave no gaps"):
        pretrain_grad_norm([_fake(8)[::2]])
    for bad in (-1.0, math.nan, math.inf, "1", True, None):
        with pytest.raises(ValueError, match="max_norm must be a finite number"):
            pretrain_clip_grad_norm([a], bad)
        with pytest.raises(ValueError, match="eps must be a finite number"):
            pretrain_clip_grad_norm([a], 1.0, eps=bad)
    with pytest.raises(ValueError, match="one tensor for each"):
        pretrain_clip_grad_norm([a], 1.0, out=[_fake(4), _fake(4)])
    with pytest.raises(ValueError, match="match tensors in shape and strides"):
        pretrain_clip_grad_norm([a], 1.0, out=[_fake(2, 2)])
    with pytest.raises(ValueError, match="must not require gradients"):
        pretrain_clip_grad_norm([_fake(4).requires_grad_()], 1.0)
    with pytest.raises(ValueError, match="tensors must not require gradients"):
        pretrain_grad_norm([a, _fake(4).requires_grad_()])
    with pytest.raises(ValueError, match="tensors must not require gradients"):
        pretrain_clip_grad_norm([_fake(4).requires_grad_()], 1.0, out=[a])
    with pytest.raises(ValueError, match="out must not require gradients"):
        pretrain_clip_grad_norm([a], 1.0, out=[_fake(4).requires_grad_()])
    flat = _fake(10)
    for tensors, out in (([a, a], None), ([flat[:6], flat[5:]], None), ([flat[:4]], [flat[2:6]]),
                         ([a, _fake(4)], [flat[:4]] * 2)):
        with pytest.raises(ValueError, match="must not overlap"):
            pretrain_clip_grad_norm(tensors, 1.0, out=out)
    with pytest.raises(ValueError, match="must keep its dtype"):
        half = a.view(torch.bfloat16)[:4]
        pretrain_clip_grad_norm([a], 1.0, out=[half])


def test_c_abi_refuses_before_any_launch():
    lib = capi.library()
    null, p = ctypes.c_void_p(), ctypes.c_void_p(0x1000)

    def error():
        return lib.frwkv_last_error().decode()

    def policy(tokens=4, sequences=0, cu=null, mask=null, x=p, old=p, a=p, per=0, low=0.2,
               high=0.2, dual=0.0, kl=0.0, reduction=1, loss=p, saved=p, bytes_=1 << 20):
        return lib.frwkv_policy_loss_forward(
            tokens, sequences, cu, mask, 0, x, 0, old, 0, a, per, 0, null, 0, null, low, high,
            dual, kl, 0.0, reduction, loss, null, 1, saved, bytes_, p, 1 << 20, null)

    for args, message in (({"tokens": 0}, "tokens must be in"), ({"tokens": 1 << 31}, "tokens must"),
                          ({"sequences": -1}, "sequences must be"), ({"x": null}, "log_probs is null"),
                          ({"sequences": 2}, "go together"), ({"cu": p}, "go together"),
                          ({"per": 1}, "cu_seqlens is null"), ({"reduction": 3}, "cu_seqlens is null"),
                          ({"reduction": 4}, "unknown reduction"), ({"low": 1.5}, "clip_low"),
                          ({"high": math.nan}, "clip_high"), ({"dual": 1.0}, "dual_clip"),
                          ({"kl": math.inf}, "finite"), ({"loss": null}, "loss is null"),
                          ({"bytes_": 8}, "saved of 8 bytes"),
                          ({"saved": ctypes.c_void_p(0x1008)}, "256-byte aligned")):
        assert policy(**args) != 0 and message in error(), (args, error())
    assert lib.frwkv_preference_loss_forward(4, 0, p, null, 0, p, 0, null, 0.1, 0.0, 0.0, 0, 0, 1,
                                             p, p, p, 1 << 20, p, 1 << 20, null) == 1
    assert lib.frwkv_preference_loss_forward(4, 1 << 62, p, null, 0, p, 0, null, 0.1, 0.0, 0.0, 0,
                                             0, 1, p, p, p, 1 << 20, p, 1 << 20, null) == 1
    assert lib.frwkv_preference_loss_forward(4, 1, p, null, 0, p, 0, null, 0.0, 0.0, 0.0, 0, 0, 1,
                                             p, p, p, 1 << 20, p, 1 << 20, null) == 1
    assert "beta" in error()
    assert lib.frwkv_policy_loss_backward(4, 0, null, null, 0.0, 1, null, p, 1 << 20, 0, p, 0,
                                          null, null) == 1 and "grad_loss" in error()
    assert lib.frwkv_linear_log_probs_backward(2, 1, 64, 5, p, 1.0, null, null, p, 1 << 20, p, p,
                                               p, 1 << 20, null) == 1
    assert lib.frwkv_linear_log_probs_forward(2, 1, 64, 5, p, p, 4, p, -100, 0.0, 1, p, null, p,
                                              1 << 20, p, 1 << 20, null) == 1
    assert "temperature" in error()


def test_byte_queries():
    lib = capi.library()
    assert lib.frwkv_policy_loss_saved_bytes(0, 0) == 0
    assert lib.frwkv_policy_loss_saved_bytes(1 << 31, 0) == 0
    assert lib.frwkv_policy_loss_saved_bytes(1000, 3) >= 4000 + 12
    assert lib.frwkv_preference_loss_saved_bytes(0) == 0
    assert lib.frwkv_preference_loss_saved_bytes(-(1 << 62)) == 0
    assert lib.frwkv_preference_loss_saved_bytes(1 << 62) == 0
    assert lib.frwkv_sequence_loss_workspace_bytes(1 << 20, 1 << 31) == 0
    rows = lib.frwkv_linear_log_probs_forward_workspace_bytes
    assert rows(100, 1000, 1) > rows(100, 1000, 0) > 0 and rows(0, 10, 1) == 0
    back = lib.frwkv_linear_log_probs_backward_workspace_bytes
    assert back(100, 64, 1000, 1, 1) > back(100, 64, 1000, 1, 0) > 0


def test_gradient_lists_through_the_c_abi():
    lib = capi.library()
    null, p = ctypes.c_void_p(), ctypes.c_void_p(0x1000)
    need = lib.frwkv_grad_norm_workspace_bytes(0, null)
    assert need >= 256

    def one(**fields):
        values = {"data": 0x1000, "out": 0x1000, "numel": 10, "dtype": 0, "out_dtype": 0, **fields}
        return (capi.Gradient * 1)(capi.Gradient(**values))

    for item, message in ((one(numel=-1), "elements"), (one(numel=1 << 41), "elements"),
                          (one(data=None), "is null"), (one(out=None), "is null"),
                          (one(dtype=7), "float32"), (one(out_dtype=3), "float32"),
                          (one(out_dtype=1), "two types")):
        assert lib.frwkv_grad_clip(1, item, 1.0, 0.0, p, p, 1 << 20, null) != 0
        assert message in lib.frwkv_last_error().decode()
    assert lib.frwkv_grad_norm(-1, null, p, p, 1 << 20, null) == 1
    assert lib.frwkv_grad_norm(1, null, p, p, 1 << 20, null) == 1
    assert lib.frwkv_grad_norm(1, one(), null, p, 1 << 20, null) == 1
    assert lib.frwkv_grad_norm(1, one(), p, p, 8, null) == 1
    assert lib.frwkv_grad_clip(1, one(), math.nan, 0.0, p, p, 1 << 20, null) == 1
    assert lib.frwkv_grad_clip(1, one(), 1.0, -1.0, p, p, 1 << 20, null) == 1

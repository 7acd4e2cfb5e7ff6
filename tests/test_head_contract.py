"""CPU tests of the training head's public layer: names, refusals before any
launch, and the C ABI's argument errors."""

from __future__ import annotations

import ctypes

import pytest
import torch

import flashrwkv_amd
from flashrwkv_amd import capi
from flashrwkv_amd.loss import pretrain_linear_cross_entropy, pretrain_linear_topk_distillation
from flashrwkv_amd.normalization import infer_layer_norm_forward_varlen, pretrain_layer_norm


def test_names_are_exported():
    for name in ("infer_layer_norm_forward_varlen", "pretrain_layer_norm",
                 "pretrain_linear_cross_entropy", "pretrain_linear_topk_distillation"):
        assert name in flashrwkv_amd.__all__ and callable(getattr(flashrwkv_amd, name))


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on the GPU: reaches the checks behind that one."""

    @property
    def is_cuda(self):
        return True


def _fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


@pytest.mark.parametrize("fn", [infer_layer_norm_forward_varlen, pretrain_layer_norm])
def test_layer_norm_refusals(fn):
    x, w = _fake(3, 8), _fake(8)
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        fn(None, w, w)
    with pytest.raises(TypeError, match="x must be float32, float16 or bfloat16"):
        fn(_fake(3, 8, dtype=torch.float64), w, w)
    with pytest.raises(ValueError, match="x must be CUDA and contiguous"):
        fn(torch.zeros(3, 8), w, w)
    with pytest.raises(ValueError, match="x must be CUDA and contiguous"):
        fn(_fake(8, 3).t(), w, w)
    with pytest.raises(ValueError, match="at most 16384 channels"):
        fn(_fake(1, 16385), w, w)
    with pytest.raises(TypeError, match="weight must have x's dtype"):
        fn(x, _fake(8, dtype=torch.float32), w)
    with pytest.raises(ValueError, match=r"bias must have shape \[C\]"):
        fn(x, w, _fake(9))
    for eps in (-1.0, float("nan"), "1", True):
        with pytest.raises(ValueError, match="eps must be a finite number"):
            fn(x, w, w, eps=eps)
    with pytest.raises(ValueError, match="residual must match x's shape"):
        fn(x, w, w, residual=_fake(8, 3))
    with pytest.raises(TypeError, match="residual must have x's dtype"):
        fn(x, w, w, residual=_fake(3, 8, dtype=torch.float16))


def test_packed_rows_are_asked_for_in_inference_only():
    w = _fake(8)
    with pytest.raises(ValueError, match="packed shape"):
        infer_layer_norm_forward_varlen(_fake(2, 3, 8), w, w)
    with pytest.raises(ValueError, match="packed shape"):
        infer_layer_norm_forward_varlen(_fake(0, 8), w, w)
    with pytest.raises(ValueError, match="at least one channel"):
        pretrain_layer_norm(_fake(3, 0), _fake(0), _fake(0))


def _ce(h, w, **kw):
    return pretrain_linear_cross_entropy(h, w, torch.zeros(3, dtype=torch.int64)
                                         .as_subclass(_Cuda), **kw)


def _distill(h, w, **kw):
    return pretrain_linear_topk_distillation(
        h, w, _fake(3, 5, dtype=torch.float32),
        torch.zeros(3, 5, dtype=torch.int64).as_subclass(_Cuda), **kw)


@pytest.mark.parametrize("fn", [_ce, _distill])
def test_head_refusals(fn):
    h, w = _fake(3, 64), _fake(10, 64)
    with pytest.raises(TypeError, match="hidden must be a torch.Tensor"):
        fn(None, w)
    with pytest.raises(TypeError, match="hidden must be float16 or bfloat16"):
        fn(_fake(3, 64, dtype=torch.float32), w)
    with pytest.raises(ValueError, match="hidden must be CUDA and contiguous"):
        fn(torch.zeros(3, 64).half(), w)
    for c in (0, 32, 100):
        with pytest.raises(ValueError, match="C a multiple of 64"):
            fn(_fake(3, c), _fake(10, c))
    with pytest.raises(TypeError, match="weight must have hidden's dtype"):
        fn(h, _fake(10, 64, dtype=torch.float16))
    with pytest.raises(ValueError, match="weight must be CUDA and contiguous"):
        fn(h, _fake(64, 10).t())
    for shape in ((10, 128), (0, 64), (64,)):
        with pytest.raises(ValueError, match=r"weight must have shape \[V,C\]"):
            fn(h, _fake(*shape))
    with pytest.raises(ValueError, match="reduction must be one of"):
        fn(h, w, reduction="max")


def test_target_refusals():
    h, w = _fake(3, 64), _fake(10, 64)

    def ce(targets, **kw):
        return pretrain_linear_cross_entropy(h, w, targets, **kw)

    with pytest.raises(TypeError, match="targets must be int32 or int64"):
        ce(_fake(3))
    with pytest.raises(ValueError, match="hidden's shape without the channels"):
        ce(_fake(4, dtype=torch.int64))
    with pytest.raises(TypeError, match="ignore_index must be an int"):
        ce(_fake(3, dtype=torch.int64), ignore_index=None)

    def kd(logits, indices, **kw):
        return pretrain_linear_topk_distillation(h, w, logits, indices, **kw)

    tokens = _fake(3, 4, dtype=torch.int64)
    with pytest.raises(TypeError, match="teacher_logits must be float32"):
        kd(tokens, tokens)
    with pytest.raises(ValueError, match="K at most 1024"):
        kd(_fake(3, 1025), _fake(3, 1025, dtype=torch.int64))
    with pytest.raises(ValueError, match="hidden's leading shape"):
        kd(_fake(2, 4), tokens)
    with pytest.raises(TypeError, match="teacher_indices must be int32 or int64"):
        kd(_fake(3, 4), _fake(3, 4))
    with pytest.raises(ValueError, match="teacher_indices must match teacher_logits"):
        kd(_fake(3, 4), _fake(3, 5, dtype=torch.int64))
    for t in (0.0, -1.0, float("inf"), float("nan"), None):
        with pytest.raises(ValueError, match="temperature must be positive and finite"):
            kd(_fake(3, 4), tokens, temperature=t)


def _last():
    return capi.library().frwkv_last_error()


def test_c_abi_rejects_bad_layer_norm_calls_without_a_gpu():
    lib = capi.library()
    null, p = ctypes.c_void_p(), ctypes.c_void_p(0x1000)
    assert lib.frwkv_layer_norm_forward(0, 1, 8, null, null, p, p, 1e-5, p, null, null, null,
                                        null) == 1
    assert b"null pointer" in _last()
    assert lib.frwkv_layer_norm_forward(0, 1, 8, p, p, p, p, 1e-5, p, null, null, null, null) == 1
    assert b"stream_out" in _last()
    for dtype, rows, c, eps, rc in ((7, 1, 8, 1e-5, 2), (0, 0, 8, 1e-5, 1), (0, 1, 16385, 1e-5, 2),
                                    (0, 1, 0, 1e-5, 2), (0, 1, 8, -1.0, 1)):
        assert lib.frwkv_layer_norm_forward(dtype, rows, c, p, null, p, p, eps, p, null, null,
                                            null, null) == rc
    assert lib.frwkv_layer_norm_backward_workspace_bytes(1, 100) == 800
    assert lib.frwkv_layer_norm_backward_workspace_bytes(0, 100) == 0
    assert lib.frwkv_layer_norm_backward(0, 1, 100, p, p, null, p, p, p, p, p, p, p, 799,
                                         null) == 1
    assert b"workspace of 799 bytes given, 800 needed" in _last()


def test_c_abi_rejects_bad_loss_calls_without_a_gpu():
    lib = capi.library()
    null, p = ctypes.c_void_p(), ctypes.c_void_p(0x1000)
    n, c, v = 300, 128, 1000
    saved = lib.frwkv_linear_loss_saved_bytes(n, c, 1)
    work = lib.frwkv_linear_loss_forward_workspace_bytes(n, v)
    back = lib.frwkv_linear_loss_backward_workspace_bytes(n, c, v, 1)
    assert saved >= 512 * c * 2 and work >= 4 * 512 * 8 and back >= 512 * 1024 * 2 + n * c * 4
    assert lib.frwkv_linear_loss_backward_workspace_bytes(n, c, v, 0) < back
    assert lib.frwkv_linear_loss_saved_bytes(0, c, 1) == 0
    assert lib.frwkv_linear_loss_saved_bytes(n, c, 1025) == 0
    assert lib.frwkv_linear_loss_forward_workspace_bytes(n, 2 ** 40) == 0
    assert lib.frwkv_linear_loss_backward_workspace_bytes(n, c, 2 ** 62, 1) == 0
    assert lib.frwkv_linear_loss_backward_workspace_bytes(2 ** 40, c, v, 1) == 0

    def forward(dtype=2, n=n, c=c, v=v, hidden=p, bytes_=8, reduction=1, saved_=saved,
                work_=work):
        return lib.frwkv_linear_cross_entropy_forward(dtype, n, c, v, hidden, p, bytes_, p, -100,
                                                      reduction, p, p, saved_, p, work_, null)

    for kw, rc, message in (
            ({"hidden": null}, 1, b"null pointer"), ({"dtype": 0}, 2, b"io dtype"),
            ({"c": 100}, 2, b"multiple of 64"), ({"n": 0}, 1, b"rows must be"),
            ({"n": 1 << 24}, 1, b"rows must be"), ({"n": 1 << 22, "v": 1 << 24}, 2, b"too large"),
            ({"v": 0}, 1, b"vocabulary"), ({"reduction": 3}, 1, b"unknown reduction"),
            ({"hidden": ctypes.c_void_p(0x1008)}, 1, b"16-byte aligned"),
            ({"saved_": saved - 1}, 1, b"saved of"), ({"work_": work - 1}, 1, b"workspace of"),
            ({"bytes_": 2}, 1, b"targets must be int32 or int64")):
        assert forward(**kw) == rc, kw
        assert message in _last(), kw

    def distill(k=4, t=1.0, dtype=0, bytes_=8):
        size = lib.frwkv_linear_loss_saved_bytes(n, c, max(k, 1))
        return lib.frwkv_linear_topk_distillation_forward(2, n, c, v, k, p, p, dtype, p, bytes_,
                                                          p, t, 1, p, p, size, p, work, null)

    for kw, rc in (({"k": 0}, 2), ({"k": 1025}, 2), ({"t": 0.0}, 1), ({"t": float("nan")}, 1),
                   ({"dtype": 5}, 1), ({"bytes_": 3}, 1)):
        assert distill(**kw) == rc, kw
    assert lib.frwkv_linear_loss_backward(2, n, c, v, 1, null, 1.0, 1, p, p, saved, p, p, p, back,
                                          null) == 1
    assert lib.frwkv_linear_loss_backward(2, n, c, v, 1, p, 1.0, 1, p, p, saved, p, p, p,
                                          back - 1, null) == 1
    assert b"workspace of" in _last()


def test_byte_queries_count_tiles_beyond_32_bits_and_give_0_for_refused_products():
    lib = capi.library()
    n, v = 1 << 16, 1 << 27  # 2^31 tiles of 64 x 64, 2^29 of 128 x 128
    assert lib.frwkv_linear_loss_forward_workspace_bytes(n, v) == (v // 128) * n * 8 + n // 32 * 4
    assert lib.frwkv_linear_loss_forward_workspace_bytes(1 << 22, 1 << 24) == 0
    assert lib.frwkv_linear_loss_backward_workspace_bytes(1 << 22, 64, 1 << 24, 1) == 0
    assert lib.frwkv_linear_loss_backward_workspace_bytes(300, 100, 1000, 1) == 0
    assert lib.frwkv_linear_loss_saved_bytes(1 << 22, 64, 1024) == 0
    assert lib.frwkv_linear_loss_saved_bytes(300, 100, 1) == 0


@pytest.mark.parametrize("c,v", [(4096, 65536), (1024, 4096), (64, 300), (2560, 200003)])
def test_backward_workspace_grows_with_rows_and_not_with_their_square(c, v):
    """dz of a piece: 512 MB, or 256 columns of all rows where that is more; fp32 slabs
    of the hidden gradient: one, or one more than the splits of a piece (at most 16).
    Splits are for products that do not fill the GPU: not for many rows."""
    lib = capi.library()
    for n in (1, 100, 4000, 8192, 30000, 65536, 131072, 262144, 1 << 20, 1 << 23):
        pad = (n + 255) // 256 * 256
        dz = max(512 << 20, pad * 512)
        rows = pad * 4 + 4096
        without = lib.frwkv_linear_loss_backward_workspace_bytes(n, c, v, 0)
        slabs = lib.frwkv_linear_loss_backward_workspace_bytes(n, c, v, 1) - without
        assert 0 < without <= dz + rows
        assert n * c * 4 <= slabs <= 17 * n * c * 4 + 256
        if n >= 65536:
            assert slabs <= 4 * n * c * 4 + 256


def test_backward_workspace_is_less_than_the_logits_it_avoids():
    lib = capi.library()
    for n in (8192, 32768, 65536, 131072, 262144):
        assert lib.frwkv_linear_loss_backward_workspace_bytes(n, 4096, 65536, 1) < n * 65536 * 2


def test_backward_plan_is_a_host_query():
    columns, pieces, splits, tile_rows = capi.linear_loss_backward_plan(8192, 4096, 65536)
    assert columns % 256 == 0 and (pieces - 1) * columns < 65536 <= pieces * columns
    assert 1 <= splits <= 16 and tile_rows in (64, 128, 256)
    lib = capi.library()
    null = ctypes.c_void_p()
    assert lib.frwkv_linear_loss_backward_plan(1, 64, 1, null, null, null, null) == 1
    assert b"null pointer" in _last()
    x = [ctypes.byref(ctypes.c_int32()) for _ in range(4)]
    assert lib.frwkv_linear_loss_backward_plan(1, 100, 1, *x) == 2
    assert b"multiple of 64" in _last()

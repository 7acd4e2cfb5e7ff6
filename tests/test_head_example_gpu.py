"""The example that runs recurrence, norm and both head losses in one step, and
the same operators through the C ABI."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

import flashrwkv_amd
from flashrwkv_amd import capi

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.fixture(scope="module", autouse=True)
def _require_native():
    if flashrwkv_amd._C is None:
        pytest.fail("flashrwkv_amd native library is not built (no fallback exists)")


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "train_head.py"
    spec = importlib.util.spec_from_file_location("train_head", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("mode,share", [("full", 0.5), ("state", 0.995)])
def test_example_learns(mode, share):
    """Full training halves the loss in 60 steps; the state alone, which can only
    shift what 192 tokens start from, lowers it."""
    losses = _example().train(mode, steps=60)
    assert all(x == x for x in losses)
    assert losses[-1] < share * losses[0], (losses[0], losses[-1])


def test_example_step_matches_logits_written_out():
    """One step's loss and the head's gradient against the same model with its
    logits written out in 64 bits."""
    example = _example()
    torch.manual_seed(1)
    model = example.Model(300, 2).to(DEV)
    ids, targets, logits, tokens = example.synthetic(300, 96, 8, DEV)
    loss = example.step_loss(model, ids, targets, logits, tokens)
    loss.backward()
    with torch.no_grad():
        rows = model.hidden(ids).double()
    head = model.head.detach().double().requires_grad_()
    z = rows @ head.t()
    keep = targets != example.IGNORE
    p = torch.softmax(logits.double() / 2, 1)
    log_q = torch.log_softmax(z / 2, 1).gather(1, tokens)
    want = 0.5 * torch.nn.functional.cross_entropy(z[keep], targets[keep]) \
        + 0.5 * 4 * (p * (p.log() - log_q)).sum(1).mean()
    want.backward()
    assert loss.item() == pytest.approx(want.item(), rel=1e-4)
    off = (model.head.grad.double() - head.grad).norm() / head.grad.norm()
    assert off < 6e-3, off
    score = example.token_log_probs(model, ids, targets.clamp_min(0))
    assert score.shape == (96,) and (score < 0).all()


def test_layer_norm_through_the_c_abi():
    gen = torch.Generator().manual_seed(2)
    x, r, dy = (torch.randn(33, 200, generator=gen).bfloat16().to(DEV) for _ in range(3))
    w, b = (torch.randn(200, generator=gen).bfloat16().to(DEV) for _ in range(2))
    y, stream = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(33, device=DEV), torch.empty(33, device=DEV)
    capi.layer_norm_forward(x, w, b, residual=r, eps=1e-5, y=y, stream_out=stream, mean=mean,
                            rstd=rstd)
    grads = [torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)]
    capi.layer_norm_backward(dy, stream, w, mean, rstd, grad_stream=None, grads=grads)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want, want_stream = flashrwkv_amd.pretrain_layer_norm(*leaves, residual=r)
    assert torch.equal(y, want) and torch.equal(stream, want_stream)
    for a, e in zip(grads, torch.autograd.grad(want, leaves, dy)):
        assert torch.equal(a, e)


def test_losses_through_the_c_abi():
    gen = torch.Generator().manual_seed(3)
    h = torch.randn(70, 128, generator=gen).half().to(DEV).requires_grad_()
    w = (torch.randn(500, 128, generator=gen) * 0.2).half().to(DEV).requires_grad_()
    targets = torch.randint(500, (70,), generator=gen).to(DEV)
    logits = torch.randn(70, 5, generator=gen).to(DEV)
    tokens = torch.randint(500, (70, 5), generator=gen, dtype=torch.int32).to(DEV)
    one = torch.ones((), device=DEV)
    loss, saved = torch.empty(1, device=DEV), None
    for kind in ("cross entropy", "distillation"):
        if kind == "cross entropy":
            saved = capi.linear_cross_entropy_forward(h, w, targets, reduction="sum", loss=loss)
            want = flashrwkv_amd.pretrain_linear_cross_entropy(h, w, targets, reduction="sum")
            extra = {"top": 1, "temperature": 1.0}
        else:
            saved = capi.linear_topk_distillation_forward(h, w, logits, tokens, temperature=2.0,
                                                          reduction="sum", loss=loss)
            want = flashrwkv_amd.pretrain_linear_topk_distillation(
                h, w, logits, tokens, temperature=2.0, reduction="sum")
            extra = {"top": 5, "temperature": 2.0}
        dh, dw = torch.empty_like(h), torch.empty_like(w)
        capi.linear_loss_backward(one, w, saved, rows=70, reduction="sum", grad_hidden=dh,
                                  grad_weight=dw, **extra)
        want_dh, want_dw = torch.autograd.grad(want, [h, w], one)
        assert torch.equal(loss[0], want) and torch.equal(dh, want_dh) and torch.equal(dw, want_dw)


def test_example_scores_with_the_whole_model():
    """token_log_probs against the model's logits written out in 64 bits, which
    come from the recurrence and not from the embedding alone."""
    example = _example()
    torch.manual_seed(3)
    model = example.Model(300, 2).to(DEV)
    ids, targets, _, _ = example.synthetic(300, 96, 8, DEV)
    targets = targets.clamp_min(0)
    with torch.no_grad():
        rows = model.hidden(ids)
    log_q = torch.log_softmax(rows.double() @ model.head.detach().double().t(), 1)
    want = log_q.gather(1, targets[:, None])[:, 0]
    got = example.token_log_probs(model, ids, targets)
    assert got.dtype == torch.float32 and not got.requires_grad
    torch.testing.assert_close(got.double(), want, rtol=0, atol=1e-4)

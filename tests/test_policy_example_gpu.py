"""The example that runs recurrence, norm, token scores, a sequence loss and gradient
clipping in one step: it runs, and its gradients are those of the same model with its
logits written out in 64 bits."""

from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import pytest
import torch

import flashrwkv_amd
from oracle import step

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.fixture(scope="module", autouse=True)
def _require_native():
    if flashrwkv_amd._C is None:
        pytest.fail("flashrwkv_amd native library is not built (no fallback exists)")


def _example(name="train_policy"):
    path = Path(__file__).resolve().parents[1] / "examples" / f"{name}.py"
    sys.path.insert(0, str(path.parent))
    try:
        spec = importlib.util.spec_from_file_location(name, path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    finally:
        sys.path.remove(str(path.parent))
    return module


@pytest.mark.parametrize("loss", ["policy", "preference"])
@pytest.mark.parametrize("mode", ["full", "state"])
def test_example_runs(loss, mode):
    seen = _example().train(loss, mode, steps=3, vocab=300, heads=2, answers=6)
    assert len(seen) == 3
    assert all(math.isfinite(x) and math.isfinite(norm) and norm > 0 for x, norm in seen)


@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_example_step_matches_logits_written_out(loss):
    """The head's gradient and that of the hidden rows from the written-out step, which
    the bf16 logit gradients (one rounding, 2^-8) and the outputs' rounding (2^-8) may move: 2^-7
    of the sum of absolute terms, and 2^-7 of the value."""
    example = _example()
    torch.manual_seed(1)
    model = example.Model(300, 2).to(DEV)
    batch = example.synthetic(model, 300, 6, DEV)
    # A policy that has moved: some ratios are clipped.
    batch["old"] = batch["old"] + 0.3 * torch.randn_like(batch["old"])
    rows = example.hidden_rows(model, batch["ids"], batch["cu_seqlens"]).detach()
    rows.requires_grad_()
    log_probs, entropy = flashrwkv_amd.pretrain_linear_log_probs(
        rows, model.head, batch["next"], temperature=example.TEMPERATURE, entropy=True)
    hidden_rows = example.hidden_rows
    example.hidden_rows = lambda *_: rows
    try:
        value = example.step_loss(model, batch, loss)
    finally:
        example.hidden_rows = hidden_rows
    d_rows, d_head = torch.autograd.grad(value, [rows, model.head])

    ref = step.scores(rows.detach(), model.head.detach(), batch["next"],
                      temperature=example.TEMPERATURE)
    torch.testing.assert_close(log_probs.double(), ref["log_probs"], rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(entropy.double(), ref["entropy"], rtol=1e-5, atol=1e-5)
    if loss == "policy":
        want = step.policy(log_probs, batch["old"], batch["advantages"],
                           reference=batch["reference"], entropy=entropy, mask=batch["answer"],
                           cu_seqlens=batch["cu_seqlens"], clip_low=0.2, clip_high=0.28,
                           kl_weight=0.02, entropy_weight=1e-3, reduction="sequence_mean")
        ups = (want["dlog_probs"].to(DEV), want["dentropy"].to(DEV))
    else:
        want = step.preference(log_probs, batch["cu_seqlens"], reference=batch["reference"],
                               mask=batch["answer"], beta=0.1)
        ups = (want["dlog_probs"].to(DEV), None)
    assert value.item() == pytest.approx(float(want["loss"]), rel=1e-5, abs=1e-6)
    ref = step.scores(rows.detach(), model.head.detach(), batch["next"],
                      temperature=example.TEMPERATURE, grad_log_probs=ups[0],
                      grad_entropy=ups[1])
    for got, name in ((d_rows, "dhidden"), (d_head, "dweight")):
        allowed = 2.0 ** -7 * (ref[f"abs_{name}"] + ref[name].abs()) + 1e-9
        assert ((got.double() - ref[name]).abs() <= allowed).all(), name
    assert d_head.any() and d_rows.any()


@pytest.mark.parametrize("mode", ["full", "state"])
def test_head_example_clips(mode):
    losses = _example("train_head").train(mode, steps=3, vocab=300, heads=2, tokens=64, top=4,
                                          max_norm=0.1)
    assert len(losses) == 3 and all(math.isfinite(x) for x in losses)


def test_head_example_gradients_are_scaled_to_the_norm():
    """Against the same gradients in 64 bits: the norm is rounded once (2^-24, twice allowed),
    a gradient by its factor, the product and its type (2 2^-24 and 2^-8)."""
    example = _example("train_head")
    torch.manual_seed(2)
    model = example.Model(300, 2).to(DEV)
    example.step_loss(model, *example.synthetic(300, 64, 4, DEV)).backward()
    grads = [p.grad for p in model.parameters()]
    assert len(grads) == 6 and {g.dtype for g in grads} == {torch.bfloat16, torch.float32}
    before = [g.clone() for g in grads]
    most = 0.5 * step.clip(before, 1.0, 0.0)[0]
    norm = flashrwkv_amd.pretrain_clip_grad_norm(grads, most)
    want, clipped = step.clip(before, most, 1e-6)
    assert abs(norm.item() - want) <= 2 ** -23 * want
    for got, value in zip(grads, clipped):
        off = 2.0 ** -23 + (2.0 ** -8 if got.dtype == torch.bfloat16 else 0.0)
        assert ((got.double() - value).abs() <= 1.01 * off * value.abs() + 2.0 ** -134).all()

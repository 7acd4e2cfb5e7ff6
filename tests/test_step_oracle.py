"""CPU pins of oracle/step.py: torch's 64-bit functions and autograd, hand-worked
cases and central differences."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import step


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(*shape, seed=0):
    return torch.randn(*shape, generator=_gen(seed), dtype=torch.float64)


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_scores_are_torch_s_distribution(temperature):
    h = _randn(9, 5, seed=1).requires_grad_()
    w = _randn(13, 5, seed=2).requires_grad_()
    targets = torch.tensor([3, -100, 0, 12, 5, 5, -100, 7, 1])
    g, e = _randn(9, seed=3), _randn(9, seed=4)
    got = step.scores(h.detach(), w.detach(), targets, temperature=temperature, grad_log_probs=g,
                      grad_entropy=e)
    q = torch.distributions.Categorical(logits=h @ w.t() / temperature)
    part = targets != -100
    log_probs = torch.where(part, q.log_prob(targets.clamp_min(0)), 0.0)
    entropy = torch.where(part, q.entropy(), 0.0)
    torch.testing.assert_close(got["log_probs"], log_probs.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(got["entropy"], entropy.detach(), rtol=1e-12, atol=1e-12)
    dh, dw = torch.autograd.grad((log_probs * g + entropy * e).sum(), [h, w])
    torch.testing.assert_close(got["dhidden"], dh, rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(got["dweight"], dw, rtol=1e-10, atol=1e-12)


def _policy_args(seed=0):
    n = 60
    x = -torch.rand(n, generator=_gen(seed), dtype=torch.float64) * 2
    return x, x + 0.4 * _randn(n, seed=seed + 1), _randn(4, seed=seed + 2), {
        "reference": x + 0.5 * _randn(n, seed=seed + 3),
        "entropy": torch.rand(n, generator=_gen(seed + 4), dtype=torch.float64),
        "mask": torch.rand(n, generator=_gen(seed + 5)) < 0.7,
        "cu_seqlens": torch.tensor([0, 20, 20, 53, 57]), "clip_low": 0.2, "clip_high": 0.3,
        "dual_clip": 1.5, "kl_weight": 0.4, "entropy_weight": 0.1}


@pytest.mark.parametrize("reduction", ["none", "mean", "sum", "sequence_mean"])
def test_policy_gradients_are_differences(reduction):
    x, old, a, args = _policy_args()
    up = _randn(60, seed=9) if reduction == "none" else torch.tensor(0.7, dtype=torch.float64)
    got = step.policy(x, old, a, reduction=reduction, upstream=up, **args)

    def total(y, entropy):
        out = step.policy(y, old, a, reduction=reduction, **{**args, "entropy": entropy})
        return float((out["loss"] * up).sum())

    for i in range(60):
        bump = torch.zeros(60, dtype=torch.float64)
        bump[i] = 1e-6
        slope = (total(x + bump, args["entropy"]) - total(x - bump, args["entropy"])) / 2e-6
        assert slope == pytest.approx(float(got["dlog_probs"][i]), abs=1e-7)
        slope = (total(x, args["entropy"] + bump) - total(x, args["entropy"] - bump)) / 2e-6
        assert slope == pytest.approx(float(got["dentropy"][i]), abs=1e-7)


def test_policy_by_hand():
    """r = 2, 1/2 and 1 with advantages 1, -1 and 3; low 0.2, high 0.5."""
    x = torch.log(torch.tensor([2.0, 0.5, 1.0], dtype=torch.float64))
    old, a = torch.zeros(3, dtype=torch.float64), torch.tensor([1.0, -1.0, 3.0])
    got = step.policy(x, old, a, clip_low=0.2, clip_high=0.5, reduction="none")
    assert got["loss"].tolist() == pytest.approx([-1.5, 0.8, -3.0])
    assert got["dlog_probs"].tolist() == pytest.approx([0.0, 0.0, -3.0])
    assert got["metrics"][:2].tolist() == pytest.approx([3.5 / 3, 2 / 3])
    got = step.policy(x[:1], old[:1], -a[:1], dual_clip=1.5, reduction="none")
    assert got["loss"].tolist() == pytest.approx([1.5])
    got = step.policy(x, old, a, mask=torch.tensor([1, 0, 1]), clip_high=0.5, reduction="mean")
    assert float(got["loss"]) == pytest.approx(-2.25)
    got = step.policy(x, old, a, cu_seqlens=torch.tensor([0, 2, 2, 3]), clip_low=0.2,
                      clip_high=0.5, reduction="sequence_mean")
    assert float(got["loss"]) == pytest.approx((-0.35 - 3.0) / 2)


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("normalize", [False, True])
def test_preference_gradients_are_differences(kind, reduction, normalize):
    x, reference = -_randn(40, seed=1).abs(), -_randn(40, seed=2).abs()
    cu = torch.tensor([0, 11, 20, 20, 25, 31, 38])
    args = {"reference": reference, "mask": torch.rand(40, generator=_gen(3)) < 0.8, "beta": 0.3,
            "margin": 0.2, "kind": kind, "normalize": normalize, "reduction": reduction,
            "label_smoothing": 0.1 if kind == "sigmoid" else 0.0}
    up = _randn(3, seed=4) if reduction == "none" else torch.tensor(0.7, dtype=torch.float64)
    got = step.preference(x, cu, upstream=up, **args)
    assert got["part"].tolist() == [True, False, True]
    for i in range(40):
        bump = torch.zeros(40, dtype=torch.float64)
        bump[i] = 1e-6
        high, low = (float((step.preference(y, cu, **args)["loss"] * up).sum())
                     for y in (x + bump, x - bump))
        assert (high - low) / 2e-6 == pytest.approx(float(got["dlog_probs"][i]), abs=1e-6)


def test_preference_by_hand():
    x = torch.tensor([-1.0, -2.0, -4.0], dtype=torch.float64)
    got = step.preference(x, torch.tensor([0, 2, 3]), beta=0.5)
    assert got["rewards"].tolist() == [[-1.5, -2.0]]
    assert float(got["loss"]) == pytest.approx(math.log(1 + math.exp(-0.5)))
    got = step.preference(x, torch.tensor([0, 2, 3]), beta=0.5, kind="hinge", margin=0.25)
    assert float(got["loss"]) == pytest.approx(0.75)
    got = step.preference(x, torch.tensor([0, 2, 3]), beta=0.5, kind="squared", normalize=True)
    assert float(got["loss"]) == pytest.approx(((0.5 * 2.5 - 0.5) / 0.5) ** 2)


def test_clip_by_hand():
    tensors = [torch.tensor([3.0, 0.0]), torch.tensor([[4.0]])]
    norm, out = step.clip(tensors, 1.0, 0.0)
    assert norm == 5.0 and out[0].tolist() == pytest.approx([0.6, 0.0])
    assert step.clip(tensors, 6.0, 0.0)[1][1].tolist() == [[4.0]]
    assert step.clip([torch.tensor([math.inf])], 1.0, 0.0)[1][0].tolist() == [math.inf]

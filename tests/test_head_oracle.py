"""The 64-bit layer norm and head losses of oracle/head.py, pinned on the CPU by
loops, hand-worked cases, central differences and torch's own 64-bit functions."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import head


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed),
                       dtype=torch.float64)


def _differences(loss, leaf, eps=1e-6):
    grad = torch.zeros_like(leaf)
    flat, out = leaf.view(-1), grad.view(-1)
    for i in range(flat.numel()):
        keep = flat[i].item()
        flat[i] = keep + eps
        plus = loss()
        flat[i] = keep - eps
        out[i] = (plus - loss()) / (2 * eps)
        flat[i] = keep
    return grad


def test_layer_norm_matches_loops_and_torch():
    x, w, b = _rand(3, 5, seed=1), _rand(5, seed=2), _rand(5, seed=3)
    got = head.layer_norm(x, w, b, 1e-3)
    for i in range(3):
        m = sum(x[i].tolist()) / 5
        var = sum((v - m) ** 2 for v in x[i].tolist()) / 5
        for c in range(5):
            want = (x[i, c].item() - m) / math.sqrt(var + 1e-3) * w[c].item() + b[c].item()
            assert got["y"][i, c].item() == pytest.approx(want, rel=1e-13)
    torch.testing.assert_close(got["y"], torch.nn.functional.layer_norm(x, (5,), w, b, 1e-3),
                               rtol=1e-12, atol=1e-12)


def test_layer_norm_gradients_match_central_differences():
    x, w, b = _rand(3, 4, seed=4), _rand(4, seed=5), _rand(4, seed=6)
    dy, ds = _rand(3, 4, seed=7), _rand(3, 4, seed=8)
    got = head.layer_norm(x, w, b, 1e-5, dy, ds)

    def loss():
        return ((head.layer_norm(x, w, b, 1e-5)["y"] * dy).sum() + (x * ds).sum()).item()

    for name, leaf in (("dx", x), ("dweight", w), ("dbias", b)):
        torch.testing.assert_close(got[name], _differences(loss, leaf), rtol=1e-5, atol=1e-7)


def test_cross_entropy_matches_torch_and_leaves_ignored_rows_out():
    h, w = _rand(6, 4, seed=9), _rand(7, 4, seed=10)
    targets = torch.tensor([3, -100, 0, 6, -100, 2])
    h[1] = math.nan
    entry = head.labels(targets, 7, -100)
    got = head.head_loss(h, w, *entry, row_weight=torch.ones(6), mean=True)
    keep = targets != -100
    logits = (h[keep] @ w.t()).requires_grad_()
    want = torch.nn.functional.cross_entropy(logits, targets[keep], reduction="none")
    torch.testing.assert_close(got["loss"][keep], want.detach(), rtol=1e-12, atol=1e-12)
    assert (got["loss"][~keep] == 0).all() and (got["dhidden"][~keep] == 0).all()
    grad, = torch.autograd.grad(want.mean(), logits)
    torch.testing.assert_close(got["dz"], grad, rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(got["dweight"], grad.t() @ h[keep], rtol=1e-10, atol=1e-12)


def test_uniform_logits_give_log_vocab_and_hand_worked_gradient():
    h, w = torch.zeros(1, 2, dtype=torch.float64), _rand(5, 2, seed=11)
    got = head.head_loss(h, w, *head.labels(torch.tensor([4]), 5, -100),
                         row_weight=torch.ones(1))
    assert got["loss"].item() == pytest.approx(math.log(5), rel=1e-14)
    assert got["dz"].tolist()[0] == pytest.approx([0.2, 0.2, 0.2, 0.2, -0.8], rel=1e-14)


def test_teacher_shares_present_entries_only():
    logits = torch.tensor([[1.0, 3.0, 0.0, -math.inf], [5.0, 1.0, 1.0, 1.0],
                           [-math.inf, 0.0, 0.0, 0.0]])
    indices = torch.tensor([[2, 5, -1, 4], [-1, -1, -1, -1], [3, -1, -1, -1]])
    index, p, present = head.teacher(logits, indices, 2.0)
    e = math.exp(0.5) + math.exp(1.5)
    assert p[0].tolist() == pytest.approx([math.exp(0.5) / e, math.exp(1.5) / e, 0, 0])
    assert present.tolist() == [[True, True, False, False], [False] * 4, [False] * 4]
    assert not p[1:].any() and (index[~present] == 0).all()


def test_distillation_is_the_divergence_and_zero_at_the_teacher():
    """Against torch's kl_div over the scattered teacher, and 0 with zero
    gradient where the teacher lists the student's own logits."""
    h, w, t = _rand(3, 4, seed=12), _rand(6, 4, seed=13), 1.7
    indices = torch.tensor([[0, 3, 5], [1, 2, -1], [4, 0, 2]])
    logits = _rand(3, 3, seed=14)
    entry = head.teacher(logits, indices, t)
    got = head.head_loss(h, w, *entry, temperature=t)
    dense = torch.zeros(3, 6, dtype=torch.float64).scatter_add(1, entry[0], entry[1])
    log_q = torch.log_softmax(h @ w.t() / t, 1)
    want = torch.nn.functional.kl_div(log_q, dense, reduction="none").sum(1) * t * t
    torch.testing.assert_close(got["loss"], want, rtol=1e-12, atol=1e-12)
    every = torch.arange(6).expand(3, 6)
    same = head.head_loss(h, w, *head.teacher(h @ w.t(), every, t), temperature=t,
                          row_weight=torch.ones(3))
    assert same["loss"].abs().max() < 1e-14 and same["dz"].abs().max() < 1e-14


@pytest.mark.parametrize("mean", [False, True])
def test_head_loss_gradients_match_central_differences(mean):
    h, w, t = _rand(3, 3, seed=15), _rand(5, 3, seed=16), 1.3
    entry = head.teacher(_rand(3, 2, seed=17), torch.tensor([[0, 2], [-1, -1], [4, 4]]), t)
    weights = torch.tensor([0.7, 2.0, -1.1], dtype=torch.float64)
    got = head.head_loss(h, w, *entry, temperature=t, row_weight=weights, mean=mean)

    def loss():
        total = (head.head_loss(h, w, *entry, temperature=t)["loss"] * weights).sum().item()
        return total / 2 if mean else total

    for name, leaf in (("dhidden", h), ("dweight", w)):
        torch.testing.assert_close(got[name], _differences(loss, leaf), rtol=1e-5, atol=1e-8)


def test_a_token_listed_four_times_hand_worked():
    """Entries are summed one by one in the loss, joined in the gradient: a uniform
    student over 5 tokens and a teacher with its four entries on one of them."""
    h, w = torch.zeros(1, 2, dtype=torch.float64), _rand(5, 2, seed=18)
    entry = head.teacher(torch.zeros(1, 4), torch.full((1, 4), 3), 2.0)
    got = head.head_loss(h, w, *entry, temperature=2.0, row_weight=torch.ones(1))
    assert got["loss"].item() == pytest.approx(4 * (math.log(5) - math.log(4)), rel=1e-14)
    assert got["dz"].tolist()[0] == pytest.approx([0.4, 0.4, 0.4, -1.6, 0.4], rel=1e-14)

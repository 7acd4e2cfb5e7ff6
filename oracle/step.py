"""Token scores, sequence losses and the gradient norm in 64 bits -- TEST
INFRASTRUCTURE ONLY.

Plain torch double from the definitions, one sequence after another: nothing
here knows tiles or pieces. Gradients are closed forms; tests/test_step_oracle.py
pins them by torch's 64-bit autograd and by central differences.
"""

from __future__ import annotations

import math

import torch


def scores(hidden, weight, targets, *, temperature=1.0, ignore_index=-100, grad_log_probs=None,
           grad_entropy=None):
    """Log probability of each row's target under softmax(h W^T / T) and the row's
    entropy; with upstream rows dh and dW, and the sums of absolute terms of both."""
    n, c = hidden.shape
    rows = (targets != ignore_index).nonzero()[:, 0]
    h, w, token = hidden.double()[rows], weight.double(), targets[rows].long()
    log_q = torch.log_softmax(h @ w.t() / temperature, 1)
    q = torch.exp(log_q)
    entropy = -(q * log_q).sum(1)

    def full(values, *shape):
        out = torch.zeros(n, *shape, dtype=torch.float64, device=hidden.device)
        out[rows] = values
        return out

    out = {"rows": rows, "log_probs": full(log_q.gather(1, token[:, None])[:, 0]),
           "entropy": full(entropy), "abs_entropy": full((q * log_q).abs().sum(1))}
    if grad_log_probs is None and grad_entropy is None:
        return out
    dz = torch.zeros_like(q)
    if grad_log_probs is not None:
        g = grad_log_probs.double()[rows, None] / temperature
        dz = dz - g * q
        dz.scatter_add_(1, token[:, None], g)
    if grad_entropy is not None:
        e = grad_entropy.double()[rows, None] / temperature
        dz = dz - e * q * (log_q + entropy[:, None])
    out |= {"dz": dz, "dhidden": full(dz @ w, c), "abs_dhidden": full(dz.abs() @ w.abs(), c),
            "dweight": dz.t() @ h, "abs_dweight": dz.abs().t() @ h.abs()}
    return out


def sequences(cu_seqlens, tokens):
    """[(first, end)] of each sequence, and the sequence of each token (-1: none)."""
    offsets = [0, tokens] if cu_seqlens is None else [int(x) for x in cu_seqlens]
    spans = list(zip(offsets[:-1], offsets[1:]))
    owner = torch.full((tokens,), -1, dtype=torch.int64)
    for b, (first, end) in enumerate(spans):
        owner[first:end] = b
    return spans, owner


def _k3(x):
    return torch.expm1(x) - x


def policy(log_probs, old, advantages, *, reference=None, entropy=None, mask=None,
           cu_seqlens=None, clip_low=0.2, clip_high=0.2, dual_clip=None, kl_weight=0.0,
           entropy_weight=0.0, reduction="mean", upstream=None):
    """Dict: loss, metrics, dlog_probs, dentropy; vectors flat."""
    x, old, a = (t.detach().cpu().double().flatten() for t in (log_probs, old, advantages))
    n = x.numel()
    spans, owner = sequences(None if cu_seqlens is None else cu_seqlens.cpu(), n)
    part = owner >= 0
    if mask is not None:
        part &= mask.cpu().flatten().bool()
    if a.numel() != n:
        a = a[owner.clamp_min(0)]
    keep = part.nonzero()[:, 0]
    x, old, a = x[keep], old[keep], a[keep]
    d = x - old
    r = torch.exp(d)
    first = r * a
    second = r.clamp(1 - clip_low, 1 + clip_high) * a
    each = -torch.minimum(first, second)
    cut = ((a > 0) & (d > math.log1p(clip_high))) | (
        (a < 0) & (d < (math.log1p(-clip_low) if clip_low < 1 else -math.inf)))
    if dual_clip is not None:
        each = torch.where(a < 0, torch.minimum(each, -dual_clip * a), each)
        cut = cut | ((a < 0) & (d > math.log(dual_clip)))
    slope = torch.where(cut, 0.0, -first)
    kl = torch.zeros_like(x)
    if reference is not None:
        t = reference.detach().cpu().double().flatten()[keep] - x
        kl = _k3(t)
        each = each + kl_weight * kl
        slope = slope - kl_weight * torch.expm1(t)
    if entropy is not None:
        each = each - entropy_weight * entropy.detach().cpu().double().flatten()[keep]
    count = max(1, keep.numel())
    share = torch.ones_like(x)
    if reduction == "mean":
        share = share / count
    elif reduction == "sequence_mean":
        counts = torch.bincount(owner[keep], minlength=len(spans)).double()
        share = 1.0 / counts[owner[keep]] / max(1, int((counts > 0).sum()))

    def full(values):
        out = torch.zeros(n, dtype=torch.float64)
        out[keep] = values
        return out

    out = {"each": full(each), "share": full(share), "part": part}
    out["loss"] = full(each) if reduction == "none" else (each * share).sum()
    means = [v.double().sum() / count for v in (r, cut, _k3(d), kl)]
    out["metrics"] = torch.stack(means)
    up = 1.0 if upstream is None else upstream.cpu().double().flatten()
    up = up[keep] if isinstance(up, torch.Tensor) and up.numel() == n else up
    out["dlog_probs"] = full(slope * share * up)
    out["dentropy"] = full(-entropy_weight * share * up)
    return out


def preference(log_probs, cu_seqlens, *, reference=None, mask=None, beta=0.1, margin=0.0,
               label_smoothing=0.0, kind="sigmoid", normalize=False, reduction="mean",
               upstream=None):
    """Dict: loss, rewards, dlog_probs; vectors flat."""
    x = log_probs.detach().cpu().double().flatten()
    n = x.numel()
    keep = torch.ones(n, dtype=torch.bool) if mask is None else mask.cpu().flatten().bool()
    ref = torch.zeros_like(x) if reference is None else reference.cpu().double().flatten()
    spans, _ = sequences(cu_seqlens.cpu(), n)
    pairs = len(spans) // 2
    rewards = torch.zeros(pairs, 2, dtype=torch.float64)
    counts = torch.zeros(pairs, 2, dtype=torch.int64)
    for b, (first, end) in enumerate(spans):
        here = keep[first:end]
        values = (x[first:end] - ref[first:end])[here]
        by = 1.0 / max(1, values.numel()) if normalize else 1.0
        rewards[b // 2, b % 2] = beta * values.sum() * by
        counts[b // 2, b % 2] = values.numel()
    part = (counts > 0).all(1)
    m = rewards[:, 0] - rewards[:, 1] - margin
    if kind == "sigmoid":
        log_sigmoid = torch.nn.functional.logsigmoid
        each = -(1 - label_smoothing) * log_sigmoid(m) - label_smoothing * log_sigmoid(-m)
        slope = label_smoothing * torch.sigmoid(m) - (1 - label_smoothing) * torch.sigmoid(-m)
    elif kind == "hinge":
        each = torch.relu(1 - m)
        slope = -(m < 1).double()
    else:
        each = ((m - 0.5) / beta) ** 2
        slope = 2 * (m - 0.5) / beta ** 2
    each, slope = (torch.where(part, t, 0.0) for t in (each, slope))
    share = 1.0 / max(1, int(part.sum())) if reduction == "mean" else 1.0
    up = torch.ones(pairs).double() if upstream is None else upstream.cpu().double()
    grad = torch.zeros(n, dtype=torch.float64)
    for b, (first, end) in enumerate(spans):
        p = b // 2
        by = 1.0 / max(1, int(counts[p, b % 2])) if normalize else 1.0
        value = slope[p] * beta * by * share * (up[p] if up.ndim else up)
        grad[first:end] = torch.where(keep[first:end], -value if b % 2 else value, 0.0)
    return {"each": each, "loss": each if reduction == "none" else each.sum() * share,
            "rewards": rewards, "m": m, "dlog_probs": grad, "part": part}


def clip(tensors, max_norm, eps):
    """(norm, [clipped]) of a list."""
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
    by = min(1.0, max_norm / (norm + eps)) if math.isfinite(norm) else 1.0
    return norm, [t.double() * by for t in tensors]

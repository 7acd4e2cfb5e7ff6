"""Layer norm and head losses in 64 bits -- TEST INFRASTRUCTURE ONLY.

Plain torch double, on whatever device the inputs are, from the definitions:
nothing here knows tiles, pieces or compaction. Beside each result that is a
sum stands the sum of its terms' absolute values, which is what a rounding
error bound of that sum is stated in.

Pinned in tests/test_head_oracle.py by explicit loops, hand-worked cases,
central differences and torch's own 64-bit log_softmax and layer_norm.
"""

from __future__ import annotations

import math

import torch


def layer_norm(x, weight, bias, eps, dy=None, ds=None):
    """x [N, C] (already the sum with a residual). Dict with y, mean, rstd; with
    dy also dx, dweight, dbias and the sums of absolute terms of the latter two."""
    x, weight, bias = x.double(), weight.double(), bias.double()
    c = x.shape[1]
    mean = x.sum(1, keepdim=True) / c
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).sum(1, keepdim=True) / c + eps)
    xhat = d * rstd
    out = {"y": xhat * weight + bias, "mean": mean[:, 0], "rstd": rstd[:, 0], "xhat": xhat}
    if dy is not None:
        dy = dy.double()
        g = dy * weight
        mg = g.sum(1, keepdim=True) / c
        mgx = (g * xhat).sum(1, keepdim=True) / c
        out["dx"] = rstd * (g - mg - xhat * mgx)
        if ds is not None:
            out["dx"] = out["dx"] + ds.double()
        out["dweight"], out["dbias"] = (dy * xhat).sum(0), dy.sum(0)
        out["abs_dweight"], out["abs_dbias"] = (dy * xhat).abs().sum(0), dy.abs().sum(0)
    return out


def labels(targets, vocab, ignore_index):
    """(index [N, 1], p [N, 1], present [N, 1]) of cross entropy targets."""
    present = (targets != ignore_index)[:, None]
    index = torch.where(present, targets[:, None].long(), 0)
    return index, present.double(), present


def teacher(logits, indices, temperature):
    """The same of a teacher's entries: softmax over the present ones."""
    x = logits.double() / temperature
    present = (indices >= 0) & (x > -math.inf)
    index = torch.where(present, indices.long(), 0)
    e = torch.where(present, x, -math.inf)
    top = torch.where(present.any(1, keepdim=True), e.amax(1, keepdim=True), 0.0)
    e = torch.exp(e - top)
    total = e.sum(1, keepdim=True)
    return index, e / torch.where(total > 0, total, 1.0), present


def head_loss(hidden, weight, index, p, present, *, temperature=1.0, row_weight=None,
              mean=False):
    """Row losses T^2 sum p (log p - log softmax(h W^T / T)) and, for upstream
    row weights, dh and dW with the sums of absolute terms. Rows without a
    present entry are taken out first."""
    n, vocab = hidden.shape[0], weight.shape[0]
    rows = present.any(1).nonzero()[:, 0]
    h, w = hidden.double()[rows], weight.double()
    index, p = index[rows], p[rows]
    z = h @ w.t()
    s = z / temperature
    top = s.amax(1, keepdim=True) if rows.numel() else s[:, :1]
    lse = torch.log(torch.exp(s - top).sum(1, keepdim=True)) + top
    log_p = torch.where(p > 0, torch.log(torch.where(p > 0, p, 1.0)), 0.0)
    terms = torch.where(p > 0, p * (log_p - (s.gather(1, index) - lse)), 0.0)
    loss = torch.zeros(n, dtype=torch.float64, device=hidden.device)
    loss[rows] = terms.sum(1) * temperature ** 2
    out = {"loss": loss, "rows": rows, "lse": lse[:, 0], "z": z}
    if row_weight is None:
        return out
    scale = row_weight.double()[rows, None] * temperature
    if mean:
        scale = scale / max(1, rows.numel())
    dz = torch.exp(s - lse)
    dz.scatter_add_(1, index, -p)
    dz = dz * scale
    out["dz"] = dz
    for name, value in (("dhidden", dz @ w), ("abs_dhidden", dz.abs() @ w.abs())):
        full = torch.zeros(n, h.shape[1], dtype=torch.float64, device=hidden.device)
        full[rows] = value
        out[name] = full
    out["dweight"] = dz.t() @ h
    out["abs_dweight"] = dz.abs().t() @ h.abs()
    return out

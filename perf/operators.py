"""Cases of the training head's operators: layer norm with the residual add,
softmax cross entropy over the vocabulary from the hidden rows, and
distillation from a teacher's top logits.

``own`` false computes them in plain torch operations in 32 bits, ``own`` true
with the entry points of ``flashrwkv_amd.normalization`` and
``flashrwkv_amd.loss``. ``exact`` restates them in 64 bits.

Definitions (rows i, channels c, vocabulary v; everything per row):

* norm: s = x + residual, rounded to the io type (the residual stream as a
  model keeps it; s = x without a residual); y = (s - mean) / sqrt(var + eps)
  weight + bias with the biased variance. Training gradients for upstream dy
  (and ds for the stream): x, residual (equal to x's), weight, bias.
* ce: z = hidden weight^T, loss = logsumexp(z) - z[target]; rows whose target
  is -100 take no part (loss 0, gradient 0, not counted by the mean).
* distill: p = softmax(teacher / T) over the row's entries with index >= 0,
  q = softmax(z / T) over the vocabulary, loss = T^2 sum p (log p - log q);
  rows without an entry take no part.
"""

import math

import torch

own = False

IGNORE = -100
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _norm(name, rows, channels, dtype, train, residual):
    return {"name": name, "op": "norm", "rows": rows, "channels": channels, "dtype": dtype,
            "train": train, "residual": residual}


def _ce(name, rows, channels, vocab, dtype, grads, reduction, masked):
    return {"name": name, "op": "ce", "rows": rows, "channels": channels, "vocab": vocab,
            "dtype": dtype, "grads": grads, "reduction": reduction, "masked": masked}


def _distill(name, rows, channels, vocab, top, dtype, grads, reduction, masked, temperature):
    return {"name": name, "op": "distill", "rows": rows, "channels": channels, "vocab": vocab,
            "top": top, "dtype": dtype, "grads": grads, "reduction": reduction,
            "masked": masked, "temperature": temperature}


def listed():
    return [
        # One decode step of one sequence (40 heads of 64): latency only.
        _norm("norm_decode_1", 1, 2560, "fp16", False, False),
        # One decode step of a full batch, with the block's residual add.
        _norm("norm_decode_256_residual", 256, 2560, "bf16", False, True),
        # A training block's norm with the residual add over 16k tokens.
        _norm("norm_train_16384_residual", 16384, 4096, "bf16", True, True),
        # fp32 rows of a width that is no power of two and a ragged row count.
        _norm("norm_train_odd", 2311, 1000, "fp32", True, False),
        # Scoring one token (per-token log probability of a serving loop).
        _ce("ce_score_1", 1, 2048, 65536, "bf16", "none", "none", 0.0),
        # Per-token losses of an evaluation batch.
        _ce("ce_score_1000", 1000, 2560, 50277, "fp16", "none", "none", 0.0),
        # A small fine-tuning step, odd sizes, a third of the rows prompt.
        _ce("ce_train_odd", 777, 768, 20011, "fp16", "both", "sum", 0.3),
        # Per-token weights from outside (policy gradient), hidden rows only:
        # the head is frozen while states or adapters are tuned.
        _ce("ce_frozen_weighted", 2048, 2560, 65536, "bf16", "hidden", "none", 0.25),
        # The head of a pretraining step.
        _ce("ce_train_8192", 8192, 4096, 65536, "bf16", "both", "mean", 0.0),
        # A short distillation step, odd sizes, ragged teacher lists.
        _distill("distill_train_odd", 333, 832, 20011, 20, "fp16", "both", "sum", 0.2, 1.0),
        # The head of a distillation step with the teacher's top 64.
        _distill("distill_train_4096", 4096, 2048, 65536, 64, "bf16", "both", "mean", 0.1, 2.0),
        # Distillation into states or adapters: the head is frozen.
        _distill("distill_frozen", 2048, 2560, 65536, 32, "bf16", "hidden", "mean", 0.0, 1.5),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _unnamed(case):
    return {key: value for key, value in case.items() if key != "name"}


def draw(rng):
    op = rng.choice(["norm", "ce", "distill"])
    if op == "norm":
        rows, channels = _log_uniform(rng, 1, 16384), _log_uniform(rng, 33, 8192)
        if rng.random() < 0.5:
            channels = 64 * max(1, channels // 64)
        rows = max(1, min(rows, 16384 * 4096 // channels))
        return _unnamed(_norm("", rows, channels, rng.choice(["bf16", "fp16", "fp32"]),
                              rng.random() < 0.7, rng.random() < 0.5))
    rows = _log_uniform(rng, 1, 8192)
    channels = 64 * _log_uniform(rng, 4, 64)
    vocab = _log_uniform(rng, 500, 65536)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    grads = rng.choice(["none", "hidden", "both", "both"])
    reduction = "none" if grads == "none" else rng.choice(["mean", "sum", "none"])
    if dtype == "fp16" and reduction == "mean":
        reduction = "sum"  # fp16 gradients of a mean come with loss scaling
    masked = rng.choice([0.0, 0.1, 0.5])
    if op == "ce":
        return _unnamed(_ce("", rows, channels, vocab, dtype, grads, reduction, masked))
    return _unnamed(_distill("", rows, channels, vocab, _log_uniform(rng, 1, 128), dtype, grads,
                             reduction, masked, rng.choice([1.0, 1.5, 2.0, 4.0])))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    dtype = DTYPES[case["dtype"]]
    n, c = case["rows"], case["channels"]
    state = {"case": case}
    if case["op"] == "norm":
        # A residual stream: a few wide channels, a mean that is not zero.
        scale = torch.exp(0.5 * randn(c))
        state["x"] = (randn(n, c) * scale + 0.3 * randn(n, 1)).to(dtype)
        state["weight"] = (1.0 + 0.2 * randn(c)).to(dtype)
        state["bias"] = (0.1 * randn(c)).to(dtype)
        if case["residual"]:
            state["residual"] = (0.5 * randn(n, c)).to(dtype)
        if case["train"]:
            state["dy"] = randn(n, c).to(dtype)
            if case["residual"]:
                state["ds"] = randn(n, c).to(dtype)
        return state
    v = case["vocab"]
    # Normalised hidden rows; logits of standard deviation about 2.5, the
    # right token up to about 9 above that.
    weight = (randn(v, c) * (2.5 / math.sqrt(c))).to(dtype)
    first = torch.randint(v, (n,), generator=gen, device="cuda")
    state["weight"] = weight
    state["hidden"] = (randn(n, c) + weight[first].float() * (1.5 * rand(n, 1))).to(dtype)
    masked = rand(n) < case["masked"]
    if case["op"] == "ce":
        state["targets"] = torch.where(masked, IGNORE, first)
    else:
        k = min(case["top"], v)
        # Distinct tokens a row (a stride of at most v / k), the likely one
        # first; lists end early in some rows, masked rows have none.
        step = 1 + (rand(n, 1) * (v // k)).long().clamp_max(v // k - 1)
        place = torch.arange(k, device="cuda")
        index = (first[:, None] + place * step) % v
        length = torch.where(rand(n) < 0.2, (rand(n) * (k + 1)).long().clamp(1, k), k)
        length = torch.where(masked, 0, length)
        state["indices"] = torch.where(place < length[:, None], index, -1)
        logits = 8.0 - 2.0 * torch.log1p(place.float()) + 0.5 * randn(n, k)
        state["teacher"] = torch.sort(logits, dim=1, descending=True).values.to(dtype)
    if case["grads"] != "none":
        # Upstream gradient: 1 for a mean or a sum, weights of both signs a row.
        per_row = case["reduction"] == "none"
        state["upstream"] = randn(n) if per_row else torch.ones((), device="cuda")
    return state


# ------------------------------------------------------------- plain forms
def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    w, b = state["weight"].float(), state["bias"].float()
    s = state["x"].float()
    out = {}
    if case["residual"]:
        stream = (s + state["residual"].float()).to(dtype)
        out["stream"] = stream
        s = stream.float()
    mean = s.mean(1, keepdim=True)
    d = s - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    xhat = d * rstd
    out["y"] = (xhat * w + b).to(dtype)
    if case["train"]:
        dy = state["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + state["ds"].float()
            out["dresidual"] = dx.to(dtype)
        out["dx"] = dx.to(dtype)
        out["dweight"] = (dy * xhat).sum(0).to(dtype)
        out["dbias"] = dy.sum(0).to(dtype)
    return out


def _plain_head(state):
    case = state["case"]
    hidden, weight = state["hidden"].float(), state["weight"].float()
    temperature = case.get("temperature", 1.0)
    z = (hidden @ weight.t()) / temperature
    top = z.max(1, keepdim=True).values
    lse = torch.log(torch.exp(z - top).sum(1, keepdim=True)) + top
    if case["op"] == "ce":
        valid = state["targets"] != IGNORE
        index = torch.where(valid, state["targets"], 0)[:, None]
        share = torch.ones_like(index, dtype=torch.float32)
        loss = (lse - z.gather(1, index))[:, 0]
    else:
        present = state["indices"] >= 0
        valid = present.any(1)
        index = torch.where(present, state["indices"], 0)
        t = torch.where(present, state["teacher"].float() / temperature, -math.inf)
        t = torch.where(valid[:, None], t, 0.0)
        t = t - t.max(1, keepdim=True).values
        e = torch.exp(t)
        total = e.sum(1, keepdim=True)
        share = torch.where(present, e / total, 0.0)
        log_share = torch.where(present, t - torch.log(total), 0.0)
        log_q = z.gather(1, index) - lse
        loss = (share * (log_share - log_q)).sum(1) * (temperature * temperature)
    loss = torch.where(valid, loss, 0.0)
    count = valid.sum().clamp_min(1)
    out = {"loss": loss}
    if case["reduction"] != "none":
        out["loss"] = loss.sum() / count if case["reduction"] == "mean" else loss.sum()
    if case["grads"] == "none":
        return out
    row = torch.where(valid, state["upstream"] * temperature, 0.0)[:, None]
    if case["reduction"] == "mean":
        row = row / count
    dz = torch.exp(z - lse)
    dz.scatter_add_(1, index, -share)
    dz *= row
    out["dhidden"] = (dz @ weight).to(state["hidden"].dtype)
    if case["grads"] == "both":
        out["dweight"] = (dz.t() @ hidden).to(state["weight"].dtype)
    return out


# ------------------------------------------------- the framework's operators
def _own_norm(state):
    from flashrwkv_amd.normalization import infer_layer_norm_forward_varlen, pretrain_layer_norm

    case = state["case"]
    args = {"eps": EPS}
    if case["residual"]:
        args["residual"] = state["residual"]
    if not case["train"]:
        got = infer_layer_norm_forward_varlen(state["x"], state["weight"], state["bias"], **args)
        return {"stream": got[1], "y": got[0]} if case["residual"] else {"y": got}
    leaves = [t.detach().requires_grad_() for t in (state["x"], state["weight"], state["bias"])]
    if not case["residual"]:
        y = pretrain_layer_norm(*leaves, **args)
        dx, dw, db = torch.autograd.grad(y, leaves, state["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    args["residual"] = state["residual"].detach().requires_grad_()
    y, stream = pretrain_layer_norm(*leaves, **args)
    dx, dw, db, dr = torch.autograd.grad((y, stream), [*leaves, args["residual"]],
                                         (state["dy"], state["ds"]))
    return {"stream": stream.detach(), "y": y.detach(), "dresidual": dr, "dx": dx, "dweight": dw,
            "dbias": db}


def _own_head(state):
    from flashrwkv_amd.loss import (pretrain_linear_cross_entropy,
                                    pretrain_linear_topk_distillation)

    case = state["case"]
    hidden = state["hidden"].detach().requires_grad_(case["grads"] != "none")
    weight = state["weight"].detach().requires_grad_(case["grads"] == "both")
    if case["op"] == "ce":
        loss = pretrain_linear_cross_entropy(hidden, weight, state["targets"],
                                             ignore_index=IGNORE, reduction=case["reduction"])
    else:
        loss = pretrain_linear_topk_distillation(
            hidden, weight, state["teacher"], state["indices"],
            temperature=case["temperature"], reduction=case["reduction"])
    out = {"loss": loss.detach()}
    if case["grads"] == "hidden":
        out["dhidden"], = torch.autograd.grad(loss, [hidden], state["upstream"])
    elif case["grads"] == "both":
        out["dhidden"], out["dweight"] = torch.autograd.grad(loss, [hidden, weight],
                                                             state["upstream"])
    return out


def run(state):
    if state["case"]["op"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_head(state) if own else _plain_head(state)


def work(case):
    n, c, e = case["rows"], case["channels"], BYTES[case["dtype"]]
    if case["op"] == "norm":
        # forward x -> y, backward dy -> dx (x is read once); with a residual
        # also r -> s, ds and the residual's gradient, which is x's own.
        planes = 2 + 2 * case["residual"] + case["train"] * (2 + case["residual"])
        vectors = 2 + 2 * case["train"]
        return {"bytes": e * (n * c * planes + c * vectors),
                "flops": n * c * (8 + 12 * case["train"])}
    v = case["vocab"]
    products = {"none": 1, "hidden": 2, "both": 3}[case["grads"]]
    rows_moved = n * c * (1 + (products > 1)) + v * c * (1 + (products > 2))
    side = n * 8 if case["op"] == "ce" else n * case["top"] * (8 + e)
    # the logits once, then a product for each gradient
    return {"bytes": e * rows_moved + side + 4 * n, "flops": 2 * n * v * c * products}


# --------------------------------------------------------------- in 64 bits
def _exact_norm(state):
    case, dtype = state["case"], state["x"].dtype
    s = state["x"].double()
    out = {}
    if case["residual"]:
        s = s + state["residual"].double()
        out["stream"] = s
        s = s.to(dtype).double()
    s.requires_grad_()
    w, b = (state[k].double().requires_grad_() for k in ("weight", "bias"))
    var, mean = torch.var_mean(s, dim=1, correction=0, keepdim=True)
    y = (s - mean) * torch.rsqrt(var + EPS) * w + b
    out["y"] = y.detach()
    if case["train"]:
        dx, dw, db = torch.autograd.grad(y, [s, w, b], state["dy"].double())
        if case["residual"]:
            dx = dx + state["ds"].double()
            out["dresidual"] = dx
        out |= {"dx": dx, "dweight": dw, "dbias": db}
    return out


def _exact_head(state):
    case = state["case"]
    distill = case["op"] == "distill"
    temperature = case["temperature"] if distill else 1.0
    if distill:
        valid = (state["indices"] >= 0).sum(1) > 0
    else:
        valid = state["targets"] != IGNORE
    rows = valid.nonzero()[:, 0]
    hidden, weight = state["hidden"].double()[rows], state["weight"].double()
    logq = torch.log_softmax((hidden @ weight.t()).div_(temperature), dim=1)
    if distill:
        index = state["indices"][rows]
        logits = state["teacher"].double()[rows] / temperature
        logp = torch.log_softmax(logits.masked_fill(index < 0, -math.inf), dim=1)
        index, p = index.clamp_min(0), torch.exp(logp)
        cross = (p * logq.gather(1, index)).sum(1)
        entropy = torch.special.entr(p).sum(1)
        part = -(cross + entropy) * temperature ** 2
    else:
        index = state["targets"][rows][:, None]
        p = torch.ones_like(index, dtype=torch.float64)
        part = -logq.gather(1, index)[:, 0]
    loss = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    loss[rows] = part
    share = 1.0
    if case["reduction"] == "mean":
        share = 1.0 / max(1, rows.numel())
    out = {"loss": loss if case["reduction"] == "none" else loss.sum() * share}
    if case["grads"] == "none":
        return out
    upstream = state["upstream"].double()
    upstream = upstream[rows] if upstream.dim() else upstream.expand(rows.numel())
    dz = torch.exp(logq).scatter_add(1, index, -p) * (upstream * (share * temperature))[:, None]
    del logq
    out["dhidden"] = torch.zeros(case["rows"], case["channels"], dtype=torch.float64,
                                 device="cuda")
    out["dhidden"][rows] = dz @ weight
    if case["grads"] == "both":
        out["dweight"] = dz.t() @ hidden
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_norm(state) if case["op"] == "norm" else _exact_head(state)

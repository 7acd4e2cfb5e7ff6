"""Cases of the operators at the end of a policy or preference training step:
log probabilities and entropies of tokens from the hidden rows, the clipped
policy loss, the preference loss of paired sequences, and the norm of all
gradients with clipping.

``own`` false computes them in plain torch operations in 32 bits (log ratios
and sums over sequences in 64), ``own`` true with the entry points of
``flashrwkv_amd.loss`` and ``flashrwkv_amd.gradients``. ``exact`` restates
them in 64 bits.

Definitions:

* logp: z = hidden weight^T / T; logp = z[target] - logsumexp(z), entropy =
  -sum p log p with p = softmax(z). Rows whose target is -100 take no part
  (both 0, gradient 0). Upstream gradients a row for both.
* policy: per token d = logp - old, r = exp(d), loss = -min(r A, clamp(r,
  1 - low, 1 + high) A) (with a dual clip at most -dual A where A < 0) +
  kl k3(ref - logp) - entropy_weight H, k3(x) = exp(x) - 1 - x. Tokens that the
  mask leaves out and those behind the last sequence take no part. Reduced by
  their mean, by the mean over sequences of each one's mean, or not.
* preference: s = sum of logp - ref over a sequence's tokens (their mean with
  ``normalize``), m = beta (s_chosen - s_rejected) - margin, loss =
  -(1 - eps) log sigmoid(m) - eps log sigmoid(-m), max(0, 1 - m) or
  ((m - 1/2) / beta)^2. A pair of which one side has no token takes no part.
* clip: norm = sqrt(sum x^2) over all tensors, y = x min(1, max / (norm + eps)).
"""

import math

import torch

own = False

IGNORE = -100
CLIP_EPS = 1e-6
LOW, HIGH, DUAL = 0.2, 0.28, 3.0
KL_WEIGHT, ENTROPY_WEIGHT = 0.05, 0.01
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _logp(name, rows, channels, vocab, dtype, grads, entropy, temperature, masked):
    return {"name": name, "op": "logp", "rows": rows, "channels": channels, "vocab": vocab,
            "dtype": dtype, "grads": grads, "entropy": entropy, "temperature": temperature,
            "masked": masked}


def _policy(name, tokens, sequences, reduction, reference, entropy, masked, per_sequence,
            dual=False, dtype="fp32", tail=0):
    return {"name": name, "op": "policy", "tokens": tokens, "sequences": sequences,
            "reduction": reduction, "reference": reference, "entropy": entropy,
            "masked": masked, "per_sequence": per_sequence, "dual": dual, "dtype": dtype,
            "tail": tail}


def _preference(name, tokens, pairs, kind, reference, normalize, masked, smoothing,
                dtype="fp32", tail=0):
    return {"name": name, "op": "preference", "tokens": tokens, "pairs": pairs, "kind": kind,
            "reference": reference, "normalize": normalize, "masked": masked,
            "smoothing": smoothing, "dtype": dtype, "tail": tail}


def _clip(name, layout, layers, channels, vocab, dtype, to, over):
    return {"name": name, "op": "clip", "layout": layout, "layers": layers,
            "channels": channels, "vocab": vocab, "dtype": dtype, "to": to, "over": over}


def listed():
    return [
        # Log probabilities and entropies of one decoded token of 8 requests.
        _logp("logp_rollout_8", 8, 2048, 65536, "bf16", "none", True, 0.7, 0.0),
        # A small policy step, odd sizes, a third of the rows prompt, with the
        # gradient of an entropy bonus.
        _logp("logp_train_odd", 777, 768, 20011, "fp16", "both", True, 1.3, 0.3),
        # The head of a policy step with the entropy beside the log probability.
        _logp("logp_train_8192", 8192, 4096, 65536, "bf16", "both", True, 1.0, 0.1),
        # One short answer.
        _policy("policy_one_300", 300, 1, "mean", False, False, 0.0, False),
        # A group of 64 answers, one advantage each, prompts masked, the mean
        # over sequences, KL to a reference and an entropy bonus; 16-bit logs of
        # the engine that sampled.
        _policy("policy_64_answers", 50001, 64, "sequence_mean", True, True, 0.3, True,
                dtype="bf16", tail=77),
        # A whole policy batch: 1024 long answers.
        _policy("policy_4m_tokens", 4194304, 1024, "mean", True, False, 0.2, False, dual=True),
        # One pair of answers.
        _preference("preference_one_pair", 1213, 1, "sigmoid", True, False, 0.2, 0.0),
        # A batch by mean log probability, without a reference.
        _preference("preference_64_normalized", 50021, 64, "sigmoid", False, True, 0.3, 0.1,
                    dtype="bf16", tail=100),
        # A whole preference batch.
        _preference("preference_2m_tokens", 2097152, 512, "sigmoid", True, False, 0.3, 0.0),
        # The states of a state-tuned model: 24 layers of 32 heads of 64 x 64,
        # under the maximum, in place.
        _clip("clip_states", "states", 24, 2048, 0, "fp32", "same", False),
        # A few ragged tensors of mixed types, over the maximum.
        _clip("clip_ragged_mixed", "ragged", 37, 1000, 0, "mixed", "new", True),
        # A model of 24 layers of 1024 channels: bf16 gradients clipped into
        # the fp32 ones that an optimizer with master weights takes.
        _clip("clip_model_master", "model", 24, 1024, 65536, "bf16", "fp32", True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _unnamed(case):
    return {key: value for key, value in case.items() if key != "name"}


def draw(rng):
    op = rng.choice(["logp", "policy", "preference", "clip"])
    if op == "logp":
        grads = rng.choice(["none", "hidden", "both", "both"])
        return _unnamed(_logp("", _log_uniform(rng, 1, 8192), 64 * _log_uniform(rng, 4, 64),
                              _log_uniform(rng, 500, 65536), rng.choice(["bf16", "bf16", "fp16"]),
                              grads, rng.random() < 0.7, rng.choice([0.6, 0.7, 1.0, 1.3]),
                              rng.choice([0.0, 0.1, 0.5])))
    if op == "clip":
        layout = rng.choice(["states", "ragged", "model"])
        layers = _log_uniform(rng, 1, 24) if layout != "ragged" else _log_uniform(rng, 1, 300)
        return _unnamed(_clip("", layout, layers, 64 * _log_uniform(rng, 2, 16),
                              _log_uniform(rng, 500, 65536),
                              "mixed" if layout == "ragged" else
                              rng.choice(["bf16", "fp16", "fp32"]),
                              rng.choice(["new", "fp32"]) if rng.random() < 0.7 else "same",
                              rng.random() < 0.7))
    tokens = _log_uniform(rng, 1, 4194304 if op == "policy" else 2097152)
    tail = rng.choice([0, 0, rng.randrange(1 + min(tokens // 4, 500))])
    masked = rng.choice([0.0, 0.2, 0.5])
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    if op == "policy":
        sequences = _log_uniform(rng, 1, max(1, tokens // 4))
        return _unnamed(_policy("", tokens, sequences,
                                rng.choice(["mean", "mean", "sequence_mean", "none"]),
                                rng.random() < 0.6, rng.random() < 0.4, masked,
                                rng.random() < 0.5, rng.random() < 0.3, dtype, tail))
    return _unnamed(_preference("", tokens, _log_uniform(rng, 1, max(1, tokens // 16)),
                                rng.choice(["sigmoid", "sigmoid", "hinge", "squared"]),
                                rng.random() < 0.7, rng.random() < 0.4, masked,
                                rng.choice([0.0, 0.1]), dtype, tail))


# --------------------------------------------------------------------- inputs
class _Random:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def randn(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda")

    def rand(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def integers(self, high, *shape):
        return torch.randint(high, shape, generator=self.gen, device="cuda")


def _prepare_logp(case, state, rng):
    n, c, v, dtype = case["rows"], case["channels"], case["vocab"], DTYPES[case["dtype"]]
    # Normalised hidden rows; logits of standard deviation about 2.5, the token
    # that was sampled up to about 9 above that.
    weight = (rng.randn(v, c) * (2.5 / math.sqrt(c))).to(dtype)
    tokens = rng.integers(v, n)
    state["weight"] = weight
    state["hidden"] = (rng.randn(n, c) + weight[tokens].float() * (1.5 * rng.rand(n, 1))).to(dtype)
    state["targets"] = torch.where(rng.rand(n) < case["masked"], IGNORE, tokens)
    if case["grads"] != "none":
        # Advantages of both signs, and a bonus of the size that they are used with.
        state["upstream"] = [rng.randn(n)]
        if case["entropy"]:
            state["upstream"].append(0.1 * (1.0 + rng.rand(n)))


def _prepare_tokens(case, state, rng, sequences):
    """Offsets of ragged sequences (a few of them empty), the mask of prompts."""
    n, used = case["tokens"], case["tokens"] - case["tail"]
    cuts = torch.sort(rng.integers(used + 1, sequences - 1)).values
    offsets = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), used)])
    state["cu_seqlens"] = offsets.to(torch.int32)
    place = torch.arange(n, device="cuda")
    sequence = torch.searchsorted(offsets, place, right=True) - 1
    inside = sequence.clamp_max(sequences - 1)
    if case["masked"]:
        prompt = rng.rand(sequences) * (2 * case["masked"] * used / sequences)
        state["mask"] = place - offsets[inside] >= prompt[inside]
    dtype = DTYPES[case["dtype"]]
    # Sampled tokens are likely ones; the policies are close to each other.
    logp = 1.2 * torch.log1p(-rng.rand(n))
    state["log_probs"] = logp
    if case["reference"]:
        state["reference"] = (logp + 0.3 * rng.randn(n)).clamp_max(0.0).to(dtype)
    return logp, dtype


def _prepare_policy(case, state, rng):
    n, b = case["tokens"], case["sequences"]
    logp, dtype = _prepare_tokens(case, state, rng, b)
    state["old"] = (logp + 0.15 * rng.randn(n)).clamp_max(0.0).to(dtype)
    state["advantages"] = rng.randn(b if case["per_sequence"] else n)
    if case["entropy"]:
        state["entropy"] = 3.0 * rng.rand(n)
    per_token = case["reduction"] == "none"
    state["upstream"] = rng.randn(n) if per_token else torch.ones((), device="cuda")


def _prepare_preference(case, state, rng):
    _prepare_tokens(case, state, rng, 2 * case["pairs"])
    state["upstream"] = torch.ones((), device="cuda")


def _shapes(case):
    """The tensors of a model's gradients, and the type of each."""
    c, layers = case["channels"], case["layers"]
    if case["layout"] == "states":
        shapes = [(c // 64, 64, 64)] * layers
    elif case["layout"] == "ragged":
        gen = torch.Generator().manual_seed(layers)
        sizes = torch.exp(torch.rand(layers, generator=gen) * math.log(100.0 * c)).long()
        return [((int(n),), ("fp32", "bf16", "fp16")[i % 3]) for i, n in enumerate(sizes)]
    else:
        block = [(c, c)] * 4 + [(4 * c, c), (c, 4 * c)] + [(c, 64), (64, c)] * 4 + [(c,)] * 14
        shapes = [(case["vocab"], c), *(block * layers), (c,), (c,), (case["vocab"], c)]
    return [(s, case["dtype"]) for s in shapes]


def _prepare_clip(case, state, rng):
    # Gradients are views of one buffer a type, as data-parallel training keeps them.
    shapes = _shapes(case)
    room, buffers, places = {}, {}, []
    for shape, dtype in shapes:
        at = room.get(dtype, 0)
        places.append(at)
        room[dtype] = at + -(-math.prod(shape) // 64) * 64
    for dtype, size in room.items():
        buffers[dtype] = (1e-2 * rng.randn(size)).to(DTYPES[dtype])

    def views(of, to):
        return [of[to or d][at: at + math.prod(s)].view(s) for at, (s, d) in zip(places, shapes)]

    state["tensors"] = views(buffers, None)
    if case["to"] == "same":
        state["flat"] = buffers
    else:
        # One buffer a type of the results; of the inputs' types, or fp32 beside.
        state["flat"] = {d: torch.zeros(size, device="cuda", dtype=torch.float32 if
                                        case["to"] == "fp32" else DTYPES[d])
                         for d, size in room.items()}
        state["out"] = views(state["flat"], None)
    count = sum(math.prod(s) for s, _ in shapes)
    state["max_norm"] = 1e-2 * math.sqrt(count) * (0.1 if case["over"] else 10.0)


def prepare(case, seed):
    state, rng = {"case": case}, _Random(seed)
    if case["op"] == "logp":
        _prepare_logp(case, state, rng)
    elif case["op"] == "policy":
        _prepare_policy(case, state, rng)
    elif case["op"] == "preference":
        _prepare_preference(case, state, rng)
    else:
        _prepare_clip(case, state, rng)
    return state


# ---------------------------------------------------------------- plain forms
def _plain_logp(state):
    case = state["case"]
    hidden, weight = state["hidden"].float(), state["weight"].float()
    scale = 1.0 / case["temperature"]
    valid = (state["targets"] != IGNORE)[:, None]
    index = torch.where(valid, state["targets"][:, None], 0)
    z = (hidden @ weight.t()) * scale
    z -= z.max(1, keepdim=True).values
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    log_total = torch.log(total)
    out = {"log_probs": torch.where(valid, z.gather(1, index) - log_total, 0.0)[:, 0]}
    p /= total
    if case["entropy"]:
        entropy = log_total - (p * z).sum(1, keepdim=True)
        out["entropy"] = torch.where(valid, entropy, 0.0)[:, 0]
    if case["grads"] == "none":
        return out
    g = torch.where(valid, state["upstream"][0][:, None] * scale, 0.0)
    if case["entropy"]:
        e = torch.where(valid, state["upstream"][1][:, None] * scale, 0.0)
        dz = p * (-g - e * (z - log_total + entropy))
    else:
        dz = p * -g
    dz.scatter_add_(1, index, g)
    out["dhidden"] = (dz @ weight).to(state["hidden"].dtype)
    if case["grads"] == "both":
        out["dweight"] = (dz.t() @ hidden).to(state["weight"].dtype)
    return out


def _part(state):
    """Which tokens take part, and each one's sequence."""
    offsets = state["cu_seqlens"].long()
    n, b = state["log_probs"].numel(), offsets.numel() - 1
    place = torch.arange(n, device="cuda")
    sequence = torch.searchsorted(offsets, place, right=True) - 1
    part = place < offsets[-1]
    if "mask" in state:
        part = part & state["mask"]
    return part, sequence.clamp_max(b - 1), offsets


def _sums(values, offsets):
    """Sums over the sequences of [tokens] values, in 64 bits."""
    total = torch.cat([values.new_zeros(1, dtype=torch.float64), values.double().cumsum(0)])
    return total[offsets[1:]] - total[offsets[:-1]]


def _plain_policy(state):
    case = state["case"]
    part, sequence, offsets = _part(state)
    logp = state["log_probs"].double()
    d = logp - state["old"].double()
    a = state["advantages"]
    a = a[sequence] if case["per_sequence"] else a
    ratio = torch.exp(d).float()
    clipped = ((a > 0) & (d > math.log1p(HIGH))) | ((a < 0) & (d < math.log1p(-LOW)))
    surrogate = torch.minimum(ratio * a, ratio.clamp(1.0 - LOW, 1.0 + HIGH) * a)
    if case["dual"]:
        clipped = clipped | ((a < 0) & (d > math.log(DUAL)))
        surrogate = torch.where(a < 0, torch.maximum(surrogate, DUAL * a), surrogate)
    loss = -surrogate
    slope = torch.where(clipped, 0.0, -ratio * a)
    reference = torch.zeros_like(loss)
    if case["reference"]:
        x = state["reference"].double() - logp
        reference = (torch.expm1(x) - x).float()
        loss = loss + KL_WEIGHT * reference
        slope = slope - KL_WEIGHT * torch.expm1(x).float()
    if case["entropy"]:
        loss = loss - ENTROPY_WEIGHT * state["entropy"]
    loss = torch.where(part, loss, 0.0)
    count = part.double().sum().clamp_min(1)
    old = (torch.expm1(d) - d).float()
    metrics = torch.stack([torch.where(part, x, 0.0).double().sum() / count
                           for x in (ratio, clipped.float(), old, reference)])
    if case["reduction"] == "none":
        share = state["upstream"].double()
    elif case["reduction"] == "mean":
        share = (1.0 / count).expand(loss.shape)
        loss = loss.double().sum() / count
    else:
        counts = _sums(part, offsets)
        each = _sums(loss, offsets) / counts.clamp_min(1)
        sequences = (counts > 0).double().sum().clamp_min(1)
        loss = each.sum() / sequences
        share = (1.0 / (counts.clamp_min(1) * sequences))[sequence]
    share = torch.where(part, share, 0.0).float()
    if case["reduction"] != "none":
        share = share * state["upstream"]
    out = {"loss": loss.float(), "metrics": metrics.float(),
           "dlog_probs": torch.where(part, slope, 0.0) * share}
    if case["entropy"]:
        out["dentropy"] = -ENTROPY_WEIGHT * share
    return out


BETA = {"sigmoid": 0.1, "hinge": 0.05, "squared": 0.1}
MARGIN = 0.2


def _plain_preference(state):
    case = state["case"]
    beta = BETA[case["kind"]]
    part, sequence, offsets = _part(state)
    d = state["log_probs"].double()
    if case["reference"]:
        d = d - state["reference"].double()
    counts = _sums(part, offsets)
    sums = _sums(torch.where(part, d, 0.0), offsets)
    by = 1.0 / counts.clamp_min(1) if case["normalize"] else torch.ones_like(counts)
    rewards = beta * (sums * by).view(-1, 2)
    m = rewards[:, 0] - rewards[:, 1] - MARGIN
    if case["kind"] == "sigmoid":
        eps = case["smoothing"]
        soft = torch.log1p(torch.exp(-m.abs()))
        loss = (1 - eps) * (soft - m.clamp_max(0.0)) + eps * (soft + m.clamp_min(0.0))
        slope = 1.0 / (1.0 + torch.exp(-m)) - (1 - eps)
    elif case["kind"] == "hinge":
        loss = (1.0 - m).clamp_min(0.0)
        slope = -(m < 1.0).double()
    else:
        loss = ((m - 0.5) / beta) ** 2
        slope = 2.0 * (m - 0.5) / (beta * beta)
    valid = (counts.view(-1, 2) > 0).all(1)
    pairs = valid.double().sum().clamp_min(1)
    slope = torch.where(valid, slope, 0.0) * (beta / pairs)
    slope = (torch.stack([slope, -slope], 1).view(-1) * by).float() * state["upstream"]
    return {"loss": (torch.where(valid, loss, 0.0).sum() / pairs).float(),
            "rewards": rewards.float(),
            "dlog_probs": torch.where(part, slope[sequence], 0.0)}


def _plain_clip(state):
    total = torch.stack([t.float().square().sum() for t in state["tensors"]]).sum()
    norm = torch.sqrt(total)
    by = (state["max_norm"] / (norm + CLIP_EPS)).clamp_max(1.0)
    [y.copy_(x.float() * by) for x, y in zip(state["tensors"], state.get("out", state["tensors"]))]
    return {"norm": norm, "gradients": state["flat"]}


# -------------------------------------------------- the framework's operators
def _own_logp(state):
    from flashrwkv_amd.loss import pretrain_linear_log_probs

    case = state["case"]
    hidden = state["hidden"].detach().requires_grad_(case["grads"] != "none")
    weight = state["weight"].detach().requires_grad_(case["grads"] == "both")
    got = pretrain_linear_log_probs(hidden, weight, state["targets"],
                                    temperature=case["temperature"], ignore_index=IGNORE,
                                    entropy=case["entropy"])
    got = got if case["entropy"] else (got,)
    out = {name: t.detach() for name, t in zip(("log_probs", "entropy"), got)}
    if case["grads"] == "hidden":
        out["dhidden"], = torch.autograd.grad(got, [hidden], state["upstream"])
    elif case["grads"] == "both":
        out["dhidden"], out["dweight"] = torch.autograd.grad(got, [hidden, weight],
                                                             state["upstream"])
    return out


def _own_policy(state):
    from flashrwkv_amd.loss import pretrain_policy_loss

    case = state["case"]
    leaves = [state["log_probs"].detach().requires_grad_()]
    more = {}
    if case["entropy"]:
        leaves.append(state["entropy"].detach().requires_grad_())
        more = {"entropy": leaves[1], "entropy_weight": ENTROPY_WEIGHT}
    if case["reference"]:
        more |= {"reference_log_probs": state["reference"], "kl_weight": KL_WEIGHT}
    loss, metrics = pretrain_policy_loss(
        leaves[0], state["old"], state["advantages"], mask=state.get("mask"),
        cu_seqlens=state["cu_seqlens"], clip_low=LOW, clip_high=HIGH,
        dual_clip=DUAL if case["dual"] else None, reduction=case["reduction"], metrics=True,
        **more)
    grads = torch.autograd.grad(loss, leaves, state["upstream"])
    out = {"loss": loss.detach(), "metrics": metrics}
    return out | dict(zip(("dlog_probs", "dentropy"), grads))


def _own_preference(state):
    from flashrwkv_amd.loss import pretrain_preference_loss

    case = state["case"]
    logp = state["log_probs"].detach().requires_grad_()
    loss, rewards = pretrain_preference_loss(
        logp, state["cu_seqlens"], reference_log_probs=state.get("reference"),
        mask=state.get("mask"), beta=BETA[case["kind"]], margin=MARGIN,
        label_smoothing=case["smoothing"] if case["kind"] == "sigmoid" else 0.0,
        kind=case["kind"], normalize=case["normalize"])
    grad, = torch.autograd.grad(loss, [logp], state["upstream"])
    return {"loss": loss.detach(), "rewards": rewards, "dlog_probs": grad}


def _own_clip(state):
    from flashrwkv_amd.gradients import pretrain_clip_grad_norm

    norm = pretrain_clip_grad_norm(state["tensors"], state["max_norm"], out=state.get("out"),
                                   eps=CLIP_EPS)
    return {"norm": norm, "gradients": state["flat"]}


def run(state):
    op = state["case"]["op"]
    if op == "logp":
        return _own_logp(state) if own else _plain_logp(state)
    if op == "policy":
        return _own_policy(state) if own else _plain_policy(state)
    if op == "preference":
        return _own_preference(state) if own else _plain_preference(state)
    return _own_clip(state) if own else _plain_clip(state)


def work(case):
    if case["op"] == "logp":
        n, c, v, e = case["rows"], case["channels"], case["vocab"], BYTES[case["dtype"]]
        products = {"none": 1, "hidden": 2, "both": 3}[case["grads"]]
        moved = n * c * (1 + (products > 1)) + v * c * (1 + (products > 2))
        sides = (1 + case["entropy"]) * (1 + (products > 1))
        return {"bytes": e * moved + n * (8 + 4 * sides), "flops": 2 * n * v * c * products}
    if case["op"] == "clip":
        shapes = _shapes(case)
        read = sum(math.prod(s) * BYTES[d] for s, d in shapes)
        count = sum(math.prod(s) for s, _ in shapes)
        written = {"same": read if case["over"] else 0, "new": read, "fp32": 4 * count}
        return {"bytes": read + written[case["to"]], "flops": 3 * count}
    n, e = case["tokens"], BYTES[case["dtype"]]
    side = 1 if case["masked"] else 0
    if case["op"] == "preference":
        each = 8 + e * case["reference"] + side
        return {"bytes": n * each + 8 * case["pairs"], "flops": 4 * n}
    each = 8 + e * (1 + case["reference"]) + 8 * case["entropy"] + side
    each += 0 if case["per_sequence"] else 4
    each += 8 if case["reduction"] == "none" else 0
    return {"bytes": n * each + 8 * case["sequences"], "flops": 30 * n}


# ----------------------------------------------------------------- in 64 bits
def _exact_logp(state):
    case = state["case"]
    rows = (state["targets"] != IGNORE).nonzero()[:, 0]
    hidden, weight = state["hidden"].double()[rows], state["weight"].double()
    token = state["targets"][rows][:, None]
    logq = torch.log_softmax((hidden @ weight.t()).div_(case["temperature"]), dim=1)
    zeros = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    out = {"log_probs": zeros.index_copy(0, rows, logq.gather(1, token)[:, 0])}
    q = torch.exp(logq)
    if case["entropy"]:
        entropy = torch.linalg.vecdot(q, logq).neg()
        out["entropy"] = zeros.index_copy(0, rows, entropy)
    if case["grads"] == "none":
        return out
    up = [u.double()[rows][:, None] / case["temperature"] for u in state["upstream"]]
    if case["entropy"]:
        dz = logq.add_(entropy[:, None]).mul_(up[1]).add_(up[0]).mul_(q).neg_()
    else:
        dz = q.mul(up[0]).neg_()
    del q, logq
    dz.scatter_add_(1, token, up[0])
    out["dhidden"] = torch.zeros(case["rows"], case["channels"], dtype=torch.float64,
                                 device="cuda")
    out["dhidden"][rows] = dz @ weight
    if case["grads"] == "both":
        out["dweight"] = dz.t() @ hidden
    return out


def _exact_lengths(state, n):
    """Sequence of each token (the last number for those behind), 64 bits."""
    lengths = state["cu_seqlens"].diff().long()
    behind = n - int(state["cu_seqlens"][-1])
    lengths = torch.cat([lengths, lengths.new_full((1,), behind)])
    return torch.arange(lengths.numel(), device="cuda").repeat_interleave(lengths)


def _exact_policy(state):
    case = state["case"]
    n, b = case["tokens"], case["sequences"]
    owner = _exact_lengths(state, n)
    keep = owner < b
    if "mask" in state:
        keep &= state["mask"]
    rows, owner = keep.nonzero()[:, 0], owner[keep]
    logp = state["log_probs"].double()[rows].requires_grad_()
    a = state["advantages"].double()
    a = a[owner] if case["per_sequence"] else a[rows]
    ratio = (logp - state["old"].double()[rows]).exp()
    plain, bounded = ratio * a, ratio.clamp(1 - LOW, 1 + HIGH) * a
    gain = torch.minimum(plain, bounded)
    cut = (bounded < plain)
    if case["dual"]:
        cut = cut | ((a < 0) & (gain < DUAL * a))
        gain = torch.where(a < 0, gain.clamp_min(DUAL * a), gain)
    each = -gain
    kl = torch.zeros_like(each)
    if case["reference"]:
        x = state["reference"].double()[rows] - logp
        kl = torch.special.expm1(x) - x
        each = each + KL_WEIGHT * kl
    entropy = None
    if case["entropy"]:
        entropy = state["entropy"].double()[rows].requires_grad_()
        each = each - ENTROPY_WEIGHT * entropy
    count = max(1, rows.numel())
    inverse = logp.detach() - state["old"].double()[rows]
    old = torch.special.expm1(inverse) - inverse
    metrics = torch.stack([t.detach().double().sum() / count for t in (ratio, cut, old, kl)])
    if case["reduction"] == "none":
        loss = torch.zeros(n, dtype=torch.float64, device="cuda").index_copy(0, rows, each)
        total = (loss * state["upstream"].double()).sum()
    elif case["reduction"] == "mean":
        total = loss = each.sum() / count
    else:
        counts = torch.bincount(owner, minlength=b).double()
        weights = 1.0 / counts[owner] / max(1, int((counts > 0).sum()))
        total = loss = (each * weights).sum()
    leaves = [logp] if entropy is None else [logp, entropy]
    out = {"loss": loss.detach(), "metrics": metrics}
    for name, grad in zip(("dlog_probs", "dentropy"), torch.autograd.grad(total, leaves)):
        out[name] = torch.zeros(n, dtype=torch.float64, device="cuda").index_copy(0, rows, grad)
    return out


def _exact_preference(state):
    case = state["case"]
    n, b = case["tokens"], 2 * case["pairs"]
    beta = BETA[case["kind"]]
    owner = _exact_lengths(state, n)
    keep = owner < b
    if "mask" in state:
        keep &= state["mask"]
    rows, owner = keep.nonzero()[:, 0], owner[keep]
    logp = state["log_probs"].double()[rows].requires_grad_()
    value = logp - state["reference"].double()[rows] if case["reference"] else logp
    counts = torch.bincount(owner, minlength=b).double()
    sums = torch.zeros(b, dtype=torch.float64, device="cuda").index_add(0, owner, value)
    if case["normalize"]:
        sums = sums / counts.clamp_min(1)
    rewards = beta * sums.view(-1, 2)
    both = counts.view(-1, 2).amin(1) > 0
    m = (rewards[:, 0] - rewards[:, 1])[both] - MARGIN
    if case["kind"] == "sigmoid":
        log_sigmoid = torch.nn.functional.logsigmoid
        eps = case["smoothing"]
        loss = -(1 - eps) * log_sigmoid(m) - eps * log_sigmoid(-m)
    elif case["kind"] == "hinge":
        loss = torch.relu(1 - m)
    else:
        loss = (m / beta - 0.5 / beta).square()
    loss = loss.sum() / max(1, m.numel())
    grad, = torch.autograd.grad(loss, [logp])
    full = torch.zeros(n, dtype=torch.float64, device="cuda").index_copy(0, rows, grad)
    return {"loss": loss.detach(), "rewards": rewards.detach(), "dlog_probs": full}


def _exact_clip(state):
    norms = torch.stack([torch.linalg.vector_norm(t.double()) for t in state["tensors"]])
    norm = torch.linalg.vector_norm(norms)
    by = min(1.0, state["max_norm"] / (float(norm) + CLIP_EPS))
    # What stands between the tensors of a buffer stays.
    out = {d: t.double() for d, t in state["flat"].items()}
    for source, target in zip(state["tensors"], state.get("out", state["tensors"])):
        buffer = next(d for d, t in state["flat"].items()
                      if t.data_ptr() <= target.data_ptr() < t.data_ptr() + t.nbytes)
        start = target.storage_offset()
        out[buffer][start: start + target.numel()] = source.double().flatten() * by
    return {"norm": norm, "gradients": out}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logp":
        return _exact_logp(state)
    if case["op"] == "policy":
        return _exact_policy(state)
    if case["op"] == "preference":
        return _exact_preference(state)
    return _exact_clip(state)

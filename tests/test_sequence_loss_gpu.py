"""GPU parity of the policy and preference losses against oracle/step.py (64 bits).

Bounds, before any run. A token's log ratio is rounded once to 32 bits, so its
exponential is off by 2^-24 |d| and that of the function and of the products after it
(8 units in all), and up to 256 tokens are added up in 32 bits (10 roundings), the rest in 64:
K 2^-24 of the sizes of the terms, K = 16 + |d|, with 4 (loss) or 2 (metrics) more
where sums are made:
  loss:      (K + 4) 2^-24 sum |terms| share + 2^-24 |ref|
  gradient:  K 2^-24 |terms of the slope| share + 4 2^-24 |ref| + u |ref|, u of the type
             of log_probs (its smallest step beside it)
  metrics:   (K + 2) 2^-24 of the mean of their terms
A preference's sums are of differences that are exact in 64 bits, and everything of
a pair is in 64 bits until its one rounding: rewards 2 2^-24 |ref|, losses and
gradients 4 2^-24 |ref| and the rounding of their type.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.utils.checkpoint

import flashrwkv_amd
from flashrwkv_amd import capi, pretrain_policy_loss, pretrain_preference_loss
from oracle import step

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
E = 2.0 ** -24
ROUND = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


@pytest.fixture(scope="module", autouse=True)
def _require_native():
    if flashrwkv_amd._C is None:
        pytest.fail("flashrwkv_amd native library is not built (no fallback exists)")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _offsets(lengths, tail=0):
    """(int32 offsets on the GPU, tokens) of sequences of these lengths."""
    cu = torch.tensor([0, *lengths]).cumsum(0)
    return cu.to(torch.int32).to(DEV), int(cu[-1]) + tail


def _logs(n, seed, dtype=torch.float32, spread=0.15):
    gen = _gen(seed)
    x = -1.2 * torch.empty(n).exponential_(generator=gen)
    old = (x + spread * torch.randn(n, generator=gen)).clamp_max(0.0)
    reference = (x + 0.4 * torch.randn(n, generator=gen)).clamp_max(0.0)
    return [t.to(dtype).to(DEV) for t in (x, old, reference)]


# Lengths that end inside and at the ends of rounds of 64 and of tiles of 128 and 512 tokens.
LAYOUTS = {
    "one token": [1],
    "one short": [300],
    "empty ones": [0, 0, 5, 0, 64, 1, 63, 65, 0, 0, 127, 128, 129, 0],
    "all empty but one": [0] * 70 + [3] + [0] * 140,
    "tiny": [1 + (i * 7) % 5 for i in range(700)],
    "rounds": [64] * 40,
    "tiles": [512, 511, 513, 1, 128, 384, 512, 1024, 7],
    "one of 8192": [8192],
    "beyond one workgroup": [8000, 193, 0, 4000, 61, 62, 500, 3, 2, 1, 0],
    "many pieces": [30000, 1, 40000, 129],
}


def _policy(layout, *, dtype=torch.float32, log_dtype=torch.float32, reduction="mean",
            tail=0, seed=0, masked=0.3, reference=True, entropy=True, per_sequence=False,
            offsets=True, dual=None, **more):
    cu, n = _offsets(layout, tail)
    x, old, ref = _logs(n, seed)
    x, old, ref = x.to(log_dtype), old.to(dtype), ref.to(dtype)
    gen = _gen(seed + 1)
    a = torch.randn(len(layout) if per_sequence else n, generator=gen)
    a[torch.rand(a.shape, generator=gen) < 0.1] = 0.0
    args = {"mask": (torch.rand(n, generator=gen) >= masked).to(DEV) if masked else None,
            "cu_seqlens": cu if offsets else None, "clip_low": 0.2, "clip_high": 0.28,
            "dual_clip": dual, "reduction": reduction, **more}
    args["reference"] = ref if reference else None
    args["kl_weight"] = 0.3 if reference else 0.0
    args["entropy"] = (3 * torch.rand(n, generator=gen)).to(log_dtype).to(DEV) if entropy else None
    args["entropy_weight"] = 0.05 if entropy else 0.0
    upstream = torch.randn(n, generator=gen).to(DEV) if reduction == "none" \
        else torch.tensor(0.7, device=DEV)
    return x, old, a.to(dtype).to(DEV), args, upstream


def _run_policy(x, old, a, args, upstream):
    args = dict(args)
    args["reference_log_probs"] = args.pop("reference")
    x = x.detach().clone().requires_grad_()
    leaves = [x]
    if args["entropy"] is not None:
        args["entropy"] = args["entropy"].detach().clone().requires_grad_()
        leaves.append(args["entropy"])
    loss, metrics = pretrain_policy_loss(x, old, a, metrics=True, **args)
    grads = torch.autograd.grad(loss, leaves, upstream)
    assert not metrics.requires_grad
    return {"loss": loss.detach(), "metrics": metrics,
            **dict(zip(("dlog_probs", "dentropy"), grads))}


def _check_policy(x, old, a, args, upstream, got):
    ref = step.policy(x, old, a, upstream=upstream, **args)
    part = ref["part"]
    d = (x.double() - old.double()).flatten().cpu()
    d = torch.where(part, d, 0.0).abs()
    k = (16 + d) * E
    adv = a.double().cpu().flatten()
    if adv.numel() != d.numel():
        _, owner = step.sequences(args["cu_seqlens"].cpu(), d.numel())
        adv = adv[owner.clamp_min(0)]
    signed = torch.where(part, (x.double() - old.double()).flatten().cpu(), 0.0)
    gain = torch.exp(signed) * adv.abs()
    kl = torch.zeros_like(gain)
    if args["reference"] is not None:
        t = torch.where(part, (args["reference"].double() - x.double()).flatten().cpu(), 0.0)
        k = k + t.abs() * E
        kl = abs(args["kl_weight"]) * (torch.exp(t) + 1 + t.abs())
    size = gain + kl
    if args["entropy"] is not None:
        size = size + abs(args["entropy_weight"]) * args["entropy"].double().cpu().flatten()
    size = torch.where(part, size, 0.0)
    up = upstream.double().cpu().flatten()
    loss = got["loss"].double().cpu()
    if args["reduction"] == "none":
        assert got["loss"].shape == x.shape
        allowed, want = k * size, ref["each"].view(x.shape)
    else:
        assert got["loss"].shape == ()
        allowed = (k * size * ref["share"]).sum() + E * ref["loss"].abs() \
            + 4 * E * (size * ref["share"]).sum()
        want = ref["loss"]
    assert ((loss - want).abs().flatten() <= allowed).all(), (
        (loss - want).abs().max(), allowed)
    count = max(1, int(part.sum()))
    means = [torch.where(part, torch.exp(signed), 0.0), part.double(),
             torch.where(part, torch.exp(signed) + 1 + d, 0.0), kl / 0.3]
    for got_mean, want_mean, terms in zip(got["metrics"].cpu(), ref["metrics"], means):
        limit = (k * torch.where(part, terms, 0.0)).sum() / count + 2 * E * want_mean.abs()
        assert abs(got_mean.double() - want_mean) <= limit
    for name, spread, like in (("dlog_probs", gain + kl, x),
                               ("dentropy", None, args["entropy"])):
        if name not in got:
            continue
        want = ref[name]
        assert got[name].dtype == like.dtype and got[name].shape == like.shape
        value = got[name].double().cpu().flatten()
        assert not value[~part].any()
        allowed = (4 * E + ROUND[like.dtype] * (1 + E)) * want.abs() + STEP[like.dtype]
        if spread is not None:
            allowed = allowed + k * torch.where(part, spread, 0.0) * ref["share"] * up.abs()
        worst = ((value - want).abs() - allowed).max().item()
        assert worst <= 0, (name, worst)


@pytest.mark.parametrize("reduction", ["mean", "sum", "sequence_mean", "none"])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_policy(layout, reduction):
    print(f"case {layout} {reduction}", flush=True)
    for per_sequence in (False, True):
        case = _policy(LAYOUTS[layout], reduction=reduction, tail=5 if per_sequence else 0,
                       per_sequence=per_sequence, seed=3, dual=2.0 if per_sequence else None)
        _check_policy(*case, _run_policy(*case))


@pytest.mark.parametrize("log_dtype", ROUND)
@pytest.mark.parametrize("dtype", ROUND)
def test_policy_types(dtype, log_dtype):
    for reduction in ("mean", "sequence_mean"):
        case = _policy(LAYOUTS["tiles"], dtype=dtype, log_dtype=log_dtype, reduction=reduction,
                       seed=4)
        _check_policy(*case, _run_policy(*case))


@pytest.mark.parametrize("masked", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("reference", [False, True])
@pytest.mark.parametrize("entropy", [False, True])
def test_policy_options(masked, reference, entropy):
    for offsets, reduction in ((False, "mean"), (False, "none"), (True, "sequence_mean")):
        case = _policy([700, 0, 301], masked=masked, reference=reference, entropy=entropy,
                       offsets=offsets, reduction=reduction, seed=5, tail=0)
        _check_policy(*case, _run_policy(*case))


@pytest.mark.parametrize("reduction", ["mean", "sequence_mean"])
@pytest.mark.parametrize("lengths", ["one", "many"])
def test_policy_large(lengths, reduction):
    """Tiles of eight rounds; one sequence of all of their pieces, or more sequences than
    waves."""
    layout = [300001] if lengths == "one" else torch.randint(
        9, (70000,), generator=_gen(6)).tolist() + [4000]
    print(f"case {lengths} {reduction} {sum(layout)} tokens", flush=True)
    case = _policy(layout, reduction=reduction, tail=3, seed=7, per_sequence=True)
    _check_policy(*case, _run_policy(*case))


def test_policy_borders_are_decided_in_64_bits():
    """Ratios next to 1 + high and 1 - low: the gradient stays or goes by the exact log
    ratio, also where both logs are large."""
    high, low = math.log1p(0.28), math.log1p(-0.2)
    old = torch.tensor([0.0, -3.0, -40.0, -900.0]).repeat_interleave(400)
    steps = torch.arange(-200, 200).repeat(4)
    for border, sign in ((high, 1.0), (low, -1.0)):
        x = (old.double() + border).float()
        x = torch.nextafter(x, torch.where(steps < 0, -math.inf, math.inf)) + steps * x.abs() * E
        a = torch.full_like(x, sign)
        args = {"clip_low": 0.2, "clip_high": 0.28, "reduction": "sum", "reference": None,
                "entropy": None, "mask": None, "cu_seqlens": None, "dual_clip": None,
                "kl_weight": 0.0, "entropy_weight": 0.0}
        case = (x.to(DEV), old.to(DEV), a.to(DEV), args, torch.tensor(1.0, device=DEV))
        got = _run_policy(*case)
        d = x.double() - old.double()
        clipped = d > border if sign > 0 else d < border
        assert clipped.any() and not clipped.all()
        assert torch.equal(got["dlog_probs"].cpu() == 0, clipped)
        assert got["metrics"][1].item() == pytest.approx(clipped.double().mean().item(), abs=1e-7)


def test_policy_of_the_same_weights_has_ratio_one():
    x, _, _ = _logs(1000, seed=8)
    a = torch.randn(1000, generator=_gen(9)).to(DEV)
    leaf = x.clone().requires_grad_()
    loss, metrics = pretrain_policy_loss(leaf, x, a, clip_low=0.0, clip_high=0.0, metrics=True)
    grad, = torch.autograd.grad(loss, [leaf])
    assert metrics.tolist() == [1.0, 0.0, 0.0, 0.0]
    assert torch.equal(grad, -a * torch.tensor(1e-3, device=DEV))


def test_small_kl_keeps_its_digits():
    """k3 of log ratios down to 1e-6, whose 1 + x + ... cancels in 32 bits."""
    x = torch.zeros(7, device=DEV)
    ref = torch.tensor([1e-6, -1e-5, 1e-4, -1e-3, 1e-2, -0.1, 0.99], device=DEV)
    leaf = x.clone().requires_grad_()
    loss = pretrain_policy_loss(leaf, x, x, reference_log_probs=ref, kl_weight=1.0,
                                reduction="none")
    grad, = torch.autograd.grad(loss.sum(), [leaf])
    t = ref.double()
    torch.testing.assert_close(loss.double(), torch.expm1(t) - t, rtol=8 * E, atol=0)
    torch.testing.assert_close(grad.double(), -torch.expm1(t), rtol=8 * E, atol=0)


def test_policy_ratios_far_out_stay_what_the_formula_says():
    """Ratios that are 0 or infinite in 32 bits: clipped where the clip bounds them."""
    old = torch.tensor([-200.0, 0.0, -math.inf, 0.0, -100.0, 0.0], device=DEV)
    x = torch.tensor([0.0, -200.0, 0.0, -math.inf, 0.0, -100.0], device=DEV)
    leaf = x.clone().requires_grad_()
    loss = pretrain_policy_loss(leaf, old, torch.ones_like(x), reduction="none")
    grad, = torch.autograd.grad(loss.sum(), [leaf])
    assert loss.tolist() == pytest.approx([-1.2, 0.0, -1.2, 0.0, -1.2, 0.0])
    assert not grad.any()
    loss = pretrain_policy_loss(leaf, old, -torch.ones_like(x), reduction="none")
    grad, = torch.autograd.grad(loss.sum(), [leaf])
    for t in (loss, grad):
        assert t.tolist() == pytest.approx([math.inf, 0.8, math.inf, 0.8, math.inf, 0.8]
                                           if t is loss else
                                           [math.inf, 0.0, math.inf, 0.0, math.inf, 0.0])
    loss = pretrain_policy_loss(leaf, x, -torch.ones_like(x), reduction="none", kl_weight=1.0,
                                reference_log_probs=torch.tensor(
                                    [-300.0, 0.0, 0.0, 0.0, 60.0, -190.0], device=DEV))
    assert loss[0].item() == 300.0 - 1.0 + 1.0
    assert loss[1].item() == math.inf and loss[2].item() == 1.0
    assert loss[4].item() == pytest.approx(math.exp(60.0) - 61.0 + 1.0, rel=64 * E)
    assert loss[5].item() == pytest.approx(90.0 - 1.0 + 1.0)


def test_policy_tokens_without_part_may_hold_anything():
    for reduction in ("mean", "sequence_mean", "none"):
        x, old, a, args, up = _policy([500, 40, 700], reduction=reduction, tail=30, seed=10)
        clean = _run_policy(x, old, a, args, up)
        out = ~args["mask"]
        out[1240:] = True
        for t, value in ((x, math.nan), (old, -math.inf), (a, math.inf),
                         (args["reference"], math.nan), (args["entropy"], -math.inf)):
            t[out] = value
        got = _run_policy(x, old, a, args, up)
        for name in got:
            assert torch.equal(got[name], clean[name]), (reduction, name)
        assert not got["dlog_probs"][out].any() and not got["dentropy"][out].any()


def test_policy_calls_repeat_bitwise_on_any_stream():
    case = _policy(LAYOUTS["many pieces"], reduction="sequence_mean", seed=11)
    first = _run_policy(*case)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = _run_policy(*case)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(first[name], other[name]) for name in first)


def test_calls_on_two_streams_at_once():
    cases = [_policy(LAYOUTS["many pieces"], reduction="sequence_mean", seed=30),
             _policy(LAYOUTS["tiny"], reduction="mean", seed=31)]
    want = [_run_policy(*case) for case in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for case, stream, out in zip(cases, streams, got):
            with torch.cuda.stream(stream):
                out.append(_run_policy(*case))
    torch.cuda.synchronize()
    for first, runs in zip(want, got):
        assert all(torch.equal(run[name], first[name]) for run in runs for name in first)


def test_policy_gradient_of_either_input_alone():
    x, old, a, args, up = _policy([100, 200], seed=12)
    full = _run_policy(x, old, a, args, up)
    more = {k: v for k, v in args.items() if k != "reference"}
    more["reference_log_probs"] = args["reference"]
    leaf = x.clone().requires_grad_()
    loss = pretrain_policy_loss(leaf, old, a, **more)
    assert torch.equal(torch.autograd.grad(loss, [leaf], up)[0], full["dlog_probs"])
    more["entropy"] = args["entropy"].clone().requires_grad_()
    loss = pretrain_policy_loss(x, old, a, **more)
    assert torch.equal(torch.autograd.grad(loss, [more["entropy"]], up)[0], full["dentropy"])
    with torch.no_grad():
        assert torch.equal(pretrain_policy_loss(x, old, a, **more), full["loss"])


def test_padded_batch_by_rows():
    """[B, T] with a mask: the rows are the sequences."""
    x, old, _ = (t.view(6, 50) for t in _logs(300, seed=13))
    a = torch.randn(6, generator=_gen(14)).to(DEV)
    length = torch.tensor([50, 1, 0, 17, 33, 49], device=DEV)
    mask = torch.arange(50, device=DEV) < length[:, None]
    cu = torch.arange(0, 301, 50, dtype=torch.int32, device=DEV)
    args = {"clip_low": 0.1, "clip_high": 0.1, "reduction": "sequence_mean", "reference": None,
            "entropy": None, "mask": mask, "cu_seqlens": cu, "dual_clip": None, "kl_weight": 0.0,
            "entropy_weight": 0.0}
    case = (x, old, a, args, torch.tensor(1.0, device=DEV))
    _check_policy(*case, _run_policy(*case))


def test_no_tokens():
    x = torch.zeros(0, device=DEV, requires_grad=True)
    cu = torch.zeros(3, dtype=torch.int32, device=DEV)
    for reduction, shape in (("mean", ()), ("none", (0,)), ("sequence_mean", ())):
        loss, metrics = pretrain_policy_loss(x, x.detach(), x.detach(), cu_seqlens=cu,
                                             reduction=reduction, metrics=True)
        assert loss.shape == shape and not loss.any() and not metrics.any()
        assert torch.autograd.grad(loss.sum(), [x])[0].shape == (0,)
    loss, rewards = pretrain_preference_loss(x, cu, reduction="none")
    assert loss.tolist() == [0.0] and rewards.tolist() == [[0.0, 0.0]]


# -------------------------------------------------------------- preference
def _run_preference(x, cu, args, upstream):
    leaf = x.detach().clone().requires_grad_()
    more = {k: v for k, v in args.items() if k != "reference"}
    loss, rewards = pretrain_preference_loss(leaf, cu, reference_log_probs=args["reference"],
                                             **more)
    grad, = torch.autograd.grad(loss, [leaf], upstream)
    assert not rewards.requires_grad
    return {"loss": loss.detach(), "rewards": rewards, "dlog_probs": grad}


def _check_preference(x, cu, args, upstream, got):
    ref = step.preference(x, cu, upstream=upstream, **args)
    torch.testing.assert_close(got["rewards"].double().cpu(), ref["rewards"], rtol=2 * E,
                               atol=1e-12)
    # m cancels: what 64 bits leave of the rewards' sum.
    slack = 1e-11 * (1 + ref["rewards"].abs().max().item() + abs(args.get("margin", 0.0)))
    steep = 2 / args.get("beta", 0.1) ** 2 * (1 + ref["m"].abs().max().item())
    torch.testing.assert_close(got["loss"].double().cpu(), ref["loss"], rtol=4 * E,
                               atol=slack * steep)
    want, value = ref["dlog_probs"], got["dlog_probs"]
    assert value.dtype == x.dtype and value.shape == x.shape
    value = value.double().cpu().flatten()
    assert not value[want == 0].any()
    allowed = (4 * E + ROUND[x.dtype] * (1 + E)) * want.abs() + STEP[x.dtype] + slack * steep * (
        want != 0)
    assert ((value - want).abs() <= allowed).all(), ((value - want).abs() - allowed).max()


PAIRED = {
    "one token": [1, 1],
    "one pair": [300, 411],
    "empty sides": [0, 5, 64, 0, 0, 0, 63, 65, 127, 129, 1, 128],
    "tiny": [1 + (i * 7) % 5 for i in range(700)],
    "rounds": [64] * 40,
    "tiles": [512, 511, 513, 1, 128, 384, 512, 1024],
    "beyond one workgroup": [8000, 193, 0, 4000, 61, 62, 500, 3],
    "many pieces": [30000, 1, 40000, 129],
}


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("layout", PAIRED)
def test_preference(layout, kind):
    print(f"case {layout} {kind}", flush=True)
    for normalize, masked, reduction in ((False, 0.0, "mean"), (True, 0.3, "mean"),
                                         (False, 0.3, "sum"), (True, 0.0, "none")):
        cu, n = _offsets(PAIRED[layout], tail=9 if masked else 0)
        x, _, reference = _logs(n, seed=len(layout))
        mask = (torch.rand(n, generator=_gen(1)) >= masked).to(DEV) if masked else None
        args = {"reference": None if normalize else reference, "mask": mask,
                "beta": 0.3 if normalize else 0.02, "margin": 0.1, "kind": kind,
                "label_smoothing": 0.1 if kind == "sigmoid" else 0.0, "normalize": normalize,
                "reduction": reduction}
        pairs = len(PAIRED[layout]) // 2
        up = torch.randn(pairs, generator=_gen(2)).to(DEV) if reduction == "none" \
            else torch.tensor(0.6, device=DEV)
        _check_preference(x, cu, args, up, _run_preference(x, cu, args, up))


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("reference_dtype", ROUND)
def test_preference_types(dtype, reference_dtype):
    cu, n = _offsets(PAIRED["tiles"])
    x, _, reference = _logs(n, seed=20)
    args = {"reference": reference.to(reference_dtype), "mask": None}
    one = torch.tensor(1.0, device=DEV)
    _check_preference(x.to(dtype), cu, args, one, _run_preference(x.to(dtype), cu, args, one))


@pytest.mark.parametrize("lengths", ["one", "many"])
def test_preference_large(lengths):
    layout = [200001, 100002] if lengths == "one" else torch.randint(
        9, (60000,), generator=_gen(21)).tolist() + [3000, 2000]
    print(f"case {lengths} {sum(layout)} tokens", flush=True)
    cu, n = _offsets(layout, tail=11)
    x, _, reference = _logs(n, seed=22)
    args = {"reference": reference, "mask": None, "beta": 0.05}
    one = torch.tensor(1.0, device=DEV)
    _check_preference(x, cu, args, one, _run_preference(x, cu, args, one))


def test_preference_far_apart_answers_keep_their_slope():
    """sigma(-m) of m up to 80, which 1 - sigma(m) has lost from 17 on in 32 bits."""
    cu, n = _offsets([1, 1] * 5)
    x = torch.zeros(n, device=DEV)
    x[1::2] = -torch.tensor([1.0, 5.0, 20.0, 40.0, 80.0], device=DEV)
    args = {"reference": None, "mask": None, "beta": 1.0, "reduction": "none"}
    up = torch.ones(5, device=DEV)
    got = _run_preference(x, cu, args, up)
    want = step.preference(x, cu, upstream=up, **args)
    torch.testing.assert_close(got["loss"].double().cpu(), want["loss"], rtol=4 * E, atol=0)
    torch.testing.assert_close(got["dlog_probs"].double().cpu(), want["dlog_probs"], rtol=4 * E,
                               atol=0)


def test_preference_tokens_without_part_may_hold_anything():
    cu, n = _offsets([500, 40, 700, 31], tail=30)
    x, _, reference = _logs(n, seed=23)
    mask = (torch.rand(n, generator=_gen(24)) >= 0.3).to(torch.uint8).to(DEV)
    args, one = {"reference": reference, "mask": mask}, torch.tensor(1.0, device=DEV)
    clean = _run_preference(x, cu, args, one)
    out = mask == 0
    out[-30:] = True
    x[out], reference[out] = math.nan, math.inf
    got = _run_preference(x, cu, args, one)
    assert all(torch.equal(got[name], clean[name]) for name in got)


def test_c_abi_writes_what_the_operators_return():
    x, old, a, args, up = _policy([700, 301], reduction="sequence_mean", seed=25)
    want = _run_policy(x, old, a, args, up)
    loss, metrics = torch.empty(1, device=DEV), torch.empty(4, device=DEV)
    saved = capi.policy_loss_forward(
        x, old, a, loss=loss, metrics=metrics, reference_log_probs=args["reference"],
        entropy=args["entropy"], mask=args["mask"], cu_seqlens=args["cu_seqlens"], clip_low=0.2,
        clip_high=0.28, kl_weight=0.3, entropy_weight=0.05, reduction="sequence_mean")
    gx, gh = torch.empty_like(x), torch.empty_like(x)
    capi.policy_loss_backward(up, saved, tokens=1001, mask=args["mask"],
                              cu_seqlens=args["cu_seqlens"], entropy_weight=0.05,
                              reduction="sequence_mean", grad_log_probs=gx, grad_entropy=gh)
    for name, t in (("loss", loss[0]), ("metrics", metrics), ("dlog_probs", gx),
                    ("dentropy", gh)):
        assert torch.equal(t, want[name]), name
    args, one = {"reference": old, "mask": None}, torch.tensor(1.0, device=DEV)
    cu = torch.tensor([0, 700, 1001], dtype=torch.int32, device=DEV)
    want = _run_preference(x, cu, args, one)
    rewards = torch.empty(1, 2, device=DEV)
    saved = capi.preference_loss_forward(x, cu, loss=loss, rewards=rewards,
                                         reference_log_probs=old)
    capi.preference_loss_backward(one, saved, cu, grad_log_probs=gx)
    for name, t in (("loss", loss[0]), ("rewards", rewards), ("dlog_probs", gx)):
        assert torch.equal(t, want[name]), name


def test_subclasses_take_the_tables():
    class Wrapped(torch.Tensor):
        pass

    case = x, old, a, args, up = _policy([300, 41], reduction="sequence_mean", seed=26)
    want = _run_policy(*case)
    got = _run_policy(x.as_subclass(Wrapped), old, a, args, up)
    for name in want:
        assert torch.equal(got[name].as_subclass(torch.Tensor), want[name]), name
    cu = torch.tensor([0, 300, 341], dtype=torch.int32, device=DEV)
    args, one = {"reference": old, "mask": None}, torch.tensor(1.0, device=DEV)
    want = _run_preference(x, cu, args, one)
    got = _run_preference(x.as_subclass(Wrapped), cu, args, one)
    for name in want:
        assert torch.equal(got[name].as_subclass(torch.Tensor), want[name]), name


def test_the_graph_is_kept_or_freed_as_asked():
    x, old, _ = _logs(20, seed=27)
    cu = torch.tensor([0, 11, 20], dtype=torch.int32, device=DEV)
    leaf = x.clone().requires_grad_()
    for loss in (pretrain_policy_loss(leaf, old, old), pretrain_preference_loss(leaf, cu)[0]):
        first, = torch.autograd.grad(loss, [leaf], retain_graph=True)
        assert torch.equal(torch.autograd.grad(loss, [leaf])[0], first)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(loss, [leaf])
    # A tensor of the caller's that the backward reads and that has changed since.
    mask = torch.ones(20, dtype=torch.bool, device=DEV)
    loss, _ = pretrain_preference_loss(leaf, cu, mask=mask)
    mask[3] = False
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("reduction", [-1, 4, 2 ** 32])
def test_ops_refuse_unknown_reductions(reduction):
    """Also one whose low 32 bits are a known one."""
    x, old, _ = _logs(20, seed=27)
    cu = torch.tensor([0, 11, 20], dtype=torch.int32, device=DEV)
    ops = torch.ops.flashrwkv2
    _, saved = ops.policy_loss_forward(x, old, old, None, None, None, None, 0.2, 0.2, 0.0, 0.0,
                                       0.0, 1, False, True)
    _, _, pair_saved = ops.preference_loss_forward(x, cu, None, None, 0.1, 0.0, 0.0, 0, False, 1)
    up = torch.ones((), device=DEV)
    for call in (
            lambda: ops.policy_loss_forward(x, old, old, None, None, None, None, 0.2, 0.2, 0.0,
                                            0.0, 0.0, reduction, False, True),
            lambda: ops.policy_loss_backward(up, saved, None, None, [20], torch.float32,
                                             torch.float32, 0.0, reduction, True, False),
            lambda: ops.preference_loss_forward(x, cu, None, None, 0.1, 0.0, 0.0, 0, False,
                                                reduction),
            lambda: ops.preference_loss_backward(up, pair_saved, cu, None, [20], torch.float32,
                                                 reduction)):
        with pytest.raises(RuntimeError, match="unknown reduction"):
            call()


def test_forward_mode_is_refused():
    x, old, _ = _logs(20, seed=27)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            pretrain_policy_loss(dual, old, old)
        cu = torch.tensor([0, 11, 20], dtype=torch.int32, device=DEV)
        for call in (lambda: pretrain_policy_loss(x, dual, old),
                     lambda: pretrain_policy_loss(x, old, dual),
                     lambda: pretrain_policy_loss(x, old, old, reference_log_probs=dual),
                     lambda: pretrain_preference_loss(x, cu, reference_log_probs=dual),
                     lambda: flashrwkv_amd.pretrain_grad_norm([x, dual]),
                     lambda: flashrwkv_amd.pretrain_clip_grad_norm([dual], 1.0, out=[old])):
            with pytest.raises(ValueError, match="must not require gradients"):
                call()
        with pytest.raises((RuntimeError, NotImplementedError)):
            pretrain_policy_loss(x, old, old, entropy=dual, entropy_weight=0.1)


def test_backward_on_a_capturing_stream_is_refused():
    x, old, _ = _logs(20, seed=27)
    leaf = x.clone().requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        loss = pretrain_policy_loss(leaf, old, old)
        one = torch.ones((), device=DEV)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="graph capture"):
                torch.autograd.grad(loss, [leaf], one)
        finally:
            graph.capture_end()


def test_second_derivatives_and_captures_are_refused():
    x, old, _ = _logs(20, seed=27)
    cu = torch.tensor([0, 11, 20], dtype=torch.int32, device=DEV)
    leaf = x.clone().requires_grad_()

    def losses():
        return (pretrain_policy_loss(leaf, old, old), pretrain_preference_loss(leaf, cu)[0])

    for loss in losses():
        grad, = torch.autograd.grad(loss, [leaf], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiat"):
            grad.sum().backward()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            for call in (lambda: pretrain_policy_loss(leaf, old, old),
                         lambda: pretrain_preference_loss(leaf, cu)):
                with pytest.raises(RuntimeError, match="graph capture"):
                    call()
        finally:
            graph.capture_end()


@pytest.mark.parametrize("offsets", [[1, 11, 20], [0, 15, 11], [0, 11, 21], [0, -900, 20],
                                     [0, 1 << 30, 20], [-3, 11, 20]])
def test_offsets_that_may_not_be_make_loss_and_gradients_nan(offsets):
    """Every index made from offsets is bounded in the kernels; what they compute is
    marked."""
    x, old, _ = _logs(20, seed=28)
    cu = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    leaf = x.clone().requires_grad_()
    for reduction in ("mean", "sum", "sequence_mean"):
        loss = pretrain_policy_loss(leaf, old, old, cu_seqlens=cu, reduction=reduction)
        assert torch.isnan(loss)
        assert torch.isnan(torch.autograd.grad(loss, [leaf])[0]).any()
    loss, _ = pretrain_preference_loss(leaf, cu)
    assert torch.isnan(loss)


@pytest.mark.parametrize("log_dtype", ROUND)
@pytest.mark.parametrize("offsets", ["start", "late fall", "beyond"])
@pytest.mark.parametrize("n,sequences", [(20, 4), (5000, 10), (5000, 2000), (300_000, 3000)])
def test_offsets_that_may_not_be_mark_every_gradient(n, sequences, offsets, log_dtype):
    """In one workgroup's form and in those of two launches, one bad offset among many:
    gradients of clipped tokens, of satisfied pairs and of masked tokens too."""
    cu = (torch.arange(sequences + 1) * n // sequences).to(torch.int32)
    if offsets == "start":
        cu[0] = 1
    elif offsets == "late fall":
        cu[-2] = cu[-3] - 1
    else:
        cu[-1] = n + 1
    cu = cu.to(DEV)
    x, old, _ = _logs(n, seed=28)
    # Half of the ratios are clipped, half have an advantage of 0; all pairs are satisfied.
    x, a = x.to(log_dtype), torch.zeros(n, device=DEV)
    old[::2], a[::2] = old[::2] - 1000.0, 1.0
    mask = (torch.rand(n, generator=_gen(29)) >= 0.3).to(DEV)
    for reduction in ("mean", "sum", "sequence_mean", "none"):
        print(f"case {n} {sequences} {offsets} {log_dtype} {reduction}", flush=True)
        leaf = x.clone().requires_grad_()
        entropy = torch.ones_like(x).requires_grad_()
        loss = pretrain_policy_loss(leaf, old, a, cu_seqlens=cu, mask=mask, entropy=entropy,
                                    entropy_weight=0.1, reduction=reduction)
        assert reduction == "none" or torch.isnan(loss)
        for grad in torch.autograd.grad(loss.sum(), [leaf, entropy]):
            assert torch.isnan(grad).all()
    for reduction in ("mean", "sum", "none"):
        for kind, margin in (("sigmoid", 0.0), ("hinge", -1e30)):
            leaf = x.clone().requires_grad_()
            loss, _ = pretrain_preference_loss(leaf, cu, mask=mask, kind=kind, margin=margin,
                                               reduction=reduction)
            assert reduction == "none" or torch.isnan(loss)
            assert torch.isnan(torch.autograd.grad(loss.sum(), [leaf])[0]).all()


SIZES = [2, 300, 2048, 2049, 4096, 4097, 262144, 262145]


@pytest.mark.parametrize("reduction", ["mean", "sum", "sequence_mean"])
@pytest.mark.parametrize("n", SIZES)
def test_policy_sums_hold_what_32_bits_do_not(n, reduction):
    """Terms that cancel, each of them exact: 2^25 at the ends and 1 between, whose sum is
    n - 2, rounded once. And ratios of 3.3e38, of which two have a mean but no sum."""
    cu, _ = _offsets([n])
    zeros = torch.zeros(n, device=DEV)
    a = -torch.ones(n, device=DEV)
    a[0], a[-1] = -2.0 ** 25, 2.0 ** 25
    loss = pretrain_policy_loss(zeros, zeros, a, cu_seqlens=cu, reduction=reduction)
    want = (n - 2) / (1 if reduction == "sum" else n)
    assert abs(loss.item() - want) <= 2 * E * want
    if reduction == "sum":
        return
    high = torch.full((n,), 88.7, device=DEV)
    d = high[0].double().item()
    loss, metrics = pretrain_policy_loss(high, zeros, torch.full_like(high, -1.0), metrics=True,
                                         cu_seqlens=cu, reduction=reduction)
    k = (16 + d) * E
    for value, want in ((loss, math.exp(d)), (metrics[0], math.exp(d)),
                        (metrics[2], math.expm1(d) - d)):
        assert abs(value.item() - want) <= k * want


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_a_rejected_answer_that_cannot_be_has_no_loss(reduction):
    """m = inf: the term that label_smoothing 0 leaves out is infinite."""
    cu, n = _offsets([3, 2, 4, 1])
    x, _, _ = _logs(n, seed=32)
    x[4] = -math.inf
    args = {"reference": None, "mask": None, "reduction": reduction}
    up = torch.ones(2 if reduction == "none" else (), device=DEV)
    got = _run_preference(x, cu, args, up)
    clean = x.clone()
    clean[4] = -1e6
    want = _run_preference(clean, cu, args, up)
    assert torch.equal(got["loss"], want["loss"]) and torch.isfinite(got["loss"]).all()
    assert torch.equal(got["dlog_probs"], want["dlog_probs"])
    assert not got["dlog_probs"][:5].any() and got["dlog_probs"][5:].all()
    assert got["rewards"][0, 1].item() == -math.inf
    # With smoothing the rejected answer's own term is there, and infinite.
    got = _run_preference(x, cu, args | {"label_smoothing": 0.1}, up)
    assert math.isinf(got["loss"].flatten()[0].item())


@pytest.mark.parametrize("reduction", ["mean", "sum", "sequence_mean", "none"])
@pytest.mark.parametrize("n", [300, 5000])
def test_terms_of_weight_zero_are_not_there(n, reduction):
    """A reference that is only looked at (metrics) and an entropy without a bonus reach
    neither loss nor gradient, whatever they hold: a reference's k3 is infinite from 89 on."""
    x, old, a, args, up = _policy([n - 100, 100], reduction=reduction, seed=33)
    args |= {"reference": None, "entropy": None, "kl_weight": 0.0, "entropy_weight": 0.0}
    want = _run_policy(x, old, a, args, up)
    taking = args["mask"].nonzero()[:, 0]
    reference = x - 0.5
    reference[taking[3]], reference[taking[7]] = 100.0, 1e30
    entropy = torch.zeros_like(x)
    entropy[taking[5]], entropy[taking[9]] = math.inf, math.nan
    got = _run_policy(x, old, a, args | {"reference": reference, "entropy": entropy}, up)
    for name in ("loss", "dlog_probs"):
        assert torch.equal(got[name], want[name]), name
    assert torch.equal(got["metrics"][:3], want["metrics"][:3])
    assert got["metrics"][3].item() == math.inf
    assert not got["dentropy"].any()


# ------------------------------------------------ at the borders of the forms
# One workgroup with tiles of 128 tokens up to 2048 and of 256 up to 4096; beyond, two launches
# with tiles of 128 up to 262144 tokens and of 256 from there on; up to 64 pieces (tiles) of a
# sequence are added by one lane, more by a wave.
BORDERS = {
    **{str(n): [n // 3, n - n // 3 - 65, 64, 1] for n in SIZES if n > 300},
    "tiles of 128": [128, 127, 129, 256, 255, 257, 1, 128, 3900, 5],
    "64 and 65 pieces": [8192, 8193, 8191, 64],
    "64 and 65 long pieces": [16384, 16385, 16383, 250000],
    "one long pair": [200001, 150002],
    "many": torch.randint(9, (80000,), generator=_gen(34)).tolist(),
}


@pytest.mark.parametrize("reduction", ["mean", "sequence_mean", "none"])
@pytest.mark.parametrize("layout", BORDERS)
def test_policy_at_the_borders_of_its_forms(layout, reduction):
    print(f"case {layout} {reduction}", flush=True)
    for per_sequence in (False, True):
        case = _policy(BORDERS[layout], reduction=reduction, per_sequence=per_sequence, seed=35)
        _check_policy(*case, _run_policy(*case))


def _pairs(x, cu, args, upstream):
    """What oracle/step.py's preference gives, without its loop over sequences, and of each
    sequence its count, the sum of its terms' sizes and the factor of its sum."""
    n, offsets = x.numel(), cu.cpu().long()
    lengths = torch.cat([offsets.diff(), n - offsets[-1:]])
    owner = torch.arange(lengths.numel()).repeat_interleave(lengths)
    part = owner < lengths.numel() - 1
    if args["mask"] is not None:
        part &= args["mask"].cpu()
    terms = x.double().cpu()
    if args["reference"] is not None:
        terms = terms - args["reference"].double().cpu()
    zeros = torch.zeros(lengths.numel() - 1, dtype=torch.float64)
    counts = zeros.index_add(0, owner[part], torch.ones(int(part.sum()), dtype=torch.float64))
    sums = zeros.index_add(0, owner[part], terms[part])
    sizes = zeros.index_add(0, owner[part], terms[part].abs())
    by = 1 / counts.clamp_min(1) if args["normalize"] else torch.ones_like(counts)
    beta, eps = args["beta"], args["label_smoothing"]
    rewards = (beta * sums * by).view(-1, 2)
    m = rewards[:, 0] - rewards[:, 1] - args["margin"]
    taking = counts.view(-1, 2).amin(1) > 0
    if args["kind"] == "sigmoid":
        log_sigmoid = torch.nn.functional.logsigmoid
        each = -(1 - eps) * log_sigmoid(m) - eps * log_sigmoid(-m)
        slope = eps * torch.sigmoid(m) - (1 - eps) * torch.sigmoid(-m)
    elif args["kind"] == "hinge":
        each, slope = torch.relu(1 - m), -(m < 1).double()
    else:
        each, slope = ((m - 0.5) / beta) ** 2, 2 * (m - 0.5) / beta ** 2
    each, slope = torch.where(taking, each, 0.0), torch.where(taking, slope, 0.0)
    share = 1 / max(1, int(taking.sum())) if args["reduction"] == "mean" else 1.0
    up = upstream.double().cpu().expand(m.numel())
    coefficient = torch.stack([slope, -slope], 1).view(-1) * by * beta * share \
        * up.repeat_interleave(2)
    grad = torch.where(part, coefficient[owner.clamp_max(lengths.numel() - 2)], 0.0)
    return {"m": m, "rewards": rewards, "each": each, "taking": taking, "share": share,
            "loss": each if args["reduction"] == "none" else each.sum() * share,
            "dlog_probs": grad, "counts": counts, "sizes": sizes, "by": by, "part": part,
            "owner": owner.clamp_max(lengths.numel() - 2)}


def _check_pairs(x, cu, args, upstream, got):
    """Within what 64 bits leave of m, and the roundings to 32 bits behind it.

    A sum of L terms is off by at most (L + 8) 2^-53 of the sum of their sizes, here and in
    the oracle, so m by delta = (L + 8) 2^-52 (beta sum |terms| + |margin|). Loss: |dl/dm|
    delta (64-bit roundings of the pairs' sum beside it) and two roundings to 32 bits.
    Gradient: |d2l/dm2| delta through beta, share and 1 / count, and the roundings of
    coefficient, share and two products to 32 bits."""
    kind, beta, margin = args["kind"], args["beta"], args["margin"]
    ref = _pairs(x, cu, args, upstream)
    if ref["m"].numel() < 100:
        plain = step.preference(x, cu, upstream=upstream, **args)
        for name in ("m", "loss", "rewards", "dlog_probs"):
            torch.testing.assert_close(ref[name], plain[name], rtol=1e-9, atol=1e-12)
    m, by, share, taking = ref["m"], ref["by"], ref["share"], ref["taking"]
    off = 2.0 ** -52 * (ref["counts"].max() + 8)
    reward_off = off * beta * ref["sizes"] * by
    delta = reward_off.view(-1, 2).sum(1) + off * abs(margin)
    want = ref["rewards"].flatten()
    value = got["rewards"].double().cpu().flatten()
    assert ((value - want).abs() <= reward_off + E * want.abs()).all()
    if kind == "sigmoid":
        steep, curved = torch.ones_like(m), torch.full_like(m, 0.25)
    elif kind == "hinge":
        steep, curved = torch.ones_like(m), torch.zeros_like(m)
        assert ((1 - m).abs() > delta)[taking].all()  # none is on the kink
    else:
        curved = torch.full_like(m, 2 / beta ** 2)
        steep = curved * ((m - 0.5).abs() + delta)
    each_off = torch.where(taking, steep * delta + 2.0 ** -49 * ref["each"].abs(), 0.0)
    value = got["loss"].double().cpu()
    if args["reduction"] == "none":
        allowed = each_off + 2 * E * ref["each"].abs()
    else:
        allowed = share * (each_off.sum() + m.numel() * 2.0 ** -52 * ref["each"].abs().sum()) \
            + 2 * E * ref["loss"].abs()
    assert ((value - ref["loss"]).abs() <= allowed).all(), (value, ref["loss"])
    up = upstream.double().cpu().abs().expand(m.numel())
    slack = (curved * delta * beta * share * up).repeat_interleave(2) * by
    want, value = ref["dlog_probs"], got["dlog_probs"].double().cpu()
    allowed = 4 * E * (1 + 4 * E) * want.abs() + STEP[x.dtype] + torch.where(
        ref["part"], slack[ref["owner"]], 0.0)
    assert ((value - want).abs() <= allowed).all(), ((value - want).abs() - allowed).max()
    # What is compared is far above what is allowed.
    largest = want.abs().argmax()
    assert want[largest].abs() >= 1e4 * allowed[largest] > 0.0


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("layout", BORDERS)
def test_preference_at_the_borders_of_its_forms(layout, kind):
    lengths = BORDERS[layout]
    print(f"case {layout} {kind} {sum(lengths)} tokens, {len(lengths)} sequences", flush=True)
    for normalize, masked, reduction in ((False, 0.0, "mean"), (True, 0.3, "mean"),
                                         (False, 0.3, "sum"), (True, 0.0, "none")):
        cu, n = _offsets(lengths, tail=9 if masked else 0)
        x, _, reference = _logs(n, seed=len(lengths) + 36)
        mask = (torch.rand(n, generator=_gen(37)) >= masked).to(DEV) if masked else None
        args = {"reference": None if normalize else reference, "mask": mask, "beta": 1.0,
                "margin": 0.1, "kind": kind, "normalize": normalize, "reduction": reduction,
                "label_smoothing": 0.1 if kind == "sigmoid" else 0.0}
        # m within 0.9, where no kind is flat or saturated.
        up = torch.randn(len(lengths) // 2, generator=_gen(38)).to(DEV) if reduction == "none" \
            else torch.tensor(0.6, device=DEV)
        args["beta"] = 0.8 / _pairs(x, cu, args, up)["rewards"].diff(dim=1).abs().max().item()
        _check_pairs(x, cu, args, up, _run_preference(x, cu, args, up))


def test_the_borders_are_those_of_the_forms():
    assert sum(BORDERS["many"]) > 262145 and len(BORDERS["many"]) > 64 * 1024
    assert sum(BORDERS["64 and 65 pieces"]) in range(4097, 262145)
    assert sum(BORDERS["64 and 65 long pieces"]) > 262144


def test_what_is_kept_may_be_moved_or_made_again():
    """Hooks on saved tensors: kept on the host between forward and backward, or made again by
    a checkpoint."""
    case = x, old, a, args, up = _policy([3000, 2100], reduction="sequence_mean", seed=39)
    cu = args["cu_seqlens"]
    pairs = {"reference": old, "mask": args["mask"]}
    for run in (lambda: _run_policy(*case), lambda: _run_preference(x, cu, pairs, up)):
        want = run()
        with torch.autograd.graph.save_on_cpu():
            got = run()
        assert all(torch.equal(got[name], want[name]) for name in want)
    leaf = x.clone().requires_grad_()

    def both(leaf):
        return (pretrain_policy_loss(leaf, old, a, cu_seqlens=cu, mask=args["mask"])
                + pretrain_preference_loss(leaf, cu, mask=args["mask"])[0])

    want, = torch.autograd.grad(both(leaf), [leaf])
    again = torch.utils.checkpoint.checkpoint(both, leaf, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(again, [leaf])[0], want)


def test_as_many_tokens_as_offsets_can_name():
    """2^31 - 1 tokens in three sequences and an empty one: ratios of 1, a ratio of 2 at the
    ends of the sequences, whose tokens are found behind 2^32 bytes."""
    n = 2 ** 31 - 1
    cu = torch.tensor([0, 5, n - 1000, n - 1000, n - 1], dtype=torch.int32, device=DEV)
    x = torch.zeros(n, device=DEV)
    x[4] = x[n - 1001] = x[n - 2] = math.log(2.0)
    x[n - 1] = math.nan  # behind the last sequence
    old = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    a = torch.tensor([-1.0, -2.0, 7.0, -4.0], device=DEV)
    leaf = x.requires_grad_()
    means = [(6.0, 5), (2.0 * (n - 1005) + 2.0, n - 1005), (4.0 * 999 + 4.0, 999)]
    for reduction, want in (("sequence_mean", sum(s / k for s, k in means) / 3),
                            ("mean", sum(s for s, _ in means) / (n - 1))):
        loss, metrics = pretrain_policy_loss(leaf, old, a, cu_seqlens=cu, reduction=reduction,
                                             metrics=True)
        assert abs(loss.item() - want) <= 24 * E * want
        assert abs(metrics[0].item() - 1.0) <= 24 * E
        grad, = torch.autograd.grad(loss, [leaf])
        for i, slope, k in ((4, 2.0, 5), (0, 1.0, 5), (5, 2.0, n - 1005), (n - 1001, 4.0, n - 1005),
                            (n - 1000, 4.0, 999), (n - 2, 8.0, 999), (n - 1, 0.0, 1)):
            share = 1 / (3 * k) if reduction == "sequence_mean" else 1 / (n - 1)
            assert abs(grad[i].item() - slope * share) <= 24 * E * slope * share
        del grad, loss
    # Pairs: the second has an empty side and takes no part.
    cu = torch.tensor([0, 5, n - 1000, n - 1000, n - 1], dtype=torch.int32, device=DEV)
    loss, rewards = pretrain_preference_loss(leaf, cu, beta=1.0)
    two = math.log(2.0)
    want = [two, two, 0.0, two]
    assert all(abs(r - w) <= 4 * E for r, w in zip(rewards.flatten().tolist(), want))
    assert abs(loss.item() - two) <= 4 * E
    grad, = torch.autograd.grad(loss, [leaf])
    for i, value in ((0, -0.5), (4, -0.5), (5, 0.5), (n - 1001, 0.5), (n - 1000, 0.0),
                     (n - 2, 0.0), (n - 1, 0.0)):
        assert abs(grad[i].item() - value) <= 4 * E
    assert grad[5:n - 1000].min().item() == grad[5:n - 1000].max().item()
    assert not grad[n - 1000:].any()

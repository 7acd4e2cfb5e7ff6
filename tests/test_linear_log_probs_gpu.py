"""GPU parity of log probabilities and entropies from hidden rows against
oracle/step.py (64 bits).

Bounds, before any run. With A = max over rows and vocabulary of sum_c |h W| a
logit is off by at most gamma A, gamma = (sqrt(C) + 16) 2^-24, and so is its log
sum; exponential and logarithm add a few 2^-24 of their exponents:
  delta = 2 gamma A / T + 8 2^-24 (1 + |z| / T + |lse|)    (relative error of q)
  log_probs: 1.5 delta.
  entropy:   its derivative in log q is -q (log q + H), so delta moves it by at most
             2 delta (sum q |log q| + H); its sums of V terms add
             (sqrt(V) + 32) 2^-24 (1 + sum q |log q|).
  gradients: dz is off by u |dz| (one rounding to 16 bits; u^2 in the two terms that up to
             32 rows keep) + delta / T (|g| (q + b) + |e| q (2 |log q + H| + 2 + H)),
             and a product of n such terms adds gamma_n sum |dz| |factor| and the output's
             rounding u |ref|. fp16 adds its smallest step.
"""

from __future__ import annotations

import math

import pytest
import torch

import flashrwkv_amd
from flashrwkv_amd import capi, pretrain_linear_cross_entropy, pretrain_linear_log_probs
from oracle import step

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
E = 2.0 ** -24
IGNORE = -100


@pytest.fixture(scope="module", autouse=True)
def _require_native():
    if flashrwkv_amd._C is None:
        pytest.fail("flashrwkv_amd native library is not built (no fallback exists)")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _case(n, c, v, dtype, seed, masked=0.3, scale=2.0, index=torch.int64):
    gen = _gen(seed)
    h = torch.randn(n, c, generator=gen).to(dtype)
    w = (torch.randn(v, c, generator=gen) * (scale / math.sqrt(c))).to(dtype)
    targets = torch.randint(v, (n,), generator=gen).to(index)
    targets[torch.rand(n, generator=gen) < masked] = IGNORE
    g = torch.randn(n, generator=gen)
    e = torch.randn(n, generator=gen)
    return [t.to(DEV) for t in (h, w, targets, g, e)]


def _check(h, w, targets, got, *, temperature, g=None, e=None):
    """got: dict of what was asked for."""
    u, least = ROUND[h.dtype], STEP[h.dtype]
    ref = step.scores(h, w, targets, temperature=temperature, grad_log_probs=g, grad_entropy=e)
    rows = ref["rows"]
    n, vocab = rows.numel(), w.shape[0]
    for name in ("log_probs", "entropy"):
        if name in got:
            assert got[name].dtype == torch.float32 and got[name].shape == targets.shape
            assert not got[name][targets == IGNORE].any()
    if n == 0:
        assert all(not t.any() for t in got.values())
        return
    z = h.double()[rows] @ w.double().t()
    a = (h.double()[rows].abs() @ w.double().abs().t()).max().item()
    gamma = (math.sqrt(h.shape[1]) + 16) * E
    log_q = torch.log_softmax(z / temperature, 1)
    lse = torch.logsumexp(z / temperature, 1).abs().max().item()
    delta = 2 * gamma * a / temperature + 8 * E * (1 + lse + z.abs().max().item() / temperature)
    entropy, spread = ref["entropy"][rows, None], ref["abs_entropy"]
    off = (got["log_probs"].double() - ref["log_probs"]).abs().max().item()
    assert off <= 1.5 * delta, (off, delta)
    if "entropy" in got:
        allowed = (2 * delta * (spread + ref["entropy"])
                   + (math.sqrt(vocab) + 32) * E * (1 + spread))
        worst = ((got["entropy"].double() - ref["entropy"]).abs() - allowed).max().item()
        assert worst <= 0, worst
    if "dhidden" not in got and "dweight" not in got:
        return
    q = torch.exp(log_q)
    b = torch.zeros_like(q).scatter_(1, targets[rows].long()[:, None], 1.0)
    gs = torch.zeros(n, 1, device=DEV).double() if g is None else g.double()[rows, None].abs()
    es = torch.zeros(n, 1, device=DEV).double() if e is None else e.double()[rows, None].abs()
    dz = ref["dz"].abs()
    terms = 2 if n <= 32 else 1
    dz_off = u ** terms * dz + delta / temperature * (
        gs * (q + b) + es * q * (2 * (log_q + entropy).abs() + 2 + entropy))
    # fp16 keeps its logit gradients on a grid of 2^-38 of the largest row's bound at worst.
    grid = 2.0 ** -38 * ((gs + es * (math.log(vocab) + 1)).max().item() / temperature)
    for name, count, factor, spent in (
            ("dhidden", vocab, w.double().abs(), dz_off @ w.double().abs()),
            ("dweight", n, h.double()[rows].abs(), dz_off.t() @ h.double()[rows].abs())):
        if name not in got:
            continue
        want, value = ref[name], got[name]
        allowed = torch.zeros_like(want)
        if name == "dhidden":
            allowed[rows] = spent
        else:
            allowed = spent
        allowed += ((math.sqrt(count) + 16) * E * ref[f"abs_{name}"] + u * want.abs() * (1 + u)
                    + least + grid * count * factor.max().item())
        assert value.dtype == h.dtype and torch.isfinite(value).all(), name
        worst = ((value.double() - want).abs() - allowed).max().item()
        assert worst <= 0, f"{name}: {worst:.3e} over its bound"


def _run(h, w, targets, g, e, *, temperature=1.0, entropy=True, hidden=True, weight=True):
    h = h.detach().clone().requires_grad_(hidden)
    w = w.detach().clone().requires_grad_(weight)
    got = pretrain_linear_log_probs(h, w, targets, temperature=temperature, entropy=entropy)
    got = got if entropy else (got,)
    out = {name: t.detach() for name, t in zip(("log_probs", "entropy"), got)}
    used = [(t, up) for t, up in zip(got, (g, e)) if up is not None]
    leaves = [(name, t) for name, t in (("dhidden", h), ("dweight", w)) if t.requires_grad]
    if used and leaves:
        grads = torch.autograd.grad([t for t, _ in used], [t for _, t in leaves],
                                    [up for _, up in used])
        out |= dict(zip([name for name, _ in leaves], grads))
    return out


SHAPES = [(1, 64, 1), (1, 64, 300), (1, 2048, 1000), (2, 128, 255), (33, 192, 256), (64, 64, 257),
          (65, 320, 513), (255, 128, 100), (257, 448, 999), (520, 1024, 770), (1100, 64, 2050)]


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("n,c,v", SHAPES)
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_scores_and_gradients(n, c, v, dtype, temperature):
    print(f"case {n}x{c} vocab {v} {dtype} T {temperature}", flush=True)
    h, w, targets, g, e = _case(n, c, v, dtype, seed=n + c + v)
    for ups in ((g, e), (g, None), (None, e)):
        got = _run(h, w, targets, *ups, temperature=temperature)
        _check(h, w, targets, got, temperature=temperature, g=ups[0], e=ups[1])
    plain = _run(h, w, targets, g, None, temperature=temperature, entropy=False)
    _check(h, w, targets, plain, temperature=temperature, g=g)
    # What is not asked for changes nothing else.
    full = _run(h, w, targets, g, e, temperature=temperature)
    for hidden, weight in ((True, False), (False, True), (False, False)):
        part = _run(h, w, targets, g, e, temperature=temperature, hidden=hidden, weight=weight)
        assert all(torch.equal(part[name], full[name]) for name in part)


def test_is_minus_the_cross_entropy_at_temperature_one():
    h, w, targets, _, _ = _case(300, 256, 1000, torch.bfloat16, seed=1)
    got = pretrain_linear_log_probs(h, w, targets)
    assert torch.equal(got, -pretrain_linear_cross_entropy(h, w, targets, reduction="none"))


@pytest.mark.parametrize("dtype", ROUND)
def test_a_large_vocabulary_in_pieces(dtype):
    """Enough rows and tokens for large and small tiles and more than one piece."""
    n, c, v = 4096, 64, 70000
    assert capi.linear_loss_backward_plan(n, c, v)[1] > 1
    h, w, targets, g, e = _case(n, c, v, dtype, seed=2, masked=0.1)
    _check(h, w, targets, _run(h, w, targets, g, e), temperature=1.0, g=g, e=e)


@pytest.mark.parametrize("n", [1, 40])
def test_a_weight_beyond_the_caches_is_read_alike(n):
    """Without a backward to follow few rows read a large weight past the caches."""
    c, v = 2048, 50000
    assert 2 * c * v > 192 << 20
    h, w, targets, _, _ = _case(n, c, v, torch.bfloat16, seed=12, masked=0.0)
    alone = pretrain_linear_log_probs(h, w, targets, entropy=True)
    followed = pretrain_linear_log_probs(h.clone().requires_grad_(), w, targets, entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(alone, followed))
    _check(h, w, targets, dict(zip(("log_probs", "entropy"), alone)), temperature=1.0)


@pytest.mark.parametrize("shape", [(), (6,), (2, 3)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_leading_shapes_and_index_types(shape, index):
    n = math.prod(shape)
    h, w, targets, g, e = _case(n, 64, 50, torch.bfloat16, seed=3, masked=0.0, index=index)
    flat = _run(h, w, targets, g, e)
    lead = _run(h.view(*shape, 64), w, targets.view(shape), g.view(shape), e.view(shape))
    for name in flat:
        assert lead[name].shape == (w.shape if name == "dweight" else
                                    (*shape, 64) if name == "dhidden" else shape)
        assert torch.equal(lead[name].flatten(), flat[name].flatten())


def test_no_rows_and_no_rows_that_take_part():
    h, w, _, _, _ = _case(4, 64, 50, torch.bfloat16, seed=4)
    none = torch.full((4,), IGNORE, device=DEV)
    ones = torch.ones(4, device=DEV)
    _check(h, w, none, _run(h, w, none, ones, ones), temperature=1.0, g=ones, e=ones)
    empty = _run(h[:0], w, none[:0], ones[:0], ones[:0])
    assert empty["log_probs"].shape == (0,) and empty["dhidden"].shape == (0, 64)
    assert not empty["dweight"].any()


def test_rows_that_take_no_part_may_hold_anything():
    h, w, targets, g, e = _case(200, 128, 300, torch.float16, seed=5)
    clean = _run(h, w, targets, g, e)
    out = targets == IGNORE
    h[out], g[out], e[out] = math.nan, math.inf, math.nan
    got = _run(h, w, targets, g, e)
    assert all(torch.equal(got[name], clean[name]) for name in got)


def test_targets_out_of_range_are_nan_in_their_row_alone():
    h, w, targets, g, e = _case(70, 64, 90, torch.bfloat16, seed=6, masked=0.0)
    clean = _run(h, w, targets, g, e)
    bad = targets.clone()
    bad[3], bad[44] = 90, -7
    got = _run(h, w, bad, g, e)
    keep = torch.ones(70, dtype=torch.bool, device=DEV)
    keep[3] = keep[44] = False
    for name in ("log_probs", "entropy", "dhidden"):
        assert torch.isnan(got[name][~keep]).all(), name
    for name in ("log_probs", "entropy"):
        assert torch.equal(got[name][keep], clean[name][keep])


def test_certain_and_uniform_rows():
    """One token far above the others has entropy 0 and no gradient; equal logits have
    log V, and gradients of the log probability alone."""
    c, v = 64, 500
    w = torch.zeros(v, c, device=DEV, dtype=torch.bfloat16)
    w[7, 0] = 1.0
    h = torch.zeros(2, c, device=DEV, dtype=torch.bfloat16)
    h[0, 0] = 30000.0
    targets = torch.tensor([7, 9], device=DEV)
    one = torch.ones(2, device=DEV)
    got = _run(h, w, targets, one, one)
    assert got["log_probs"][0] == 0 and got["entropy"][0] == 0
    assert abs(got["entropy"][1].item() - math.log(v)) <= 16 * E * math.log(v)
    assert abs(got["log_probs"][1].item() + math.log(v)) <= 16 * E * math.log(v)
    assert not got["dhidden"][0].any() and torch.isfinite(got["dweight"]).all()
    _check(h, w, targets, got, temperature=1.0, g=one, e=one)


@pytest.mark.parametrize("temperature", [1e-3, 50.0])
def test_extreme_temperatures_stay_finite(temperature):
    h, w, targets, g, e = _case(40, 128, 300, torch.bfloat16, seed=7)
    got = _run(h, w, targets, g, e, temperature=temperature)
    _check(h, w, targets, got, temperature=temperature, g=g, e=e)


def test_calls_repeat_bitwise_on_any_stream():
    h, w, targets, g, e = _case(300, 256, 1500, torch.bfloat16, seed=8)
    first = _run(h, w, targets, g, e)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = _run(h, w, targets, g, e)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(first[name], other[name]) for name in first)


def test_c_abi_writes_what_the_operator_returns():
    h, w, targets, g, e = _case(90, 128, 400, torch.bfloat16, seed=9)
    want = _run(h, w, targets, g, e, temperature=0.8)
    log_probs, entropy = torch.empty(90, device=DEV), torch.empty(90, device=DEV)
    saved = capi.linear_log_probs_forward(h, w, targets, log_probs=log_probs, entropy=entropy,
                                          temperature=0.8)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    capi.linear_log_probs_backward(g, e, w, saved, rows=90, temperature=0.8, grad_hidden=dh,
                                   grad_weight=dw)
    for name, t in (("log_probs", log_probs), ("entropy", entropy), ("dhidden", dh),
                    ("dweight", dw)):
        assert torch.equal(t, want[name]), name


def test_subclasses_and_modes_take_the_tables():
    class Wrapped(torch.Tensor):
        pass

    h, w, targets, g, e = _case(20, 64, 90, torch.bfloat16, seed=10)
    want = _run(h, w, targets, g, e)
    leaf = h.detach().clone().as_subclass(Wrapped).requires_grad_()
    log_probs, entropy = pretrain_linear_log_probs(leaf, w, targets, entropy=True)
    grad, = torch.autograd.grad([log_probs, entropy], [leaf], [g, e])
    assert torch.equal(log_probs.as_subclass(torch.Tensor), want["log_probs"])
    assert torch.equal(grad.as_subclass(torch.Tensor), want["dhidden"])


def test_second_derivatives_and_captures_are_refused():
    h, w, targets, _, _ = _case(5, 64, 90, torch.bfloat16, seed=11, masked=0.0)
    h.requires_grad_()
    grad, = torch.autograd.grad(pretrain_linear_log_probs(h, w, targets).sum(), [h],
                                create_graph=True)
    with pytest.raises(RuntimeError, match="differentiat"):
        grad.sum().backward()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="graph capture"):
                pretrain_linear_log_probs(h, w, targets)
        finally:
            graph.capture_end()


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("n", [3, 300])
@pytest.mark.parametrize("temperature", [1.1e-30, 1e-10])
def test_certain_rows_at_the_least_temperatures(temperature, n, dtype):
    """A token's distance from the others in units of the temperature, times the tokens of
    a sum, is beyond fp32: such rows have entropy 0 and no gradient. Rows of equal logits
    between them have log V. Upstream gradients of the temperature's size cancel 1 / T."""
    c, v = 64, 65536
    w = torch.zeros(v, c, device=DEV, dtype=dtype)
    w[7, 0] = 1.0
    h = torch.zeros(n, c, device=DEV, dtype=dtype)
    h[0::3, 0], h[1::3, 0] = 30000.0, 1.0
    targets = torch.full((n,), 7, device=DEV)
    up = torch.full((n,), temperature, device=DEV)
    got = _run(h, w, targets, up, up, temperature=temperature)
    for first in (0, 1):
        for name in ("log_probs", "entropy", "dhidden"):
            assert not got[name][first::3].any(), name
    # Sums of V equal terms and their logarithm.
    limit = (math.sqrt(v) + 32) * E * (1 + math.log(v))
    assert (got["entropy"][2::3] - math.log(v)).abs().max() <= limit
    assert (got["log_probs"][2::3] + math.log(v)).abs().max() <= limit
    # dz of the target is 1 - 1 / V, rounded once as an operand and once as an output.
    dhidden = got["dhidden"][2::3].double()
    assert (dhidden[:, 0] - (1 - 1 / v)).abs().max() <= 2 * ROUND[dtype] + limit
    assert not dhidden[:, 1:].any()
    # The rows with a gradient hold zeros.
    assert not got["dweight"].any()


@pytest.mark.parametrize("v", [65536, 90000])
def test_cross_entropy_with_and_without_a_backward_to_follow(v):
    """The hint that the weight is not read again soon changes no bits. Weights that are read
    past the caches without a backward, and with one too."""
    c = 2048
    assert 2 * c * v > (248 if v == 65536 else 320) << 20
    h, w, targets, _, _ = _case(5, c, v, torch.bfloat16, seed=13, masked=0.3)
    for reduction in ("none", "mean", "sum"):
        alone = pretrain_linear_cross_entropy(h, w, targets, reduction=reduction)
        leaf = h.clone().requires_grad_()
        followed = pretrain_linear_cross_entropy(leaf, w, targets, reduction=reduction)
        assert torch.equal(alone, followed.detach()) and followed.requires_grad
        for follows in (True, False):
            loss = torch.empty(5 if reduction == "none" else 1, device=DEV)
            capi.linear_cross_entropy_forward(h, w, targets, loss=loss, reduction=reduction,
                                              backward_follows=follows)
            assert torch.equal(loss.view(alone.shape), alone)
        want, = torch.autograd.grad(followed.sum(), [leaf])
        # What the call without one leaves serves a backward as well.
        saved = capi.linear_cross_entropy_forward(h, w, targets, loss=loss, reduction=reduction,
                                                  backward_follows=False)
        grad = torch.empty_like(h)
        capi.linear_loss_backward(torch.ones(5 if reduction == "none" else 1, device=DEV), w,
                                  saved, rows=5, top=1, reduction=reduction, grad_hidden=grad)
        assert torch.equal(grad, want)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("v", [65536, 90000])
def test_scores_from_weights_that_no_cache_keeps(n, v):
    """Read past the caches without a backward to follow, and the larger one with one too."""
    c = 2048
    assert 2 * c * v > (248 if v == 65536 else 320) << 20
    h, w, targets, _, _ = _case(n, c, v, torch.bfloat16, seed=14, masked=0.0)
    alone = pretrain_linear_log_probs(h, w, targets, entropy=True)
    followed = pretrain_linear_log_probs(h.clone().requires_grad_(), w, targets, entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(alone, followed))
    _check(h, w, targets, dict(zip(("log_probs", "entropy"), alone)), temperature=1.0)


@pytest.mark.parametrize("n", [3, 300])
def test_a_weight_beyond_32_bits_of_bytes(n):
    """300000 tokens of 8192 channels, 4.9 GB, all of logit 0 but the first and the last two:
    what is read or written at the end is found behind 2^32 bytes."""
    c, v = 8192, 300_000
    w = torch.zeros(v, c, device=DEV, dtype=torch.bfloat16)
    w[0], w[v - 2], w[v - 1] = 2.0 ** -11, 2.0 ** -12, 2.0 ** -10
    h = torch.ones(n, c, device=DEV, dtype=torch.bfloat16)
    targets = (v - 1 - torch.arange(n) % 2).to(DEV)
    z = torch.zeros(v, dtype=torch.float64)
    z[0], z[v - 2], z[v - 1] = 4.0, 2.0, 8.0
    log_q = torch.log_softmax(z, 0)
    q, entropy = log_q.exp(), -(log_q.exp() * log_q).sum()
    # Sums of V terms and the logarithms of them; logits are exact.
    delta = (math.sqrt(v) + 32) * E * (1 + math.log(v))
    got = pretrain_linear_log_probs(h, w, targets, entropy=True)
    assert (got[0].double().cpu() - log_q[targets.cpu()]).abs().max() <= delta
    assert (got[1].double().cpu() - entropy).abs().max() <= 2 * delta * (1 + entropy)
    up, ue = torch.ones(n, device=DEV), torch.full((n,), 0.5, device=DEV)
    out = _run(h, w, targets, up, ue)
    assert torch.equal(out["log_probs"], got[0]) and torch.equal(out["entropy"], got[1])
    b = torch.zeros(n, v, dtype=torch.float64)
    b[torch.arange(n), targets.cpu()] = 1.0
    dz = b - q - 0.5 * q * (log_q + entropy)
    # One or two roundings of dz to 16 bits and one of the gradient; what the scores are off by.
    u = ROUND[torch.bfloat16]
    off = dz.abs() * 2 * u + delta * (b + 2 * q * (1 + log_q.abs() + entropy))
    weights = w[[0, v - 2, v - 1], 0].double().cpu()
    rows = [0, v - 2, v - 1]
    value, want = out["dhidden"].double().cpu(), dz[:, rows] @ weights
    allowed = off[:, rows] @ weights + 2 * u * want.abs()
    assert ((value - want[:, None]).abs() <= allowed[:, None]).all()
    want, allowed = dz.sum(0), off.sum(0) + 2 * u * dz.sum(0).abs()
    for first in (0, v // 2, 262144 - 64, v - 128):
        value = out["dweight"][first:first + 128].double().cpu()
        there = slice(first, first + 128)
        assert ((value - want[there, None]).abs() <= allowed[there, None]).all(), first

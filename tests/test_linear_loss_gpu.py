"""GPU parity of the head losses against oracle/head.py (64 bits).

Bounds, before any run. With A = max over rows and vocabulary of
sum_c |h W|, an fp32 dot product of C terms is off by at most
gamma A, gamma = (sqrt(C) + 16) 2^-24 (rounding errors of either sign; the worst
case C 2^-24 A does not occur), and so is the log sum; the exponential and the
logarithm add a few 2^-24 of the exponent in base 2. So
  loss:     |off| <= T^2 (3 gamma A / T + 8 2^-24 (1 + |lse| + |z| / T))
  p:        relative delta = 2 gamma A / T + 8 2^-24 (1 + |z| / T + |lse|)
  gradient: each logit gradient is rounded once to 16 bits (u), its p is off by
            delta p <= delta (|dz| + w T b); then a product of n terms with
            fp32 sums, and the output's own rounding:
            |off| <= (u + delta + gamma_n) sum |dz| |factor| (+ delta of the
            target entries) + u |ref|.
fp16 adds its smallest step (outputs below 2^-14 lose digits).
"""

from __future__ import annotations

import math

import pytest
import torch

import flashrwkv_amd
from flashrwkv_amd import capi
from flashrwkv_amd.loss import pretrain_linear_cross_entropy, pretrain_linear_topk_distillation
from oracle import head

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
E = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _require_native():
    if flashrwkv_amd._C is None:
        pytest.fail("flashrwkv_amd native library is not built (no fallback exists)")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _head(n, c, v, dtype, seed, scale=2.0):
    gen = _gen(seed)
    h = torch.randn(n, c, generator=gen)
    w = torch.randn(v, c, generator=gen) * (scale / math.sqrt(c))
    return h.to(dtype).to(DEV), w.to(dtype).to(DEV)


def _teacher(n, k, v, seed, empty=0.2, dtype=torch.float32, index=torch.int64):
    """Distinct tokens a row; some entries absent in either way, some rows empty."""
    gen = _gen(seed)
    tokens = torch.stack([torch.randperm(v, generator=gen)[:k] for _ in range(n)])
    logits = (torch.randn(n, k, generator=gen) * 2).to(dtype)
    tokens[torch.rand(n, k, generator=gen) < 0.15] = -1
    logits[torch.rand(n, k, generator=gen) < 0.1] = -math.inf
    tokens[torch.rand(n, generator=gen) < empty] = -1
    return logits.to(DEV), tokens.to(index).to(DEV)


def _bounds(h, w, ref, temperature):
    rows = ref["rows"]
    a = (h.double()[rows].abs() @ w.double().abs().t()).max().item() if rows.numel() else 0.0
    gamma = (math.sqrt(h.shape[1]) + 16) * E
    z = ref["z"].abs().max().item() if rows.numel() else 0.0
    lse = ref["lse"].abs().max().item() if rows.numel() else 0.0
    loss = temperature ** 2 * (3 * gamma * a / temperature + 8 * E * (1 + lse + z / temperature))
    delta = 2 * gamma * a / temperature + 8 * E * (1 + lse + z / temperature)
    return loss, delta


def _check(h, w, entry, got, *, temperature=1.0, row_weight, reduction, terms_of_dz=1):
    """got: loss, dhidden, dweight (the gradients may be None). terms_of_dz: the 16-bit
    terms that a logit gradient is kept in; each leaves u of what the one before left."""
    dtype = h.dtype
    u, step = ROUND[dtype], STEP[dtype]
    ref = head.head_loss(h, w, *entry, temperature=temperature, row_weight=row_weight,
                         mean=reduction == "mean")
    n = ref["rows"].numel()
    loss_off, delta = _bounds(h, w, ref, temperature)
    want = ref["loss"]
    if reduction == "mean":
        want = want.sum() / max(1, n)
    if reduction == "sum":
        want, loss_off = want.sum(), loss_off * n + 16 * E * want.abs().sum().item()
    assert got[0].dtype == torch.float32 and got[0].shape == want.shape
    assert ((got[0].double() - want).abs() <= loss_off + 1e-7 * want.abs()).all(), \
        ((got[0].double() - want).abs().max().item(), loss_off)
    if n == 0:
        assert all(g is None or not g.any() for g in got[1:])
        return ref
    # What the target entries' p is off beyond their |dz|.
    index, p = entry[0][ref["rows"]], entry[1][ref["rows"]]
    by = row_weight.double()[ref["rows"], None].abs() * temperature
    by = by / n if reduction == "mean" else by
    extra_h = torch.zeros_like(ref["dhidden"])
    extra_h[ref["rows"]] = ((p * by)[:, :, None] * w.double().abs()[index]).sum(1)
    extra_w = torch.zeros_like(ref["dweight"])
    hs = h.double()[ref["rows"]].abs()
    for j in range(index.shape[1]):
        extra_w.index_add_(0, index[:, j], (p * by)[:, j:j + 1] * hs)
    # fp16 logit gradients: at most 2^-25 of the largest row weight's scale off, far below.
    grid = 2.0 ** -38 * float(by.max())
    for name, value, extra, terms, factor in (
            ("dhidden", got[1], extra_h, w.shape[0], w), ("dweight", got[2], extra_w, n, h)):
        if value is None:
            continue
        gamma = (math.sqrt(terms) + 16) * E
        allowed = ((u ** terms_of_dz + delta + gamma) * ref[f"abs_{name}"] + delta * extra
                   + u * ref[name].abs() * (1 + u) + step
                   + grid * terms * float(factor.double().abs().max()))
        off = (value.double().view(ref[name].shape) - ref[name]).abs()
        assert value.dtype == dtype and torch.isfinite(value).all(), name
        worst = (off - allowed).max().item()
        assert worst <= 0, f"{name}: {worst:.3e} over its bound (largest off {off.max():.3e})"
    return ref


def _grads(call, h, w, upstream, hidden=True, weight=True):
    h = h.clone().requires_grad_(hidden)
    w = w.clone().requires_grad_(weight)
    loss = call(h, w)
    leaves = [t for t in (h, w) if t.requires_grad]
    grads = list(torch.autograd.grad(loss, leaves, upstream)) if leaves else []
    return (loss.detach(), grads.pop(0) if hidden else None, grads.pop(0) if weight else None)


def _upstream(reduction, n, seed):
    if reduction == "none":
        return torch.randn(n, generator=_gen(seed)).to(DEV)
    return torch.tensor(1.0 if reduction == "mean" else 0.37, device=DEV)


def _row_weight(upstream, n):
    return upstream if upstream.dim() else upstream.expand(n)


SHAPES = [(1, 64, 1), (1, 64, 300), (1, 2048, 1000), (2, 128, 255), (63, 192, 256), (64, 64, 257),
          (65, 320, 513), (255, 128, 100), (256, 64, 1024), (257, 448, 999), (520, 1024, 770)]


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("n,c,v", SHAPES)
@pytest.mark.parametrize("masked,reduction", [(0.0, "mean"), (0.4, "sum"), (0.4, "none")])
def test_cross_entropy(n, c, v, dtype, masked, reduction):
    print(f"case {n}x{c} vocab {v} {dtype} masked {masked} {reduction}", flush=True)
    h, w = _head(n, c, v, dtype, seed=n + c + v)
    targets = torch.randint(v, (n,), generator=_gen(n))
    targets[torch.rand(n, generator=_gen(n + 1)) < masked] = -100
    targets = targets.to(DEV)
    upstream = _upstream(reduction, n, seed=n + 2)

    def call(a, b):
        return pretrain_linear_cross_entropy(a, b, targets, reduction=reduction)

    got = _grads(call, h, w, upstream)
    _check(h, w, head.labels(targets, v, -100), got, row_weight=_row_weight(upstream, n),
           reduction=reduction)
    for hidden, weight in ((True, True), (True, False), (False, True), (False, False)):
        part = _grads(call, h, w, upstream, hidden, weight)
        for a, b in zip(got, part):
            assert b is None or torch.equal(a, b)


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("n,c,v,k,t,reduction", [
    (1, 64, 40, 1, 1.0, "mean"), (3, 128, 300, 7, 0.5, "sum"), (65, 192, 512, 64, 2.0, "mean"),
    (130, 64, 700, 65, 1.5, "none"), (40, 64, 1100, 1024, 4.0, "mean"),
    (300, 576, 260, 130, 1.0, "none")])
def test_distillation(n, c, v, k, t, reduction, dtype):
    print(f"case {n}x{c} vocab {v} top {k} T {t} {dtype} {reduction}", flush=True)
    h, w = _head(n, c, v, dtype, seed=n + k)
    logits, tokens = _teacher(n, k, v, seed=k)
    upstream = _upstream(reduction, n, seed=n + 2)
    got = _grads(lambda a, b: pretrain_linear_topk_distillation(
        a, b, logits, tokens, temperature=t, reduction=reduction), h, w, upstream)
    _check(h, w, head.teacher(logits, tokens, t), got, temperature=t,
           row_weight=_row_weight(upstream, n), reduction=reduction)


@pytest.mark.parametrize("logit_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_teacher_types(logit_dtype, index):
    h, w = _head(20, 64, 90, torch.bfloat16, seed=4)
    logits, tokens = _teacher(20, 9, 90, seed=5, dtype=logit_dtype, index=index)
    one = torch.ones((), device=DEV)
    got = _grads(lambda a, b: pretrain_linear_topk_distillation(a, b, logits, tokens,
                                                                reduction="sum"), h, w, one)
    _check(h, w, head.teacher(logits, tokens, 1.0), got, row_weight=one.expand(20),
           reduction="sum")


def test_a_token_listed_twice_counts_with_both_shares():
    h, w = _head(3, 64, 50, torch.float16, seed=6)
    tokens = torch.tensor([[4, 9, 4, 4], [1, 1, -1, 2], [7, 7, 7, 7]], device=DEV)
    logits = torch.tensor([[1.0, 2.0, 0.5, 0.1], [0.0, 1.0, 9.0, 2.0], [3.0, 2.0, 1.0, 0.0]],
                          device=DEV)
    one = torch.ones((), device=DEV)
    got = _grads(lambda a, b: pretrain_linear_topk_distillation(
        a, b, logits, tokens, temperature=2.0, reduction="sum"), h, w, one)
    _check(h, w, head.teacher(logits, tokens, 2.0), got, temperature=2.0,
           row_weight=one.expand(3), reduction="sum")


def test_teacher_of_lowest_values_and_one_that_is_the_student():
    """Entries all at the type's lowest finite value are a uniform teacher;
    a teacher that lists the student's own logits gives a loss and gradients
    that are only rounding."""
    h, w = _head(8, 64, 33, torch.float16, seed=7)
    low = torch.full((8, 3), torch.finfo(torch.float32).min, device=DEV)
    tokens = torch.tensor([[0, 11, 32]], device=DEV).expand(8, 3).contiguous()
    even = pretrain_linear_topk_distillation(h, w, torch.zeros_like(low), tokens)
    assert torch.equal(even, pretrain_linear_topk_distillation(h, w, low, tokens))
    z = (h.double() @ w.double().t()).float()
    every = torch.arange(33, device=DEV).expand(8, 33).contiguous()
    one = torch.ones((), device=DEV)
    loss, dh, dw = _grads(lambda a, b: pretrain_linear_topk_distillation(
        a, b, z, every, reduction="sum"), h, w, one)
    assert abs(loss.item()) < 8 * 2e-5
    assert dh.abs().max() < 1e-5 and dw.abs().max() < 1e-4


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_masked_rows_hold_reaches_nothing(bad):
    h, w = _head(150, 128, 300, torch.bfloat16, seed=8)
    targets = torch.randint(300, (150,), generator=_gen(9)).to(DEV)
    masked = torch.rand(150, generator=_gen(10)).to(DEV) < 0.5
    targets[masked] = -100
    one = torch.ones((), device=DEV)

    def call(a, b):
        return pretrain_linear_cross_entropy(a, b, targets)

    clean = _grads(call, h, w, one)
    h[masked] = bad
    dirty = _grads(call, h, w, one)
    assert all(torch.equal(a, b) for a, b in zip(clean, dirty))
    assert torch.isfinite(dirty[2]).all() and not dirty[1][masked].any()


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_no_row_left(reduction):
    h, w = _head(70, 64, 130, torch.bfloat16, seed=11)
    targets = torch.full((70,), 5, dtype=torch.int32, device=DEV)
    upstream = _upstream(reduction, 70, seed=1)
    got = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets, ignore_index=5,
                                                            reduction=reduction), h, w, upstream)
    assert not got[0].any() and not got[1].any() and not got[2].any()
    none = torch.full((70, 3), -1, device=DEV)
    got = _grads(lambda a, b: pretrain_linear_topk_distillation(
        a, b, torch.zeros(70, 3, device=DEV), none, reduction=reduction), h, w, upstream)
    assert not got[0].any() and not got[1].any() and not got[2].any()


def test_no_row_at_all():
    h, w = _head(4, 64, 130, torch.bfloat16, seed=12)
    h = h[:0].clone().requires_grad_()
    w = w.requires_grad_()
    targets = torch.empty(0, dtype=torch.int64, device=DEV)
    loss = pretrain_linear_cross_entropy(h, w, targets)
    dh, dw = torch.autograd.grad(loss, [h, w])
    assert loss.item() == 0 and dh.shape == (0, 64) and dw.shape == w.shape and not dw.any()
    assert pretrain_linear_cross_entropy(h, w, targets, reduction="none").shape == (0,)


def test_targets_out_of_range_make_their_rows_nan():
    h, w = _head(10, 64, 100, torch.bfloat16, seed=13)
    targets = torch.randint(100, (10,), generator=_gen(14)).to(DEV)
    clean = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets, reduction="none"),
                   h, w, torch.ones(10, device=DEV))
    bad = targets.clone()
    bad[3], bad[7] = 100, -1
    got = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, bad, reduction="none"), h, w,
                 torch.ones(10, device=DEV))
    keep = [0, 1, 2, 4, 5, 6, 8, 9]
    assert torch.isnan(got[0][[3, 7]]).all() and torch.equal(got[0][keep], clean[0][keep])
    assert torch.isnan(got[1][[3, 7]]).all() and torch.equal(got[1][keep], clean[1][keep])
    assert torch.isnan(got[2]).all()
    huge = targets.clone()
    huge[0] = 2 ** 40
    assert torch.isnan(pretrain_linear_cross_entropy(h, w, huge))
    tokens = torch.tensor([[1, 100]], device=DEV).expand(10, 2).contiguous()
    loss = pretrain_linear_topk_distillation(h, w, torch.zeros(10, 2, device=DEV), tokens,
                                             reduction="none")
    assert torch.isnan(loss).all()


@pytest.mark.parametrize("dtype", ROUND)
def test_large_logits_stay_finite(dtype):
    """Logits of several hundred: the maximum is taken out before the
    exponential, in the tiles and where they are joined."""
    h, w = _head(40, 256, 600, dtype, seed=15, scale=150.0)
    targets = torch.randint(600, (40,), generator=_gen(16)).to(DEV)
    one = torch.ones((), device=DEV)
    got = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets), h, w, one)
    _check(h, w, head.labels(targets, 600, -100), got, row_weight=one.expand(40),
           reduction="mean")


@pytest.mark.parametrize("scale", [1e-6, 1.0, 3e4])
def test_upstream_scales(scale):
    """bf16 gradients follow any scale of the upstream weights, among rows too."""
    h, w = _head(90, 64, 200, torch.bfloat16, seed=17)
    targets = torch.randint(200, (90,), generator=_gen(18)).to(DEV)
    upstream = (torch.randn(90, generator=_gen(19)) * scale).to(DEV)
    upstream[::7] = 0
    upstream[1] = 1000 * scale
    got = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets, reduction="none"), h,
                 w, upstream)
    _check(h, w, head.labels(targets, 200, -100), got, row_weight=upstream, reduction="none")
    assert not got[1][::7].any()


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("n,c,v,masked", [
    (520, 768, 25000, 0.0), (520, 768, 25000, 0.3), (300, 64, 20000, 0.5), (60, 128, 20000, 0.5),
    (50, 128, 40000, 0.1), (700, 64, 20000, 0.97), (130, 640, 5000, 0.2), (250, 320, 7000, 0.0)])
def test_wide_vocabularies(n, c, v, masked, dtype):
    """More tiles than CUs, the last ones smaller; dz W split over the vocabulary,
    into more parts the fewer rows take part."""
    h, w = _head(n, c, v, dtype, seed=n + c)
    targets = torch.randint(v, (n,), generator=_gen(n))
    targets[torch.rand(n, generator=_gen(n + 1)) < masked] = -100
    targets[-1] = v - 1
    targets = targets.to(DEV)
    upstream = _upstream("none", n, seed=n + 2)
    got = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets, reduction="none"), h,
                 w, upstream)
    _check(h, w, head.labels(targets, v, -100), got, row_weight=upstream, reduction="none")
    again = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets, reduction="none"), h,
                   w, upstream)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("n,c,v,k", [(1, 512, 300, 1), (3, 64, 1000, 1), (31, 320, 257, 1),
                                     (32, 1024, 700, 1), (20, 128, 400, 9), (32, 128, 20000, 1),
                                     (5, 64, 40000, 1), (17, 192, 70001, 3)])
def test_few_rows_lose_nothing_to_their_logit_gradients(n, c, v, k, dtype):
    """Up to 32 rows keep them in two terms, with per-row weights as well."""
    h, w = _head(n, c, v, dtype, seed=31 + n)
    upstream = _upstream("none", n, seed=n + 2)
    if k == 1:
        targets = torch.randint(v, (n,), generator=_gen(n)).to(DEV)
        targets[n // 2] = -100 if n > 1 else 7
        entry = head.labels(targets, v, -100)

        def call(a, b):
            return pretrain_linear_cross_entropy(a, b, targets, reduction="none")
    else:
        logits, tokens = _teacher(n, k, v, seed=32)
        entry = head.teacher(logits, tokens, 1.0)

        def call(a, b):
            return pretrain_linear_topk_distillation(a, b, logits, tokens, reduction="none")

    _check(h, w, entry, _grads(call, h, w, upstream), row_weight=upstream, reduction="none",
           terms_of_dz=2)


def test_several_pieces_of_the_vocabulary():
    """4096 rows and 70000 tokens need several pieces of logit gradients; a target
    list that reaches into both, and the last piece ragged."""
    n, c, v = 4096, 64, 70000
    h, w = _head(n, c, v, torch.bfloat16, seed=20)
    logits, tokens = _teacher(1, 6, v, seed=21, empty=0.0)
    logits = logits.expand(n, 6).contiguous()
    logits[logits == -math.inf] = 0.0
    tokens = torch.randint(v, (n, 6), generator=_gen(22)).to(DEV)
    tokens[:, 1], tokens[:, 2] = 3, v - 1
    one = torch.ones((), device=DEV)
    got = _grads(lambda a, b: pretrain_linear_topk_distillation(a, b, logits, tokens), h, w, one)
    _check(h, w, head.teacher(logits, tokens, 1.0), got, row_weight=one.expand(n),
           reduction="mean")


@pytest.mark.parametrize("n", [1023, 1024, 1025, 2113])
@pytest.mark.parametrize("last", [True, False])
def test_rows_are_numbered_in_order(n, last):
    """Up to 1024 rows each workgroup numbers them for itself; the last row alone,
    or with others that are left after two of three were masked."""
    h, w = _head(n, 64, 130, torch.bfloat16, seed=n)
    targets = torch.randint(130, (n,), generator=_gen(n))
    targets[torch.arange(n) % 3 != 1] = -100
    if last:
        targets[:-1] = -100
    targets[-1] = 7
    targets = targets.to(DEV)
    upstream = _upstream("none", n, seed=n + 2)
    entry = head.labels(targets, 130, -100)
    got = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets, reduction="none"), h,
                 w, upstream)
    _check(h, w, entry, got, row_weight=upstream, reduction="none")
    tokens = torch.where(targets < 0, -1, targets)[:, None].expand(n, 2).contiguous()
    tokens[:, 1] = -1
    one = torch.ones((), device=DEV)
    got = _grads(lambda a, b: pretrain_linear_topk_distillation(
        a, b, torch.zeros(n, 2, device=DEV), tokens), h, w, one)
    _check(h, w, entry, got, row_weight=one.expand(n), reduction="mean")


def test_offsets_beyond_32_bits():
    """A weight of more than 2^31 elements, and its gradient; references by blocks."""
    n, c, v, block = 3, 4096, 530001, 53000
    gen = torch.Generator(device=DEV).manual_seed(33)
    h = torch.randn(n, c, generator=gen, device=DEV).bfloat16()
    w = torch.empty(v, c, dtype=torch.bfloat16, device=DEV)
    for at in range(0, v, block):
        part = w[at:at + block]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV) * (2 / math.sqrt(c)))
    targets = torch.tensor([v - 1, 5, v - block - 1], device=DEV)
    upstream = torch.tensor([1.0, -2.0, 0.5], device=DEV)
    loss, dh, dw = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets,
                                                                     reduction="none"),
                          h, w, upstream)
    hd = h.double()
    z = torch.cat([hd @ w[at:at + block].double().t() for at in range(0, v, block)], 1)
    lse = torch.logsumexp(z, 1, keepdim=True)
    rows = torch.arange(n, device=DEV)
    a = (hd.abs().amax() * w.abs().sum(1).max().double()).item()
    gamma = (math.sqrt(c) + 16) * E
    size = 1 + lse.abs().max().item() + z.abs().max().item()
    want = lse[:, 0] - z[rows, targets]
    assert ((loss.double() - want).abs() <= 3 * gamma * a + 8 * E * size).all()
    dz = torch.exp(z - lse)
    dz[rows, targets] -= 1
    dz *= upstream.double()[:, None]
    u = ROUND[torch.bfloat16]
    delta = 2 * gamma * a + 8 * E * size
    by = upstream.double().abs()
    ref, scale = torch.zeros_like(hd), torch.zeros_like(hd)
    for at in range(0, v, block):
        part = w[at:at + block].double()
        ref += dz[:, at:at + block] @ part
        scale += dz[:, at:at + block].abs() @ part.abs()
    sums = (math.sqrt(v) + 16) * E
    allowed = ((u * u + delta + sums) * scale + delta * by[:, None] * w[targets].double().abs()
               + u * ref.abs() * (1 + u))
    assert ((dh.double() - ref).abs() <= allowed).all()
    some = torch.cat([torch.arange(0, v, 4999, device=DEV), targets])
    ref = dz[:, some].t() @ hd
    target = torch.zeros(n, v, dtype=torch.float64, device=DEV)
    target[rows, targets] = by
    allowed = ((u * u + delta + 32 * E) * (dz[:, some].abs().t() @ hd.abs())
               + delta * (target[:, some].t() @ hd.abs()) + u * ref.abs() * (1 + u))
    assert ((dw[some].double() - ref).abs() <= allowed).all()


def test_gradient_matches_differences_of_the_operator():
    """Central differences of the operator's own loss along directions in which
    the fp16 inputs move exactly (multiples of 1/16): truncation h^2 of a
    smooth function whose steps are small against the logits' scale."""
    gen = _gen(23)
    h = (torch.randint(-16, 17, (12, 64), generator=gen) / 16).half().to(DEV)
    w = (torch.randint(-16, 17, (50, 64), generator=gen) / 64).half().to(DEV)
    targets = torch.randint(50, (12,), generator=gen).to(DEV)
    one = torch.ones((), device=DEV)

    def call(a, b):
        return pretrain_linear_cross_entropy(a, b, targets, reduction="sum")

    _, dh, dw = _grads(call, h, w, one)
    for grad, which, step in ((dh, 0, 1 / 16), (dw, 1, 1 / 64)):
        move = (torch.randint(-1, 2, grad.shape, generator=gen)).half().to(DEV)
        plus, minus = [h, w], [h, w]
        plus[which] = plus[which] + step * move
        minus[which] = minus[which] - step * move
        slope = ((call(*plus).double() - call(*minus).double()) / (2 * step)).item()
        want = (grad.double() * move.double()).sum().item()
        scale = (grad.double().norm() * move.double().norm()).item()
        assert abs(slope - want) <= 0.02 * scale, (slope, want, scale)


def test_shapes_repeats_and_other_streams():
    """Leading shapes, the same bits on a repeat, and inputs made on the stream
    that the call runs on."""
    h, w = _head(120, 128, 700, torch.bfloat16, seed=24)
    targets = torch.randint(700, (120,), generator=_gen(25)).to(DEV)
    one = torch.ones((), device=DEV)
    flat = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets), h, w, one)
    deep = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets.view(4, 30)),
                  h.view(4, 30, 128), w, one)
    assert torch.equal(flat[0], deep[0]) and torch.equal(flat[1], deep[1].view(120, 128))
    assert torch.equal(flat[2], deep[2]) and deep[1].shape == (4, 30, 128)
    rows = pretrain_linear_cross_entropy(h.view(4, 30, 128), w, targets.view(4, 30),
                                         reduction="none")
    assert rows.shape == (4, 30)
    torch.testing.assert_close(rows.mean(), flat[0], rtol=1e-6, atol=0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets.clone()),
                       h.clone(), w.clone(), one.clone())
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(flat, again))


class _Sub(torch.Tensor):
    """A tensor subclass: no whole call, the wrapper's own tables and autograd function."""


@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_calls_that_are_not_plain_give_the_same_bits(reduction):
    h, w = _head(50, 128, 300, torch.float16, seed=26)
    targets = torch.randint(300, (50,), generator=_gen(27)).to(DEV)
    logits, tokens = _teacher(50, 8, 300, seed=28)
    upstream = _upstream(reduction, 50, seed=29)
    for call in (lambda a, b: pretrain_linear_cross_entropy(a, b, targets, reduction=reduction),
                 lambda a, b: pretrain_linear_topk_distillation(
                     a, b, logits, tokens, temperature=2, reduction=reduction)):
        plain = _grads(call, h, w, upstream)
        other = _grads(call, h.as_subclass(_Sub), w.as_subclass(_Sub), upstream)
        assert all(torch.equal(a, b.as_subclass(torch.Tensor)) for a, b in zip(plain, other))


@pytest.mark.parametrize("kind", [torch.Tensor, _Sub])
def test_differentiating_twice_raises(kind):
    h, w = _head(5, 64, 30, torch.bfloat16, seed=30)
    h = h.as_subclass(kind).requires_grad_()
    loss = pretrain_linear_cross_entropy(h, w, torch.zeros(5, dtype=torch.int64, device=DEV))
    dh, = torch.autograd.grad(loss, h, torch.ones((), device=DEV, requires_grad=True),
                              create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dh.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [0.1, 0.5, 3.0])
def test_only_minus_infinity_is_absent_whatever_the_temperature(t, dtype):
    """Rows whose logits are all the type's lowest finite value are a uniform
    teacher at any temperature and count in a mean; beside an ordinary logit such
    an entry has no share; -inf is absent."""
    n, v, low = 9, 70, torch.finfo(dtype).min
    h, w = _head(n, 64, v, torch.bfloat16, seed=40)
    logits = torch.randn(n, 4, generator=_gen(41)).to(dtype)
    logits[0] = low
    logits[1, 1:] = low
    logits[2, 0], logits[2, 1:] = low, -math.inf
    logits[3] = -math.inf
    logits = logits.to(DEV)
    tokens = torch.stack([torch.randperm(v, generator=_gen(42 + i))[:4] for i in range(n)]).to(DEV)
    one = torch.ones((), device=DEV)
    entry = head.teacher(logits, tokens, t)
    assert entry[2].any(1).sum() == n - 1
    for reduction in ("mean", "none"):
        upstream = one if reduction == "mean" else _upstream("none", n, seed=43)
        got = _grads(lambda a, b: pretrain_linear_topk_distillation(
            a, b, logits, tokens, temperature=t, reduction=reduction), h, w, upstream)
        _check(h, w, entry, got, temperature=t, row_weight=_row_weight(upstream, n),
               reduction=reduction)
    even = logits.clone()
    even[0] = 0
    rows = [pretrain_linear_topk_distillation(h, w, x, tokens, temperature=t, reduction="none")
            for x in (logits, even)]
    assert torch.equal(*rows)


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan, 3e38])
def test_a_row_weight_beyond_the_others_range_stays_with_its_row(bad, dtype):
    """The other rows' losses and hidden gradients are within their bounds."""
    h, w = _head(90, 128, 300, dtype, seed=44)
    targets = torch.randint(300, (90,), generator=_gen(45)).to(DEV)
    upstream = (torch.randn(90, generator=_gen(46)) * 20).to(DEV)
    upstream[11] = bad
    loss, dh, _ = _grads(lambda a, b: pretrain_linear_cross_entropy(a, b, targets,
                                                                    reduction="none"),
                         h, w, upstream)
    keep = [i for i in range(90) if i != 11]
    entry = head.labels(targets[keep], 300, -100)
    _check(h[keep], w, entry, (loss[keep], dh[keep], None), row_weight=upstream[keep],
           reduction="none")


@pytest.mark.parametrize("t", [1e-25, 1e25])
def test_losses_at_extreme_temperatures_neither_vanish_nor_overflow(t):
    """The loss is of the size of T at a small T; one token has the loss 0 at a
    large T, whose square is beyond fp32. Logits are whole numbers apart."""
    h = torch.zeros(3, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(4 if t < 1 else 1, 64, dtype=torch.bfloat16, device=DEV)
    h[:, 0] = 1
    w[:, 0] = torch.arange(w.shape[0], device=DEV)
    tokens = torch.zeros(3, 1, dtype=torch.int64, device=DEV)
    loss = pretrain_linear_topk_distillation(h, w, torch.zeros(3, 1, device=DEV), tokens,
                                             temperature=t, reduction="none")
    want = 3 * t if t < 1 else 0.0
    assert ((loss.double() - want).abs() <= 1e-5 * want).all(), loss


def test_more_rows_than_a_call_takes_are_refused_with_their_count():
    """Before anything is allocated for them."""
    n = 2 ** 23 + 1
    h = torch.zeros(n, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    targets = torch.zeros(n, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match=r"rows must be in \[1, 2\^23\], got 8388609"):
        pretrain_linear_cross_entropy(h, w, targets, reduction="sum")
    with pytest.raises(RuntimeError, match=r"rows must be in \[1, 2\^23\], got 8388609"):
        pretrain_linear_topk_distillation(h, w, torch.zeros(n, 1, device=DEV), targets[:, None])


@pytest.mark.parametrize("n,c,v,masked", [(16500, 128, 20011, 0.0), (17001, 320, 20300, 0.6)])
def test_many_rows_in_several_pieces(n, c, v, masked):
    """Each piece of the vocabulary adds to the slabs of the hidden gradient that the
    pieces before it left; the last piece is ragged, and so is the last row tile."""
    h, w = _head(n, c, v, torch.bfloat16, seed=50 + n)
    targets = torch.randint(v, (n,), generator=_gen(n))
    targets[torch.rand(n, generator=_gen(n + 1)) < masked] = -100
    targets = targets.to(DEV)
    upstream = _upstream("none", n, seed=n + 2)

    def call(a, b):
        return pretrain_linear_cross_entropy(a, b, targets, reduction="none")

    got = _grads(call, h, w, upstream)
    _check(h, w, head.labels(targets, v, -100), got, row_weight=upstream, reduction="none")
    assert all(torch.equal(a, b) for a, b in zip(got, _grads(call, h, w, upstream)))
    frozen = _grads(call, h, w, upstream, weight=False)
    assert torch.equal(frozen[1], got[1])


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("n,c,v,left", [(40, 64, 300, 10), (100, 512, 700, 32), (300, 320, 3001, 1),
                                        (1030, 512, 3001, 9), (2500, 192, 20011, 20),
                                        (600, 512, 40000, 31)])
def test_few_rows_left_by_masks_are_few_rows(n, c, v, left, dtype):
    """A row's gradient is as exact with masked rows beside it as without them."""
    h, w = _head(n, c, v, dtype, seed=47 + n)
    keep = torch.randperm(n, generator=_gen(n))[:left].to(DEV)
    targets = torch.full((n,), -100, device=DEV)
    targets[keep] = torch.randint(v, (left,), generator=_gen(n + 1)).to(DEV)
    upstream = _upstream("none", n, seed=n + 2)
    entry = head.labels(targets, v, -100)

    def call(a, b):
        return pretrain_linear_cross_entropy(a, b, targets, reduction="none")

    got = _grads(call, h, w, upstream)
    _check(h, w, entry, got, row_weight=upstream, reduction="none", terms_of_dz=2)
    assert all(torch.equal(a, b) for a, b in zip(got, _grads(call, h, w, upstream)))


def test_a_token_listed_four_times_hand_worked():
    """A uniform student over 5 tokens, four equal entries on one of them: the loss is
    T^2 (log 5 - log 4), the gradient that of one entry with all of p."""
    h = torch.zeros(1, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(5, 64, dtype=torch.bfloat16, device=DEV)
    w[:, :5] = 4 * torch.eye(5)
    four = torch.full((1, 4), 3, device=DEV)
    loss, dh, dw = _grads(lambda a, b: pretrain_linear_topk_distillation(
        a, b, torch.zeros(1, 4, device=DEV), four, temperature=2.0, reduction="sum"), h, w,
        torch.ones((), device=DEV))
    assert loss.item() == pytest.approx(4 * (math.log(5) - math.log(4)), rel=1e-5)
    want = torch.tensor([1.6, 1.6, 1.6, -6.4, 1.6], device=DEV)
    torch.testing.assert_close(dh[0, :5].float(), want, rtol=2.0 ** -8, atol=0)
    assert not dh[0, 5:].any() and not dw.any()
    with_far_ahead = h.clone()
    with_far_ahead[0, 3] = 16  # z = 64 at the token, 0 elsewhere: q is 1 there
    loss = pretrain_linear_topk_distillation(with_far_ahead, w, torch.zeros(1, 4, device=DEV),
                                             four, reduction="sum")
    assert loss.item() == pytest.approx(-math.log(4), rel=1e-5)


# Rows, channels, tokens, masked share and whether one piece holds the vocabulary: the
# hidden gradient goes through 256 x 256 tiles in several splits. Ragged: rows, the last
# tile of channels, the last split and the last piece.
LARGE = [(700, 1088, 20011, 0.0, True), (700, 1088, 20011, 0.5, True),
         (2047, 576, 20011, 0.2, True), (4095, 576, 70001, 0.0, False),
         (4095, 832, 70001, 0.4, False)]


def _require_large_tiles(n, c, v, one_piece):
    columns, pieces, splits, tile_rows = capi.linear_loss_backward_plan(n, c, v)
    print(f"pieces of {columns}: {pieces}, splits {splits}, tile rows {tile_rows}", flush=True)
    assert tile_rows == 256 and splits > 1 and (pieces == 1) == one_piece
    assert c % 256 and v % columns and n % 256


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("n,c,v,masked,one_piece", LARGE)
def test_large_tiles_cross_entropy(n, c, v, masked, one_piece, dtype):
    _require_large_tiles(n, c, v, one_piece)
    h, w = _head(n, c, v, dtype, seed=60 + n + c)
    targets = torch.randint(v, (n,), generator=_gen(n))
    targets[torch.rand(n, generator=_gen(n + 1)) < masked] = -100
    targets[-1] = v - 1
    targets = targets.to(DEV)
    upstream = _upstream("none", n, seed=n + 2)

    def call(a, b):
        return pretrain_linear_cross_entropy(a, b, targets, reduction="none")

    got = _grads(call, h, w, upstream)
    _check(h, w, head.labels(targets, v, -100), got, row_weight=upstream, reduction="none")
    assert all(torch.equal(a, b) for a, b in zip(got, _grads(call, h, w, upstream)))
    frozen = _grads(call, h, w, upstream, weight=False)
    assert torch.equal(frozen[1], got[1])


@pytest.mark.parametrize("n,c,v,masked,one_piece", LARGE)
def test_large_tiles_distillation(n, c, v, masked, one_piece):
    _require_large_tiles(n, c, v, one_piece)
    h, w = _head(n, c, v, torch.bfloat16, seed=61 + n + c)
    gen = torch.Generator(device=DEV).manual_seed(n)
    first = torch.randint(v, (n, 1), generator=gen, device=DEV)
    tokens = (first + torch.arange(5, device=DEV) * (v // 5)) % v  # in every piece
    tokens[torch.rand(n, generator=gen, device=DEV) < masked] = -1
    logits = torch.randn(n, 5, generator=gen, device=DEV)
    one = torch.ones((), device=DEV)
    got = _grads(lambda a, b: pretrain_linear_topk_distillation(
        a, b, logits, tokens, temperature=1.5, reduction="sum"), h, w, one)
    _check(h, w, head.teacher(logits, tokens, 1.5), got, temperature=1.5,
           row_weight=one.expand(n), reduction="sum")

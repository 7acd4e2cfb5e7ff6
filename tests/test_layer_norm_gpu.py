"""GPU parity of the layer norm operators against oracle/head.py (64 bits).

Bounds, elementwise, before any run: an output rounded to a type of unit
roundoff u is off by at most u |ref|, plus what the fp32 arithmetic inside adds.
Inside, a row's mean is off by a few 2^-24 of the row's largest value A (sums of
partial sums; 16 for depth and conditioning), xhat therefore by 16 2^-24 (A
rstd + |xhat|); y by that times |weight|; dx by the same share of its terms'
magnitudes; dweight by 32 2^-24 of the sum of its terms' absolute values plus
what the xhat in them is off.
"""

from __future__ import annotations

import pytest
import torch

import flashrwkv_amd
from flashrwkv_amd.normalization import infer_layer_norm_forward_varlen, pretrain_layer_norm
from oracle import head

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-38, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-38}
INNER = 16 * 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _require_native():
    if flashrwkv_amd._C is None:
        pytest.fail("flashrwkv_amd native library is not built (no fallback exists)")


def _inputs(rows, c, dtype, seed, residual=False, loc=0.3):
    gen = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    out = {"x": randn(rows, c) + loc, "weight": 1 + 0.3 * randn(c), "bias": 0.2 * randn(c),
           "dy": randn(rows, c)}
    if residual:
        out |= {"residual": randn(rows, c), "ds": randn(rows, c)}
    return {k: v.to(dtype).to(DEV) for k, v in out.items()}


def _within(name, got, want, allowed):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), name
    worst = (off - allowed).max().item()
    assert worst <= 0, f"{name}: {worst:.3e} over its bound"


def _check(case, eps, y, grads=None):
    """y, and grads (dx, dweight, dbias) against the oracle; case["s"] was normed."""
    dtype = y.dtype
    u, tiny = ROUND[dtype], TINY[dtype]
    s, w = case["s"], case["weight"].double()
    ref = head.layer_norm(s, w, case["bias"], eps, case["dy"], case.get("ds"))
    rstd = ref["rstd"][:, None]
    big = s.double().abs().amax(1, keepdim=True)
    xhat_off = INNER * (big * rstd + ref["xhat"].abs())
    allowed = u * ref["y"].abs() + xhat_off * w.abs() + INNER * case["bias"].double().abs() + tiny
    _within("y", y, ref["y"], allowed)
    if grads is None:
        return
    g = (case["dy"].double() * w).abs()
    mean_g = g.mean(1, keepdim=True)
    x_abs = ref["xhat"].abs()
    mean_gx = (g * x_abs).mean(1, keepdim=True)
    mean_off = (g * xhat_off).mean(1, keepdim=True)
    inner = rstd * (INNER * (g + mean_g + 2 * x_abs * mean_gx) + xhat_off * mean_gx
                    + x_abs * mean_off)
    ds = case["ds"].double().abs() if "ds" in case else 0.0
    _within("dx", grads[0], ref["dx"], u * ref["dx"].abs() + inner * (1 + INNER * big * rstd)
            + INNER * ds + tiny)
    dy_abs = case["dy"].double().abs()
    _within("dweight", grads[1], ref["dweight"],
            u * ref["dweight"].abs() + 2 * INNER * ref["abs_dweight"]
            + (dy_abs * xhat_off).sum(0) + tiny)
    _within("dbias", grads[2], ref["dbias"],
            u * ref["dbias"].abs() + 2 * INNER * ref["abs_dbias"] + tiny)


SHAPES = [(1, 1), (4, 2), (1, 64), (3, 100), (9, 1023), (9, 1024), (5, 1025), (2, 4096), (3, 4097),
          (2, 16384), (1300, 264), (2051, 40), (700, 2560)]


@pytest.mark.parametrize("dtype", ROUND)
@pytest.mark.parametrize("rows,c", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_forward_and_gradients(rows, c, dtype, residual):
    print(f"case {rows}x{c} {dtype} residual {residual}", flush=True)
    case = _inputs(rows, c, dtype, seed=rows + c, residual=residual)
    eps = 1e-5
    names = ("x", "weight", "bias", "residual") if residual else ("x", "weight", "bias")
    leaves = {n: case[n].clone().requires_grad_() for n in names}
    out = pretrain_layer_norm(leaves["x"], leaves["weight"], leaves["bias"], eps=eps,
                              residual=leaves.get("residual"))
    if residual:
        y, stream = out
        want = (case["x"].double() + case["residual"].double()).float().to(dtype)
        torch.testing.assert_close(stream.detach(), want, rtol=2 * ROUND[dtype], atol=0)
        case["s"] = stream.detach()
        grads = torch.autograd.grad((y, stream), list(leaves.values()), (case["dy"], case["ds"]))
        assert torch.equal(grads[0], grads[3])
        served = infer_layer_norm_forward_varlen(case["x"], case["weight"], case["bias"], eps=eps,
                                                 residual=case["residual"])
        assert torch.equal(served[0], y) and torch.equal(served[1], stream)
    else:
        y, case["s"] = out, case["x"]
        grads = torch.autograd.grad(y, list(leaves.values()), case["dy"])
        assert torch.equal(y, infer_layer_norm_forward_varlen(case["x"], case["weight"],
                                                              case["bias"], eps=eps))
    _check(case, eps, y.detach(), grads)
    again = pretrain_layer_norm(leaves["x"], leaves["weight"], leaves["bias"], eps=eps,
                                residual=leaves.get("residual"))
    again = torch.autograd.grad(again, list(leaves.values()),
                                (case["dy"], case["ds"]) if residual else case["dy"])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the first and last rows, and the sums over all."""
    rows, c, dtype = 530003, 4096, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(5)
    x, dy = (torch.empty(rows, c, dtype=dtype, device=DEV).normal_(generator=gen)
             for _ in range(2))
    small = _inputs(1, c, dtype, seed=6)
    weight = small["weight"].clone().requires_grad_()
    bias = small["bias"].clone().requires_grad_()
    leaf = x.requires_grad_()
    y = pretrain_layer_norm(leaf, weight, bias)
    grads = torch.autograd.grad(y, [leaf, weight, bias], dy)
    y = y.detach()
    for part in (slice(0, 3), slice(rows // 2, rows // 2 + 3), slice(rows - 3, rows)):
        case = {"x": x.detach()[part], "weight": small["weight"], "bias": small["bias"],
                "dy": dy[part]}
        alone = {k: case[k].clone().requires_grad_() for k in ("x", "weight", "bias")}
        want = pretrain_layer_norm(alone["x"], alone["weight"], alone["bias"])
        dx, = torch.autograd.grad(want, [alone["x"]], case["dy"])
        case["s"] = case["x"]
        _check(case, 1e-5, want.detach())
        assert torch.equal(y[part], want) and torch.equal(grads[0][part], dx)
    dbias, abs_dbias = 0.0, 0.0
    for at in range(0, rows, 53000):
        part = dy[at:at + 53000].double()
        dbias, abs_dbias = dbias + part.sum(0), abs_dbias + part.abs().sum(0)
    _within("dbias", grads[2], dbias, ROUND[dtype] * dbias.abs() + 2 * INNER * abs_dbias)


@pytest.mark.parametrize("dtype", ROUND)
def test_tensors_off_16_byte_boundaries(dtype):
    """Contiguous views that start one element into their storage take the
    path of unaligned rows and give the aligned call's result."""
    case = _inputs(37, 192, dtype, seed=3)
    case["s"] = case["x"]

    def shifted(t):
        buffer = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        buffer[1:] = t.reshape(-1)
        return buffer[1:].view(t.shape)

    args = [shifted(case[n]).requires_grad_() for n in ("x", "weight", "bias")]
    y = pretrain_layer_norm(*args)
    grads = torch.autograd.grad(y, args, shifted(case["dy"]))
    _check(case, 1e-5, y.detach(), grads)


def test_constant_rows_and_a_large_mean():
    """Zero variance gives y = bias (rstd = 1/sqrt(eps) times 0); a mean of
    1000 with a deviation of 1 keeps the deviation (variance about the mean)."""
    case = _inputs(4, 512, torch.float32, seed=5)
    x = torch.full((4, 512), 3.0, device=DEV)
    y = infer_layer_norm_forward_varlen(x, case["weight"], case["bias"])
    assert torch.equal(y, case["bias"].expand(4, 512))
    case["x"] = case["x"] + 1000.0
    case["s"] = case["x"]
    _check(case, 1e-5, infer_layer_norm_forward_varlen(case["x"], case["weight"], case["bias"]))


def test_non_finite_rows_stay_alone():
    case = _inputs(6, 320, torch.bfloat16, seed=6)
    clean = infer_layer_norm_forward_varlen(case["x"], case["weight"], case["bias"])
    case["x"][2, 7], case["x"][4, 0] = float("nan"), float("inf")
    x = case["x"].requires_grad_()
    y = pretrain_layer_norm(x, case["weight"], case["bias"])
    dx, = torch.autograd.grad(y, x, case["dy"])
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], clean[keep]) and torch.isfinite(dx[keep]).all()
    assert torch.isnan(y[[2, 4]]).all() and torch.isnan(dx[[2, 4]]).all()


def test_partial_upstream_gradients_and_frozen_parameters():
    """Only the stream's gradient, only y's, and parameters that need none."""
    case = _inputs(70, 256, torch.float32, seed=7, residual=True)
    names = ("x", "residual", "weight", "bias")
    leaves = [case[n].clone().requires_grad_() for n in names]
    y, stream = pretrain_layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    grads = torch.autograd.grad(stream, leaves, case["ds"], allow_unused=True, retain_graph=True)
    assert torch.equal(grads[0], case["ds"]) and torch.equal(grads[1], case["ds"])
    assert grads[2] is None and grads[3] is None
    case["s"] = stream.detach()
    del case["ds"]
    grads = torch.autograd.grad(y, leaves, case["dy"])
    _check(case, 1e-5, y.detach(), (grads[0], grads[2], grads[3]))
    x = case["x"].clone().requires_grad_()
    y = pretrain_layer_norm(x, case["weight"], case["bias"])
    assert y.requires_grad and torch.autograd.grad(y, x, case["dy"])[0].shape == x.shape


def test_gradient_matches_differences_of_the_operator():
    """Along random directions, fp32, central differences of the operator's own
    output: truncation about h^2, rounding about 2^-24 sqrt(N C) / h."""
    case = _inputs(5, 96, torch.float32, seed=8)
    leaves = [case[n].clone().requires_grad_() for n in ("x", "weight", "bias")]
    y = pretrain_layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, case["dy"])
    h = 2.0 ** -7
    for i, grad in enumerate(grads):
        move = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV)

        def value(sign):
            args = [t.detach() + (sign * h * move if j == i else 0) for j, t in enumerate(leaves)]
            return (pretrain_layer_norm(*args).double() * case["dy"].double()).sum()

        slope = ((value(1) - value(-1)) / (2 * h)).item()
        want = (grad.double() * move.double()).sum().item()
        scale = (grad.double().norm() * move.double().norm()).item()
        assert abs(slope - want) <= 2e-3 * scale


def test_leading_shapes_empty_rows_and_other_streams():
    case = _inputs(24, 128, torch.bfloat16, seed=9)
    flat = pretrain_layer_norm(case["x"], case["weight"], case["bias"])
    deep = pretrain_layer_norm(case["x"].view(2, 3, 4, 128), case["weight"], case["bias"])
    assert torch.equal(deep.view(24, 128), flat)
    assert torch.equal(pretrain_layer_norm(case["x"][0], case["weight"], case["bias"]), flat[0])
    empty = case["x"][:0].clone().requires_grad_()
    weight = case["weight"].clone().requires_grad_()
    y = pretrain_layer_norm(empty, weight, case["bias"])
    grads = torch.autograd.grad(y, [empty, weight], torch.empty_like(y))
    assert y.shape == (0, 128) and grads[0].shape == (0, 128) and not grads[1].any()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x = case["x"].clone()
        got = pretrain_layer_norm(x, case["weight"], case["bias"])
    stream.synchronize()
    assert torch.equal(got, flat)


def test_inference_form_under_graph_capture():
    """Captured with the residual, replayed with other data and the program's
    own work between the replays; every replay equals the eager call."""
    case = _inputs(16, 2560, torch.float16, seed=10, residual=True)

    def step():
        return infer_layer_norm_forward_varlen(case["x"], case["weight"], case["bias"],
                                               residual=case["residual"])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stream = step()
    for seed in range(4):
        fresh = _inputs(16, 2560, torch.float16, seed=20 + seed, residual=True)
        case["x"].copy_(fresh["x"])
        case["residual"].copy_(fresh["residual"])
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(stream, want[1])


class _Sub(torch.Tensor):
    """A tensor subclass: no whole call, the wrapper's own tables and autograd function."""


def test_calls_that_are_not_plain_give_the_same_bits():
    case = _inputs(40, 384, torch.float16, seed=30, residual=True)
    names = ("x", "weight", "bias", "residual")
    plain = [case[n].clone().requires_grad_() for n in names]
    y, stream = pretrain_layer_norm(*plain[:3], residual=plain[3])
    grads = torch.autograd.grad((y, stream), plain, (case["dy"], case["ds"]))
    sub = [case[n].clone().as_subclass(_Sub).requires_grad_() for n in names]
    y2, stream2 = pretrain_layer_norm(*sub[:3], residual=sub[3])
    grads2 = torch.autograd.grad((y2, stream2), sub, (case["dy"], case["ds"]))
    for a, b in zip((y, stream, *grads), (y2, stream2, *grads2)):
        assert torch.equal(a, b.as_subclass(torch.Tensor))


@pytest.mark.parametrize("kind", [torch.Tensor, _Sub])
def test_differentiating_twice_raises(kind):
    case = _inputs(4, 64, torch.float32, seed=31)
    x = case["x"].clone().as_subclass(kind).requires_grad_()
    y = pretrain_layer_norm(x, case["weight"], case["bias"])
    dx, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dx.sum().backward()

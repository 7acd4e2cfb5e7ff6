"""GPU parity of the gradient norm and clipping against 64 bits.

Bounds, before any run: squares and sums are in 64 bits (relative error far below
2^-40) and the norm is rounded once to 32: 2^-24 of it, 2 2^-24 allowed. The factor is
rounded once to 32 bits, the product once to 32 bits and once to the output's type:
2 2^-24 |y| (1 + u) + u |y| and the type's smallest step.
"""

from __future__ import annotations

import math

import pytest
import torch

import flashrwkv_amd
from flashrwkv_amd import capi, pretrain_clip_grad_norm, pretrain_grad_norm
from oracle import step

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
E = 2.0 ** -24
ROUND = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
TYPES = list(ROUND)


@pytest.fixture(scope="module", autouse=True)
def _require_native():
    if flashrwkv_amd._C is None:
        pytest.fail("flashrwkv_amd native library is not built (no fallback exists)")


def _tensors(shapes, seed, scale=1.0, types=TYPES):
    gen = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(s, generator=gen)).to(types[i % len(types)]).to(DEV)
            for i, s in enumerate(shapes)]


def _check(tensors, got, norm, max_norm, eps=1e-6):
    want, clipped = step.clip(tensors, max_norm, eps)
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(norm.item() - want) <= 2 * E * want
    for y, x in zip(got, clipped):
        u = ROUND[y.dtype]
        allowed = (2 * E * (1 + u) + u) * x.abs() + STEP[y.dtype]
        assert ((y.double() - x).abs() <= allowed).all()


LISTS = {
    "one element": [(1,)],
    "one scalar": [()],
    "small": [(3,), (64, 5), (1, 1, 1), (0,), (7, 0, 3), (8191,), (8192,), (8193,)],
    "chunks": [(3 * 8192,), (2, 8192 + 8), (50000,), (77,)],
    "many": [(1 + (i * 37) % 400,) for i in range(500)],
    "large": [(5_000_003,), (300, 4096), (17,)],
    # Lists that stand in memory: units that are read together and alone, and a tensor
    # of more units than are summed at a time.
    "long list": [(1 + (i * 2477) % 30000,) for i in range(230)],
    "one of many units": [(40_000_001,), (2048,), (2049,)],
}


@pytest.mark.parametrize("over", [True, False])
@pytest.mark.parametrize("name", LISTS)
def test_clip_in_place_and_into_others(name, over):
    print(f"case {name} over {over}", flush=True)
    tensors = _tensors(LISTS[name], seed=1)
    norm = step.clip(tensors, 1.0, 0.0)[0]
    most = norm * (0.3 if over else 1.5)
    assert abs(pretrain_grad_norm(tensors).item() - norm) <= 2 * E * norm
    before = [t.clone() for t in tensors]
    for types in ([torch.float32], [torch.bfloat16, torch.float16, torch.float32]):
        out = [torch.full_like(t, math.nan, dtype=types[i % len(types)])
               for i, t in enumerate(tensors)]
        _check(tensors, out, pretrain_clip_grad_norm(tensors, most, out=out), most)
        assert all(torch.equal(a, b) for a, b in zip(tensors, before))
    got = pretrain_clip_grad_norm(tensors, most)
    _check(before, tensors, got, most)
    if not over:
        assert all(torch.equal(a, b) for a, b in zip(tensors, before))


def test_more_than_the_last_level_cache():
    """300 MB in bf16 and fp32, read past the caches, 16-byte places or not."""
    gen = torch.Generator(device=DEV).manual_seed(8)
    flat = torch.randn(40_000_007, generator=gen, device=DEV)
    tensors = [flat[3:], torch.randn(70_000_001, generator=gen, device=DEV).bfloat16()]
    before = [t.clone() for t in tensors]
    out = [torch.empty_like(t, dtype=torch.float32) for t in tensors]
    most = 0.1 * math.sqrt(110_000_005)
    _check(before, out, pretrain_clip_grad_norm(tensors, most, out=out), most)
    _check(before, tensors, pretrain_clip_grad_norm(tensors, most), most)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 3, 8])
def test_views_off_16_byte_places(dtype, offset):
    """Views of one buffer; what stands between them stays."""
    gen = torch.Generator().manual_seed(offset)
    flat = torch.randn(60000, generator=gen).to(dtype).to(DEV)
    spans = [(offset, 5000), (5000 + offset, 20001), (20003 + offset, 20004 + offset),
             (30000, 50000 - offset)]
    views = [flat[a:b] for a, b in spans]
    before, kept = flat.clone(), torch.ones(60000, dtype=torch.bool, device=DEV)
    for a, b in spans:
        kept[a:b] = False
    norm = pretrain_clip_grad_norm(views, 5.0)
    _check([before[a:b] for a, b in spans], views, norm, 5.0)
    assert torch.equal(flat[kept], before[kept])


def test_orders_of_dimensions():
    a = torch.randn(30, 70, device=DEV).t()
    b = torch.randn(4, 6, 5, 8, device=DEV).to(memory_format=torch.channels_last).bfloat16()
    before = [a.clone(), b.clone()]
    out = [torch.empty_strided(t.shape, t.stride(), device=DEV) for t in (a, b)]
    _check(before, out, pretrain_clip_grad_norm([a, b], 2.0, out=out), 2.0)
    _check(before, [a, b], pretrain_clip_grad_norm((a, b), 2.0), 2.0)


def test_values_whose_squares_32_bits_do_not_hold():
    for value in (1e25, 1e-30):
        t = torch.full((10000,), value, device=DEV)
        want = float(t[0].double()) * 100
        assert abs(pretrain_grad_norm([t]).item() - want) <= 2 * E * want
        assert pretrain_clip_grad_norm([t], want / 4, eps=0.0).item() == pytest.approx(want)
        assert torch.allclose(t, torch.full_like(t, value / 4), rtol=4 * E, atol=0)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_norm_that_is_not_finite_scales_nothing(bad):
    tensors = _tensors([(100,), (9000,)], seed=3)
    tensors[1][77] = bad
    before = [t.clone() for t in tensors]
    norm = pretrain_clip_grad_norm(tensors, 1e-3)
    assert not math.isfinite(norm.item())
    out = [torch.zeros_like(t) for t in tensors]
    pretrain_clip_grad_norm(tensors, 1e-3, out=out)
    for x, y, z in zip(before, tensors, out):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))
        assert torch.equal(x.nan_to_num(7.0), z.nan_to_num(7.0))


@pytest.mark.parametrize("count", [4, 300])
def test_a_norm_beyond_32_bits_scales_nothing(count):
    """Each value is fp32's, their norm (2e38 sqrt(count)) is not: the returned norm is
    infinite, by which a caller skips the step, so the tensors are left alone too."""
    tensors = [torch.full((1,), 2e38, device=DEV) for _ in range(count)]
    norm = pretrain_clip_grad_norm(tensors, 1.0)
    assert norm.item() == math.inf == pretrain_grad_norm(tensors).item()
    assert all(t.item() == torch.tensor(2e38).item() for t in tensors)


def test_zeros_and_a_maximum_of_zero():
    t = torch.zeros(100, device=DEV)
    assert pretrain_clip_grad_norm([t], 1.0).item() == 0.0
    assert pretrain_clip_grad_norm([t], 0.0, eps=0.0).item() == 0.0 and not t.any()
    u = torch.ones(100, device=DEV)
    assert pretrain_clip_grad_norm([u], 0.0).item() == 10.0
    assert not u.any()


def test_writes_count_as_such():
    t = torch.ones(10, device=DEV)
    version = t._version
    pretrain_clip_grad_norm([t], 1.0)
    assert t._version > version
    p = torch.ones(10, device=DEV, requires_grad=True)
    y = p * t
    pretrain_clip_grad_norm([t], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals_that_need_a_gpu():
    a, b = torch.ones(10, device=DEV), torch.ones(10, device=DEV)
    assert pretrain_grad_norm([a, a]).item() == pytest.approx(math.sqrt(20))
    for tensors, out in (([a, a], None), ([a[:6], a[5:]], None), ([a, b], [b, a]),
                         ([a, b], [a, a]), ([a[:5]], [a[2:7]])):
        with pytest.raises(ValueError, match="overlap"):
            pretrain_clip_grad_norm(tensors, 1.0, out=out)
    assert torch.equal(a, b)
    with pytest.raises(ValueError, match="gaps"):
        pretrain_grad_norm([a[::2]])
    with pytest.raises(ValueError, match="gaps"):
        pretrain_grad_norm([a[:1].expand(4)])
    with pytest.raises(ValueError, match="negated"):
        pretrain_clip_grad_norm([torch._neg_view(a)], 1.0)
    leaf = torch.ones(4, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="must not require gradients"):
        pretrain_clip_grad_norm([leaf], 1.0)
    with torch.no_grad():
        pretrain_clip_grad_norm([leaf], 1.0)
    assert leaf[0].item() == pytest.approx(0.5)
    with pytest.raises(ValueError, match="share the first tensor's device|CUDA"):
        pretrain_grad_norm([a, torch.ones(3)])
    with pytest.raises(ValueError, match="shape and strides"):
        pretrain_clip_grad_norm([torch.ones(3, 4, device=DEV)], 1.0,
                                out=[torch.ones(4, 3, device=DEV).t()])


def test_calls_repeat_bitwise_on_any_stream_and_in_graphs():
    tensors = _tensors([(100_003,), (50, 1000)], seed=5)
    out = [torch.zeros_like(t) for t in tensors]
    first = pretrain_clip_grad_norm(tensors, 1.0, out=out)
    kept = [t.clone() for t in out]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = pretrain_clip_grad_norm(tensors, 1.0, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            norm = pretrain_clip_grad_norm(tensors, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(first, again)
    for k in range(4):
        for t in tensors:
            t.mul_(1.0 + k)
        graph.replay()
        torch.cuda.synchronize()
        got, seen = norm.clone(), [t.clone() for t in out]
        want = pretrain_clip_grad_norm(tensors, 1.0, out=out)
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(out, seen))
        if k == 0:
            assert torch.equal(got, first) and all(torch.equal(a, b) for a, b in zip(kept, seen))


def test_two_graphs_of_long_lists_in_one_pool():
    """Lists that stand in the calls' own memory, replayed in turn with eager calls between."""
    lists = [_tensors(LISTS["long list"], seed=7), _tensors(LISTS["many"], seed=8)]
    outs = [[torch.zeros_like(t, dtype=torch.float32) for t in tensors] for tensors in lists]
    graphs, norms, pool = [], [], None
    for tensors, out in zip(lists, outs):
        pretrain_clip_grad_norm(tensors, 1.0, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            norms.append(pretrain_clip_grad_norm(tensors, 1.0, out=out))
        pool = graph.pool()
        graphs.append(graph)
    for k in range(3):
        for tensors, out, graph, norm in zip(lists, outs, graphs, norms):
            tensors[k].mul_(1.5 + k)
            graph.replay()
            torch.cuda.synchronize()
            _check(tensors, out, norm, 1.0)
            eager = [torch.zeros_like(t) for t in out]
            assert torch.equal(pretrain_clip_grad_norm(tensors, 1.0, out=eager), norm)
            assert all(torch.equal(x, y) for x, y in zip(eager, out))


def test_c_abi_writes_what_the_operators_return():
    tensors = _tensors([(5000,), (0,), (33, 3)], seed=6)
    out = [torch.zeros_like(t) for t in tensors]
    want = pretrain_clip_grad_norm(tensors, 1.0, out=out)
    norm, got = torch.empty(1, device=DEV), [torch.zeros_like(t) for t in tensors]
    capi.grad_norm(tensors, norm=norm)
    assert torch.equal(norm[0], want)
    capi.grad_clip(tensors, 1.0, norm=norm, out=got)
    assert torch.equal(norm[0], want) and all(torch.equal(a, b) for a, b in zip(got, out))
    capi.grad_norm([], norm=norm)
    assert norm.item() == 0.0


def test_subclasses_take_the_tables():
    class Wrapped(torch.Tensor):
        pass

    t = torch.ones(100, device=DEV).as_subclass(Wrapped)
    assert pretrain_grad_norm([t]).item() == 10.0
    assert pretrain_clip_grad_norm([t], 5.0, eps=0.0).item() == 10.0
    assert torch.equal(t.as_subclass(torch.Tensor), torch.full((100,), 0.5, device=DEV))


@pytest.mark.parametrize("sizes", [[100, 31], [9_000_000], [77] * 200])
def test_factors_that_32_bits_do_not_hold(sizes):
    """A norm so far above the maximum that their quotient is not a normal number of 32 bits,
    or not one at all, while its products with the elements are."""
    gen = torch.Generator().manual_seed(9)
    tensors = [(1e34 * torch.randn(n, generator=gen)).to(DEV) for n in sizes]
    norm = step.clip(tensors, 1.0, 0.0)[0]
    for by in (3e-41, 2e-47):
        for dtype in (torch.float32, torch.bfloat16):
            out = [torch.empty_like(t, dtype=dtype) for t in tensors]
            _check(tensors, out, pretrain_clip_grad_norm(tensors, norm * by, out=out), norm * by)
            assert all(t.any() for t in out)
        copies = [t.clone() for t in tensors]
        _check(tensors, copies, pretrain_clip_grad_norm(copies, norm * by), norm * by)


def test_tensors_that_share_memory_until_they_are_written():
    """A lazy copy's own memory is written, not the one that it shares until then."""
    for out in (False, True):
        a = torch.ones(100, device=DEV)
        lazy = torch._lazy_clone(a)
        norm = pretrain_clip_grad_norm([a.clone() if out else lazy], 1.0, eps=0.0,
                                       out=[lazy] if out else None)
        assert norm.item() == 10.0
        assert torch.equal(a, torch.ones_like(a))
        assert torch.allclose(lazy, torch.full_like(a, 0.1))


def _long_list(seed, sizes, offset):
    """Views of one buffer a type, `offset` elements off 16-byte places, with gaps between."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    room = {dtype: 0 for dtype in TYPES}
    places = []
    for i, n in enumerate(sizes):
        dtype = TYPES[i % len(TYPES)]
        places.append((dtype, room[dtype] + offset, n))
        room[dtype] += (n + offset + 63) // 64 * 64
    flat = {dtype: torch.randn(n, generator=gen, device=DEV).to(dtype)
            for dtype, n in room.items()}
    return flat, [flat[dtype][at:at + n] for dtype, at, n in places]


def _stands_in_memory(tensors):
    """Whether the call's memory holds the units' owners, beside at most 17 KB of sums."""
    units = sum((t.numel() + 2047) // 2048 for t in tensors)
    need = capi.library().frwkv_grad_norm_workspace_bytes(
        len(tensors), capi._gradients(tensors, tensors))
    return len(tensors) > 112 and need >= 4 * units + 32 * len(tensors)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("large", [True, False])
def test_long_lists_of_many_units(large, offset):
    """Lists that stand in memory, of more units than are summed at a time, beyond the
    last-level cache and within it; in place and into other types, over the maximum and under."""
    sizes = [(1_200_000 if large else 150_000) + 1237 * (i % 50) for i in range(120)]
    sizes[7::10] = [1 + (i * 311) % 5000 for i in range(len(sizes[7::10]))]
    flat, tensors = _long_list(10, sizes, offset)
    total = sum(t.numel() for t in tensors)
    assert total > 4 * 2048 * 2048 * (1 if not large else 4) and _stands_in_memory(tensors)
    assert (sum(t.numel() * t.element_size() for t in tensors) > 256 << 20) == large
    norm = step.clip(tensors, 1.0, 0.0)[0]
    before = {dtype: t.clone() for dtype, t in flat.items()}
    for by in (0.3, 1.5):
        out = [torch.full_like(t, math.nan, dtype=TYPES[(i + i // 3) % 3])
               for i, t in enumerate(tensors)]
        _check(tensors, out, pretrain_clip_grad_norm(tensors, norm * by, out=out), norm * by)
        del out
    assert all(torch.equal(before[dtype], t) for dtype, t in flat.items())
    assert abs(pretrain_clip_grad_norm(tensors, norm * 1.5).item() - norm) <= 2 * E * norm
    assert all(torch.equal(before[dtype], t) for dtype, t in flat.items())
    sources = [before[t.dtype][t.storage_offset():t.storage_offset() + t.numel()]
               for t in tensors]
    _check(sources, tensors, pretrain_clip_grad_norm(tensors, norm * 0.3), norm * 0.3)
    # What stands between the tensors stays.
    for dtype, t in flat.items():
        kept = torch.ones(t.numel(), dtype=torch.bool, device=DEV)
        for x in tensors:
            if x.dtype == dtype:
                kept[x.storage_offset():x.storage_offset() + x.numel()] = False
        assert torch.equal(t[kept], before[dtype][kept])


@pytest.mark.parametrize("offset", [0, 3])
def test_few_tensors_beyond_the_last_level_cache(offset):
    """A list in the kernels' arguments, read through the caches whatever its size."""
    flat, tensors = _long_list(11, [45_000_001, 30_000_007, 20_000_000, 2049], offset)
    assert not _stands_in_memory(tensors)
    assert sum(t.numel() * t.element_size() for t in tensors) > 256 << 20
    norm = step.clip(tensors, 1.0, 0.0)[0]
    out = [torch.empty_like(t, dtype=torch.float32) for t in tensors]
    _check(tensors, out, pretrain_clip_grad_norm(tensors, norm * 0.1, out=out), norm * 0.1)
    before = [t.clone() for t in tensors]
    _check(before, tensors, pretrain_clip_grad_norm(tensors, norm * 0.1), norm * 0.1)


def test_offsets_of_elements_beyond_32_bits():
    """One tensor of 2^31 elements and some, whose last units stand behind 2^32 bytes."""
    n = 2 ** 31 + 4099
    t = torch.full((n,), 0.5, device=DEV, dtype=torch.bfloat16)
    t[-1], t[2 ** 31] = 1000.0, -2000.0
    norm = math.sqrt(0.25 * (n - 2) + 1000.0 ** 2 + 2000.0 ** 2)
    assert abs(pretrain_grad_norm([t]).item() - norm) <= 2 * E * norm
    assert abs(pretrain_clip_grad_norm([t], norm / 4, eps=0.0).item() - norm) <= 2 * E * norm
    # A quarter of each, within a rounding of the norm and one of the factor and the product.
    assert t[-1].item() == 250.0 and t[2 ** 31].item() == -500.0
    t[-1], t[2 ** 31] = 0.125, 0.125
    assert t.min().item() == t.max().item() == 0.125

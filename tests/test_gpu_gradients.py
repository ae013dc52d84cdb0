"""gradient_norm and clip_gradients against 64 bits on the CPU.

The squares' sum is fp64 on both sides: the norm is off by its one rounding to fp32, 2^-24
of it, and n 2^-53.  The factor carries the rounding of its own fp32 value, the product one
more, and the result's type its rounding v: 2 u + v of each value."""

import math

import pytest
import torch

import sdfoam_amd

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: (2.0 ** -24, 2.0 ** -126), torch.float16: (2.0 ** -11, 2.0 ** -24),
         torch.bfloat16: (2.0 ** -8, 2.0 ** -126)}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def say(*a):
    print(*a, flush=True)


def expected(tensors, max_norm, scale):
    norm = scale * math.sqrt(sum(float(t.double().pow(2).sum()) for t in tensors))
    return norm, scale * min(1.0, max_norm / (norm + 1e-6))


def check(got, g, factor):
    v, tiny = ROUND[got.dtype]
    ref = g.double() * factor
    off = (got.cpu().double() - ref).abs()
    assert torch.all(off <= (2 * U + v) * 1.01 * ref.abs() + tiny)


SHAPES = [
    [(1,)], [(0,), (3,)], [(7,), (), (2, 0, 3), (5, 9)], [(16_385,), (16_384,), (8,)],
    [(300, 49), (64, 3, 3, 3), (1,), (100_003,)], [(3,)] * 250, [(40_000,)] * 97 + [(1,)],
    [(3_000_001,)], [(17, 1000)] * 20,
]


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16", "mixed"])
@pytest.mark.parametrize("shapes", SHAPES, ids=range(len(SHAPES)))
def test_clip(dev, shapes, kind):
    say("clip", len(shapes), shapes[:3], kind)
    g = torch.Generator().manual_seed(len(shapes))
    types = TYPES if kind == "mixed" else [getattr(torch, kind)]
    tensors = [torch.randn(s, generator=g).to(types[k % len(types)]) for k, s in enumerate(shapes)]
    for max_norm, scale in ((0.5, 1.0), (1e9, 1.0), (2.0, 0.125), (1e9, 0.25), (0.0, 1.0)):
        norm, factor = expected(tensors, max_norm, scale)
        own = [t.to(dev) for t in tensors]
        got = sdfoam_amd.gradient_norm(own, scale)
        assert got.dtype == torch.float32 and got.shape == ()
        assert abs(float(got) - norm) <= 2 * U * norm
        before = [t._version for t in own]
        again = sdfoam_amd.clip_gradients(own, max_norm, scale)
        assert torch.equal(again, got)
        assert all(t._version > b for t, b in zip(own, before))
        for t, ref in zip(own, tensors):
            check(t, ref, factor)
            if factor == 1.0:
                assert torch.equal(t.cpu(), ref)
        for out_type in (torch.float32, None):
            own = [t.to(dev) for t in tensors]
            flat = torch.full((sum(t.numel() for t in tensors) + 1,), 7.0, device=dev)
            if out_type is None:
                out = [torch.empty_like(t) for t in own]
            else:  # one buffer, one result behind the other, from an odd element on
                out, at = [], 1
                for t in own:
                    out.append(flat[at:at + t.numel()].view(t.shape))
                    at += t.numel()
            got = sdfoam_amd.clip_gradients(own, max_norm, scale, out=out)
            assert torch.equal(got, again) and float(flat[0]) == 7.0
            for t, o, ref in zip(own, out, tensors):
                assert torch.equal(t.cpu(), ref)
                check(o, ref, factor)


def test_layouts_and_none(dev):
    g = torch.Generator().manual_seed(3)
    a = torch.randn((30, 20), generator=g)
    b = torch.randn((2, 8, 5, 5), generator=g)
    turned = a.to(dev).t()
    last = b.to(dev).to(memory_format=torch.channels_last)
    norm, factor = expected([a, b], 1.0, 1.0)
    got = sdfoam_amd.clip_gradients((k for k in (None, turned, last, None)), 1.0)
    assert abs(float(got) - norm) <= 2 * U * norm
    check(turned.t(), a, factor)
    check(last, b, factor)
    one = torch.randn(100, generator=g)
    own = one.to(dev)
    assert abs(float(sdfoam_amd.gradient_norm(own)) - float(one.double().norm())) <= 2 * U * 20
    # twice the same counts twice
    assert abs(float(sdfoam_amd.gradient_norm([own, own])) -
               math.sqrt(2.0) * float(one.double().norm())) <= 2 * U * 20
    empty = torch.empty((0, 4), device=dev)
    assert float(sdfoam_amd.clip_gradients([empty], 1.0)) == 0.0


def test_slices_of_one_buffer(dev):
    """Gradients that are neighbours in memory are scaled each by itself, and nothing
    between or beside them is written."""
    flat = torch.arange(1.0, 1001.0, device=dev)
    parts = [flat[1:4], flat[4:500], flat[501:999]]
    ref = [p.cpu() for p in parts]
    norm, factor = expected(ref, 3.0, 1.0)
    sdfoam_amd.clip_gradients(parts, 3.0)
    for p, r in zip(parts, ref):
        check(p, r, factor)
    for k, v in ((0, 1.0), (500, 501.0), (999, 1000.0)):
        assert float(flat[k]) == v


def test_far_sizes(dev):
    """Squares that fp32 does not hold."""
    for size in (1e-30, 1e30):
        t = torch.full((1000,), size)
        own = t.to(dev)
        norm = math.sqrt(1000.0) * float(t.double()[0])
        got = sdfoam_amd.clip_gradients([own], 1.0)
        assert abs(float(got) - norm) <= 2 * U * norm
        check(own, t, min(1.0, 1.0 / (norm + 1e-6)))


def test_not_finite(dev):
    t = torch.tensor([1.0, math.inf, -2.0], device=dev)
    u = torch.ones(4, device=dev)
    assert float(sdfoam_amd.clip_gradients([t, u], 1.0)) == math.inf
    assert torch.equal(u, torch.zeros(4, device=dev)) and torch.isnan(t[1]) and float(t[0]) == 0.0
    t = torch.tensor([1.0, math.nan], device=dev)
    u = torch.ones(4, device=dev)
    assert math.isnan(float(sdfoam_amd.clip_gradients([t, u], 1.0)))
    assert torch.isnan(t).all() and torch.isnan(u).all()


def test_same_on_every_run(dev):
    g = torch.Generator().manual_seed(1)
    t = [torch.randn(n, generator=g).to(dev) for n in (999_983, 5, 70_001)]
    first = sdfoam_amd.gradient_norm(t)
    for _ in range(3):
        assert torch.equal(sdfoam_amd.gradient_norm(t), first)


def test_refusals_of_memory(dev):
    t = torch.ones(100, device=dev)
    with pytest.raises(RuntimeError, match="twice, or results overlap"):
        sdfoam_amd.clip_gradients([t, t], 1.0)
    with pytest.raises(RuntimeError, match="twice, or results overlap"):
        sdfoam_amd.clip_gradients([t[:50], t[49:]], 1.0)
    with pytest.raises(RuntimeError, match="must not overlap another gradient"):
        sdfoam_amd.clip_gradients([t[:50], t[50:]], 1.0,
                                  out=[t[50:], torch.empty(50, device=dev)])
    with pytest.raises(RuntimeError, match="overlap"):
        sdfoam_amd.clip_gradients([t[:50]], 1.0, out=[t[1:51]])
    with pytest.raises(RuntimeError, match="without gaps or overlaps"):
        sdfoam_amd.clip_gradients([t[:1].expand(5)], 1.0)
    with pytest.raises(RuntimeError, match="without gaps or overlaps"):
        sdfoam_amd.clip_gradients([t[::2]], 1.0)
    half = torch.ones(64, device=dev).half()
    over = torch.empty(0, device=dev).set_(half.untyped_storage(), 0, (32,))
    with pytest.raises(RuntimeError, match="overlap"):
        sdfoam_amd.clip_gradients([half[:32]], 1.0, out=[over])
    assert torch.equal(t, torch.ones(100, device=dev))


def test_label_field_clips(dev):
    """The example trains with clipped gradients."""
    import importlib.util
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location(
        "label_field", os.path.join(root, "examples", "label_field.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(points=3000, labels=32, features=8, size=32, cameras=3, batch=1024, steps=3,
                     max_norm=0.01, log=None)
    assert all(math.isfinite(x) for x in r["loss"])


def test_in_a_graph(dev):
    g = torch.Generator().manual_seed(4)
    ref = [torch.randn(n, generator=g) for n in (5000, 33, 1)] * 40
    own = [t.to(dev) for t in ref]
    out = [torch.empty_like(t) for t in own]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sdfoam_amd.clip_gradients(own, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = sdfoam_amd.clip_gradients(own, 1.0, out=out)
    for k in range(3):
        for t in own:
            t.mul_(0.9)
        eager = [torch.empty_like(t) for t in own]
        want = sdfoam_amd.clip_gradients(own, 1.0, out=eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("size,max_norm,scale", [
    (1e37, 1e-6, 1.0), (1e37, 1e-3, 1.0), (3e36, 1.0, 2.0 ** -20), (1e37, 1e-38, 1.0),
    (1e30, 1e-20, 1e-10), (1.0, 1e9, 1e-41)])
def test_factors_below_the_range(dev, size, max_norm, scale):
    """Factors that float32 holds with few bits or none, whose products it holds."""
    say("small factors", size, max_norm, scale)
    g = torch.Generator().manual_seed(7)
    scale = float(torch.tensor(scale))  # as the call takes them
    max_norm = float(torch.tensor(max_norm))
    for own_type, out_type in ((torch.float32, None), (torch.bfloat16, None),
                               (torch.bfloat16, torch.float32)):
        t = (size * (1.0 + torch.rand(777, generator=g))).to(own_type)
        norm, factor = expected([t], max_norm, scale)
        own = t.to(dev)
        out = None if out_type is None else [torch.empty_like(own, dtype=out_type)]
        got = sdfoam_amd.clip_gradients([own], max_norm, scale, out=out)
        if norm < 2.0 ** 128:
            assert abs(float(got) - norm) <= 2 * U * norm + 2.0 ** -149
        else:  # past float32's largest, 2^128 (1 - 2^-24), by more than half a step
            assert float(got) == math.inf
        check(own if out is None else out[0], t, factor)


def test_norms_past_the_range(dev):
    """Finite gradients whose norm float32 does not hold: it is returned as infinite, and the
    gradients are clipped by what it is."""
    for kind in (torch.float32, torch.bfloat16):
        t, u = torch.full((1000,), 3e38).to(kind), torch.full((33,), -2e38).to(kind)
        norm, factor = expected([t, u], 2.0, 1.0)
        a, b = t.to(dev), u.to(dev)
        assert float(sdfoam_amd.gradient_norm([a, b])) == math.inf
        assert float(sdfoam_amd.clip_gradients([a, b], 2.0)) == math.inf
        check(a, t, factor)
        check(b, u, factor)
        assert abs(float(sdfoam_amd.gradient_norm([a, b])) - 2.0) <= 2.0 * (3 * U + ROUND[kind][0])
        # an infinite gradient is another matter
        a[5] = math.inf
        assert float(sdfoam_amd.clip_gradients([a, b], 2.0)) == math.inf
        assert torch.isnan(a[5]) and not a[:5].any() and not b.any()
    a = torch.tensor([1.0, -2.0], device=dev)
    sdfoam_amd.clip_gradients([a], math.inf, 0.5)
    assert torch.equal(a.cpu(), torch.tensor([0.5, -1.0]))
    a[0] = math.inf
    assert float(sdfoam_amd.clip_gradients([a], math.inf)) == math.inf and torch.isnan(a).all()


def test_one_tensor_into_another(dev):
    """One gradient and one result, neither in a list."""
    g = torch.Generator().manual_seed(6)
    for shape in ((40,), (5, 8), (1, 40), ()):
        t = torch.randn(shape, generator=g).to(torch.bfloat16)
        own, out = t.to(dev), torch.full(shape, math.nan, device=dev)
        got = sdfoam_amd.clip_gradients(own, 0.25, out=out)
        want = torch.empty_like(out)
        assert torch.equal(got, sdfoam_amd.clip_gradients([own], 0.25, out=[want]))
        assert torch.equal(out, want) and torch.equal(own.cpu(), t)
    # the rows of a matrix are results too
    rows = [torch.randn(8, generator=g).to(dev) for _ in range(3)]
    matrix = torch.empty((3, 8), device=dev)
    sdfoam_amd.clip_gradients(rows, 0.25, out=matrix)
    sdfoam_amd.clip_gradients(rows, 0.25)
    assert torch.equal(matrix, torch.stack(rows))

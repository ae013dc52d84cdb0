"""The heads' operators (expert_order, expert_rows, expert_combine, expert_linear,
adapter_linear and their gradients) against plain statements of their formulas in 64 bits,
on the CPU.

Bounds, from the arithmetic alone.  u = 2^-24 is fp32's rounding, v that of the output's
type (2^-24, 2^-11, 2^-8), each with the type's smallest step below its normal range.

* a sum of n products in fp32, in any order and with up to two roundings a term (the product
  and the sum): 2 n u times the sum of the products' sizes; 8 more for the joining of parts
  and the scale; then v for the result;
* an adapter's inner values carry such an error into every product that they enter: the
  bound of the inner sum times the size of the other factor, summed.
"""

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


def near(got, ref, tol, dtype):
    """|got - ref| <= tol and the rounding to dtype, the same infinities and NaN."""
    assert got.dtype == dtype
    got = got.detach().cpu().double()
    v, tiny = ROUND[dtype]
    assert got.shape == ref.shape
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    off = (got - ref).abs()
    lim = tol + v * ref.abs() * 1.01 + tiny
    assert torch.all((off <= lim)[fine]), float((off - lim)[fine].max())


def bound(n):
    return (2 * n + 8) * U


def ids_as(ids, dtype, dev):
    """int64 ids on the device as `dtype` (-1 is 0xffffffff in uint32)."""
    if dtype == torch.uint32:
        return ids.to(torch.int32).to(dev).view(torch.uint32)
    return ids.to(dtype).to(dev)


ID_TYPES = [torch.int64, torch.uint32, torch.int32]


def some_ids(shape, groups, seed, none=0.1, spread="any"):
    g = torch.Generator().manual_seed(seed)
    if groups == 0 or spread == "none":
        return torch.full(shape, -1, dtype=torch.int64)
    if spread == "one":
        ids = torch.full(shape, groups // 2, dtype=torch.int64)
    elif spread == "few":
        ids = torch.where(torch.rand(shape, generator=g) < 0.8,
                          torch.randint(min(2, groups), shape, generator=g),
                          torch.randint(groups, shape, generator=g))
    else:
        ids = torch.randint(groups, shape, generator=g)
    ids[torch.rand(shape, generator=g) < none] = -1
    return ids


def order_reference(ids, groups):
    flat = ids.reshape(-1)
    named = (flat >= 0) & (flat < groups)
    key = torch.where(named, flat, groups)
    order = torch.sort(key, stable=True).indices
    places = torch.empty_like(flat)
    places[order] = torch.arange(flat.numel())
    places = torch.where(named, places, -1 - places).reshape(ids.shape)
    count = torch.bincount(key, minlength=groups + 1)[:groups]
    return places, torch.cat([torch.zeros(1, dtype=torch.int64), count.cumsum(0)])


# ---- the order -------------------------------------------------------------------------------

ORDERS = [  # rows, choices, experts, spread
    (1, 1, 1, "any"), (1, 4, 64, "any"), (0, 3, 5, "any"), (7, 0, 5, "any"), (9, 2, 0, "none"),
    (63, 1, 2, "any"), (65, 2, 3, "few"), (1000, 3, 31, "any"), (4096, 1, 64, "one"),
    (4097, 1, 63, "any"), (2048, 8, 2048, "any"), (50_000, 2, 1023, "few"),
    (300_001, 1, 17, "any"), (70_000, 8, 300, "few"), (300_000, 1, 2048, "none"),
]


@pytest.mark.parametrize("rows,choices,experts,spread", ORDERS)
def test_order(dev, rows, choices, experts, spread):
    say("order", rows, choices, experts, spread)
    ids = some_ids((rows, choices), experts, 3, spread=spread)
    if experts:  # too large names none as well
        ids[::7] = torch.where(ids[::7] == 0, experts + 5, ids[::7])
    places, offsets = order_reference(ids, experts)
    for t in ID_TYPES:
        order = sdfoam_amd.expert_order(ids_as(ids, t, dev), experts)
        assert order.places.dtype == order.offsets.dtype == torch.int32
        assert torch.equal(order.places.cpu().long(), places)
        assert torch.equal(order.offsets.cpu().long(), offsets)


# ---- rows and back ---------------------------------------------------------------------------

SPREADS = [  # rows, choices, experts, width
    (1, 1, 1, 1), (1, 4, 8, 2048), (3, 2, 5, 7), (33, 3, 4, 49), (65, 1, 9, 8), (100, 8, 16, 130),
    (257, 2, 3, 1024), (1000, 4, 64, 5), (5000, 2, 7, 33), (17, 2, 3, 4099), (40, 3, 5, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,choices,experts,width", SPREADS)
def test_rows_and_back(dev, rows, choices, experts, width, dtype):
    say("rows and back", rows, choices, experts, width, dtype)
    ids = some_ids((rows, choices), experts, rows + width)
    g = torch.Generator().manual_seed(width)
    x = torch.randn((rows, width), generator=g).to(dtype)
    y = torch.randn((rows * choices, width), generator=g).to(dtype)
    w = torch.rand((rows, choices), generator=g)
    grad = torch.randn((rows, width), generator=g).to(dtype)
    places, _ = order_reference(ids, experts)
    at = torch.where(places < 0, -1 - places, places)
    named = (places >= 0).double()
    order = sdfoam_amd.expert_order(ids.to(dev), experts)

    out = sdfoam_amd.expert_rows(x.to(dev), order)
    ref = torch.zeros((rows * choices, width), dtype=torch.float64)
    ref[at.reshape(-1)] = (x.double()[:, None] * named[..., None]).flatten(0, 1)
    assert out.dtype == dtype and torch.equal(out.cpu().double(), ref)

    for use in (w, None):
        f = named * (1.0 if use is None else use.double())
        terms = f[..., None] * y.double()[at]
        got = sdfoam_amd.expert_combine(y.to(dev), order, None if use is None else use.to(dev))
        near(got, terms.sum(1), bound(choices) * terms.abs().sum(1), dtype)
        rows_grad, weight_grad = sdfoam_amd.expert_combine_backward(
            grad.to(dev), y.to(dev), order, None if use is None else use.to(dev))
        ref = torch.empty((rows * choices, width), dtype=torch.float64)
        ref[at.reshape(-1)] = (f[..., None] * grad.double()[:, None]).flatten(0, 1)
        near(rows_grad, ref, U * ref.abs(), dtype)
        terms = named[..., None] * y.double()[at] * grad.double()[:, None]
        near(weight_grad, terms.sum(2), bound(width) * terms.abs().sum(2), torch.float32)
        alone, nothing = sdfoam_amd.expert_combine_backward(
            grad.to(dev), None, order, None if use is None else use.to(dev))
        assert nothing is None and torch.equal(alone, rows_grad)

    # through autograd; the rows' copies add up
    xg = x.to(dev).requires_grad_()
    got, = torch.autograd.grad(sdfoam_amd.expert_rows(xg, order), xg, y.to(dev))
    assert torch.equal(got, sdfoam_amd.expert_combine(y.to(dev), order))
    yg, wg = y.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    got = torch.autograd.grad(sdfoam_amd.expert_combine(yg, order, wg), (yg, wg), grad.to(dev))
    for a, b in zip(got, sdfoam_amd.expert_combine_backward(grad.to(dev), y.to(dev), order,
                                                            w.to(dev))):
        assert torch.equal(a, b)


def test_rows_strided_and_of_any_shape(dev):
    g = torch.Generator().manual_seed(0)
    ids = some_ids((3, 5, 2), 4, 1).to(dev)
    wide = torch.randn((3, 5, 40), generator=g).to(dev)
    order = sdfoam_amd.expert_order(ids, 4)
    x = wide[..., 3:30]
    out = sdfoam_amd.expert_rows(x, order)
    assert torch.equal(out, sdfoam_amd.expert_rows(x.contiguous(), order))
    back = sdfoam_amd.expert_combine(torch.cat([out, out], 1)[:, 27:], order)
    assert back.shape == (3, 5, 27)
    assert torch.equal(back, x * (ids >= 0).sum(-1, keepdim=True))
    assert torch.equal(sdfoam_amd.expert_combine(out, order),
                       sdfoam_amd.expert_combine(out.t().contiguous().t(), order))
    # order of transposed ids is of the ids as they are read
    t = ids.transpose(0, 1)
    assert torch.equal(sdfoam_amd.expert_order(t, 4).places,
                       sdfoam_amd.expert_order(t.contiguous(), 4).places)


def test_places_outside_are_left_out(dev):
    places = torch.tensor([[0, 7], [-9, 1], [2 ** 31 - 1, -2 ** 31]], dtype=torch.int32)
    order = sdfoam_amd.ExpertOrder(places.to(dev), torch.tensor([0, 6], dtype=torch.int32).to(dev))
    x = torch.arange(1.0, 13.0).reshape(3, 4).to(dev)
    out = sdfoam_amd.expert_rows(x, order)
    assert torch.equal(out[0], x[0]) and torch.equal(out[1], x[1])
    y = torch.arange(24.0).reshape(6, 4).to(dev)
    assert torch.equal(sdfoam_amd.expert_combine(y, order).cpu(),
                       torch.stack([y[0], y[1], torch.zeros_like(y[0])]).cpu())
    rows_grad, weight_grad = sdfoam_amd.expert_combine_backward(x, y, order)
    assert torch.equal(rows_grad[0], x[0]) and torch.equal(rows_grad[1], x[1])
    dots = torch.stack([(x[0] * y[0]).sum(), (x[1] * y[1]).sum()]).cpu()
    assert torch.equal(weight_grad.cpu(), torch.tensor([[dots[0], 0.0], [0.0, dots[1]], [0.0, 0.0]]))


def test_values_of_unnamed_places_stay_out(dev):
    ids = torch.tensor([[0, -1], [-1, -1], [1, 0]]).to(dev)
    order = sdfoam_amd.expert_order(ids, 2)
    y = torch.full((6, 9), math.nan, device=dev)
    y[:3] = 1.0
    w = torch.tensor([[2.0, math.nan], [math.inf, math.nan], [3.0, 4.0]], device=dev)
    out = sdfoam_amd.expert_combine(y, order, w)
    assert torch.equal(out.cpu()[:, 0], torch.tensor([2.0, 0.0, 7.0]))
    rows_grad, weight_grad = sdfoam_amd.expert_combine_backward(torch.ones(3, 9, device=dev), y,
                                                                order, w)
    assert torch.equal(rows_grad[3:], torch.zeros(3, 9, device=dev))
    assert torch.equal(weight_grad.cpu(), torch.tensor([[9.0, 0.0], [0.0, 0.0], [9.0, 9.0]]))


# ---- the experts' products -------------------------------------------------------------------


def offsets_of(counts, rows):
    o = torch.tensor([0] + list(counts), dtype=torch.int64).cumsum(0)
    assert o[-1] <= rows
    return o


LINEARS = [  # rows, counts, width, out
    (1, [1], 1, 1), (5, [2, 0, 1], 7, 9), (64, [1] * 64, 64, 128), (130, [129], 64, 33),
    (300, [0, 128, 0, 0, 129, 3], 65, 130), (257, [1, 255], 200, 17), (40, [], 5, 6),
    (33, [0, 0, 0], 16, 40), (1000, [999], 49, 201), (700, [100, 500, 90], 1031, 300),
    (16, [3, 13], 4097, 260), (3000, [2900, 60], 24, 40), (2048, [2000, 48], 8, 8),
    (20, [20], 0, 5), (20, [4, 15], 6, 0), (0, [0, 0], 4, 4), (64, [10, 6, 0, 33], 1024, 500),
    (17, [1, 2, 3, 4, 5], 2050, 70),
    # large tiles, each way, whole pieces of 16 bytes and not
    (8200, [5000, 3100], 264, 1288), (8200, [4000, 4100], 1288, 264), (8195, [8000], 301, 1289),
    (300, [150, 149], 2056, 2064), (300, [150, 149], 2059, 2061),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,counts,width,out", LINEARS)
def test_linear(dev, rows, counts, width, out, dtype):
    say("linear", rows, counts[:8], width, out, dtype)
    g = torch.Generator().manual_seed(rows + width)
    experts = len(counts)
    offsets = offsets_of(counts, rows)
    x = torch.randn((rows, width), generator=g).to(dtype)
    w = torch.randn((experts, out, width), generator=g).to(dtype)
    d = torch.randn((rows, out), generator=g).to(dtype)
    y, size = (torch.zeros((rows, out), dtype=torch.float64) for _ in range(2))
    dx, dx_size = (torch.zeros((rows, width), dtype=torch.float64) for _ in range(2))
    dw, dw_size = (torch.zeros((experts, out, width), dtype=torch.float64) for _ in range(2))
    for e in range(experts):
        p = slice(int(offsets[e]), int(offsets[e + 1]))
        xe, we, de = x[p].double(), w[e].double(), d[p].double()
        y[p], size[p] = xe @ we.T, xe.abs() @ we.abs().T
        dx[p], dx_size[p] = de @ we, de.abs() @ we.abs()
        dw[e], dw_size[e] = de.T @ xe, de.abs().T @ xe.abs()
    o = offsets.to(torch.int32).to(dev)
    X, W, D = x.to(dev), w.to(dev), d.to(dev)
    got = sdfoam_amd.expert_linear(X, W, o)
    near(got, y, bound(width) * size, dtype)
    rows_grad, weight_grad = sdfoam_amd.expert_linear_backward(D, X, W, o)
    near(rows_grad, dx, bound(out) * dx_size, dtype)
    near(weight_grad, dw, bound(max(counts, default=0)) * dw_size, dtype)
    only, none = sdfoam_amd.expert_linear_backward(D, X, W, o, need_weight=False)
    assert none is None and torch.equal(only, rows_grad)
    none, only = sdfoam_amd.expert_linear_backward(D, X, W, o, need_rows=False)
    assert none is None and torch.equal(only, weight_grad)
    Xg, Wg = X.clone().requires_grad_(), W.clone().requires_grad_()
    for a, b in zip(torch.autograd.grad(sdfoam_amd.expert_linear(Xg, Wg, o), (Xg, Wg), D),
                    (rows_grad, weight_grad)):
        assert torch.equal(a, b)
    # strided rows, read in place
    pad = torch.full((rows, width + 3), math.nan, dtype=dtype, device=dev)
    pad[:, 1:1 + width] = X
    assert torch.equal(sdfoam_amd.expert_linear(pad[:, 1:1 + width], W, o), got)


def test_no_choices(dev):
    order = sdfoam_amd.expert_order(torch.zeros((5, 0), dtype=torch.int64, device=dev), 3)
    assert torch.equal(order.offsets.cpu(), torch.zeros(4, dtype=torch.int32))
    assert sdfoam_amd.expert_rows(torch.ones((5, 6), device=dev), order).shape == (0, 6)
    out = sdfoam_amd.expert_combine(torch.ones((0, 6), device=dev), order)
    assert torch.equal(out, torch.zeros((5, 6), device=dev))


def test_more_than_2_to_32_elements(dev):
    """Rows whose elements pass 32 bits.  Small whole numbers: every sum is exact."""
    rows, width = (1 << 21) + 133, 2056
    at = torch.arange(rows, device=dev)
    x = ((at % 5) - 2).to(torch.bfloat16)[:, None].expand(rows, width)
    ids = (at % 3 == 0).long()[:, None]
    order = sdfoam_amd.expert_order(ids, 2)
    sorted_rows = sdfoam_amd.expert_rows(x, order)
    p = order.places[:, 0].long()
    assert torch.equal(sorted_rows[p[-1000:]], x[-1000:])
    w = torch.ones((2, 16, width), dtype=torch.bfloat16, device=dev)
    w[1] = -1.0
    y = sdfoam_amd.expert_linear(sorted_rows, w, order.offsets)
    want = (x[:, 0].float() * width * torch.where(ids[:, 0] == 1, -1.0, 1.0)).to(torch.bfloat16)
    assert torch.equal(y[p], want[:, None].expand(rows, 16))
    back = sdfoam_amd.expert_combine(sorted_rows, order)
    assert torch.equal(back[-1000:], x[-1000:]) and torch.equal(back[:1000], x[:1000])
    d = torch.ones((rows, 16), dtype=torch.bfloat16, device=dev)
    dx, dw = sdfoam_amd.expert_linear_backward(d, sorted_rows, w, order.offsets)
    sums = torch.stack([x[:, 0].float()[ids[:, 0] == e].sum() for e in (0, 1)]).to(torch.bfloat16)
    assert torch.equal(dw, sums[:, None, None].expand(2, 16, width))
    assert torch.equal(dx[p[-5:], 0].float().cpu(),
                       torch.where(ids[-5:, 0] == 1, -16.0, 16.0).cpu())


def test_linear_keeps_values_apart(dev):
    """What is not finite in one expert's rows or weights, or behind all experts' rows,
    reaches no other expert's results."""
    for dtype in TYPES:
        g = torch.Generator().manual_seed(5)
        x = torch.randn((200, 40), generator=g).to(dtype).to(dev)
        w = torch.randn((3, 50, 40), generator=g).to(dtype).to(dev)
        d = torch.randn((200, 50), generator=g).to(dtype).to(dev)
        o = torch.tensor([0, 70, 75, 190], dtype=torch.int32, device=dev)
        clean = sdfoam_amd.expert_linear(x, w, o), *sdfoam_amd.expert_linear_backward(d, x, w, o)
        x[70:75], w[1], d[70:75] = math.nan, math.inf, math.nan
        x[190:], d[190:] = math.nan, math.inf
        y = sdfoam_amd.expert_linear(x, w, o)
        dx, dw = sdfoam_amd.expert_linear_backward(d, x, w, o)
        for a, b in ((y, clean[0]), (dx, clean[1])):
            assert torch.equal(a[:70], b[:70]) and torch.equal(a[75:], b[75:])
            assert torch.isnan(a[70:75]).all()
        assert torch.equal(dw[0], clean[2][0]) and torch.equal(dw[2], clean[2][2])


def test_linear_against_differences(dev):
    """The product is linear in each of its factors: differences are exact but for fp32's
    roundings of the losses, each at most bound(terms) times the sum of their sizes."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn((50, 12), generator=g).to(dev)
    w = torch.randn((3, 9, 12), generator=g).to(dev)
    d = torch.randn((50, 9), generator=g).to(dev)
    o = torch.tensor([0, 20, 20, 47], dtype=torch.int32, device=dev)
    dx, dw = sdfoam_amd.expert_linear_backward(d, x, w, o)

    def loss(x, w):
        y = sdfoam_amd.expert_linear(x, w, o).double()
        return float((y * d.double()).sum()), float((y * d.double()).abs().sum())

    sizes = float((d[:47].double().abs().sum()) * 12 * 16.0)  # |x| and |w| are below 4
    for at in ((0, 0), (19, 5), (46, 11), (49, 3)):
        up, low = x.clone(), x.clone()
        up[at] += 1.0
        low[at] -= 1.0
        diff = (loss(up, w)[0] - loss(low, w)[0]) / 2
        assert abs(diff - float(dx[at])) <= 2 * bound(12) * sizes
    for at in ((0, 0, 0), (1, 3, 3), (2, 8, 11)):
        up, low = w.clone(), w.clone()
        up[at] += 1.0
        low[at] -= 1.0
        diff = (loss(x, up)[0] - loss(x, low)[0]) / 2
        assert abs(diff - float(dw[at])) <= 2 * bound(50) * sizes


# ---- adapters --------------------------------------------------------------------------------


def adapter_reference(x, w, ids, down, up, scale, d):
    """Results in 64 bits and what bounds their errors."""
    x, w, down, up, d = (t.double() for t in (x, w, down, up, d))
    rows, width = x.shape
    out, rank = w.shape[0], down.shape[1]
    y, y_tol = x @ w.T, bound(width) * (x.abs() @ w.abs().T)
    dx, dx_tol = d @ w, bound(out) * (d.abs() @ w.abs())
    dw, dw_tol = d.T @ x, bound(rows) * (d.abs().T @ x.abs())
    dd, du, dd_tol, du_tol = (torch.zeros_like(t) for t in (down, up, down, up))
    for a in range(down.shape[0]):
        i = torch.nonzero(ids == a)[:, 0]
        n = i.numel()
        if n == 0:
            continue
        h = scale * (x[i] @ down[a].T)
        h_tol = bound(width) * abs(scale) * (x[i].abs() @ down[a].abs().T)
        b = scale * (d[i] @ up[a])
        b_tol = bound(out) * abs(scale) * (d[i].abs() @ up[a].abs())
        h_size, b_size = h.abs() + h_tol, b.abs() + b_tol
        y[i] += h @ up[a].T
        y_tol[i] += h_tol @ up[a].abs().T + bound(rank + width) * (h_size @ up[a].abs().T)
        dx[i] += b @ down[a]
        dx_tol[i] += b_tol @ down[a].abs() + bound(rank + out) * (b_size @ down[a].abs())
        dd[a] = b.T @ x[i]
        dd_tol[a] = b_tol.T @ x[i].abs() + bound(n) * (b_size.T @ x[i].abs())
        du[a] = d[i].T @ h
        du_tol[a] = d[i].abs().T @ h_tol + bound(n) * (d[i].abs().T @ h_size)
    return (y, dx, dw, dd, du), (y_tol, dx_tol, dw_tol, dd_tol, du_tol)


ADAPTERS = [  # rows, adapters, rank, width, out, spread
    (1, 1, 1, 1, 1, "any"), (1, 3, 16, 300, 70, "one"), (3, 256, 8, 64, 128, "any"),
    (17, 4, 5, 33, 47, "any"), (64, 64, 16, 130, 257, "any"), (65, 9, 4, 64, 512, "any"),
    (200, 200, 17, 40, 90, "any"), (300, 3, 64, 100, 31, "few"), (1000, 2, 130, 50, 20, "any"),
    (2500, 7, 4, 8, 24, "any"), (400, 5, 16, 1030, 260, "none"), (31, 0, 4, 9, 10, "none"),
    (50, 6, 0, 21, 22, "any"), (0, 3, 4, 5, 6, "any"), (40, 2, 3, 0, 7, "any"),
    (40, 2, 3, 7, 0, "any"), (4100, 12, 8, 17, 41, "few"), (150, 2048, 2, 24, 16, "any"),
    (60, 2, 32, 2100, 64, "any"), (33, 40, 256, 64, 72, "any"),
    # rows whose adapters are added one by one: in the order they come, in order of adapters,
    # in parts, along a short inner dimension
    (60, 7, 5, 40, 100, "any"), (1500, 1500, 4, 70, 90, "any"), (1300, 700, 16, 1100, 130, "any"),
    (1500, 1200, 9, 30, 70, "any"), (900, 300, 20, 600, 1100, "any"),
]


def adapter_case(rows, adapters, rank, width, out, spread, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + rows + width)

    def randn(*shape, scale=1.0):
        return (scale * torch.randn(shape, generator=g)).to(dtype)

    ids = some_ids((rows,), adapters, rows + out, spread=spread)
    s = max(width, 1) ** -0.5
    return (randn(rows, width), randn(out, width, scale=s), ids,
            randn(adapters, rank, width, scale=s),
            randn(adapters, out, rank, scale=max(rank, 1) ** -0.5), randn(rows, out))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,adapters,rank,width,out,spread", ADAPTERS)
def test_adapters(dev, rows, adapters, rank, width, out, spread, dtype):
    say("adapters", rows, adapters, rank, width, out, spread, dtype)
    x, w, ids, down, up, d = adapter_case(rows, adapters, rank, width, out, spread, dtype)
    scale = 1.75
    refs, tols = adapter_reference(x, w, ids, down, up, scale, d)
    X, W, A, B, D = (t.to(dev) for t in (x, w, down, up, d))
    c = ids_as(ids, ID_TYPES[(rows + rank) % 3], dev)
    y = sdfoam_amd.adapter_linear(X, W, c, A, B, scale)
    near(y, refs[0], tols[0], dtype)
    grads = sdfoam_amd.adapter_linear_backward(D, X, W, c, A, B, scale)
    for got, ref, tol in zip(grads, refs[1:], tols[1:]):
        near(got, ref, tol, dtype)
    frozen = sdfoam_amd.adapter_linear_backward(D, X, W, c, A, B, scale, need_weight=False)
    assert frozen[1] is None
    for k in (0, 2, 3):
        assert torch.equal(frozen[k], grads[k])
    alone = sdfoam_amd.adapter_linear_backward(D, X, W, c, A, B, scale, need_adapters=False)
    assert alone[2] is None and alone[3] is None
    assert torch.equal(alone[0], grads[0]) and torch.equal(alone[1], grads[1])
    leaves = [t.clone().requires_grad_() for t in (X, W, A, B)]
    z = sdfoam_amd.adapter_linear(leaves[0], leaves[1], c, leaves[2], leaves[3], scale)
    assert torch.equal(z, y)
    for a, b in zip(torch.autograd.grad(z, leaves, D), grads):
        assert torch.equal(a, b)


def test_adapters_of_any_shape_and_stride(dev):
    x, w, ids, down, up, d = adapter_case(42, 5, 6, 29, 35, "any", torch.float16)
    c = ids.to(dev)
    X, W, A, B, D = (t.to(dev) for t in (x, w, down, up, d))
    y = sdfoam_amd.adapter_linear(X, W, c, A, B)
    wide = torch.full((42, 40), math.nan, dtype=torch.float16, device=dev)
    wide[:, 5:34] = X
    tall = torch.full((35, 31), math.nan, dtype=torch.float16, device=dev)
    tall[:, 1:30] = W
    got = sdfoam_amd.adapter_linear(wide[:, 5:34], tall[:, 1:30], c, A, B)
    assert torch.equal(got, y)
    got = sdfoam_amd.adapter_linear(X.reshape(6, 7, 29), W, c.reshape(6, 7), A, B)
    assert got.shape == (6, 7, 35) and torch.equal(got.reshape(42, 35), y)
    got = sdfoam_amd.adapter_linear(X.t().contiguous().t(), W.t().contiguous().t(), c,
                                    A.transpose(1, 2).contiguous().transpose(1, 2),
                                    B.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(got, y)
    one = sdfoam_amd.adapter_linear(X[0], W, c[0], A, B)
    assert one.shape == (35,)
    grads = sdfoam_amd.adapter_linear_backward(D, X, W, c, A, B)
    other = sdfoam_amd.adapter_linear_backward(D.reshape(2, 21, 35), X.reshape(2, 21, 29), W,
                                               c.reshape(2, 21), A, B)
    assert torch.equal(other[0].reshape(42, 29), grads[0])
    for a, b in zip(other[1:], grads[1:]):
        assert torch.equal(a, b)
    # a gradient broadcast over the rows
    same = sdfoam_amd.adapter_linear_backward(D[:1].expand(42, 35), X, W, c, A, B)
    full = sdfoam_amd.adapter_linear_backward(D[:1].repeat(42, 1), X, W, c, A, B)
    for a, b in zip(same, full):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [7, 40, 64, 65, 300])
def test_adapters_keep_values_apart(dev, rows):
    """An adapter that holds what is not finite reaches its own rows alone, forward and
    back, wherever they stand among the others."""
    for dtype in TYPES:
        x, w, ids, down, up, d = adapter_case(rows, 4, 8, 48, 100, "any", dtype)
        ids[1] = 2
        X, W, A, B, D = (t.to(dev) for t in (x, w, down, up, d))
        c = ids.to(dev)
        y = sdfoam_amd.adapter_linear(X, W, c, A, B)
        dx, _, dd, du = sdfoam_amd.adapter_linear_backward(D, X, W, c, A, B, need_weight=False)
        A[2, 3], B[2, 5] = math.nan, math.inf
        z = sdfoam_amd.adapter_linear(X, W, c, A, B)
        ex, _, ed, eu = sdfoam_amd.adapter_linear_backward(D, X, W, c, A, B, need_weight=False)
        other = c != 2
        assert torch.equal(z[other], y[other]) and torch.equal(ex[other], dx[other])
        assert torch.isnan(z[~other]).all()
        for a in (0, 1, 3):
            assert torch.equal(ed[a], dd[a]) and torch.equal(eu[a], du[a])


def test_adapters_against_differences(dev):
    """Each factor enters linearly: differences of the loss are exact but for roundings,
    bounded by those of all terms of the loss."""
    x, w, ids, down, up, d = adapter_case(70, 3, 4, 12, 9, "any", torch.float32)
    c = ids.to(dev)
    t = {"x": x.to(dev), "w": w.to(dev), "down": down.to(dev), "up": up.to(dev)}
    D = d.to(dev)
    grads = sdfoam_amd.adapter_linear_backward(D, t["x"], t["w"], c, t["down"], t["up"])

    def loss(t):
        y = sdfoam_amd.adapter_linear(t["x"], t["w"], c, t["down"], t["up"]).double()
        return float((y * D.double()).sum())

    _, tols = adapter_reference(x, w, ids, down, up, 1.0, d)
    # a changed entry moves its factor by 1: sizes grow by at most that of the gradient's
    noise = float((tols[0] * d.double().abs()).sum()) + sum(float(k.max()) for k in tols[1:])
    noise += U * float(d.double().abs().sum()) * 16.0  # results below 16, rounded to fp32
    for name, grad, at in (("x", grads[0], (3, 5)), ("x", grads[0], (69, 11)),
                           ("w", grads[1], (8, 0)), ("down", grads[2], (1, 3, 7)),
                           ("down", grads[2], (2, 0, 11)), ("up", grads[3], (0, 8, 3)),
                           ("up", grads[3], (2, 4, 1))):
        high, low = dict(t), dict(t)
        high[name], low[name] = t[name].clone(), t[name].clone()
        high[name][at] += 0.5
        low[name][at] -= 0.5
        assert abs(loss(high) - loss(low) - float(grad[at])) <= 4 * noise, name


# ---- together --------------------------------------------------------------------------------


def mixture(x, ids, gate, w1, w2, base, cams, down, up):
    """A head of experts: two layers of each, and an adapted projection behind them."""
    order = sdfoam_amd.expert_order(ids, w1.shape[0])
    h = sdfoam_amd.expert_linear(sdfoam_amd.expert_rows(x, order), w1, order.offsets)
    y = sdfoam_amd.expert_linear(torch.relu(h), w2, order.offsets)
    y = sdfoam_amd.expert_combine(y, order, gate)
    return sdfoam_amd.adapter_linear(y, base, cams, down, up, 2.0)


def mixture_reference(x, ids, gate, w1, w2, base, cams, down, up):
    y = torch.zeros((x.shape[0], w2.shape[1]), dtype=x.dtype)
    for k in range(ids.shape[1]):
        for e in range(w1.shape[0]):
            i = torch.nonzero(ids[:, k] == e)[:, 0]
            y = y.index_add(0, i, gate[i, k, None] * (torch.relu(x[i] @ w1[e].T) @ w2[e].T))
    out = y @ base.T
    for a in range(down.shape[0]):
        i = torch.nonzero(cams == a)[:, 0]
        out = out.index_add(0, i, 2.0 * (y[i] @ down[a].T) @ up[a].T)
    return out


def mixture_case(seed, rows=300):
    g = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g) * shape[-1] ** -0.5

    ids = some_ids((rows, 2), 5, seed)
    cams = some_ids((rows,), 3, seed + 1)
    return [randn(rows, 24), torch.rand((rows, 2), generator=g), randn(5, 40, 24),
            randn(5, 16, 40), randn(30, 16), randn(3, 4, 16), randn(3, 30, 4)], ids, cams


def test_together(dev):
    """A whole head forward and back, against 64 bits.  Five layers of sums with at most 40
    terms of order 1: results are off by less than the sum of their bounds, 1e-4 of the
    largest."""
    leaves, ids, cams = mixture_case(1)
    ref_leaves = [t.double().requires_grad_() for t in leaves]
    x, gate, *rest = ref_leaves
    ref = mixture_reference(x, ids, gate, rest[0], rest[1], rest[2], cams, rest[3], rest[4])
    seed = torch.randn(ref.shape, generator=torch.Generator().manual_seed(9))
    ref_grads = torch.autograd.grad(ref, ref_leaves, seed.double())
    own = [t.to(dev).requires_grad_() for t in leaves]
    x, gate, *rest = own
    out = mixture(x, ids.to(dev), gate, rest[0], rest[1], rest[2], cams.to(dev), rest[3], rest[4])
    grads = torch.autograd.grad(out, own, seed.to(dev))
    for got, want in zip((out, *grads), (ref, *ref_grads)):
        off = (got.detach().cpu().double() - want.detach()).abs().max()
        assert off <= 1e-4 * want.detach().abs().max()


def test_captured_and_replayed(dev):
    """Forward and backward calls in a graph, replayed on other inputs with eager work
    between: each replay as the eager calls."""
    leaves, ids, cams = mixture_case(2, rows=200)
    x, gate, w1, w2, base, down, up = (t.to(dev) for t in leaves)
    ids, cams = ids.to(dev), cams.to(dev)
    d = torch.randn((200, 30), device=dev)

    def step():
        order = sdfoam_amd.expert_order(ids, 5)
        s = sdfoam_amd.expert_rows(x, order)
        h = sdfoam_amd.expert_linear(s, w1, order.offsets)
        r = torch.relu(h)
        y = sdfoam_amd.expert_linear(r, w2, order.offsets)
        z = sdfoam_amd.expert_combine(y, order, gate)
        out = sdfoam_amd.adapter_linear(z, base, cams, down, up, 2.0)
        dz, dbase, ddown, dup = sdfoam_amd.adapter_linear_backward(d, z, base, cams, down, up, 2.0)
        dy, dgate = sdfoam_amd.expert_combine_backward(dz, y, order, gate)
        dr, dw2 = sdfoam_amd.expert_linear_backward(dy, r, w2, order.offsets)
        ds, dw1 = sdfoam_amd.expert_linear_backward(dr * (h > 0), s, w1, order.offsets)
        dx = sdfoam_amd.expert_combine(ds, order)
        grads = [dx, dgate, dw1, dw2, dbase, ddown, dup]
        norm = sdfoam_amd.clip_gradients(grads, 1.0)
        return [out, norm, *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.mul_(-0.5).add_(0.1 * k)
            ids.copy_(some_ids((200, 2), 5, 100 + k).to(dev))
            cams.copy_(some_ids((200,), 3, 200 + k).to(dev))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b), k
        step()


def test_on_another_stream(dev):
    """Calls go to the current stream, and two streams' calls do not meet in scratch."""
    cases = [adapter_case(500, 6, 8, 64, 200, "any", torch.bfloat16, seed) for seed in (1, 2)]
    on = [[t.to(dev) for t in c] for c in cases]
    want = [sdfoam_amd.adapter_linear(x, w, i, a, b) for x, w, i, a, b, _ in on]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, w, i, a, b, _ = on[k]
                got[k].append(sdfoam_amd.adapter_linear(x, w, i, a, b))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert torch.equal(g, want[k])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,out", [(300, 6, 1024), (300, 1024, 6), (300, 2056, 1030),
                                            (7, 1024, 1024)])
def test_no_experts(dev, rows, width, out, dtype):
    """No experts: zeros, also where the inner dimension is cut in parts."""
    say("no experts", rows, width, out, dtype)
    x = torch.ones((rows, width), dtype=dtype, device=dev).requires_grad_()
    w = torch.empty((0, out, width), dtype=dtype, device=dev).requires_grad_()
    o = torch.zeros(1, dtype=torch.int32, device=dev)
    d = torch.ones((rows, out), dtype=dtype, device=dev)
    y = sdfoam_amd.expert_linear(x, w, o)
    assert y.shape == (rows, out) and not y.any()
    for dx, dw in (sdfoam_amd.expert_linear_backward(d, x.detach(), w.detach(), o),
                   torch.autograd.grad(y, (x, w), d)):
        assert dx.shape == x.shape and not dx.any() and dw.shape == w.shape


LAST_COLUMNS = [  # rows, adapters, rank, width, out: many adapters in every 32 rows
    (1100, 400, 4, 70, 65), (1100, 400, 4, 65, 129),  # tiles of 128 x 128, both ways
    (1100, 400, 5, 30, 95), (1100, 400, 16, 8, 1),    # a short inner dimension
    (1100, 400, 16, 1100, 70), (1100, 400, 8, 70, 1100),  # in parts, forward and back
    (4100, 1500, 4, 264, 2180), (4100, 1500, 4, 2180, 264),  # tiles of 256 x 256
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,adapters,rank,width,out", LAST_COLUMNS)
def test_adapters_last_columns(dev, rows, adapters, rank, width, out, dtype):
    """Rows whose adapters are added one by one, where fewer than 32 columns are left for a
    wavefront: where each row goes, and its adapter, lie in lanes past the last column."""
    test_adapters(dev, rows, adapters, rank, width, out, "any", dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,out", [(264, 2180), (2180, 264)])
def test_adapters_in_large_tiles(dev, width, out, dtype):
    """Few adapters in every 32 rows, added by the matrix units in tiles of 256 x 256."""
    test_adapters(dev, 4100, 3, 16, width, out, "any", dtype)


# ---- results of more tiles, and of more rows, than one launch takes ------------------------------
# Small whole numbers: every sum is exact.


@pytest.fixture
def much_memory(dev):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("not enough free memory")
    yield dev
    torch.cuda.empty_cache()


def soil(dev, *shape, dtype=torch.bfloat16):
    """Memory that the next tensor of this size takes holds NaN."""
    torch.full(shape, math.nan, dtype=dtype, device=dev)


def test_many_experts_of_many_columns(much_memory):
    dev, experts, each, width, out = much_memory, 2048, 16, 8, 65_600
    say("many tiles of few rows")
    rows = experts * each
    x = (torch.arange(rows * width, device=dev) % 5 - 2).to(torch.bfloat16).reshape(rows, width)
    c = ((torch.arange(experts, device=dev)[:, None] * 7 + torch.arange(out, device=dev) * 3) % 5 -
         2).to(torch.bfloat16)
    w = c[..., None].expand(experts, out, width).contiguous()
    o = torch.arange(experts + 1, device=dev, dtype=torch.int32) * each
    soil(dev, rows, out)
    y = sdfoam_amd.expert_linear(x, w, o).view(experts, each, out)
    sums = x.float().sum(1).to(torch.bfloat16).view(experts, each, 1)
    for e in range(0, experts, 256):
        assert torch.equal(y[e:e + 256], sums[e:e + 256] * c[e:e + 256, None])


def test_narrow_rows_past_2_to_30(much_memory):
    dev, rows = much_memory, (1 << 30) + 300
    say("many narrow rows")
    x = torch.empty(rows, dtype=torch.bfloat16, device=dev)
    parts = [slice(k, min(k + (1 << 27), rows)) for k in range(0, rows, 1 << 27)]
    for p in parts:
        x[p] = (torch.arange(p.start, p.stop, device=dev) % 5 - 2).to(torch.bfloat16)
    o = torch.tensor([0, (1 << 29) + 7, rows - 50], dtype=torch.int32, device=dev)
    w = torch.tensor([3.0, -5.0], dtype=torch.bfloat16, device=dev).reshape(2, 1, 1)

    def check(got, times):
        for p in parts:
            at = torch.arange(p.start, p.stop, device=dev)
            f = torch.where(at < (1 << 29) + 7, times[0], times[1]) * (at < rows - 50)
            assert torch.equal(got[p, 0], x[p] * f.to(torch.bfloat16))

    soil(dev, rows, 1)
    check(sdfoam_amd.expert_linear(x[:, None], w, o), (3.0, -5.0))
    # 65 elements, the same row again and again
    one = torch.ones((1, 65), dtype=torch.bfloat16, device=dev)
    long = w.expand(2, 1, 65).contiguous()
    soil(dev, rows, 1)
    y = sdfoam_amd.expert_linear(one.expand(rows, 65), long, o)
    x.fill_(1.0)
    # -325 lies halfway between 162 and 163 steps of 2: the even one, -324, as `to` rounds it
    check(y, (195.0, -325.0))
    del y
    soil(dev, rows, 1)
    dx, none = sdfoam_amd.expert_linear_backward(one[:, :1].expand(rows, 1), x[:, None], w, o,
                                                 need_weight=False)
    assert none is None
    check(dx, (3.0, -5.0))
    del dx
    # the same rows with an adapter each
    ids = torch.zeros(rows, dtype=torch.int32, device=dev)
    ids[(1 << 29) + 7:] = 1
    ids[rows - 50:] = -1
    up = torch.tensor([1.0, -7.0], dtype=torch.bfloat16, device=dev).reshape(2, 1, 1)
    shared = torch.zeros((1, 1), dtype=torch.bfloat16, device=dev)
    soil(dev, rows, 1)
    y = sdfoam_amd.adapter_linear(x[:, None], shared, ids, torch.ones_like(up), up, 2.0)
    check(y, (2.0, -14.0))


def test_many_adapters_of_many_columns(much_memory):
    """The gradient of `up`: a tile of 128 x 32 for each adapter and part of its matrix."""
    dev, adapters, out, rank = much_memory, 2048, 1 << 18, 33
    say("many adapters")
    up = torch.zeros((adapters, out, rank), dtype=torch.bfloat16, device=dev)
    down = torch.ones((adapters, rank, 4), dtype=torch.bfloat16, device=dev)
    down[:, 32] = -2.0
    ids = torch.tensor([2047, 0, 2047, 700, -1], device=dev)
    x = torch.ones((5, 4), dtype=torch.bfloat16, device=dev)
    x[2] = 2.0
    d = (torch.arange(5 * out, device=dev) % 7 - 3).to(torch.bfloat16).reshape(5, out)
    w = torch.zeros((out, 4), dtype=torch.bfloat16, device=dev)
    soil(dev, adapters, out, rank)
    _, _, _, up_grad = sdfoam_amd.adapter_linear_backward(d, x, w, ids, down, up,
                                                          need_rows=False, need_weight=False)
    h = down[0].float().sum(1)
    for a, column in ((0, d[1].float()), (700, d[3].float()), (2047, d[0].float() + 2 * d[2].float())):
        assert torch.equal(up_grad[a].float(), column[:, None] * h)
        up_grad[a] = 0
    for a in range(0, adapters, 64):
        assert not up_grad[a:a + 64].any()


def test_rows_past_2_to_25(much_memory):
    """Rows of 64 lanes each, four a block."""
    dev, rows, width = much_memory, (1 << 25) + 77, 132
    say("many rows")
    at = torch.arange(rows, device=dev)
    x = torch.arange(width, device=dev, dtype=torch.float32).repeat(rows, 1)
    x += (at % 65_521)[:, None]
    ids = (at % 3).int()
    ids[at % 1000 == 5] = -1
    order = sdfoam_amd.expert_order(ids[:, None], 3)
    soil(dev, rows, width, dtype=torch.float32)
    y = sdfoam_amd.expert_rows(x, order)
    p = order.places[:, 0].long()
    named = p >= 0
    parts = [slice(k, min(k + (1 << 22), rows)) for k in range(0, rows, 1 << 22)]
    for s in parts:
        assert torch.equal(y[torch.where(named[s], p[s], -1 - p[s])], x[s] * named[s, None])
    gate = torch.where(at % 2 == 0, 2.0, -1.0)[:, None]
    back = sdfoam_amd.expert_combine(y, order, gate)
    for s in parts:
        assert torch.equal(back[s], x[s] * (gate[s] * named[s, None]))
    del back
    soil(dev, rows, width, dtype=torch.float32)
    rows_grad, gate_grad = sdfoam_amd.expert_combine_backward(
        torch.ones((1, width), device=dev).expand(rows, width), y, order, gate)
    for s in parts:
        assert torch.equal(gate_grad[s, 0], x[s].sum(1) * named[s])
        want = (gate[s] * named[s, None]).expand(-1, width)
        assert torch.equal(rows_grad[torch.where(named[s], p[s], -1 - p[s])], want)


# ---- values that are not finite, and values below the normal range --------------------------------


def same(got, ref, tol, dtype):
    """near(), and infinite where the reference is, with its sign."""
    near(got, ref, tol, dtype)
    got = got.detach().cpu().double()
    infinite = torch.isinf(ref)
    assert torch.equal(got[infinite], ref[infinite])


INFINITE_ADAPTERS = [  # rows, adapters, rank, width, out
    (7, 2, 1, 40, 50), (7, 2, 5, 40, 50), (64, 3, 1, 600, 130), (40, 3, 9, 70, 70),
    (300, 4, 1, 40, 30), (300, 4, 3, 30, 90), (1100, 400, 1, 1100, 70), (1100, 400, 2, 20, 70),
    (900, 300, 1, 600, 1100),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,adapters,rank,width,out", INFINITE_ADAPTERS)
def test_adapters_infinite(dev, rows, adapters, rank, width, out, dtype):
    """An infinite scale, and infinite elements: infinite results have their sign, sums of
    both signs are NaN, and what only fills up a rank adds nothing."""
    say("infinite", rows, adapters, rank, width, out, dtype)
    x, w, ids, down, up, d = adapter_case(rows, adapters, rank, width, out, "any", dtype)
    ids[0], ids[1] = 0, -1
    c = ids.to(dev)
    for scale in (math.inf, -math.inf, 1.5):
        if scale == 1.5:
            x[0, width // 2], d[0, out // 2] = math.inf, -math.inf
            x[1, 0] = -math.inf
        refs, tols = adapter_reference(x, w, ids, down, up, scale, d)
        tols = [torch.nan_to_num(t, nan=0.0, posinf=0.0) if scale != 1.5 else t for t in tols]
        X, W, A, B, D = (t.to(dev) for t in (x, w, down, up, d))
        got = [sdfoam_amd.adapter_linear(X, W, c, A, B, scale),
               *sdfoam_amd.adapter_linear_backward(D, X, W, c, A, B, scale)]
        if scale != 1.5:  # rows without an adapter, and the projection's gradient: finite
            n = ids < 0
            same(got[0].cpu()[n], refs[0][n], bound(width) * (x.double().abs() @ w.double().abs().T)[n], dtype)
            same(got[2], refs[2], bound(rows) * (d.double().abs().T @ x.double().abs()), dtype)
        for k, (a, ref) in enumerate(zip(got, refs)):
            if k == 2 and scale != 1.5:
                continue
            fine = torch.isfinite(ref)
            a = a.cpu().double()
            assert torch.equal(torch.isnan(a), torch.isnan(ref)), (scale, k)
            assert torch.equal(a[torch.isinf(ref)], ref[torch.isinf(ref)]), (scale, k)
            assert torch.isfinite(a[fine]).all(), (scale, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_and_combine_infinite(dev, dtype):
    g = torch.Generator().manual_seed(4)
    for rows, counts, width, out in ((6, [2, 4], 40, 20), (300, [100, 150], 30, 70),
                                     (300, [100, 150], 600, 70), (130, [130], 1031, 90)):
        say("infinite", rows, counts, width, out, dtype)
        x, d = (torch.randn((rows, k), generator=g).to(dtype) for k in (width, out))
        w = torch.randn((len(counts), out, width), generator=g).to(dtype)
        x[1, 0], x[3, width - 1], d[0, out - 1], w[0, 5, 7] = math.inf, -math.inf, math.inf, math.inf
        o = offsets_of(counts, rows)
        refs = [torch.zeros((rows, out), dtype=torch.float64), torch.zeros((rows, width), dtype=torch.float64),
                torch.zeros(w.shape, dtype=torch.float64)]
        sizes = [torch.zeros_like(t) for t in refs]
        for e in range(len(counts)):
            p = slice(int(o[e]), int(o[e + 1]))
            xe, we, de = x[p].double(), w[e].double(), d[p].double()
            refs[0][p], sizes[0][p] = xe @ we.T, xe.abs() @ we.abs().T
            refs[1][p], sizes[1][p] = de @ we, de.abs() @ we.abs()
            refs[2][e], sizes[2][e] = de.T @ xe, de.abs().T @ xe.abs()
        off = o.to(torch.int32).to(dev)
        X, W, D = x.to(dev), w.to(dev), d.to(dev)
        got = [sdfoam_amd.expert_linear(X, W, off), *sdfoam_amd.expert_linear_backward(D, X, W, off)]
        for a, ref, size, n in zip(got, refs, sizes, (width, out, max(counts))):
            same(a, ref, bound(n) * size, dtype)

    y = torch.randn((6, 37), generator=g).to(dtype)
    y[0, 3], y[4, 36], y[5, 0] = math.inf, -math.inf, math.nan
    gate = torch.tensor([[1.0, -2.0], [0.5, 0.25], [math.inf, 3.0]])
    places = torch.tensor([[0, 1], [-6, 4], [2, 3]], dtype=torch.int32)
    order = sdfoam_amd.ExpertOrder(places.to(dev), torch.tensor([0, 5], dtype=torch.int32).to(dev))
    live = (places >= 0).double()[..., None]
    terms = torch.where(live > 0, gate.double()[..., None] * y.double()[places.clamp(min=0).long()], 0.0)
    same(sdfoam_amd.expert_combine(y.to(dev), order, gate.to(dev)), terms.sum(1),
         bound(2) * terms.abs().sum(1), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,out", [(3, 64, 32), (40, 64, 64), (300, 200, 136), (300, 201, 137),
                                            (200, 16, 70), (8200, 264, 2056)])
def test_below_the_normal_range(dev, rows, width, out, dtype):
    """Operands below their type's normal range are not taken for 0.  Whole multiples of the
    type's smallest step times powers of two: every sum is exact."""
    say("below the normal range", rows, width, out, dtype)
    step = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[dtype]
    lift = {torch.float32: 2.0 ** 100, torch.float16: 2.0 ** 10, torch.bfloat16: 2.0 ** 100}[dtype]
    g = torch.Generator().manual_seed(rows)
    k = torch.randint(-2, 3, (rows, width), generator=g).double()
    sign = torch.randint(0, 2, (out, width), generator=g).double() * 2 - 1
    sign *= torch.rand((out, width), generator=g) < 8.0 / width  # sums below 2^8
    x, w = (k * step).to(dtype), (sign * lift).to(dtype)
    assert torch.equal(x.double(), k * step)
    y = (k @ sign.T) * (step * lift)
    assert torch.equal(y.to(dtype).double(), y)
    o = torch.tensor([0, rows], dtype=torch.int32, device=dev)
    assert torch.equal(sdfoam_amd.expert_linear(x.to(dev), w.to(dev)[None], o).cpu().double(), y)
    # the same products as the gradient of the rows, and the other operand small
    dx, _ = sdfoam_amd.expert_linear_backward(x.to(dev), torch.empty((rows, out), dtype=dtype, device=dev),
                                              w.t().contiguous().to(dev)[None], o, need_weight=False)
    assert torch.equal(dx.cpu().double(), y)
    small, large = (sign * step).to(dtype), (k * lift).to(dtype)
    assert torch.equal(sdfoam_amd.expert_linear(large.to(dev), small.to(dev)[None], o).cpu().double(), y)
    # as an adapter beside a projection of zeros
    none = torch.zeros((out, width), dtype=dtype, device=dev)
    c = torch.zeros(rows, dtype=torch.int64, device=dev)
    n = min(out, 32)
    z = sdfoam_amd.adapter_linear(x.to(dev), none, c, w[:n].to(dev)[None],
                                  torch.eye(out, n, dtype=dtype, device=dev)[None])
    assert torch.equal(z.cpu().double()[:, :n], y[:, :n]) and not z[:, n:].any()
    # as the gradient of the matrix: sums over few of the rows
    few = torch.zeros((rows, 8), dtype=torch.float64)
    few[:min(rows, 50)] = torch.randint(-1, 2, (min(rows, 50), 8), generator=g).double()
    _, dw = sdfoam_amd.expert_linear_backward((few * lift).to(dtype).to(dev), x.to(dev),
                                              torch.empty((1, 8, width), dtype=dtype, device=dev), o,
                                              need_rows=False)
    assert torch.equal(dw.cpu().double()[0], (few.T @ k) * (step * lift))

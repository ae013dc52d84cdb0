"""The label operators (cell_rows, distill_loss, label_log_probs and their gradients)
against plain statements of their formulas in 64 bits, on the CPU.

Bounds, from the arithmetic alone.  u = 2^-24 is fp32's rounding, v that of the output's
type (2^-24, 2^-11, 2^-8), each with the type's smallest step below its normal range.

* rows: one product of scale and weight, one with the value, one rounding: (2 u + v) |x|.
* a sum of n fp32 terms in any order: n u times the sum of their sizes, n + 3 with the
  terms' own roundings; then v for the result.
* a softmax: x - m has one rounding, times 1 / (T ln 2) three more, so an exponential is off
  by 4 u |x - m| and the 2 u of exp2 itself; the sum adds the roundings of its chains, no
  longer than labels / 256 + 32 terms each.  E = u (16 + 8 R + labels / 256), R the largest
  |x - m| of a label that counts (60 at most: beyond that an exponential is below 1e-26),
  bounds every log probability up to its own size, and every probability relative to it.
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


def near(got, ref, tol, dtype=torch.float32):
    """|got - ref| <= tol and the rounding to dtype, the same infinities and NaN."""
    got = got.detach().cpu().double()
    v, tiny = ROUND[dtype]
    assert got.shape == ref.shape
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    other = ~fine & ~torch.isnan(ref)
    assert torch.equal(got[other], ref[other])
    off = (got - ref).abs()
    lim = tol + v * ref.abs() * 1.01 + tiny
    assert torch.all((off <= lim)[fine]), float((off - lim)[fine].max())


def ids_as(ids, dtype, dev):
    """int64 ids on the device as `dtype` (-1 is 0xffffffff in uint32)."""
    if dtype == torch.uint32:
        return ids.to(torch.int32).to(dev).view(torch.uint32)
    return ids.to(dtype).to(dev)


# ---- rows of cells -----------------------------------------------------------------------


def rows_case(cells, count, width, spread, seed=0):
    g = torch.Generator().manual_seed(seed)
    if spread == "one":
        ids = torch.full((count,), cells // 2, dtype=torch.int64)
    elif spread == "none":
        ids = torch.full((count,), -1, dtype=torch.int64)
    elif spread == "sorted":
        ids = torch.randint(cells, (count,), generator=g).sort().values
    elif spread == "few":  # long runs and lone ids
        ids = torch.where(torch.rand(count, generator=g) < 0.7,
                          torch.randint(min(3, cells), (count,), generator=g),
                          torch.randint(cells, (count,), generator=g))
    else:
        ids = torch.randint(cells, (count,), generator=g)
        ids[torch.rand(count, generator=g) < 0.2] = -1
    return ids, torch.rand(count, generator=g)


def rows_reference(grad, ids, cells, weight, scale):
    """table_grad in 64 bits, the sum of its terms' sizes and their number."""
    f = torch.full(ids.shape, float(scale), dtype=torch.float64)
    if weight is not None:
        f = f * weight.double()
    live = ids >= 0
    terms = (grad.double() * f[:, None])[live]
    out = torch.zeros((cells, grad.shape[1]), dtype=torch.float64)
    size = torch.zeros_like(out)
    out.index_add_(0, ids[live], terms)
    size.index_add_(0, ids[live], terms.abs())
    number = torch.bincount(ids[live], minlength=cells).double()[:, None]
    return out, size, number


ROWS = [  # cells, ids, width, spread
    (1, 1, 1, "one"), (1, 65, 3, "one"), (7, 1, 64, "any"), (33, 64, 49, "any"),
    (100, 1000, 8, "few"), (1000, 63, 130, "sorted"), (1000, 5000, 1, "few"),
    (257, 4097, 17, "any"), (70_000, 20_001, 16, "any"), (70_000, 300, 49, "none"),
    (300, 70_000, 5, "one"), (5, 9000, 33, "few"), (100_003, 257, 100, "sorted"),
    (4104, 8192, 1024, "few"), (50, 12_345, 2, "any"), (17_000_000, 3000, 2, "any"),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cells,count,width,spread", ROWS)
def test_rows_and_gradients(dev, cells, count, width, spread, dtype):
    say("rows", cells, count, width, spread, dtype)
    ids, weight = rows_case(cells, count, width, spread)
    g = torch.Generator().manual_seed(1)
    scale = 1.7
    table = torch.randn((min(cells, 200_000), width), generator=g).to(dtype)
    if table.shape[0] < cells:  # a large table: the same values again and again
        table = table.repeat(cells // table.shape[0], 1)
        cells = table.shape[0]
        ids = torch.where(ids < cells, ids, -1)
    grad = torch.randn((count, width), generator=g).to(dtype)
    t, w, dg = table.to(dev), weight.to(dev), grad.to(dev)
    id_type = [torch.int64, torch.uint32, torch.int32][(cells + count) % 3]
    c = ids_as(ids, id_type, dev)
    v = ROUND[dtype][0]
    for use in (None, w):
        f = scale * (1.0 if use is None else weight.double())
        ref = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)].double(), 0.0)
        ref = ref * (f if use is None else f[:, None])
        out = sdfoam_amd.cell_rows(t, c, use, scale)
        assert out.dtype == dtype
        near(out, ref, 2 * U * ref.abs(), dtype)
        tg, wg = sdfoam_amd.cell_rows_backward(dg, c, cells, use, scale,
                                               table=t if use is not None else None)
        ref, size, number = rows_reference(grad, ids, cells, weight if use is not None else None,
                                           scale)
        assert tg.dtype == dtype
        near(tg, ref, (number + 3) * U * size, dtype)
        again, _ = sdfoam_amd.cell_rows_backward(dg, c, cells, use, scale)
        assert torch.equal(tg.cpu(), again.cpu())
        if use is None:
            assert wg is None
            continue
        prod = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)].double(), 0.0) * grad.double()
        near(wg, scale * prod.sum(1), (width + 3) * U * scale * prod.abs().sum(1))


def test_rows_layouts(dev):
    """Shapes, strided rows, an odd start, broadcast gradients, autograd."""
    g = torch.Generator().manual_seed(2)
    for dtype in TYPES:
        base = torch.randn((40, 23), generator=g).to(dtype)
        wide = base.to(dev)
        table = wide[1:, 3:16]  # rows 23 apart, starting at an odd element
        ids = torch.randint(39, (4, 6), generator=g)
        ids[1, 2] = -1
        ref = torch.where((ids >= 0)[..., None], base[1:, 3:16][ids.clamp(min=0)], 0.0)
        out = sdfoam_amd.cell_rows(table, ids.to(dev))
        assert out.shape == (4, 6, 13)
        assert torch.equal(out.cpu(), ref.to(dtype))
        assert torch.equal(sdfoam_amd.cell_rows(wide.t()[:, 1:].t(), ids.to(dev)).cpu(),
                           torch.where((ids >= 0)[..., None], base[1:][ids.clamp(min=0)], 0.0).to(dtype))
        # ids of another stride; a single id
        assert torch.equal(sdfoam_amd.cell_rows(table, ids.to(dev).t()).cpu(),
                           ref.to(dtype).transpose(0, 1))
        assert torch.equal(sdfoam_amd.cell_rows(table, torch.tensor(3, device=dev)).cpu(),
                           base[4, 3:16])
        one = torch.ones((), dtype=dtype, device=dev)
        tg, _ = sdfoam_amd.cell_rows_backward(one.expand(4, 6, 13), ids.to(dev), 39)
        number = torch.bincount(ids[ids >= 0], minlength=39)
        assert torch.equal(tg.cpu(), number[:, None].expand(39, 13).to(dtype))
        big = torch.randn((24, 30), generator=g).to(dtype)
        part = big.to(dev)[:, 5:18]
        tg, _ = sdfoam_amd.cell_rows_backward(part, ids.reshape(-1).to(dev), 39)
        ref, size, n = rows_reference(big[:, 5:18], ids.reshape(-1), 39, None, 1.0)
        near(tg, ref, (n + 3) * U * size, dtype)


def test_rows_empty(dev):
    z = torch.zeros
    ids = z(0, dtype=torch.int64, device=dev)
    assert sdfoam_amd.cell_rows(z(5, 4, device=dev), ids).shape == (0, 4)
    tg, wg = sdfoam_amd.cell_rows_backward(z(0, 4, device=dev), ids, 5, z(0, device=dev),
                                           table=z(5, 4, device=dev))
    assert torch.equal(tg.cpu(), z(5, 4)) and wg.shape == (0,)
    none = torch.full((3,), -1, device=dev)
    out = sdfoam_amd.cell_rows(z(0, 4, device=dev), none)
    assert torch.equal(out.cpu(), z(3, 4))
    tg, wg = sdfoam_amd.cell_rows_backward(torch.ones(3, 4, device=dev), none, 0,
                                           torch.ones(3, device=dev), table=z(0, 4, device=dev))
    assert tg.shape == (0, 4) and torch.equal(wg.cpu(), z(3))
    assert sdfoam_amd.cell_rows(z(5, 0, device=dev), none).shape == (3, 0)
    tg, wg = sdfoam_amd.cell_rows_backward(z(3, 0, device=dev), none, 5, torch.ones(3, device=dev),
                                           table=z(5, 0, device=dev))
    assert tg.shape == (5, 0) and torch.equal(wg.cpu(), z(3))


def test_rows_ids_past_the_table(dev):
    table = torch.arange(12.0, device=dev).reshape(4, 3)
    ids = torch.tensor([3, 4, -1, 2 ** 31, 2 ** 32, -2 ** 40, 0], device=dev)
    out = sdfoam_amd.cell_rows(table, ids).cpu()
    ref = torch.zeros(7, 3)
    ref[0], ref[6] = table[3].cpu(), table[0].cpu()
    assert torch.equal(out, ref)
    # what no id names stays out of the gradients, whatever stands in its rows
    grad = torch.ones(7, 3, device=dev)
    grad[1:6] = math.nan
    tg, wg = sdfoam_amd.cell_rows_backward(grad, ids, 4, torch.ones(7, device=dev), table=table)
    assert torch.equal(tg.cpu(), torch.tensor([[1.0] * 3, [0.0] * 3, [0.0] * 3, [1.0] * 3]))
    assert torch.equal(wg.cpu(), torch.tensor([30.0, 0, 0, 0, 0, 0, 3.0]))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_autograd(dev, dtype):
    g = torch.Generator().manual_seed(3)
    table = torch.randn((50, 12), generator=g).to(dtype)
    weight = torch.rand((8, 9), generator=g)
    ids = torch.randint(-1, 50, (8, 9), generator=g)
    grad = torch.randn((8, 9, 12), generator=g).to(dtype)
    t = table.to(dev).requires_grad_()
    w = weight.to(dev).requires_grad_()
    sdfoam_amd.cell_rows(t, ids.to(dev), w, 0.5).backward(grad.to(dev))
    tg, wg = sdfoam_amd.cell_rows_backward(grad.to(dev), ids.to(dev), 50, weight.to(dev), 0.5,
                                           table=table.to(dev))
    assert torch.equal(t.grad, tg) and torch.equal(w.grad, wg)
    # only one of the two is asked for
    w2 = weight.to(dev).requires_grad_()
    sdfoam_amd.cell_rows(table.to(dev), ids.to(dev), w2, 0.5).backward(grad.to(dev))
    assert torch.equal(w2.grad, wg)
    t2 = table.to(dev).requires_grad_()
    sdfoam_amd.cell_rows(t2, ids.to(dev), weight.to(dev), 0.5).backward(grad.to(dev))
    assert torch.equal(t2.grad, tg)


def test_rows_differences(dev):
    """<gradient, direction> against differences of the outputs themselves: rows are linear
    in the table and in the weights, so a difference of any length is exact but for the
    outputs' roundings (2 u of each side, over 2 h = 2, summed over the outputs)."""
    g = torch.Generator().manual_seed(4)
    table, weight = torch.randn((30, 9), generator=g), torch.rand(200, generator=g)
    ids = torch.randint(-1, 30, (200,), generator=g).to(dev)
    up = torch.randn((200, 9), generator=g).to(dev)
    dt, dw = torch.randn((30, 9), generator=g), torch.randn(200, generator=g)
    tg, wg = sdfoam_amd.cell_rows_backward(up, ids, 30, weight.to(dev), 1.3, table=table.to(dev))
    for gradient, d, sides in (
            (tg, dt, [sdfoam_amd.cell_rows((table + h * dt).to(dev), ids, weight.to(dev), 1.3)
                      for h in (1, -1)]),
            (wg, dw, [sdfoam_amd.cell_rows(table.to(dev), ids, (weight + h * dw).to(dev), 1.3)
                      for h in (1, -1)])):
        diff = float((up.double() * (sides[0].double() - sides[1].double())).sum() / 2)
        size = float((up.abs().double() * (sides[0].abs() + sides[1].abs()).double()).sum())
        assert abs(diff - float((gradient.cpu().double() * d.double()).sum())) <= 40 * U * size


@pytest.mark.parametrize("cells", [900, 2000, 70_000])
@pytest.mark.parametrize("count", [16_384, 16_385, 262_144, 262_145])
def test_rows_gradient_at_the_sorts_limits(dev, cells, count):
    """Whole numbers, so that every sum is exact: the counts at which the sort of the ids
    takes another form, with one and two digits a thread and one and two passes."""
    say("rows, sort", cells, count)
    g = torch.Generator().manual_seed(count + cells)
    ids = torch.randint(-1, cells, (count,), generator=g)
    up = torch.randint(-9, 10, (count, 3), generator=g).float()
    weight = torch.randint(1, 4, (count,), generator=g).float()
    got, _ = sdfoam_amd.cell_rows_backward(up.to(dev), ids.to(dev), cells, weight.to(dev))
    sums = torch.zeros((cells + 1, 3)).index_add_(0, torch.where(ids < 0, cells, ids),
                                                  up * weight[:, None])
    assert torch.equal(got.cpu(), sums[:cells])


@pytest.mark.parametrize("width", [1, 3, 8, 24, 61, 200, 700])
def test_rows_gradient_of_long_runs(dev, width):
    """Whole numbers, so that every sum is exact: cells that 1 to 6,000 ids name, the ids of
    a cell beside each other and spread."""
    say("rows, runs", width)
    g = torch.Generator().manual_seed(width)
    runs = torch.cat([torch.arange(1, 40), torch.arange(40, 800, 37),
                      torch.tensor([511, 512, 513, 519, 520, 527, 528, 1023, 6000, 1, 3000])])
    cells = len(runs)
    ids = torch.repeat_interleave(torch.arange(cells), runs)
    up = torch.randint(-9, 10, (len(ids), width), generator=g).float()
    for order in (torch.arange(len(ids)), torch.randperm(len(ids), generator=g)):
        for dtype in (torch.float32, torch.bfloat16):
            got, _ = sdfoam_amd.cell_rows_backward(up[order].to(dtype).to(dev),
                                                   ids[order].to(dev), cells)
            sums = torch.zeros((cells, width)).index_add_(0, ids, up)
            assert torch.equal(got.cpu(), sums.to(dtype))


def test_rows_past_32_bits(dev):
    """Tables and gradients of more than 2^32 bytes and 2^31 elements."""
    cells, width = 1_100_003, 2048
    say("rows past 32 bits")
    table = torch.zeros((cells, width), dtype=torch.bfloat16, device=dev)
    ids = torch.tensor([cells - 1, 5, 1_048_577, cells - 1], device=dev)
    table[ids] = torch.arange(width, dtype=torch.bfloat16, device=dev) % 97
    out = sdfoam_amd.cell_rows(table, ids)
    assert torch.equal(out, table[ids])
    tg, _ = sdfoam_amd.cell_rows_backward(out, ids, cells)
    assert torch.equal(tg[cells - 1], 2 * out[0]) and torch.equal(tg[5], out[1])
    assert torch.equal(tg[1_048_577], out[2])
    assert int((tg != 0).any(1).sum()) == 3


def test_rows_of_more_than_one_launch(dev):
    """More rows than one launch takes: 270,000 of 8,192 elements, and the weights' gradient
    alone of 1.1 million ids."""
    say("rows of more than one launch")
    g = torch.Generator().manual_seed(5)
    table = torch.randn((50, 8192), generator=g).to(torch.bfloat16).to(dev)
    ids = torch.randint(-1, 50, (270_000,), generator=g).to(dev)
    out = sdfoam_amd.cell_rows(table, ids)
    ref = torch.cat([table, torch.zeros((1, 8192), dtype=torch.bfloat16, device=dev)])
    for k in range(0, 270_000, 30_000):
        assert torch.equal(out[k:k + 30_000], ref[ids[k:k + 30_000]])
    del out
    table = torch.randn((50, 3), generator=g)
    ids = torch.randint(-1, 50, (1_100_000,), generator=g)
    up = torch.randn((1_100_000, 3), generator=g)
    w = torch.rand(1_100_000, generator=g).to(dev).requires_grad_()
    sdfoam_amd.cell_rows(table.to(dev), ids.to(dev), w).backward(up.to(dev))
    prod = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)].double(), 0.0) * up.double()
    near(w.grad, prod.sum(1), 6 * U * prod.abs().sum(1))


def test_weights_gradient_alone_takes_no_workspace(dev):
    """The weights' gradient by itself allocates that gradient and nothing beside it."""
    g = torch.Generator().manual_seed(6)
    table, up = torch.randn((50, 512), generator=g), torch.randn((20_000, 512), generator=g)
    ids = torch.randint(-1, 50, (20_000,), generator=g)
    w = torch.rand(20_000, generator=g).to(dev).requires_grad_()
    out = sdfoam_amd.cell_rows(table.to(dev), ids.to(dev), w)
    ud = up.to(dev)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out.backward(ud)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= 4 * 20_000 + 4096
    prod = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)].double(), 0.0) * up.double()
    near(w.grad, prod.sum(1), 515 * U * prod.abs().sum(1))


@pytest.mark.parametrize("width", [3, 64, 1000])
def test_rows_of_no_cell_at_any_scale(dev, width):
    """A scale that has overflown reaches the rows of cells, and those of no cell stay 0."""
    ids = torch.tensor([1, -1, 0, 7, -1], device=dev)
    none = (ids < 0) | (ids >= 4)
    table, up = torch.ones((4, width), device=dev), torch.ones((5, width), device=dev)
    for scale in (math.inf, math.nan):
        w = torch.ones(5, device=dev).requires_grad_()
        out = sdfoam_amd.cell_rows(table, ids, w, scale)
        assert not out[none].any() and not out[~none].isfinite().any()
        out.backward(up)  # the weights' gradient by itself
        tg, wg = sdfoam_amd.cell_rows_backward(up, ids, 4, w.detach(), scale, table=table)
        for x in (wg, w.grad):
            assert not x[none].any() and not x[~none].isfinite().any()
        assert not tg[2:].any() and not tg[:2].isfinite().any()


@pytest.mark.parametrize("count", [4096, 4097, 10_001, 16_383, 16_384, 16_385])
def test_rows_gradient_beside_a_large_table(dev, count):
    """Whole numbers, so that every sum is exact.  50,000 x 1,024 floats are cleared (195
    MiB): beside so much one block sorts up to 16,384 ids, 16 a thread."""
    say("rows, one block beside a large table", count)
    g = torch.Generator().manual_seed(count)
    cells, width = 50_000, 1024
    up = torch.randint(-9, 10, (count, width), generator=g).float()
    weight = torch.randint(1, 4, (count,), generator=g).float()
    few = torch.randint(3, (count,), generator=g) * 20_000
    for ids in (torch.randint(-1, cells, (count,), generator=g),
                torch.where(torch.rand(count, generator=g) < 0.6, few,
                            torch.randint(-3000, cells, (count,), generator=g)),
                torch.arange(count).flip(0) * 3, torch.full((count,), cells - 1)):
        for w in (None, weight):
            got, _ = sdfoam_amd.cell_rows_backward(up.to(dev), ids.to(dev), cells,
                                                   None if w is None else w.to(dev))
            live = ids >= 0
            sums = torch.zeros((cells, width), device=dev)
            terms = up if w is None else up * w[:, None]
            sums.index_add_(0, ids[live].to(dev), terms[live].to(dev))
            assert torch.equal(got, sums)


# ---- logits ------------------------------------------------------------------------------


def logits_case(rows, labels, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed + rows + labels)
    z = (spread * torch.randn((rows, labels), generator=g)).to(dtype)
    return z, g


def softmax64(z, temperature):
    """log probabilities in 64 bits (a row of -inf alone: zeros), which rows have any label,
    and E."""
    x = z.double() / temperature
    live = (x > -math.inf).any(1) | torch.isnan(x).any(1)
    x = torch.where(live[:, None], x, 0.0)
    m = x.amax(1, keepdim=True)
    far = torch.where(x > -math.inf, (m - x).clamp(max=60.0), 0.0).nan_to_num(0.0).amax(1)
    err = U * (16 + 8 * far + z.shape[1] / 256)
    x = x - m  # first: a row may be of the type's lowest value
    return x - x.exp().sum(1, keepdim=True).log(), live, err


def distill_reference(z, ids, t, temperature, weight, reduction, up=None):
    """loss, gradient, and bounds for each, in 64 bits."""
    labels = z.shape[1]
    log_p, live, err = softmax64(z, temperature)
    ok = (ids >= 0) & (ids < labels)
    t = t.double() / temperature
    ok &= ~(t == -math.inf)
    counts = live & ok.any(1)
    weight = torch.ones(z.shape[0], dtype=torch.float64) if weight is None else weight.double()
    counts &= weight != 0
    tt = torch.where(ok, t, -math.inf)
    tt = torch.where(counts[:, None], tt, 0.0)
    log_q = tt - torch.logsumexp(tt, 1, keepdim=True)
    q = torch.where(ok & counts[:, None], log_q.exp(), 0.0)
    at = ids.clamp(0, labels - 1)
    lp = log_p.gather(1, at)
    far_t = torch.where(ok & counts[:, None], (tt.amax(1, keepdim=True) - tt).clamp(max=60.0), 0.0)
    err = err + U * (16 + 8 * far_t.nan_to_num(0.0).amax(1) + ids.shape[1] / 64)
    # below fp32's smallest exponential the kernel's share is 0
    used = q > 1e-37
    terms = torch.where(used, q * (log_q - lp), 0.0)
    size = torch.where(used, q * (2 + log_q.abs() + lp.abs()), 0.0).sum(1)
    f = torch.where(counts, weight * temperature ** 2, 0.0)
    loss = torch.where(counts, f * terms.sum(1), 0.0)
    loss_tol = torch.where(counts, f.abs() * 4 * err * size, 0.0)
    coef = torch.where(counts, weight * temperature, 0.0)
    if reduction == "mean":
        coef = coef / z.shape[0]
    if up is not None:
        coef = coef * up
    coef = torch.where(counts, coef, 0.0)
    mass = torch.zeros(z.shape, dtype=torch.float64).scatter_add_(1, at, q)
    p = torch.where(counts[:, None], log_p.exp(), 0.0)
    grad = torch.where(counts[:, None], coef[:, None] * (p - mass), 0.0)
    grad_tol = torch.where(counts[:, None],
                           coef.abs()[:, None] * 4 * err[:, None] * (p + mass + 2.0 ** -100), 0.0)
    if reduction != "none":
        n = len(loss)
        scale = 1.0 / n if reduction == "mean" else 1.0
        loss_tol = (loss_tol.sum() + 2 * U * loss.abs().sum()) * scale
        loss = loss.sum() * scale
    return loss, grad, loss_tol, grad_tol


def teacher_case(rows, labels, top, g, dtype=torch.float32):
    ids = torch.randint(labels, (rows, top), generator=g)
    t = (2.0 * torch.randn((rows, top), generator=g)).to(dtype)
    u = torch.rand((rows, top), generator=g)
    ids[u < 0.05] = -1
    t[(u >= 0.05) & (u < 0.1)] = -math.inf
    t[u < 0.02] = math.nan  # under a label that is none
    if rows > 2:
        ids[rows // 2] = -1
    return ids, t


SHAPES = [  # rows, labels, teacher's entries
    (1, 1, 1), (3, 2, 2), (5, 20, 4), (70, 63, 8), (3, 64, 8), (9, 65, 8), (130, 121, 5),
    (2, 257, 16), (33, 1000, 32), (4, 1024, 64), (5, 1025, 64), (6, 2049, 33), (7, 4099, 64),
    (3, 8191, 1000), (2, 16_384, 100), (3, 33_001, 64), (1, 65_536, 8), (300, 5003, 7),
    (2, 65_537, 8), (1, 131_072, 64), (3, 131_075, 128), (1, 262_147, 20), (600, 300, 3),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,labels,top", SHAPES)
def test_distill(dev, rows, labels, top, dtype):
    say("distill", rows, labels, top, dtype)
    z, g = logits_case(rows, labels, dtype)
    teacher_type = TYPES[(labels + top) % 3]
    ids, t = teacher_case(rows, labels, top, g, teacher_type)
    weight = torch.rand(rows, generator=g) + 0.5
    weight[torch.rand(rows, generator=g) < 0.2] = 0.0
    id_type = [torch.int64, torch.uint32, torch.int32][(rows + labels) % 3]
    zd, td, jd = z.to(dev), t.to(dev), ids_as(ids, id_type, dev)
    for reduction, temperature, w in (("mean", 1.0, None), ("none", 2.0, weight),
                                      ("sum", 0.7, weight)):
        up = torch.randn(rows, generator=g) if reduction == "none" else torch.tensor(3.0)
        loss, grad, lt, gt = distill_reference(z, ids, t, temperature, w, reduction, up.double())
        wd = None if w is None else w.to(dev)
        got, dz = sdfoam_amd.distill_loss_and_grad(zd, jd, td, temperature, wd, reduction,
                                                   up.to(dev))
        near(got, loss, lt)
        near(dz, grad, gt, dtype)
        assert dz.dtype == dtype
        only = sdfoam_amd.distill_loss(zd, jd, td, temperature, wd, reduction)
        near(only, loss, lt)
        leaf = zd.clone().requires_grad_()
        auto = sdfoam_amd.distill_loss(leaf, jd, td, temperature, wd, reduction)
        auto.backward(up.to(dev))
        near(auto, loss, lt)
        near(leaf.grad, grad, gt, dtype)
        again, dz2 = sdfoam_amd.distill_loss_and_grad(zd, jd, td, temperature, wd, reduction,
                                                      up.to(dev))
        assert torch.equal(got, again) and torch.equal(dz, dz2)


@pytest.mark.parametrize("labels", [37, 1000, 5003, 70_001])
def test_distill_masks(dev, labels):
    """Masked labels, by -inf and by the type's lowest value, rows that are masked whole,
    rows without an entry, rows of weight 0 that hold NaN, labels named twice."""
    say("distill masks", labels)
    for dtype in TYPES:
        z, g = logits_case(9, labels, dtype, seed=5)
        low = torch.finfo(dtype).min
        ids = torch.randint(labels, (9, 12), generator=g)
        t = torch.randn((9, 12), generator=g)
        keep = torch.zeros((9, labels), dtype=torch.bool).scatter_(1, ids, True)
        z[0][~keep[0]] = -math.inf
        z[1] = -math.inf
        z[2][~keep[2]] = low
        z[3] = low
        ids[4] = -1
        t[4] = math.nan
        z[4] = math.nan
        weight = torch.ones(9)
        weight[5] = 0.0
        z[5] = math.nan
        z[5, 0] = math.inf
        ids[6, 1:] = ids[6, 0]  # one label, twelve times
        z[7, ids[7, 3]] = -math.inf  # a label that the teacher names is masked
        t[8] = -math.inf
        t[8, 5] = 1.0
        loss, grad, lt, gt = distill_reference(z, ids, t, 1.5, weight, "none")
        assert loss[7] == math.inf and loss[1] == 0 and loss[4] == 0 and loss[5] == 0
        got, dz = sdfoam_amd.distill_loss_and_grad(z.to(dev), ids.to(dev), t.to(dev), 1.5,
                                                   weight.to(dev), "none")
        near(got, loss, lt)
        near(dz, grad, gt, dtype)
        leaf = z.to(dev).requires_grad_()
        sdfoam_amd.distill_loss(leaf, ids.to(dev), t.to(dev), 1.5, weight.to(dev),
                                "none").backward(torch.ones(9, device=dev))
        near(leaf.grad, grad, gt, dtype)


@pytest.mark.parametrize("top", [1, 2, 3, 5, 7, 65, 255, 1022, 1024])
def test_distill_labels_named_often(dev, top):
    """Teachers whose entries name a few labels over and over, at odd counts of entries."""
    say("distill named often", top)
    for labels, named in ((40, 3), (3001, 40), (70_001, 500)):
        z, g = logits_case(5, labels, torch.float32, seed=top)
        ids = torch.randint(named, (5, top), generator=g) * (labels // named)
        t = torch.randn((5, top), generator=g)
        loss, grad, lt, gt = distill_reference(z, ids, t, 1.5, None, "none")
        got, dz = sdfoam_amd.distill_loss_and_grad(z.to(dev), ids.to(dev), t.to(dev), 1.5,
                                                   reduction="none")
        near(got, loss, lt)
        # a sum of up to `top` shares, one after the other, may be off by top U of it; gt
        # holds 64 U of it at least
        near(dz, grad, gt * (1 + top / 64), torch.float32)


@pytest.mark.parametrize("labels", [37, 5003, 70_001])
def test_distill_nan_reaches_the_loss(dev, labels):
    for at in (0, labels // 2, labels - 1):
        for bad in (math.nan, math.inf):
            z, g = logits_case(3, labels, torch.float32)
            z[1, at] = bad
            ids = torch.randint(labels, (3, 4), generator=g)
            t = torch.randn((3, 4), generator=g)
            got, dz = sdfoam_amd.distill_loss_and_grad(z.to(dev), ids.to(dev), t.to(dev),
                                                       reduction="none")
            assert got.isnan().tolist() == [False, True, False]
            assert dz[1].isnan().all() and not dz[0].isnan().any() and not dz[2].isnan().any()
    z[1] = math.nan
    got, dz = sdfoam_amd.distill_loss_and_grad(z.to(dev), ids.to(dev), t.to(dev), reduction="none")
    assert got.isnan().tolist() == [False, True, False] and dz[1].isnan().all()
    t[0, 0] = math.nan
    got = sdfoam_amd.distill_loss(z.to(dev), ids.to(dev), t.to(dev), reduction="none")
    assert got.isnan().tolist() == [True, True, False]


def test_distill_layouts(dev):
    """Leading dimensions, padded rows read in place, an odd start, other orders."""
    for dtype in TYPES:
        z, g = logits_case(24, 333, dtype)
        ids, t = teacher_case(24, 333, 6, g)
        loss, grad, lt, gt = distill_reference(z, ids, t, 1.0, None, "mean")
        padded = torch.full((2, 12, 351), math.nan, dtype=dtype, device=dev)
        padded[..., 7:340] = z.to(dev).reshape(2, 12, 333)
        turned = z.to(dev).t().contiguous().t()
        for zd in (padded[..., 7:340], turned):
            shape = zd.shape[:-1]
            got, dz = sdfoam_amd.distill_loss_and_grad(zd, ids.to(dev).reshape(*shape, 6),
                                                       t.to(dev).reshape(*shape, 6))
            near(got, loss, lt)
            assert dz.shape == zd.shape and dz.is_contiguous()
            near(dz.reshape(24, 333), grad, gt, dtype)
        same = z[:1].to(dev).expand(24, 333)
        loss, grad, lt, gt = distill_reference(z[:1].expand(24, 333), ids, t, 1.0, None, "none")
        got, dz = sdfoam_amd.distill_loss_and_grad(same, ids.to(dev), t.to(dev), reduction="none")
        near(got, loss, lt)
        near(dz, grad, gt, dtype)
    one = sdfoam_amd.distill_loss(z[0].to(dev), ids[0].to(dev), t[0].to(dev), reduction="none")
    assert one.shape == ()


def test_distill_empty(dev):
    z = torch.randn(5, 40, device=dev)
    none = torch.zeros((5, 0), dtype=torch.int64, device=dev)
    loss, dz = sdfoam_amd.distill_loss_and_grad(z, none, none.float())
    assert float(loss) == 0 and not dz.any()
    loss, dz = sdfoam_amd.distill_loss_and_grad(z[:0], none[:0], none[:0].float(), reduction="sum")
    assert float(loss) == 0 and dz.shape == (0, 40)
    assert sdfoam_amd.distill_loss(z[:0], none[:0], none[:0].float(), reduction="none").shape == (0,)


def test_distill_differences(dev):
    """<gradient, direction> against differences of the loss.  With |d| = 1 per row the third
    derivative of a softmax's logarithm is below 1, so a difference over 2 h is off by h^2 / 6
    and by the loss's own bound over h."""
    h = 1.0 / 64
    for labels in (50, 3001):
        z, g = logits_case(20, labels, torch.float32, spread=2.0)
        ids, t = teacher_case(20, labels, 8, g)
        d = torch.randn((20, labels), generator=g)
        d /= d.norm(dim=1, keepdim=True)
        _, grad = sdfoam_amd.distill_loss_and_grad(z.to(dev), ids.to(dev), t.to(dev), 1.0, None,
                                                   "none")
        sides = [sdfoam_amd.distill_loss((z + s * h * d).to(dev), ids.to(dev), t.to(dev), 1.0, None,
                                         "none").cpu().double() for s in (1, -1)]
        _, _, lt, _ = distill_reference(z, ids, t, 1.0, None, "none")
        diff = (sides[0] - sides[1]) / (2 * h)
        got = (grad.cpu().double() * d.double()).sum(1)
        assert torch.all((diff - got).abs() <= h * h / 6 + 2 * (lt + 8 * U) / h)


def best_reference(z, top):
    """Labels by falling logit, ties to the lowest; -1 where none above -inf is left."""
    x = z.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    v, i = x.sort(dim=1, descending=True, stable=True)
    v, i = v[:, :top], i[:, :top]
    i = torch.where(v > -math.inf, i, -1)
    if i.shape[1] < top:
        i = torch.cat([i, torch.full((i.shape[0], top - i.shape[1]), -1)], 1)
    return i


def check_answer(dev, z, y, top, temperature, dtype, id_type=torch.int64, grads=True):
    rows, labels = z.shape
    log_p, live, err = softmax64(z, temperature)
    named = (y >= 0) & (y < labels)
    at = y.clamp(0, labels - 1)[:, None]
    lp = log_p.gather(1, at)[:, 0]
    lp = torch.where(live, lp, -math.inf)
    lp = torch.where(named, lp, 0.0)
    p = log_p.exp()
    some = torch.where(p > 0, log_p, 0.0)
    entropy = torch.where(live, -(p * some).sum(1), 0.0)
    best = best_reference(z, top)
    best_lp = log_p.gather(1, best.clamp(min=0))
    best_lp = torch.where(best >= 0, best_lp, -math.inf)
    a = sdfoam_amd.label_log_probs(z.to(dev), ids_as(y, id_type, dev), top, temperature)
    near(a.log_prob, lp, 2 * err * (2 + lp.abs().nan_to_num(0.0, 0.0, 0.0)))
    far = (p * some.abs()).sum(1)
    near(a.entropy, entropy, 4 * err * (2 + far))
    if top:
        assert torch.equal(a.top_labels.cpu(), best)
        near(a.top_log_probs, best_lp,
             2 * err[:, None] * (2 + best_lp.abs().nan_to_num(0.0, 0.0, 0.0)))
    else:
        assert a.top_labels is None and a.top_log_probs is None
    if not grads:
        return
    g = torch.Generator().manual_seed(rows + labels)
    gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    for use_l, use_h in ((gl, gh), (gl, None), (None, gh)):
        leaf = z.to(dev).requires_grad_()
        a = sdfoam_amd.label_log_probs(leaf, ids_as(y, id_type, dev), top, temperature)
        outs = [o for o, u in ((a.log_prob, use_l), (a.entropy, use_h)) if u is not None]
        ups = [u.to(dev) for u in (use_l, use_h) if u is not None]
        dz, = torch.autograd.grad(outs, leaf, ups)
        cl = torch.where(named & live, gl.double() * (use_l is not None), 0.0)
        ch = torch.where(live, gh.double() * (use_h is not None), 0.0)
        ref = -p * (cl[:, None] + ch[:, None] * (some + entropy[:, None]))
        ref = torch.where(p > 0, ref, 0.0)
        ref.scatter_add_(1, at, cl[:, None])
        ref = torch.where(live[:, None], ref / temperature, 0.0)
        size = p * (cl.abs()[:, None] + ch.abs()[:, None] * (2 + some.abs() + entropy[:, None]))
        size = size.scatter_add(1, at, cl.abs()[:, None])
        near(dz, ref, 8 * err[:, None] * (size + 2.0 ** -100) / temperature, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,labels,top", SHAPES)
def test_answers(dev, rows, labels, top, dtype):
    say("answers", rows, labels, top, dtype)
    z, g = logits_case(rows, labels, dtype, seed=7)
    y = torch.randint(labels, (rows,), generator=g)
    y[torch.rand(rows, generator=g) < 0.1] = -1
    id_type = [torch.int64, torch.uint32, torch.int32][(rows + labels) % 3]
    check_answer(dev, z, y, min(top, 64), [1.0, 0.7, 2.0][labels % 3], dtype, id_type)
    check_answer(dev, z, y, 0, 1.0, dtype, id_type, grads=False)


@pytest.mark.parametrize("labels", [12, 121, 1000, 5003, 70_001, 140_000])
def test_answers_ties(dev, labels):
    """Ties go to the lowest label: rows of one value, of few values, of both zeros; and
    rows that fall or rise."""
    say("ties", labels)
    for dtype in TYPES:
        z, g = logits_case(8, labels, dtype)
        z[0] = 1.5
        z[1] = torch.randint(3, (labels,), generator=g).to(dtype)
        z[2] = torch.where(torch.rand(labels, generator=g) < 0.5, 0.0, -0.0).to(dtype)
        z[3] = torch.linspace(-3, 3, labels).to(dtype)
        z[4] = torch.linspace(3, -3, labels).to(dtype)
        z[5] = torch.finfo(dtype).min
        z[6] = 0.0
        z[6, -1] = 1.0
        y = torch.randint(labels, (8,), generator=g)
        for top in (1, 5, 64):
            check_answer(dev, z, y, top, 1.0, dtype, grads=False)


@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_distill_sums_of_many_rows(dev, reduction):
    """300,000 rows: the sum of the rows' own losses, each rounded to fp32, in 64 bits."""
    g = torch.Generator().manual_seed(3)
    z = torch.randn((300_000, 7), generator=g).to(dev)
    j = torch.randint(-1, 7, (300_000, 2), generator=g).to(dev)
    t = torch.randn((300_000, 2), generator=g).to(dev)
    rows = sdfoam_amd.distill_loss(z, j, t, reduction="none").double().sum().cpu()
    got = sdfoam_amd.distill_loss(z, j, t, reduction=reduction)
    near(got, rows if reduction == "sum" else rows / 300_000, 2 * U * rows.abs()
         if reduction == "sum" else 2 * U * rows.abs() / 300_000)


def test_answers_first_of_many_equal(dev):
    """The largest logit many times over, its first labels late in the row."""
    for labels in (5003, 70_001, 100_003):
        for dtype in TYPES:
            z, g = logits_case(4, labels, dtype)
            z[0, labels // 3:] = 20.0
            z[1, labels - 700:] = 20.0
            z[2, ::3] = 20.0
            z[3] = -5.0
            y = torch.randint(labels, (4,), generator=g)
            big = z.repeat(200, 1)
            for top in (1, 8, 64):
                check_answer(dev, z, y, top, 1.0, dtype, grads=False)
                a = sdfoam_amd.label_log_probs(big.to(dev), y.repeat(200).to(dev), top)
                assert torch.equal(a.top_labels.cpu(), best_reference(z, top).repeat(200, 1))


@pytest.mark.parametrize("labels", [37, 1000, 5003, 70_001, 140_000])
def test_answers_masks(dev, labels):
    """Few labels allowed, spread or side by side; none; the label itself masked."""
    say("answer masks", labels)
    for dtype in TYPES:
        z, g = logits_case(8, labels, dtype)
        y = torch.randint(labels, (8,), generator=g)
        low = torch.finfo(dtype).min
        keep = torch.rand(labels, generator=g) < 20.0 / labels
        z[0][~keep] = -math.inf
        z[1] = -math.inf
        z[2, 30:] = -math.inf
        z[3][~keep] = low
        z[4] = -math.inf
        z[4, labels - 1] = -2.0
        y[4] = labels - 1
        z[5, y[5]] = -math.inf
        z[6, : labels // 2] = -math.inf
        y[7] = -1
        for top in (0, 3, 40):
            check_answer(dev, z, y, top, 1.3, dtype)


@pytest.mark.parametrize("labels", [37, 5003, 140_000])
def test_answers_nan(dev, labels):
    for bad in (math.nan, math.inf):
        z, g = logits_case(3, labels, torch.float32)
        z[1, labels // 3] = bad
        y = torch.randint(labels, (3,), generator=g)
        a = sdfoam_amd.label_log_probs(z.to(dev), y.to(dev), 4)
        assert a.log_prob.isnan().tolist() == [False, True, False]
        assert a.entropy.isnan().tolist() == [False, True, False]
        assert a.top_log_probs[1].isnan().all() and not a.top_log_probs[0].isnan().any()
        assert torch.equal(a.top_labels.cpu(), best_reference(z, 4))
    z[1] = math.nan
    a = sdfoam_amd.label_log_probs(z.to(dev), y.to(dev), 4)
    assert a.log_prob.isnan().tolist() == [False, True, False]
    assert a.top_labels[1].tolist() == [-1] * 4


def test_answers_layouts(dev):
    for dtype in TYPES:
        z, g = logits_case(24, 1777, dtype)
        y = torch.randint(1777, (24,), generator=g)
        ref = sdfoam_amd.label_log_probs(z.to(dev), y.to(dev), 5)
        padded = torch.full((2, 12, 1801), math.nan, dtype=dtype, device=dev)
        padded[..., 3:1780] = z.to(dev).reshape(2, 12, 1777)
        a = sdfoam_amd.label_log_probs(padded[..., 3:1780], y.to(dev).reshape(2, 12), 5)
        assert a.top_labels.shape == (2, 12, 5) and a.log_prob.shape == (2, 12)
        _, _, err = softmax64(z, 1.0)
        near(a.log_prob.reshape(24), ref.log_prob.cpu().double(), 80 * err)
        assert torch.equal(a.top_labels.reshape(24, 5), ref.top_labels)
        one = sdfoam_amd.label_log_probs(z[0].to(dev), y[0].to(dev), 5)
        assert one.log_prob.shape == () and one.top_labels.tolist() == ref.top_labels[0].tolist()
    none = sdfoam_amd.label_log_probs(z[:0].to(dev), y[:0].to(dev), 5)
    assert none.log_prob.shape == (0,) and none.top_labels.shape == (0, 5)


def test_answers_differences(dev):
    """As for the loss: the third derivatives of log p and of the entropy along a direction
    of length 1 are below 1 and 16."""
    h = 1.0 / 64
    for labels in (50, 3001):
        z, g = logits_case(20, labels, torch.float32, spread=2.0)
        y = torch.randint(labels, (20,), generator=g)
        d = torch.randn((20, labels), generator=g)
        d /= d.norm(dim=1, keepdim=True)
        leaf = z.to(dev).requires_grad_()
        a = sdfoam_amd.label_log_probs(leaf, y.to(dev))
        one = torch.ones(20, device=dev)
        for k, third in ((0, 1.0), (1, 16.0)):
            grad, = torch.autograd.grad(a[k], leaf, one, retain_graph=True)
            sides = [sdfoam_amd.label_log_probs((z + s * h * d).to(dev), y.to(dev))[k]
                     .cpu().double() for s in (1, -1)]
            diff = (sides[0] - sides[1]) / (2 * h)
            got = (grad.cpu().double() * d.double()).sum(1)
            _, _, err = softmax64(z, 1.0)
            assert torch.all((diff - got).abs() <= third * h * h / 6 + 2 * err * 40 / h)


def test_logits_past_32_bits(dev):
    """Logits of more than 2^32 bytes and 2^31 elements: the last rows as if alone."""
    rows, labels = 17_000, 131_073
    say("logits past 32 bits")
    z = torch.zeros((rows, labels), dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(1)
    tail = (3.0 * torch.randn((4, labels), generator=g)).to(torch.bfloat16).to(dev)
    z[-4:] = tail
    y = torch.randint(labels, (rows,), generator=g).to(dev)
    a = sdfoam_amd.label_log_probs(z, y, 4)
    b = sdfoam_amd.label_log_probs(tail, y[-4:], 4)
    assert torch.equal(a.top_labels[-4:], b.top_labels)
    assert torch.equal(a.top_labels[0].cpu(), torch.arange(4))
    assert torch.allclose(a.log_prob[-4:], b.log_prob, rtol=1e-5)
    del a
    ids = torch.randint(labels, (rows, 4), generator=g).to(dev)
    t = torch.randn((rows, 4), generator=g).to(dev)
    la, da = sdfoam_amd.distill_loss_and_grad(z, ids, t, reduction="none")
    lb, db = sdfoam_amd.distill_loss_and_grad(tail, ids[-4:], t[-4:], reduction="none")
    assert torch.allclose(la[-4:], lb, rtol=1e-5)
    # one rounding of bf16 apart at most
    assert torch.all((da[-4:].float() - db.float()).abs() <= 2.0 ** -7 * db.float().abs() + 1e-30)


def test_rows_of_logits_of_more_than_one_launch(dev):
    """4.2 million rows of 5 labels: the last rows as if alone."""
    say("more rows than a launch takes")
    rows, labels = (1 << 22) + 77, 5
    g = torch.Generator().manual_seed(2)
    z = torch.randn((rows, labels), generator=g).to(dev)
    j = torch.randint(-1, labels, (rows, 2), generator=g).to(dev)
    t = torch.randn((rows, 2), generator=g).to(dev)
    w = torch.rand(rows, generator=g).to(dev)
    up = torch.randn(rows, generator=g).to(dev)
    y = j[:, 0].contiguous()
    last = slice(rows - 100, rows)

    def work(s):
        loss, dz = sdfoam_amd.distill_loss_and_grad(z[s], j[s], t[s], 1.0, w[s], "none", up[s])
        leaf = z[s].detach().requires_grad_()
        a = sdfoam_amd.label_log_probs(leaf, y[s], 3)
        back, = torch.autograd.grad((a.log_prob, a.entropy), leaf, (up[s], w[s]))
        other = z[s].detach().requires_grad_()
        sdfoam_amd.distill_loss(other, j[s], t[s], 1.0, w[s], "none").backward(up[s])
        return [loss, dz, a.log_prob, a.entropy, a.top_log_probs, a.top_labels, back, other.grad]

    for x, alone in zip(work(slice(0, rows)), work(last)):
        assert torch.equal(x[last], alone)


def test_distill_few_long_rows_after_a_full_launch(dev):
    """77 rows more than one launch takes, of a length at which 77 rows by themselves are cut
    into slices: the call's scratch holds none.  One row's logits, expanded, so that they
    take no memory; an entry a row, of share 1: its loss is -log p of its label."""
    rows, labels = (1 << 22) + 77, 8200
    say("distill, few long rows after a full launch")
    z, g = logits_case(1, labels, torch.bfloat16)
    j = torch.randint(labels, (rows, 1), generator=g)
    log_p, _, err = softmax64(z, 1.0)
    loss = -log_p[0][j[:, 0]]
    tol = 4 * (err + 17 * U) * (2 + loss.abs())
    zd, jd = z.to(dev).expand(rows, labels), j.to(dev)
    t = torch.zeros((rows, 1), device=dev)
    near(sdfoam_amd.distill_loss(zd, jd, t, reduction="none"), loss, tol)
    for reduction, scale in (("sum", 1.0), ("mean", 1.0 / rows)):
        got = sdfoam_amd.distill_loss(zd, jd, t, reduction=reduction)
        near(got, loss.sum() * scale, (tol.sum() + 2 * U * loss.abs().sum()) * scale)


def test_tangents_that_reach_a_backward(dev):
    """Inputs without a tangent, gradients with one: refused, not lost."""
    from torch.autograd import forward_ad

    j = torch.zeros((3, 2), dtype=torch.int64, device=dev)
    y = j[:, 0].contiguous()
    calls = [lambda x: sdfoam_amd.cell_rows(x, y),
             lambda x: sdfoam_amd.distill_loss(x, j, j.float(), reduction="none"),
             lambda x: sdfoam_amd.label_log_probs(x, y).log_prob,
             lambda x: sdfoam_amd.label_log_probs(x, y).entropy]
    for call in calls:
        x = torch.randn((3, 7), device=dev).requires_grad_()
        out = call(x)
        with forward_ad.dual_level():
            one = torch.ones_like(out)
            with pytest.raises(RuntimeError, match="has no forward-mode derivative for gradient"):
                out.backward(forward_ad.make_dual(one, one))
        call(x).backward(one)
        assert x.grad is not None


@pytest.mark.parametrize("labels", [40, 5003, 70_001])
def test_distill_far_temperatures(dev, labels):
    """Temperatures whose square fp32 does not hold, or barely: the loss is that of the
    formula where fp32 holds it."""
    say("distill, far temperatures", labels)
    z, g = logits_case(5, labels, torch.float32)
    ids = torch.randint(labels, (5, 6), generator=g)
    t = torch.randn((5, 6), generator=g)
    weight = torch.tensor([1.0, 0.5, 0.0, 2.0, 1.5])
    for temperature in (1e-36, 1e-30, 1e-20, 1e10, 1e18):
        loss, grad, lt, gt = distill_reference(z, ids, t, temperature, weight, "none")
        args = (z.to(dev), ids.to(dev), t.to(dev), temperature, weight.to(dev), "none")
        got, dz = sdfoam_amd.distill_loss_and_grad(*args)
        near(got, loss, lt)
        near(dz, grad, gt)
        near(sdfoam_amd.distill_loss(*args), loss, lt)
    # one label: no distance, at any temperature
    one = torch.zeros((3, 1), dtype=torch.int64, device=dev)
    for temperature in (1e-38, 1e20, 3e38):
        loss, dz = sdfoam_amd.distill_loss_and_grad(one + 2.5, one, one.float(), temperature)
        assert float(loss) == 0 and not dz.any()


@pytest.mark.parametrize("top", [341, 342, 682, 683, 1024])
def test_distill_more_entries_than_labels(dev, top):
    """Short rows whose teacher's entries fill LDS: labels named often, entries that name
    none, and rows that end inside a block."""
    say("distill, more entries than labels", top)
    for dtype, sizes in ((torch.float32, (1, 5, 31, 32, 33, 100)), (torch.bfloat16, (64, 120))):
        for labels in sizes:
            for rows in (1, 77):
                z, g = logits_case(rows, labels, dtype, seed=top)
                ids, t = teacher_case(rows, labels, top, g)
                loss, grad, lt, gt = distill_reference(z, ids, t, 1.5, None, "none")
                zd = z.to(dev).requires_grad_()
                args = (ids.to(dev), t.to(dev), 1.5, None, "none")
                got, dz = sdfoam_amd.distill_loss_and_grad(zd.detach(), *args)
                near(got, loss, lt)
                # (a sum of up to `top` shares: as above)
                near(dz, grad, gt * (1 + top / 64), dtype)
                sdfoam_amd.distill_loss(zd, *args).backward(torch.ones(rows, device=dev))
                near(zd.grad, grad, gt * (1 + top / 64), dtype)


# ---- streams and graphs ----------------------------------------------------------------------


def test_another_stream(dev):
    """Inputs made, used and freed on a stream that is not the default one."""
    g = torch.Generator().manual_seed(11)
    z, table = torch.randn((64, 9001), generator=g), torch.randn((500, 32), generator=g)
    ids = torch.randint(500, (3000,), generator=g)
    j, t = torch.randint(9001, (64, 8), generator=g), torch.randn((64, 8), generator=g)

    def work():
        zd, td, jd, tt = z.to(dev), table.to(dev), j.to(dev), t.to(dev)
        rows = sdfoam_amd.cell_rows(td, ids.to(dev))
        tg, _ = sdfoam_amd.cell_rows_backward(rows, ids.to(dev), 500)
        loss, dz = sdfoam_amd.distill_loss_and_grad(zd, jd, tt)
        a = sdfoam_amd.label_log_probs(zd, jd[:, 0].contiguous(), 3)
        return [rows, tg, loss, dz, a.log_prob, a.entropy, a.top_log_probs, a.top_labels]

    ref = work()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        outs = [work() for _ in range(3)]
    side.synchronize()
    for out in outs:
        for x, y in zip(out, ref):
            assert torch.equal(x, y)


def test_graph_replays(dev):
    """Captured once, replayed on new inputs, with eager work between the replays."""
    g = torch.Generator().manual_seed(12)
    z, table = torch.empty((37, 5003), device=dev), torch.empty((700, 24), device=dev)
    ids = torch.empty(9000, dtype=torch.int64, device=dev)
    j, t = torch.empty((37, 8), dtype=torch.int64, device=dev), torch.empty((37, 8), device=dev)

    def fill():
        z.copy_(torch.randn(z.shape, generator=g))
        table.copy_(torch.randn(table.shape, generator=g))
        ids.copy_(torch.randint(-1, 700, ids.shape, generator=g))
        j.copy_(torch.randint(5003, j.shape, generator=g))
        t.copy_(torch.randn(t.shape, generator=g))

    def work():
        rows = sdfoam_amd.cell_rows(table, ids)
        tg, _ = sdfoam_amd.cell_rows_backward(rows, ids, 700)
        loss, dz = sdfoam_amd.distill_loss_and_grad(z, j, t)
        a = sdfoam_amd.label_log_probs(z, j[:, 0].contiguous(), 3)
        return [rows, tg, loss, dz, a.log_prob, a.entropy, a.top_log_probs, a.top_labels]

    fill()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for _ in range(4):
        fill()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for x, y in zip(got, work()):
            assert torch.equal(x, y)

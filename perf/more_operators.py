"""The operators of a label field's head beyond one linear layer, as a program that trains
and serves one calls them.

* spread / back: ``expert_order`` and ``expert_rows`` put rows in the order of the experts
  that a router chose for them, ``expert_combine`` and ``expert_combine_backward`` bring the
  experts' rows back, weighted, and form the gradients;
* product / product_grad: ``expert_linear`` and ``expert_linear_backward``, each expert's
  product with its own rows, and the gradients of rows and weights;
* adapt / adapt_grad: ``adapter_linear`` and ``adapter_linear_backward``, a shared projection
  with a low-rank adapter of each row's own beside it (a camera's, a teacher's, a
  request's), and the gradients of rows and adapters under a frozen projection;
* clip: ``clip_gradients``, the norm of all gradients of a step and the gradients scaled
  to at most a given one, into the optimizer's float32 copies.

``run`` computes each in elementary operations in 32 bits where ``own`` is false, and
through this package where it is true.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2}


def _experts(name, kind, rows, choices, experts, width, dtype):
    return {"name": name, "kind": kind, "rows": rows, "choices": choices, "experts": experts,
            "width": width, "dtype": dtype}


def _product(name, kind, rows, choices, experts, width, out, dtype):
    return {"name": name, "kind": kind, "rows": rows, "choices": choices, "experts": experts,
            "width": width, "out": out, "dtype": dtype}


def _adapt(name, kind, rows, adapters, rank, width, out, spread, dtype):
    return {"name": name, "kind": kind, "rows": rows, "adapters": adapters, "rank": rank,
            "width": width, "out": out, "spread": spread, "dtype": dtype}


def _clip(name, tensors, elements, dtype, scale):
    return {"name": name, "kind": "clip", "tensors": tensors, "elements": elements,
            "dtype": dtype, "scale": scale}


def listed():
    return [
        # one token of an answer and its four experts: the least a router's rows take
        _experts("spread_one", "spread", 1, 4, 64, 2048, "bfloat16"),
        # a step's rows, copied to eight of many experts each
        _experts("spread_step", "spread", 16_384, 8, 128, 1024, "bfloat16"),
        # a batch of 65,536 rays, two experts each, brought back with all gradients
        _experts("back_rays", "back", 65_536, 2, 16, 256, "float32"),
        # sixteen answers at once: few rows an expert, the experts' weights are what is read
        _product("product_serve", "product", 16, 4, 64, 1024, 2048, "bfloat16"),
        # every pixel of the 400x400 image, rows as wide as a cell's attributes at SH degree
        # 3, an expert for each part of the scene, a segmenter's labels
        _product("product_image", "product", 160_000, 1, 8, 49, 201, "float32"),
        # the gradients of a training step's experts
        _product("product_step", "product_grad", 16_384, 2, 16, 1024, 2048, "bfloat16"),
        # one row with its adapter: the shared weights are read once, latency counts
        _adapt("adapt_one", "adapt", 1, 256, 16, 4096, 4096, "random", "bfloat16"),
        # 64 requests, an adapter each, and a vocabulary of ordinary size
        _adapt("adapt_serve", "adapt", 64, 256, 16, 2048, 32_768, "random", "bfloat16"),
        # every pixel of the 400x400 image over 64 features, an adapter for each camera
        _adapt("adapt_image", "adapt", 160_000, 8, 4, 64, 512, "runs", "float16"),
        # the gradients of a step over twelve teachers' adapters, at odd sizes
        _adapt("adapt_step", "adapt_grad", 8_192, 12, 8, 1_000, 5_003, "random", "float16"),
        # the tensors of a small label field: rows of cells, a head, the foam itself
        _clip("clip_field", 5, 813_000, "float32", 1.0),
        # the many tensors of a large head, summed in 16 bits under a loss scale
        _clip("clip_many", 300, 500_000_000, "bfloat16", 2.0 ** -10),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _width(rng, lo, hi):
    """A width: most are multiples of 8 or 64, as layers' are, and some are odd."""
    n = _log(rng, lo, hi)
    step = rng.choice([1, 8, 8, 64])
    return n if n < step else min(n // step * step, hi)


def draw(rng):
    kind = rng.choice(["spread", "back", "product", "product", "product_grad", "adapt", "adapt",
                       "adapt_grad", "clip"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    if kind == "clip":
        case = _clip("", _log(rng, 1, 400), _log(rng, 1_000, 200_000_000), dtype,
                     rng.choice([1.0, 2.0 ** -10]))
    elif kind in ("spread", "back"):
        choices = rng.choice([1, 2, 4, 8])
        width = _width(rng, 8, 4096)
        rows = _log(rng, 1, min(200_000, 60_000_000 // (choices * width)))
        case = _experts("", kind, rows, choices, _log(rng, choices, 512), width, dtype)
    else:
        # operations of one product: fewer where the type's matrix units are slower
        most = 2e10 if dtype == "float32" else 1e11
        if kind in ("product", "product_grad"):
            choices = rng.choice([1, 2, 4])
            width, out = _width(rng, 16, 4096), _width(rng, 16, 4096)
            experts = _log(rng, choices, min(128, max(choices, 200_000_000 // (width * out))))
            most = int(min(most / (2 * width * out), 100_000_000 / max(width, out)) / choices)
            case = _product("", kind, _log(rng, 1, max(1, min(200_000, most))), choices, experts,
                            width, out, dtype)
        else:
            width, out = _width(rng, 16, 4096), _width(rng, 16, 32_768)
            rank = rng.choice([4, 5, 8, 16, 16, 32, 64])
            adapters = _log(rng, 1, min(512, max(1, 100_000_000 // (rank * max(width, out)))))
            most = int(min(most / (2 * width * out), 100_000_000 / max(width, out)))
            case = _adapt("", kind, _log(rng, 1, max(1, min(200_000, most))), adapters, rank,
                          width, out, rng.choice(["random", "runs"]), dtype)
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------


def _chosen(case, gen, dev):
    """The experts that a router chose: distinct in a row, some experts more often than
    others, and none in a row out of fifty (a ray that ends in no cell)."""
    rows, k, n = case["rows"], case["choices"], case["experts"]
    u = torch.rand((rows, 1), generator=gen, device=dev, dtype=torch.float64)
    first = (u ** 1.5 * n).long().clamp(max=n - 1)
    step = torch.randint(1, n // k + 1, (rows, 1), generator=gen, device=dev)
    ids = (first + step * torch.arange(k, device=dev)) % n
    none = torch.rand((rows, 1), generator=gen, device=dev) < 0.02
    none[0] = False
    return torch.where(none, -1, ids)


def _adapters_of(case, gen, dev):
    """The rows' adapters: of requests in no order, or in runs (the pixels of a camera, the
    tokens of a prompt); one row in fifty has none."""
    rows, n = case["rows"], case["adapters"]
    if case["spread"] == "runs":
        at = torch.arange(rows, device=dev) * n // rows
        ids = torch.randperm(n, generator=gen, device=dev)[at]
    else:
        ids = torch.randint(n, (rows,), generator=gen, device=dev)
    none = torch.rand(rows, generator=gen, device=dev) < 0.02
    none[0] = False
    return torch.where(none, -1, ids)


def _tensor_sizes(case):
    """Matrices and vectors of a model with so many elements in all: sizes that fall by
    powers of a common factor, the last takes what is left."""
    n, total = case["tensors"], case["elements"]
    share = [0.97 ** k if k % 3 else 0.01 * 0.97 ** k for k in range(1, n)] + [1.0]
    sizes = [max(1, int((total - n) * f / sum(share))) for f in share]
    sizes[-1] += total - sum(sizes)
    return sizes


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    kind = case["kind"]
    s = {"case": dict(case)}

    def randn(*shape, scale=1.0, dtype=dtype):
        return torch.randn(shape, generator=gen, device=dev, dtype=dtype).mul_(scale)

    if kind == "clip":
        # the norm is several times the largest that is wanted, times the loss scale
        size = 8.0 / (math.sqrt(case["elements"]) * case["scale"])
        s["gradients"] = [randn(n, scale=size) for n in _tensor_sizes(case)]
        # the optimizer's float32 copies lie in one buffer, one behind the other
        s["flat"] = torch.empty(case["elements"], device=dev)
        s["out"] = list(s["flat"].split([g.numel() for g in s["gradients"]]))
        return s
    if kind in ("adapt", "adapt_grad"):
        width, out, rank, n = case["width"], case["out"], case["rank"], case["adapters"]
        s["adapters"] = _adapters_of(case, gen, dev)
        s["rows"] = randn(case["rows"], width)
        s["weight"] = randn(out, width, scale=width ** -0.5)
        s["down"] = randn(n, rank, width, scale=width ** -0.5)
        s["up"] = randn(n, out, rank, scale=0.5 * rank ** -0.5)
        s["scale"] = 2.0
        if kind == "adapt_grad":
            s["grad"] = randn(case["rows"], out, scale=out ** -0.5)
        return s

    ids = _chosen(case, gen, dev)
    s["experts"] = ids
    rows, k, width = case["rows"], case["choices"], case["width"]
    if kind == "spread":
        s["rows"] = randn(rows, width)
        return s
    # what a program holds by then: its router's order, and the rows in it
    places, offsets = _plain_order(ids, case["experts"])
    s["places"], s["offsets"] = places, offsets
    if kind == "back":
        gate = torch.softmax(randn(rows, k, dtype=torch.float32), 1)
        s["weight"] = gate
        s["sorted"] = randn(rows * k, width)
        s["grad"] = randn(rows, width)
        return s
    s["sorted"] = randn(rows * k, width)
    s["weight"] = randn(case["experts"], case["out"], width, scale=width ** -0.5)
    if kind == "product_grad":
        s["grad"] = randn(rows * k, case["out"], scale=case["out"] ** -0.5)
    return s


# ---- the plain form ---------------------------------------------------------------------


def _plain_order(ids, groups):
    """Where each entry stands once all are in their groups' order, those of one group as
    they came (an entry of no group behind all others, as -1 - place), and where each group
    begins."""
    flat = ids.reshape(-1)
    named = (flat >= 0) & (flat < groups)
    key, order = torch.sort(torch.where(named, flat, groups), stable=True)
    at = torch.arange(flat.numel(), device=flat.device)
    places = torch.empty_like(at)
    places[order] = at
    places = torch.where(named, places, -1 - places)
    offsets = torch.searchsorted(key, torch.arange(groups + 1, device=flat.device))
    return places.to(torch.int32).reshape(ids.shape), offsets.to(torch.int32)


def _plain_spread(s):
    c = s["case"]
    places, offsets = _plain_order(s["experts"], c["experts"])
    rows = s["rows"]
    k, p = c["choices"], places.reshape(-1).long()
    out = torch.zeros((c["rows"] * k, c["width"]), dtype=rows.dtype, device=rows.device)
    source = torch.where((p >= 0)[:, None], rows.repeat_interleave(k, 0), 0)
    out[torch.where(p >= 0, p, -1 - p)] = source
    return [places, offsets, out]


def _plain_back(s):
    c = s["case"]
    p = s["places"].long()
    named = p >= 0
    at = torch.where(named, p, -1 - p)
    x, grad = s["sorted"].float(), s["grad"].float()
    w = torch.where(named, s["weight"], 0.0)
    out = torch.zeros_like(grad)
    rows_grad = torch.empty_like(x)
    weight_grad = torch.empty_like(w)
    for k in range(c["choices"]):
        y = x[at[:, k]]
        out += w[:, k, None] * y
        rows_grad[at[:, k]] = w[:, k, None] * grad
        weight_grad[:, k] = torch.where(named[:, k], (y * grad).sum(1), 0.0)
    dtype = s["sorted"].dtype
    return [out.to(dtype), rows_grad.to(dtype), weight_grad]


def _parts(offsets):
    """(group, first row, row behind the last) of the groups that have rows."""
    o = offsets.tolist()
    return [(g, o[g], o[g + 1]) for g in range(len(o) - 1) if o[g + 1] > o[g]]


def _plain_product(s):
    c = s["case"]
    x, weight = s["sorted"], s["weight"]
    parts = _parts(s["offsets"])
    if c["kind"] == "product":
        out = torch.zeros((x.shape[0], c["out"]), dtype=x.dtype, device=x.device)
        for g, a, b in parts:
            out[a:b] = (x[a:b].float() @ weight[g].float().t()).to(x.dtype)
        return out
    grad = s["grad"]
    rows_grad, weight_grad = torch.zeros_like(x), torch.zeros_like(weight)
    for g, a, b in parts:
        d = grad[a:b].float()
        rows_grad[a:b] = (d @ weight[g].float()).to(x.dtype)
        weight_grad[g] = (d.t() @ x[a:b].float()).to(x.dtype)
    return [rows_grad, weight_grad]


def _plain_adapt(s):
    c = s["case"]
    x, weight, down, up, scale = s["rows"], s["weight"], s["down"], s["up"], s["scale"]
    key, order = torch.sort(torch.where(s["adapters"] < 0, c["adapters"], s["adapters"]),
                            stable=True)
    parts = _parts(torch.searchsorted(key, torch.arange(c["adapters"] + 1, device=x.device)))
    x32, w32 = x.float(), weight.float()
    if c["kind"] == "adapt":
        out = x32 @ w32.t()
        for a, lo, hi in parts:
            i = order[lo:hi]
            out[i] += scale * ((x32[i] @ down[a].float().t()) @ up[a].float().t())
        return out.to(x.dtype)
    grad = s["grad"].float()
    rows_grad = grad @ w32
    down_grad, up_grad = torch.zeros_like(down), torch.zeros_like(up)
    for a, lo, hi in parts:
        i = order[lo:hi]
        xi, gi = x32[i], scale * grad[i]
        inner = gi @ up[a].float()
        rows_grad[i] += inner @ down[a].float()
        down_grad[a] = (inner.t() @ xi).to(x.dtype)
        up_grad[a] = (gi.t() @ (xi @ down[a].float().t())).to(x.dtype)
    return [rows_grad.to(x.dtype), down_grad, up_grad]


MAX_NORM = 1.0


def _plain_clip(s):
    scale = s["case"]["scale"]
    squares = [g.double().pow(2).sum() for g in s["gradients"]]
    norm = torch.stack(squares).sum().sqrt().mul(scale).float()
    factor = scale * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
    for g, o in zip(s["gradients"], s["out"]):
        torch.mul(g.float(), factor, out=o)
    return [norm, s["flat"]]


# ---- this package -----------------------------------------------------------------------


def _own(s):
    import sdfoam_amd

    c = s["case"]
    kind = c["kind"]
    if kind == "spread":
        order = sdfoam_amd.expert_order(s["experts"], c["experts"])
        return [order.places, order.offsets, sdfoam_amd.expert_rows(s["rows"], order)]
    if kind == "back":
        order = sdfoam_amd.ExpertOrder(s["places"], s["offsets"])
        out = sdfoam_amd.expert_combine(s["sorted"], order, s["weight"])
        return [out, *sdfoam_amd.expert_combine_backward(s["grad"], s["sorted"], order,
                                                         s["weight"])]
    if kind == "product":
        return sdfoam_amd.expert_linear(s["sorted"], s["weight"], s["offsets"])
    if kind == "product_grad":
        return list(sdfoam_amd.expert_linear_backward(s["grad"], s["sorted"], s["weight"],
                                                      s["offsets"]))
    if kind == "adapt":
        return sdfoam_amd.adapter_linear(s["rows"], s["weight"], s["adapters"], s["down"],
                                         s["up"], s["scale"])
    if kind == "adapt_grad":
        rows_grad, _, down_grad, up_grad = sdfoam_amd.adapter_linear_backward(
            s["grad"], s["rows"], s["weight"], s["adapters"], s["down"], s["up"], s["scale"],
            need_weight=False)
        return [rows_grad, down_grad, up_grad]
    norm = sdfoam_amd.clip_gradients(s["gradients"], MAX_NORM, scale=c["scale"], out=s["out"])
    return [norm, s["flat"]]


def run(s):
    if own:
        return _own(s)
    return {"spread": _plain_spread, "back": _plain_back, "product": _plain_product,
            "product_grad": _plain_product, "adapt": _plain_adapt, "adapt_grad": _plain_adapt,
            "clip": _plain_clip}[s["case"]["kind"]](s)


# ---- what a pass cannot do without --------------------------------------------------------


def _met(groups, entries):
    """How many of the groups so many entries meet, at most on average."""
    return groups * -math.expm1(entries * math.log1p(-1.0 / groups)) if groups > 1 else 1


def work(case):
    kind, e = case["kind"], SIZES[case["dtype"]]
    if kind == "clip":
        return {"bytes": case["elements"] * (e + 4), "flops": 3 * case["elements"]}
    n, width = case["rows"], case["width"]
    if kind == "spread":
        entries = n * case["choices"]
        return {"bytes": entries * (8 + 4 + width * e) + n * width * e + 4 * case["experts"],
                "flops": entries}
    if kind == "back":
        entries = n * case["choices"]
        return {"bytes": 2 * (entries + n) * width * e + 12 * entries,
                "flops": 5 * entries * width}
    out = case["out"]
    if kind in ("product", "product_grad"):
        entries = n * case["choices"]
        # experts that have rows: few rows name few
        used = max(_met(case["experts"], entries), case["choices"])
        weights = used * width * out * e
        if kind == "product":
            return {"bytes": entries * (width + out) * e + weights,
                    "flops": 2 * entries * width * out}
        return {"bytes": entries * (2 * width + out) * e + weights
                + case["experts"] * width * out * e,
                "flops": 4 * entries * width * out}
    used, rank = case["adapters"], case["rank"]
    if case["spread"] == "random":
        used = _met(used, n)
    used = min(used, n)
    adapters = used * rank * (width + out) * e
    if kind == "adapt":
        return {"bytes": n * ((width + out) * e + 8) + width * out * e + adapters,
                "flops": 2 * n * (width * out + rank * (width + out))}
    return {"bytes": n * ((2 * width + out) * e + 8) + width * out * e + adapters
            + case["adapters"] * rank * (width + out) * e,
            "flops": 2 * n * (width * out + 3 * rank * (width + out))}


# ---- the definition in 64 bits ------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "clip":
        total = sum(float((g.double() * g.double()).sum()) for g in s["gradients"])
        norm = case["scale"] * math.sqrt(total)
        factor = case["scale"] * min(1.0, MAX_NORM / (norm + 1e-6))
        return [torch.tensor(norm, dtype=torch.float64, device="cuda"),
                torch.cat([g.double() for g in s["gradients"]]) * factor]
    if kind in ("adapt", "adapt_grad"):
        ids = s["adapters"]
        x, w, down, up = (s[k].double() for k in ("rows", "weight", "down", "up"))
        scale = s["scale"]
        if kind == "adapt":
            out = torch.matmul(x, w.t())
        else:
            g = s["grad"].double()
            rows_grad = torch.matmul(g, w)
            down_grad, up_grad = torch.zeros_like(down), torch.zeros_like(up)
        for a in range(case["adapters"]):
            i = torch.nonzero(ids == a)[:, 0]
            if i.numel() == 0:
                continue
            inner = torch.matmul(x[i], down[a].t())
            if kind == "adapt":
                out[i] += scale * torch.matmul(inner, up[a].t())
                continue
            back = scale * torch.matmul(g[i], up[a])
            rows_grad[i] += torch.matmul(back, down[a])
            down_grad[a] = torch.matmul(back.t(), x[i])
            up_grad[a] = scale * torch.matmul(g[i].t(), inner)
        return out if kind == "adapt" else [rows_grad, down_grad, up_grad]

    ids = s["experts"].reshape(-1)
    groups, k = case["experts"], case["choices"]
    if kind == "spread":
        out = torch.zeros((ids.numel(), case["width"]), dtype=torch.float64, device=ids.device)
        first = 0
        for g in range(groups):
            i = torch.nonzero(ids == g)[:, 0]
            out[first:first + i.numel()] = s["rows"].double()[i // k]
            first += i.numel()
        return [None, None, out]
    if kind == "back":
        x, g, w = s["sorted"].double(), s["grad"].double(), s["weight"].double()
        p = s["places"].long().reshape(-1)
        live = torch.nonzero(p >= 0)[:, 0]
        row = live // k
        out = torch.zeros_like(g).index_add_(0, row, w.reshape(-1)[live, None] * x[p[live]])
        rows_grad, weight_grad = torch.zeros_like(x), torch.zeros_like(w)
        rows_grad[p[live]] = w.reshape(-1)[live, None] * g[row]
        weight_grad.view(-1)[live] = (x[p[live]] * g[row]).sum(1)
        return [out, rows_grad, weight_grad]
    x, offsets = s["sorted"].double(), s["offsets"].tolist()
    if kind == "product":
        out = torch.zeros((x.shape[0], case["out"]), dtype=torch.float64, device=x.device)
    else:
        d = s["grad"].double()
        rows_grad = torch.zeros_like(x)
        weight_grad = torch.zeros(s["weight"].shape, dtype=torch.float64, device=x.device)
    for g in range(groups):
        part = slice(offsets[g], offsets[g + 1])
        if offsets[g + 1] == offsets[g]:
            continue
        w = s["weight"][g].double()
        if kind == "product":
            out[part] = torch.matmul(x[part], w.t())
        else:
            rows_grad[part] = torch.matmul(d[part], w)
            weight_grad[g] = torch.matmul(d[part].t(), x[part])
    return out if kind == "product" else [rows_grad, weight_grad]

"""The operators of a label field, as a program that trains one and asks it calls them.

A label field is a foam whose cells carry a learned row each.  A trace says in which cell
a ray ends (``depth_indices``), a head makes logits over labels of that cell's row, and

* rows / rows_grad: ``cell_rows``, the rows of the rays' cells, scaled (and weighted by the
  ray's opacity), and ``cell_rows_backward``, the gradients of the table and the weights.
  With tokens for cells it is an embedding and its gradient;
* distill / distill_value: ``distill_loss_and_grad`` and ``distill_loss``, the distance
  from a teacher's best few logits per row, with the gradient of the logits or without;
* answer: ``label_log_probs``, the log probability of a given label per row, the entropy
  and the best labels;
* score: the same with the gradient of log probability and entropy, as a policy's loss
  asks for it.

``run`` computes each in elementary operations in 32 bits where ``own`` is false, and
through this package where it is true.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2}
ID_SIZES = {"uint32": 4, "int64": 8}


def _rows(name, kind, cells, count, width, dtype, ids, spread, weighted, scale):
    return {"name": name, "kind": kind, "cells": cells, "count": count, "width": width,
            "dtype": dtype, "ids": ids, "spread": spread, "weighted": weighted, "scale": scale}


def _distill(name, kind, rows, labels, top, dtype, temperature, weighted):
    return {"name": name, "kind": kind, "rows": rows, "labels": labels, "top": top,
            "dtype": dtype, "temperature": temperature, "weighted": weighted}


def _answer(name, kind, rows, labels, top, dtype, temperature):
    return {"name": name, "kind": kind, "rows": rows, "labels": labels, "top": top,
            "dtype": dtype, "temperature": temperature}


def listed():
    return [
        # three tokens of a prompt's end: the least work a lookup has, where latency counts
        _rows("rows_three", "rows", 100_003, 3, 1024, "bfloat16", "int64", "uniform", False, 32.0),
        # every ray of the 1600x1200 image over one million cells, rows as wide as a cell's
        # attributes at SH degree 3, weighted by opacity
        _rows("rows_image", "rows", 1_000_000, 1_920_000, 49, "float32", "uint32", "image",
              True, 1.0),
        # the gradient of a training batch's 2^20 rays, rows of 64 features
        _rows("rows_grad_rays", "rows_grad", 1_000_000, 1 << 20, 64, "bfloat16", "uint32",
              "rays", True, 1.0),
        # the gradient of a text batch's embedding, tokens as frequent as words are
        _rows("rows_grad_tokens", "rows_grad", 65_536, 16_381, 2048, "float16", "int64",
              "tokens", False, math.sqrt(2048.0)),
        # a step over the 64x64 rays of the smallest image and a segmenter's few labels
        _distill("distill_small", "distill", 4_096, 201, 8, "float32", 1.0, False),
        # a step over 4,096 tokens or rays and a vocabulary of ordinary size, some rows masked
        _distill("distill_step", "distill", 4_096, 32_768, 64, "bfloat16", 2.0, True),
        # the widest vocabulary, of an odd size: no two rows start at the same alignment
        _distill("distill_wide", "distill", 2_048, 262_147, 128, "bfloat16", 1.5, True),
        # the validation loss of many rows, without a gradient
        _distill("distill_value", "distill_value", 8_192, 50_021, 32, "float16", 1.0, False),
        # one token's answer while serving
        _answer("answer_one", "answer", 1, 131_072, 20, "bfloat16", 1.0),
        # every pixel of the 400x400 image, a segmenter's labels
        _answer("answer_image", "answer", 160_000, 121, 5, "float16", 1.0),
        # the scores of a long text
        _answer("answer_text", "answer", 8_192, 100_003, 8, "bfloat16", 0.7),
        # log probability and entropy with their gradient
        _answer("score_step", "score", 2_048, 50_021, 0, "float32", 1.0),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "rows_grad", "rows_grad", "distill", "distill", "distill_value",
                       "answer", "answer", "score"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if kind in ("rows", "rows_grad"):
        count = _log(rng, 1, 2_000_000)
        cells = _log(rng, 4_000, 2_000_000)
        most = 100_000_000 // max(count, cells if kind == "rows_grad" else cells // 4)
        width = _log(rng, 1, max(1, min(4096, most)))
        case = _rows("", kind, cells, count, width, dtype, rng.choice(["uint32", "int64"]),
                     rng.choice(["uniform", "image", "rays", "tokens"]), rng.random() < 0.5,
                     rng.choice([1.0, 1.0, math.sqrt(width)]))
    else:
        labels = _log(rng, 20, 262_144)
        rows = _log(rng, 1, max(1, min(200_000, 250_000_000 // labels)))
        temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
        if kind in ("distill", "distill_value"):
            top = min(labels // 2, _log(rng, 1, 128))
            case = _distill("", kind, rows, labels, top, dtype, temperature, rng.random() < 0.5)
        else:
            top = 0 if kind == "score" else min(labels // 2, rng.choice([0, 1, 5, 8, 20, 50]))
            case = _answer("", kind, rows, labels, top, dtype, temperature)
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------


def _cells_of(case, gen, dev):
    """Ids as they are met: pixels of one cell beside each other ("image"), rays of many
    cameras that end in some cells more often than in others ("rays"), words ("tokens")."""
    n, cells = case["count"], case["cells"]
    u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
    if case["spread"] == "uniform":
        k = (u * cells).long()
    elif case["spread"] == "image":
        at = torch.arange(n, device=dev)
        at = at % 1600 // 3 + at // 1600 // 3 * 534  # 3x3 pixels of a 1600 wide image
        k = at + (torch.rand(1, generator=gen, device=dev, dtype=torch.float64) * cells).long()
    elif case["spread"] == "rays":
        k = (u.pow(3) * 0.3 * cells).long()
    else:
        k = (torch.exp(u * math.log(cells)) - 1).long()
    ids = (k % cells) * 2654435761 % cells
    if case["ids"] == "uint32":  # rays that end in no cell
        none = torch.rand(n, generator=gen, device=dev) < 0.03
        return torch.where(none, -1, ids).to(torch.int32).view(torch.uint32)
    return ids


def _teacher(case, gen, dev):
    """Ids and logits of the teacher's best labels: distinct in a row, the best first; one
    row in sixteen has only half of them and one in a hundred none."""
    rows, labels, top = case["rows"], case["labels"], case["top"]
    k = torch.arange(top, device=dev)
    first = torch.randint(labels, (rows, 1), generator=gen, device=dev)
    step = torch.randint(1, labels // top + 1, (rows, 1), generator=gen, device=dev)
    ids = (first + k * step) % labels
    t = 8.0 - 1.5 * torch.log1p(k) + 0.5 * torch.randn((rows, top), generator=gen, device=dev)
    u = torch.rand((rows, 1), generator=gen, device=dev)
    ids = torch.where((u < 0.0625) & (k >= (top + 1) // 2), -1, ids)
    ids = torch.where(u < 0.01, -1, ids)
    return ids, t


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    s = {"case": dict(case)}

    def randn(*shape, dtype=dtype):
        return torch.randn(shape, generator=gen, device=dev, dtype=dtype)

    if case["kind"] in ("rows", "rows_grad"):
        s["cells"] = _cells_of(case, gen, dev)
        if case["kind"] == "rows" or case["weighted"]:
            s["table"] = randn(case["cells"], case["width"])
        if case["weighted"]:
            s["weight"] = torch.rand(case["count"], generator=gen, device=dev)
        if case["kind"] == "rows_grad":
            s["grad"] = randn(case["count"], case["width"])
        return s

    rows, labels = case["rows"], case["labels"]
    logits = randn(rows, labels).mul_(2.5)
    at = torch.arange(rows, device=dev)
    if case["kind"] in ("distill", "distill_value"):
        ids, t = _teacher(case, gen, dev)
        logits[at, ids.clamp(min=0)[:, 0]] += 6.0  # a student that has begun to learn
        s["teacher_labels"], s["teacher_logits"] = ids, t.to(dtype)
        if case["weighted"]:  # a third of the rows are prompt or padding
            u = torch.rand(rows, generator=gen, device=dev)
            s["row_weight"] = torch.where(u < 0.33, 0.0, 1.0 + u)
    else:
        y = torch.randint(labels, (rows,), generator=gen, device=dev)
        logits[at, y] += 6.0
        none = torch.rand(rows, generator=gen, device=dev) < 0.03
        s["labels"] = torch.where(none & (at > 0), -1, y)
        if case["kind"] == "score":
            s["log_prob_grad"] = randn(rows, dtype=torch.float32)
            s["entropy_grad"] = 0.01 * randn(rows, dtype=torch.float32)
    s["logits"] = logits
    return s


# ---- the plain form ---------------------------------------------------------------------


def _plain_ids(cells):
    """Ids as int64, and which of them name a cell (all others are -1 here)."""
    ids = cells.view(torch.int32).long() if cells.dtype == torch.uint32 else cells
    return ids, ids >= 0


def _plain_rows(s):
    c = s["case"]
    ids, named = _plain_ids(s["cells"])
    factor = torch.where(named, c["scale"], 0.0)
    if c["weighted"]:
        factor = factor * s["weight"]
    ids = ids.clamp(min=0)
    if c["kind"] == "rows":
        return (s["table"][ids].float() * factor[:, None]).to(s["table"].dtype)
    grad = s["grad"].float()
    sums = torch.zeros((c["cells"], c["width"]), dtype=torch.float32, device=grad.device)
    sums.index_add_(0, ids, grad * factor[:, None])
    out = [sums.to(s["grad"].dtype)]
    if c["weighted"]:
        dot = (s["table"][ids].float() * grad).sum(1)
        out.append(torch.where(named, c["scale"], 0.0) * dot)
    return out


def _plain_lse(x):
    m = x.amax(1, keepdim=True)
    return m + (x - m).exp().sum(1, keepdim=True).log()


def _plain_distill(s):
    c = s["case"]
    temperature = c["temperature"]
    x = s["logits"].float() / temperature
    ids = s["teacher_labels"]
    valid = ids >= 0
    t = torch.where(valid, s["teacher_logits"].float() / temperature, -math.inf)
    any_valid = valid.any(1, keepdim=True)
    t = torch.where(any_valid, t, 0.0)
    tlse = _plain_lse(t)
    weight = any_valid.float()
    if c["weighted"]:
        weight = weight * s["row_weight"][:, None]
    q = torch.where(valid, (t - tlse).exp(), 0.0)
    at = ids.clamp(min=0)
    lse = _plain_lse(x)
    log_p = x.gather(1, at) - lse
    terms = torch.where(valid, q * (t - tlse - log_p), 0.0)
    loss = weight[:, 0] * temperature ** 2 * terms.sum(1)
    if c["kind"] == "distill_value":
        return loss
    grad = (x - lse).exp()
    grad.scatter_add_(1, at, -q)
    grad *= weight * (temperature / c["rows"])
    return [loss.sum() / c["rows"], grad.to(s["logits"].dtype)]


def _plain_answer(s):
    c = s["case"]
    z = s["logits"].float()
    x = z / c["temperature"]
    log_p = x - _plain_lse(x)
    y = s["labels"]
    at = y.clamp(min=0)[:, None]
    lp = torch.where(y >= 0, log_p.gather(1, at)[:, 0], 0.0)
    p = log_p.exp()
    entropy = -(p * log_p).sum(1)
    out = [lp, entropy]
    if c["kind"] == "score":
        g = s["log_prob_grad"] * (y >= 0)
        grad = -p * (g[:, None] + s["entropy_grad"][:, None] * (log_p + entropy[:, None]))
        grad.scatter_add_(1, at, g[:, None])
        return out + [(grad / c["temperature"]).to(s["logits"].dtype)]
    if c["top"]:
        # whole keys: the logit's order above, the index from the end below
        bits = z.view(torch.int32).long()
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        key = bits * (1 << 32) + ((1 << 32) - 1 - torch.arange(z.shape[1], device=z.device))
        best = (1 << 32) - 1 - (key.topk(c["top"], 1).values & ((1 << 32) - 1))
        out += [log_p.gather(1, best), best]
    return out


# ---- this package -----------------------------------------------------------------------


def _own(s):
    import sdfoam_amd

    c = s["case"]
    kind = c["kind"]
    if kind == "rows":
        return sdfoam_amd.cell_rows(s["table"], s["cells"], s.get("weight"), c["scale"])
    if kind == "rows_grad":
        table_grad, weight_grad = sdfoam_amd.cell_rows_backward(
            s["grad"], s["cells"], c["cells"], s.get("weight"), c["scale"], table=s.get("table"))
        return [table_grad, weight_grad] if c["weighted"] else [table_grad]
    if kind == "distill_value":
        return sdfoam_amd.distill_loss(s["logits"], s["teacher_labels"], s["teacher_logits"],
                                       c["temperature"], s.get("row_weight"), reduction="none")
    if kind == "distill":
        return list(sdfoam_amd.distill_loss_and_grad(
            s["logits"], s["teacher_labels"], s["teacher_logits"], c["temperature"],
            s.get("row_weight"), reduction="mean"))
    if kind == "answer":
        a = sdfoam_amd.label_log_probs(s["logits"], s["labels"], c["top"], c["temperature"])
        out = [a.log_prob, a.entropy]
        return out + [a.top_log_probs, a.top_labels] if c["top"] else out
    logits = s["logits"].detach().requires_grad_()
    a = sdfoam_amd.label_log_probs(logits, s["labels"], 0, c["temperature"])
    grad, = torch.autograd.grad((a.log_prob, a.entropy), logits,
                                (s["log_prob_grad"], s["entropy_grad"]))
    return [a.log_prob.detach(), a.entropy.detach(), grad]


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind in ("rows", "rows_grad"):
        return _plain_rows(s)
    if kind in ("distill", "distill_value"):
        return _plain_distill(s)
    return _plain_answer(s)


# ---- what a pass cannot do without --------------------------------------------------------


def work(case):
    if case["kind"] in ("rows", "rows_grad"):
        n, width, cells, e = case["count"], case["width"], case["cells"], SIZES[case["dtype"]]
        u = ID_SIZES[case["ids"]] + (4 if case["weighted"] else 0)
        # rows that are read, each once: no more than there are, nor than are asked for
        used = min(n, cells)
        if case["spread"] == "image":
            used = min(used, n // 9 + 1)
        elif case["spread"] == "rays":
            used = min(used, int(0.3 * cells) + 1)
        if case["kind"] == "rows":
            return {"bytes": n * (u + width * e) + used * width * e, "flops": n * width}
        if case["weighted"]:
            return {"bytes": n * (u + 4 + width * e) + (used + cells) * width * e,
                    "flops": 4 * n * width}
        return {"bytes": n * (u + width * e) + cells * width * e, "flops": 2 * n * width}
    rows, labels, e = case["rows"], case["labels"], SIZES[case["dtype"]]
    if case["kind"] in ("distill", "distill_value"):
        # a row of weight 0 needs no reading; its gradient is written all the same
        read = rows * (0.67 if case["weighted"] else 1.0) * 0.99
        small = rows * (case["top"] * (8 + e) + 4)
        if case["kind"] == "distill":
            return {"bytes": (read + rows) * labels * e + small, "flops": 8 * read * labels}
        return {"bytes": read * labels * e + small, "flops": 4 * read * labels}
    small = rows * (16 + 12 * case["top"])
    if case["kind"] == "score":
        return {"bytes": 2 * rows * labels * e + small + 8 * rows, "flops": 14 * rows * labels}
    return {"bytes": rows * labels * e + small, "flops": 6 * rows * labels}


# ---- the definition in 64 bits ------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] in ("rows", "rows_grad"):
        ids = s["cells"]
        ids = ids.view(torch.int32).long() if ids.dtype == torch.uint32 else ids
        live = torch.nonzero(ids >= 0)[:, 0]
        weight = s["weight"].double() if c["weighted"] else torch.ones(
            c["count"], dtype=torch.float64, device=ids.device)
        table = s["table"].double() if "table" in s else None
        if c["kind"] == "rows":
            out = torch.zeros((c["count"], c["width"]), dtype=torch.float64, device=ids.device)
            out[live] = table[ids[live]] * weight[live, None] * c["scale"]
            return out
        grad = s["grad"].double()
        sums = torch.zeros((c["cells"], c["width"]), dtype=torch.float64, device=ids.device)
        sums.index_put_((ids[live],), grad[live] * (weight[live, None] * c["scale"]),
                        accumulate=True)
        if not c["weighted"]:
            return [sums]
        dw = torch.zeros(c["count"], dtype=torch.float64, device=ids.device)
        dw[live] = torch.einsum("nd,nd->n", table[ids[live]], grad[live]) * c["scale"]
        return [sums, dw]

    rows = c["rows"]
    z = s["logits"].double().requires_grad_(c["kind"] in ("distill", "score"))
    log_p = torch.log_softmax(z / c["temperature"], 1)
    if c["kind"] in ("distill", "distill_value"):
        ids = s["teacher_labels"]
        live = ids >= 0
        t = (s["teacher_logits"].double() / c["temperature"]).masked_fill(~live, -math.inf)
        q = torch.softmax(t, 1).nan_to_num(0.0)
        cross = -(q * log_p.gather(1, ids.clamp(min=0))).sum(1)
        loss = (torch.special.xlogy(q, q).sum(1) + cross) * c["temperature"] ** 2
        if c["weighted"]:
            loss = loss * s["row_weight"].double()
        if c["kind"] == "distill_value":
            return loss
        loss = loss.sum() / rows
        grad, = torch.autograd.grad(loss, z)
        return [loss.detach(), grad]
    y = s["labels"]
    lp = log_p.gather(1, y.clamp(min=0)[:, None])[:, 0] * (y >= 0)
    entropy = -(log_p.exp() * log_p).sum(1)
    if c["kind"] == "score":
        grad, = torch.autograd.grad((lp, entropy), z, (s["log_prob_grad"].double(),
                                                       s["entropy_grad"].double()))
        return [lp.detach(), entropy.detach(), grad]
    out = [lp, entropy]
    return out + [log_p.topk(c["top"], 1).values, None] if c["top"] else out

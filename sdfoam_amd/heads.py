"""Heads of label fields beyond one linear layer: experts, and adapters beside it.

Between a label field's rows (``cell_rows``) and its logits' loss (``distill_loss``) stands
a head.  Two kinds that one matrix does not make:

* a mixture of experts: a router names some experts per row.  ``expert_order`` finds the
  order of the rows by expert, ``expert_rows`` puts them in it, ``expert_linear`` multiplies
  each expert's rows by its own matrix, and ``expert_combine`` brings them back, weighted;
* a shared projection with low-rank adapters: ``adapter_linear`` adds to each row's product
  what the row's own adapter gives -- a camera's, a teacher's, a request's.

Each has its gradients through autograd, and as a call of its own (``*_backward``) for
training loops that call the backward themselves.  The reference has no counterpart.

The work runs in libsdfoam_hip.so on torch's current stream.  Rows and matrices are float32,
float16 or bfloat16, all of one type; every sum is held in float32 and rounded to that type
once.  Experts and adapters are uint32, int32 or int64; one that is negative, 0xffffffff or
too large names none.  Rows may be strided (a slice of padded rows is read in place), as the
shared projection's may; other layouts are copied.  Results are the same on every run: no
sum's order is left to chance.  Derivatives are reverse-mode and of the first order; tensors
with a forward-mode tangent are refused.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import ptr
from .labels import (_ID_TYPES, _TYPES, _call, _check_devices, _check_float32, _check_shape,
                     _element_type, _id_type, _no_tangent, _rows, _scratch, _wants_gradient)
from .pipeline import _c10

MAX_EXPERTS = 2048
MAX_ADAPTERS = 2048
MAX_RANK = 256  # of an adapter
MAX_WIDTH = 1 << 18  # elements of a row


class ExpertOrder(NamedTuple):
    """The order of rows by expert, as ``expert_order`` finds it.

    places (int32, the shape of the experts): the row of ``expert_rows`` that stands for
    each choice; -1 - row for a choice that names no expert.  offsets (int32
    [num_experts + 1]): expert g's rows are offsets[g] to offsets[g + 1]; those from
    offsets[num_experts] on, of choices that name none, are zeros."""

    places: torch.Tensor
    offsets: torch.Tensor


def _check_width(call: str, *widths: int) -> None:
    for width in widths:
        if width > MAX_WIDTH:
            raise RuntimeError(f"{call} takes rows of at most 2^18 elements")


def _check_entries(call: str, count: int) -> None:
    if count >= 1 << 31:
        raise RuntimeError(f"{call} takes fewer than 2^31 entries")


def _check_same_type(first: str, t: torch.Tensor, **others) -> None:
    for name, o in others.items():
        if o.dtype != t.dtype:
            raise RuntimeError(f"{name} had dtype {_c10(o.dtype)}, expected {_c10(t.dtype)} "
                               f"as {first}")


def _check_int32(name: str, t: torch.Tensor) -> None:
    if t.dtype != torch.int32:
        raise RuntimeError(f"{name} had dtype {_c10(t.dtype)}, expected int32")


def expert_order(experts: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The order of a router's choices by expert, those of one expert as they came.

    experts [..., K]: the K experts that each row goes to (more than once, if it is named
    more than once).  At most 2048 experts, fewer than 2^31 choices."""
    _id_type("experts", experts)
    if experts.dim() < 1:
        raise RuntimeError("experts must have at least 1 dimension")
    num_experts = int(num_experts)
    if not 0 <= num_experts <= MAX_EXPERTS:
        raise RuntimeError(f"num_experts must be from 0 to {MAX_EXPERTS}")
    _check_entries("expert_order", experts.numel())
    _check_devices("experts", experts)
    e = experts.contiguous()
    dev = experts.device
    places = torch.empty(experts.shape, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    L = _lib.lib()
    nbytes = L.sdf_expert_order_scratch_bytes(e.numel(), num_experts)
    keep, base = _scratch(nbytes, dev)
    _call(L.sdf_expert_order, e, _ID_TYPES[e.dtype], e.data_ptr(), e.numel(), num_experts,
          places.data_ptr(), offsets.data_ptr(), base, nbytes)
    return ExpertOrder(places, offsets)


def _places_of(call: str, order: ExpertOrder) -> torch.Tensor:
    places = order.places
    _check_int32("order.places", places)
    if places.dim() < 1:
        raise RuntimeError("order.places must have at least 1 dimension")
    _check_entries(call, places.numel())
    return places


# ---- rows by expert, and back ----------------------------------------------------------------


def _spread(rows, places):
    p = places.contiguous()
    x = _rows(rows)
    count, width, choices = x.size(0), x.size(1), p.size(-1)
    out = torch.empty((count * choices, width), dtype=rows.dtype, device=rows.device)
    _call(_lib.lib().sdf_expert_rows, x, _TYPES[x.dtype], x.data_ptr(), x.stride(0), count,
          choices, width, p.data_ptr(), out.data_ptr())
    return out


def _combine(rows, places, weight):
    p = places.contiguous()
    y = _rows(rows)
    w = None if weight is None else weight.contiguous()
    width, choices = y.size(1), p.size(-1)
    out = torch.empty((*places.shape[:-1], width), dtype=rows.dtype, device=rows.device)
    count = 1
    for k in places.shape[:-1]:
        count *= k
    _call(_lib.lib().sdf_expert_combine, y, _TYPES[y.dtype], y.data_ptr(), y.stride(0), count,
          choices, width, p.data_ptr(), ptr(w), out.data_ptr())
    return out


def _combine_backward(out_grad, rows, places, weight, need_rows, need_weight):
    p = places.contiguous()
    g = _rows(out_grad)
    y = _rows(rows) if need_weight else None
    w = None if weight is None else weight.contiguous()
    width, choices, dev = g.size(1), p.size(-1), out_grad.device
    rows_grad = weight_grad = None
    if need_rows:
        rows_grad = torch.empty((p.numel(), width), dtype=out_grad.dtype, device=dev)
    if need_weight:
        weight_grad = torch.empty(places.shape, dtype=torch.float32, device=dev)
    _call(_lib.lib().sdf_expert_combine_backward, g, _TYPES[g.dtype], g.data_ptr(), g.stride(0),
          ptr(y), 0 if y is None else y.stride(0), g.size(0), choices, width, p.data_ptr(),
          ptr(w), ptr(rows_grad), ptr(weight_grad))
    return rows_grad, weight_grad


class _ExpertRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, places):
        ctx.save_for_backward(places)
        return _spread(rows, places)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _no_tangent("expert_rows", gradient=grad)
        places, = ctx.saved_tensors
        return _combine(grad, places, None), None


class _ExpertCombine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, places, weight):
        # the rows are read again only for the weights' gradient
        ctx.save_for_backward(places, weight, rows if ctx.needs_input_grad[2] else None)
        return _combine(rows, places, weight)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _no_tangent("expert_combine", gradient=grad)
        places, weight, rows = ctx.saved_tensors
        rows_grad, weight_grad = _combine_backward(grad, rows, places, weight,
                                                   ctx.needs_input_grad[0], rows is not None)
        return rows_grad, None, weight_grad


def expert_rows(rows: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """``rows`` in the order of their experts: [P, D], P the number of choices, row
    ``order.places[i, k]`` a copy of row i; zeros for choices that name no expert.

    rows [..., D] where the experts were [..., K].  Differentiable in ``rows``; the gradient
    is ``expert_combine(grad, order)``."""
    _element_type("rows", rows)
    if rows.dim() < 1:
        raise RuntimeError("rows must have at least 1 dimension")
    places = _places_of("expert_rows", order)
    if places.shape[:-1] != rows.shape[:-1]:
        raise RuntimeError(f"rows had shape {list(rows.shape)}, expected "
                           f"{list(places.shape[:-1])} and a last dimension")
    _check_width("expert_rows", rows.size(-1))
    _no_tangent("expert_rows", rows=rows)
    _check_devices("rows", rows, "order.places", places)
    if _wants_gradient(rows):
        return _ExpertRows.apply(rows, places)
    return _spread(rows, places)


def _check_combine(call, rows, places, weight):
    _element_type("rows", rows)
    if rows.dim() != 2:
        raise RuntimeError("rows must have 2 dimensions")
    if rows.size(0) != places.numel():
        raise RuntimeError(f"rows had shape {list(rows.shape)}, expected {places.numel()} rows, "
                           "one for each of the order's places")
    _check_width(call, rows.size(1))
    if weight is not None:
        _check_float32("weight", weight, places.shape)


def expert_combine(rows: torch.Tensor, order: ExpertOrder,
                   weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows in their experts' order brought back: ``sum over k of weight[i, k] *
    rows[order.places[i, k]]``, choices that name no expert left out: [..., D] of the rows'
    type.

    rows [P, D], P the number of choices; weight (optional): float32 of the shape of the
    experts, for instance a router's probabilities.  Differentiable in ``rows`` and
    ``weight``."""
    places = _places_of("expert_combine", order)
    _check_combine("expert_combine", rows, places, weight)
    _no_tangent("expert_combine", rows=rows, weight=weight)
    _check_devices("rows", rows, "order.places", places, "weight", weight)
    if _wants_gradient(rows, weight):
        return _ExpertCombine.apply(rows, places, weight)
    return _combine(rows, places, weight)


def expert_combine_backward(out_grad: torch.Tensor, rows: Optional[torch.Tensor],
                            order: ExpertOrder, weight: Optional[torch.Tensor] = None):
    """Gradients of ``expert_combine``: ``(rows_grad, weight_grad)``.

    out_grad [..., D]; rows_grad [P, D] of its type, zeros for choices that name no expert;
    weight_grad (float32, the shape of the experts) where ``rows`` is given, else None.
    Neither carries a graph."""
    _element_type("out_grad", out_grad)
    places = _places_of("expert_combine_backward", order)
    if out_grad.dim() != places.dim() or out_grad.shape[:-1] != places.shape[:-1]:
        raise RuntimeError(f"out_grad had shape {list(out_grad.shape)}, expected "
                           f"{list(places.shape[:-1])} and a last dimension")
    _check_width("expert_combine_backward", out_grad.size(-1))
    if rows is not None:
        _check_same_type("out_grad", out_grad, rows=rows)
        _check_shape("rows", rows, (places.numel(), out_grad.size(-1)))
    if weight is not None:
        _check_float32("weight", weight, places.shape)
    _no_tangent("expert_combine_backward", out_grad=out_grad, rows=rows, weight=weight)
    _check_devices("out_grad", out_grad, "rows", rows, "order.places", places, "weight", weight)
    return _combine_backward(out_grad, rows, places, weight, True, rows is not None)


# ---- the experts' products -------------------------------------------------------------------


def _linear(rows, weight, offsets):
    x, w, o = _rows(rows), weight.contiguous(), offsets.contiguous()
    experts, out_width, width = w.shape
    count, dev = x.size(0), rows.device
    out = torch.empty((count, out_width), dtype=rows.dtype, device=dev)
    L = _lib.lib()
    nbytes = L.sdf_expert_linear_scratch_bytes(count, experts, width, out_width)
    keep, base = _scratch(nbytes, dev)
    _call(L.sdf_expert_linear, x, _TYPES[x.dtype], x.data_ptr(), x.stride(0), count, experts,
          width, out_width, w.data_ptr(), o.data_ptr(), out.data_ptr(), base, nbytes)
    return out


def _linear_backward(out_grad, rows, weight, offsets, need_rows, need_weight):
    g, o = _rows(out_grad), offsets.contiguous()
    experts, out_width, width = weight.shape
    x = _rows(rows) if need_weight else None
    w = weight.contiguous() if need_rows else None
    count, dev = g.size(0), out_grad.device
    rows_grad = weight_grad = None
    if need_rows:
        rows_grad = torch.empty((count, width), dtype=out_grad.dtype, device=dev)
    if need_weight:
        weight_grad = torch.empty((experts, out_width, width), dtype=out_grad.dtype, device=dev)
    L = _lib.lib()
    nbytes = L.sdf_expert_linear_backward_scratch_bytes(count, experts, width, out_width)
    keep, base = _scratch(nbytes, dev)
    _call(L.sdf_expert_linear_backward, g, _TYPES[g.dtype], g.data_ptr(), g.stride(0), ptr(x),
          0 if x is None else x.stride(0), count, experts, width, out_width, ptr(w),
          o.data_ptr(), ptr(rows_grad), ptr(weight_grad), base, nbytes)
    return rows_grad, weight_grad


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weight, offsets):
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weight, offsets)
        return _linear(rows, weight, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _no_tangent("expert_linear", gradient=grad)
        rows, weight, offsets = ctx.saved_tensors
        rows_grad, weight_grad = _linear_backward(grad, rows, weight, offsets,
                                                  ctx.needs_input_grad[0], rows is not None)
        return rows_grad, weight_grad, None


def _check_linear(call, rows, weight, offsets):
    _element_type("rows", rows)
    if rows.dim() != 2:
        raise RuntimeError("rows must have 2 dimensions")
    if weight.dim() != 3:
        raise RuntimeError("weight must have 3 dimensions")
    _check_same_type("rows", rows, weight=weight)
    if weight.size(2) != rows.size(1):
        raise RuntimeError(f"weight had shape {list(weight.shape)}, expected a last dimension of "
                           f"{rows.size(1)}, the rows' width")
    if weight.size(0) > MAX_EXPERTS:
        raise RuntimeError(f"at most {MAX_EXPERTS} experts")
    _check_width(call, weight.size(1), weight.size(2))
    _check_entries(call, rows.size(0))
    _check_int32("offsets", offsets)
    _check_shape("offsets", offsets, (weight.size(0) + 1,))


def expert_linear(rows: torch.Tensor, weight: torch.Tensor,
                  offsets: torch.Tensor) -> torch.Tensor:
    """Each expert's product with its own rows: ``rows[p] @ weight[g].T`` for the rows p of
    expert g, offsets[g] to offsets[g + 1], zeros for rows past the last expert's: [P, O].

    rows [P, D] in their experts' order (``expert_rows``); weight [num_experts, O, D];
    offsets: ``ExpertOrder.offsets``, on the device: nothing is read back.  Offsets are in
    ascending order from 0; for others the result is undefined.  Differentiable in ``rows``
    and ``weight``."""
    _check_linear("expert_linear", rows, weight, offsets)
    _no_tangent("expert_linear", rows=rows, weight=weight)
    _check_devices("rows", rows, "weight", weight, "offsets", offsets)
    if _wants_gradient(rows, weight):
        return _ExpertLinear.apply(rows, weight, offsets)
    return _linear(rows, weight, offsets)


def expert_linear_backward(out_grad: torch.Tensor, rows: torch.Tensor, weight: torch.Tensor,
                           offsets: torch.Tensor, need_rows: bool = True,
                           need_weight: bool = True):
    """Gradients of ``expert_linear``: ``(rows_grad, weight_grad)``, either None where it is
    not needed.

    out_grad [P, O]; rows_grad [P, D], zeros for rows past the last expert's; weight_grad
    [num_experts, O, D], zeros for an expert without rows.  Neither carries a graph."""
    _check_linear("expert_linear_backward", rows, weight, offsets)
    _check_same_type("rows", rows, out_grad=out_grad)
    _check_shape("out_grad", out_grad, (rows.size(0), weight.size(1)))
    _no_tangent("expert_linear_backward", out_grad=out_grad, rows=rows, weight=weight)
    _check_devices("out_grad", out_grad, "rows", rows, "weight", weight, "offsets", offsets)
    return _linear_backward(out_grad, rows, weight, offsets, need_rows, need_weight)


# ---- adapters beside a shared projection -----------------------------------------------------


def _adapter_args(rows, weight, adapters, down, up, scale):
    """The arguments that both directions share: first what has to stay alive until the call
    is queued."""
    x, w, a = _rows(rows), _rows(weight), adapters.contiguous()
    d, u = down.contiguous(), up.contiguous()
    n, rank, width = d.shape
    out_width = w.size(0)
    return (x, w, a, d, u), (
        x.data_ptr(), x.stride(0), x.size(0), width, out_width, w.data_ptr(), w.stride(0),
        _ID_TYPES[a.dtype], a.data_ptr(), n, rank, d.data_ptr(), u.data_ptr(), scale)


def _adapt(rows, weight, adapters, down, up, scale):
    keep, args = _adapter_args(rows, weight, adapters, down, up, scale)
    dev = rows.device
    out = torch.empty((*rows.shape[:-1], weight.size(0)), dtype=rows.dtype, device=dev)
    L = _lib.lib()
    nbytes = L.sdf_adapter_linear_scratch_bytes(args[2], args[3], args[4], args[9], args[10])
    scratch, base = _scratch(nbytes, dev)
    _call(L.sdf_adapter_linear, rows, _TYPES[rows.dtype], *args, out.data_ptr(), base, nbytes)
    return out


def _adapt_backward(out_grad, rows, weight, adapters, down, up, scale, need):
    keep, args = _adapter_args(rows, weight, adapters, down, up, scale)
    g, dev = _rows(out_grad), rows.device
    grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) if n else None
             for t, n in zip((rows, weight, down, up), need)]
    L = _lib.lib()
    nbytes = L.sdf_adapter_linear_backward_scratch_bytes(args[2], args[3], args[4], args[9],
                                                         args[10])
    scratch, base = _scratch(nbytes, dev)
    _call(L.sdf_adapter_linear_backward, rows, _TYPES[rows.dtype], g.data_ptr(), g.stride(0),
          *args, *(ptr(t) for t in grads), base, nbytes)
    return tuple(grads)


class _AdapterLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weight, adapters, down, up, scale):
        ctx.save_for_backward(rows, weight, adapters, down, up)
        ctx.scale = scale
        return _adapt(rows, weight, adapters, down, up, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _no_tangent("adapter_linear", gradient=grad)
        rows, weight, adapters, down, up = ctx.saved_tensors
        n = ctx.needs_input_grad
        rows_grad, weight_grad, down_grad, up_grad = _adapt_backward(
            grad, rows, weight, adapters, down, up, ctx.scale, (n[0], n[1], n[3], n[4]))
        return rows_grad, weight_grad, None, down_grad, up_grad, None


def _check_adapter(call, rows, weight, adapters, down, up, scale) -> float:
    _element_type("rows", rows)
    if rows.dim() < 1:
        raise RuntimeError("rows must have at least 1 dimension")
    if weight.dim() != 2:
        raise RuntimeError("weight must have 2 dimensions")
    if down.dim() != 3:
        raise RuntimeError("down must have 3 dimensions")
    _check_same_type("rows", rows, weight=weight, down=down, up=up)
    out_width, width = weight.shape
    n, rank = down.shape[:2]
    if rows.size(-1) != width:
        raise RuntimeError(f"rows had shape {list(rows.shape)}, expected a last dimension of "
                           f"{width}, the weight's")
    _check_shape("down", down, (n, rank, width))
    _check_shape("up", up, (n, out_width, rank))
    _id_type("adapters", adapters)
    _check_shape("adapters", adapters, rows.shape[:-1])
    if n > MAX_ADAPTERS:
        raise RuntimeError(f"at most {MAX_ADAPTERS} adapters")
    if rank > MAX_RANK:
        raise RuntimeError(f"adapters of rank at most {MAX_RANK}")
    _check_width(call, out_width, width)
    _check_entries(call, adapters.numel())
    return float(scale)


def adapter_linear(rows: torch.Tensor, weight: torch.Tensor, adapters: torch.Tensor,
                   down: torch.Tensor, up: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """A shared projection with low-rank adapters of the rows' own beside it:
    ``rows @ weight.T``, plus for each row ``scale * (row @ down[a].T) @ up[a].T`` where
    ``adapters`` names its adapter a: [..., O].

    rows [..., D]; weight [O, D]; adapters [...], in any order; down [A, r, D] and
    up [A, O, r], A up to 2048 and r up to 256.  The inner r values are held in float32.  An
    adapter's values reach its own rows alone.  Differentiable in ``rows``, ``weight``,
    ``down`` and ``up``."""
    scale = _check_adapter("adapter_linear", rows, weight, adapters, down, up, scale)
    _no_tangent("adapter_linear", rows=rows, weight=weight, down=down, up=up)
    _check_devices("rows", rows, "weight", weight, "adapters", adapters, "down", down, "up", up)
    if _wants_gradient(rows, weight, down, up):
        return _AdapterLinear.apply(rows, weight, adapters, down, up, scale)
    return _adapt(rows, weight, adapters, down, up, scale)


def adapter_linear_backward(out_grad: torch.Tensor, rows: torch.Tensor, weight: torch.Tensor,
                            adapters: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                            scale: float = 1.0, need_rows: bool = True,
                            need_weight: bool = True, need_adapters: bool = True):
    """Gradients of ``adapter_linear``: ``(rows_grad, weight_grad, down_grad, up_grad)`` of
    their tensors' shapes and type, None where they are not needed (a frozen projection's:
    ``need_weight=False``).  Adapters without rows have gradients of 0.  None carries a
    graph."""
    scale = _check_adapter("adapter_linear_backward", rows, weight, adapters, down, up, scale)
    _check_same_type("rows", rows, out_grad=out_grad)
    _check_shape("out_grad", out_grad, (*rows.shape[:-1], weight.size(0)))
    _no_tangent("adapter_linear_backward", out_grad=out_grad, rows=rows, weight=weight, down=down,
                up=up)
    _check_devices("out_grad", out_grad, "rows", rows, "weight", weight, "adapters", adapters,
                   "down", down, "up", up)
    return _adapt_backward(out_grad, rows, weight, adapters, down, up, scale,
                           (need_rows, need_weight, need_adapters, need_adapters))


__all__ = ["ExpertOrder", "expert_order", "expert_rows", "expert_combine",
           "expert_combine_backward", "expert_linear", "expert_linear_backward",
           "adapter_linear", "adapter_linear_backward"]

"""Label fields: a foam whose cells carry learned rows, trained on a teacher's labels.

A trace says in which cell each ray ends (``trace_forward``'s ``depth_indices``), a head
makes logits over labels -- a segmenter's classes, a vocabulary -- of that cell's row, and

* ``cell_rows`` gives the rows of the rays' cells, scaled and weighted, with gradients for
  the table and the weights (``cell_rows_backward``);
* ``distill_loss`` is the distance of the logits from a teacher's best few per ray, with
  the logits' gradient; ``distill_loss_and_grad`` gives both in one pass over the logits,
  for training loops that call the backward themselves;
* ``label_log_probs`` answers: the log probability of given labels, the entropy, and the
  best labels with theirs; the first two have gradients.

The reference has no counterpart.  The work runs in libsdfoam_hip.so on torch's current
stream.  Tables and logits are float32, float16 or bfloat16; every sum and softmax is held
in float32 and rounded to the output's type once.  Cells and labels are uint32, int32 or
int64; one that is negative, 0xffffffff (what the trace writes for a ray that ends in no
cell) or too large names none.  Rows of a table or of logits may be strided (a slice of
padded rows is read in place); other layouts are copied.  Results are the same on every
run: no sum's order is left to chance.  Derivatives are reverse-mode and of the first order;
tensors with a forward-mode tangent are refused.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, ptr
from .pipeline import _c10

_TYPES = {torch.float32: _lib.SDF_TYPE_F32, torch.float16: _lib.SDF_TYPE_F16,
          torch.bfloat16: _lib.SDF_TYPE_BF16}
_ID_TYPES = {torch.uint32: _lib.SDF_ID_U32, torch.int32: _lib.SDF_ID_I32,
             torch.int64: _lib.SDF_ID_I64}
_REDUCTIONS = {"none": _lib.SDF_REDUCE_NONE, "sum": _lib.SDF_REDUCE_SUM,
               "mean": _lib.SDF_REDUCE_MEAN}

MAX_TEACHER = 1024  # a teacher's logits per row
MAX_TOP = 64  # best labels per row
MAX_WIDTH = 1 << 18  # elements of a cell's row


def _element_type(name: str, t: torch.Tensor) -> int:
    st = _TYPES.get(t.dtype)
    if st is None:
        raise RuntimeError(f"{name} had dtype {_c10(t.dtype)}, "
                           "expected float32, float16 or bfloat16")
    return st


def _id_type(name: str, t: torch.Tensor) -> int:
    st = _ID_TYPES.get(t.dtype)
    if st is None:
        raise RuntimeError(f"{name} had dtype {_c10(t.dtype)}, expected uint32, int32 or int64")
    return st


def _check_shape(name: str, t: torch.Tensor, shape) -> None:
    if t.shape != shape:
        raise RuntimeError(f"{name} had shape {list(t.shape)}, expected {list(shape)}")


def _check_float32(name: str, t: torch.Tensor, shape) -> None:
    if t.dtype != torch.float32:
        raise RuntimeError(f"{name} had dtype {_c10(t.dtype)}, expected float32")
    _check_shape(name, t, shape)


def _check_devices(first: str, t: torch.Tensor, *others) -> None:
    """others: name, tensor or None, name, ..."""
    device = t.get_device()
    if device < 0:
        raise RuntimeError(f"{first} must be on CUDA device")
    for k in range(1, len(others), 2):
        o = others[k]
        if o is not None and o.get_device() != device:
            raise RuntimeError(f"{others[k - 1]} must be on the device of {first}")


def _no_gradient(call: str, **tensors) -> None:
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{call} has no gradient for {name}: detach it")


def _no_tangent(call: str, **tensors) -> None:
    """Refuses dual tensors: their tangents would not reach the results, and requires_grad
    does not show them."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside of every dual_level
        return
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{call} has no forward-mode derivative for {name}: detach it")


def _wants_gradient(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., D] as [R, D] whose rows are contiguous, without a copy where the layout
    allows it."""
    shape = t.shape
    d = shape[-1]
    if d > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    if len(shape) == 2:
        return t
    rows = 1
    for k in shape[:-1]:
        rows *= k
    return t.reshape(rows, d)


def _like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and type, not written."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _call(function, t: torch.Tensor, *args) -> None:
    """The library call on the current stream of t's device."""
    index = t.get_device()
    if index == torch.cuda.current_device():
        status = function(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(*args, _raw_stream(index))
    if status:
        check(status)


# the stream's handle alone, without the Stream object around it (2 us of a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _lib.stream_handle)


def _scratch(nbytes: int, device: torch.device):
    """Scratch memory (kept alive by the first value) and its 256-byte aligned start.  It
    may go once the call is queued: torch gives it out again only to later work on the
    same stream."""
    if nbytes == 0:
        return None, None
    t = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
    return t, (t.data_ptr() + 255) & ~255


# ---- rows of cells ------------------------------------------------------------------------


def _check_width(call: str, width: int) -> None:
    if width > MAX_WIDTH:  # here: the library's argument has 32 bits
        raise RuntimeError(f"{call} takes rows of at most 2^18 elements")


def _check_weight(weight, cells) -> None:
    if weight is not None:
        _check_float32("weight", weight, cells.shape)


def _rows_forward(table, cells, weight, scale) -> torch.Tensor:
    device, (num_cells, width) = table.device, table.shape
    rows = torch.empty((*cells.shape, width), dtype=table.dtype, device=device)
    t = _rows(table)
    c = cells.contiguous()
    w = None if weight is None else weight.contiguous()
    _call(_lib.lib().sdf_cell_rows, t, _TYPES[table.dtype], t.data_ptr(), t.stride(0),
          num_cells, width, _ID_TYPES[cells.dtype], c.data_ptr(), c.numel(), ptr(w), scale,
          rows.data_ptr())
    return rows


def _rows_backward(rows_grad, cells, num_cells, weight, scale, table, need_table):
    width = rows_grad.size(-1)
    g = _rows(rows_grad)
    c = cells.contiguous()
    w = None if weight is None else weight.contiguous()
    t = None if table is None else _rows(table)
    dev = rows_grad.device
    table_grad = None
    if need_table:
        table_grad = torch.empty((num_cells, width), dtype=rows_grad.dtype, device=dev)
    weight_grad = None
    if table is not None:
        weight_grad = torch.empty(cells.shape, dtype=torch.float32, device=dev)
    L = _lib.lib()
    nbytes = 0
    if need_table:
        nbytes = int(L.sdf_cell_rows_backward_scratch_bytes(num_cells, width, c.numel()))
    keep, base = _scratch(nbytes, dev)
    _call(L.sdf_cell_rows_backward, g, _TYPES[rows_grad.dtype], ptr(g), g.stride(0), ptr(t),
          0 if t is None else t.stride(0), num_cells, width, _ID_TYPES[cells.dtype], ptr(c),
          c.numel(), ptr(w), scale, ptr(table_grad), ptr(weight_grad), base, nbytes)
    return table_grad, weight_grad


class _CellRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, cells, weight, scale):
        ctx.num_cells, ctx.scale = table.size(0), scale
        # the table is read again only for the weights' gradient
        ctx.save_for_backward(cells, weight, table if ctx.needs_input_grad[2] else None)
        return _rows_forward(table, cells, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, rows_grad):
        _no_tangent("cell_rows", gradient=rows_grad)
        cells, weight, table = ctx.saved_tensors
        table_grad, weight_grad = _rows_backward(rows_grad, cells, ctx.num_cells, weight,
                                                 ctx.scale, table, ctx.needs_input_grad[0])
        return table_grad, None, weight_grad, None


def cell_rows(table: torch.Tensor, cells: torch.Tensor, weight: Optional[torch.Tensor] = None,
              scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[i] * table[cells[i]]`` for cells of any shape: [*cells.shape, D] of
    the table's type; zeros where ``cells`` names no cell.

    table [N, D]; weight (optional): float32 of the shape of ``cells``, for instance the
    rays' opacity.  Differentiable in ``table`` and ``weight``."""
    if table.dim() != 2:
        raise RuntimeError("table must have 2 dimensions")
    _element_type("table", table)
    _id_type("cells", cells)
    _check_width("cell_rows", table.size(1))
    _check_weight(weight, cells)
    _no_tangent("cell_rows", table=table, weight=weight)
    _check_devices("table", table, "cells", cells, "weight", weight)
    if _wants_gradient(table, weight):
        return _CellRows.apply(table, cells, weight, float(scale))
    return _rows_forward(table, cells, weight, float(scale))


def cell_rows_backward(rows_grad: torch.Tensor, cells: torch.Tensor, num_cells: int,
                       weight: Optional[torch.Tensor] = None, scale: float = 1.0,
                       table: Optional[torch.Tensor] = None):
    """Gradients of ``cell_rows``: ``(table_grad, weight_grad)``.

    rows_grad [*cells.shape, D]; table_grad [num_cells, D] of its type, zeros for cells that
    no id names; weight_grad (float32, the shape of ``cells``) where ``table`` is given,
    else None.  Neither carries a graph."""
    _element_type("rows_grad", rows_grad)
    _id_type("cells", cells)
    if rows_grad.dim() != cells.dim() + 1 or rows_grad.shape[:-1] != cells.shape:
        raise RuntimeError(f"rows_grad had shape {list(rows_grad.shape)}, "
                           f"expected {list(cells.shape)} and a last dimension")
    _check_width("cell_rows_backward", rows_grad.size(-1))
    num_cells = int(num_cells)
    if num_cells < 0:
        raise RuntimeError("num_cells must not be negative")
    _check_weight(weight, cells)
    if table is not None:
        if table.dtype != rows_grad.dtype:
            raise RuntimeError("table and rows_grad must have the same dtype")
        _check_shape("table", table, (num_cells, rows_grad.size(-1)))
    _no_tangent("cell_rows_backward", rows_grad=rows_grad, weight=weight, table=table)
    _check_devices("rows_grad", rows_grad, "cells", cells, "weight", weight, "table", table)
    return _rows_backward(rows_grad, cells, num_cells, weight, float(scale), table, True)


# ---- distillation ----------------------------------------------------------------------------


def _check_logits(logits, temperature) -> float:
    _element_type("logits", logits)
    if logits.dim() < 1:
        raise RuntimeError("logits must have at least 1 dimension")
    if logits.size(-1) == 0:
        raise RuntimeError("logits must have at least one label")
    temperature = float(temperature)
    if not 1.0e-38 <= temperature <= 3.0e38:
        raise RuntimeError("temperature must be positive and finite, as its reciprocal in float32")
    return temperature


def _check_distill(call, logits, teacher_labels, teacher_logits, temperature, row_weight,
                   reduction):
    temperature = _check_logits(logits, temperature)
    _id_type("teacher_labels", teacher_labels)
    _element_type("teacher_logits", teacher_logits)
    shape, lead = teacher_labels.shape, logits.shape[:-1]
    if shape[:-1] != lead or not shape:
        raise RuntimeError(f"teacher_labels had shape {list(shape)}, expected {list(lead)} "
                           "and a last dimension")
    _check_shape("teacher_logits", teacher_logits, shape)
    if shape[-1] > MAX_TEACHER:
        raise RuntimeError(f"at most {MAX_TEACHER} teacher logits per row")
    if row_weight is not None:
        _check_float32("row_weight", row_weight, lead)
    if reduction not in _REDUCTIONS:
        raise RuntimeError("reduction must be 'none', 'sum' or 'mean'")
    if teacher_logits.requires_grad or (row_weight is not None and row_weight.requires_grad):
        _no_gradient(call, teacher_logits=teacher_logits, row_weight=row_weight)
    _no_tangent(call, logits=logits, teacher_logits=teacher_logits, row_weight=row_weight)
    _check_devices("logits", logits, "teacher_labels", teacher_labels, "teacher_logits",
                   teacher_logits, "row_weight", row_weight)
    return temperature


def _distill_args(logits, teacher_labels, teacher_logits, temperature, row_weight, reduction):
    """The arguments that both directions share, laid out for the library: first what has
    to stay alive until the call is queued."""
    z, ids, t = _rows(logits), teacher_labels.contiguous(), teacher_logits.contiguous()
    w = None if row_weight is None else row_weight.contiguous()
    rows, labels = z.shape
    return (z, ids, t, w), (
        _TYPES[z.dtype], z.data_ptr(), rows, labels, z.stride(0), _ID_TYPES[ids.dtype],
        ids.data_ptr(), _TYPES[t.dtype], t.data_ptr(), ids.size(-1), temperature, ptr(w),
        _REDUCTIONS[reduction])


def _distill_forward(logits, teacher_labels, teacher_logits, temperature, row_weight, reduction,
                     loss_grad=None, stats=None, logits_grad=None) -> torch.Tensor:
    keep, args = _distill_args(logits, teacher_labels, teacher_logits, temperature, row_weight,
                               reduction)
    dev = logits.device
    loss = torch.empty(logits.shape[:-1] if reduction == "none" else (), dtype=torch.float32,
                       device=dev)
    L = _lib.lib()
    nbytes = L.sdf_distill_scratch_bytes(args[2], args[3], args[12])
    scratch, base = _scratch(nbytes, dev)
    _call(L.sdf_distill, logits, *args, ptr(loss_grad), loss.data_ptr(), ptr(stats),
          ptr(logits_grad), base, nbytes)
    return loss


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_labels, teacher_logits, temperature, row_weight, reduction):
        rows = logits.numel() // logits.size(-1)
        stats = torch.empty((rows, 2), dtype=torch.float32, device=logits.device)
        loss = _distill_forward(logits, teacher_labels, teacher_logits, temperature, row_weight,
                                reduction, stats=stats)
        ctx.save_for_backward(logits, teacher_labels, teacher_logits, row_weight, stats)
        ctx.temperature, ctx.reduction = temperature, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, loss_grad):
        _no_tangent("distill_loss", gradient=loss_grad)
        logits, teacher_labels, teacher_logits, row_weight, stats = ctx.saved_tensors
        keep, args = _distill_args(logits, teacher_labels, teacher_logits, ctx.temperature,
                                   row_weight, ctx.reduction)
        g = loss_grad.contiguous()
        logits_grad = _like(logits)
        _call(_lib.lib().sdf_distill_backward, logits, *args, ptr(g), ptr(stats),
              ptr(logits_grad))
        return logits_grad, None, None, None, None, None


def distill_loss(logits: torch.Tensor, teacher_labels: torch.Tensor,
                 teacher_logits: torch.Tensor, temperature: float = 1.0,
                 row_weight: Optional[torch.Tensor] = None,
                 reduction: str = "mean") -> torch.Tensor:
    """Kullback-Leibler distance of the logits' distribution from the one that a teacher's
    best logits give, both over ``temperature``, times its square (so that gradients keep
    their size).

    logits [..., V]; teacher_labels, teacher_logits [..., K] with K up to 1024: the
    teacher's distribution is the softmax of a row's logits whose label names one and that
    are above -inf, and of no others.  row_weight (float32 [...]): a row of weight 0 is not
    read.  A row without an entry, or whose logits are all -inf, has loss 0 and no gradient.
    Returns float32: the rows' losses ("none"), their "sum", or their "mean" over all rows.
    Differentiable in ``logits``."""
    temperature = _check_distill("distill_loss", logits, teacher_labels, teacher_logits,
                                 temperature, row_weight, reduction)
    if _wants_gradient(logits):
        return _DistillLoss.apply(logits, teacher_labels, teacher_logits, temperature, row_weight,
                                  reduction)
    return _distill_forward(logits, teacher_labels, teacher_logits, temperature, row_weight,
                            reduction)


def distill_loss_and_grad(logits: torch.Tensor, teacher_labels: torch.Tensor,
                          teacher_logits: torch.Tensor, temperature: float = 1.0,
                          row_weight: Optional[torch.Tensor] = None, reduction: str = "mean",
                          loss_grad: Optional[torch.Tensor] = None):
    """``distill_loss`` and its gradient, in one pass over the logits: ``(loss,
    logits_grad)``, logits_grad of the logits' shape and type.

    loss_grad (float32, the shape of the loss; default 1) is the gradient that reaches the
    loss from above, such as a loss scale: it is applied before the gradient is rounded.
    Neither result carries a graph."""
    if loss_grad is not None:
        _no_tangent("distill_loss_and_grad", loss_grad=loss_grad)
    temperature = _check_distill("distill_loss_and_grad", logits, teacher_labels, teacher_logits,
                                 temperature, row_weight, reduction)
    if loss_grad is not None:
        _check_float32("loss_grad", loss_grad, logits.shape[:-1] if reduction == "none" else ())
        _check_devices("logits", logits, "loss_grad", loss_grad)
        loss_grad = loss_grad.contiguous()
    logits_grad = _like(logits)
    return _distill_forward(logits, teacher_labels, teacher_logits, temperature, row_weight,
                            reduction, loss_grad, None, logits_grad), logits_grad


# ---- answers ---------------------------------------------------------------------------------


class LabelLogProbs(NamedTuple):
    """What ``label_log_probs`` returns; the last two are None where no best labels were
    asked for."""

    log_prob: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: Optional[torch.Tensor]
    top_labels: Optional[torch.Tensor]


def _answer(logits, labels, top, temperature, stats=None):
    z = _rows(logits)
    y = labels.contiguous()
    dev, shape = logits.device, labels.shape
    rows, count = z.shape
    log_prob = torch.empty(shape, dtype=torch.float32, device=dev)
    entropy = torch.empty_like(log_prob)
    best = best_labels = None
    if top:
        best = torch.empty((*shape, top), dtype=torch.float32, device=dev)
        best_labels = torch.empty((*shape, top), dtype=torch.int64, device=dev)
    L = _lib.lib()
    nbytes = L.sdf_label_log_probs_scratch_bytes(rows, count, top)
    keep, base = _scratch(nbytes, dev)
    _call(L.sdf_label_log_probs, z, _TYPES[z.dtype], z.data_ptr(), rows, count, z.stride(0),
          _ID_TYPES[y.dtype], y.data_ptr(), top, temperature, log_prob.data_ptr(),
          entropy.data_ptr(), ptr(best), ptr(best_labels), ptr(stats), base, nbytes)
    return log_prob, entropy, best, best_labels


class _LabelLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, top, temperature):
        ctx.set_materialize_grads(False)
        rows = labels.numel()
        stats = torch.empty((rows, 2), dtype=torch.float32, device=logits.device)
        log_prob, entropy, best, best_labels = _answer(logits, labels, top, temperature, stats)
        ctx.save_for_backward(logits, labels, entropy, stats)
        ctx.temperature = temperature
        if top:
            ctx.mark_non_differentiable(best, best_labels)
        return log_prob, entropy, best, best_labels

    @staticmethod
    @once_differentiable
    def backward(ctx, log_prob_grad, entropy_grad, best_grad, best_labels_grad):
        if log_prob_grad is None and entropy_grad is None:
            return None, None, None, None
        for g in (log_prob_grad, entropy_grad):
            _no_tangent("label_log_probs", gradient=g)
        logits, labels, entropy, stats = ctx.saved_tensors
        z = _rows(logits)
        y = labels.contiguous()
        g = None if log_prob_grad is None else log_prob_grad.contiguous()
        h = None if entropy_grad is None else entropy_grad.contiguous()
        logits_grad = _like(logits)
        _call(_lib.lib().sdf_label_log_probs_backward, logits, _TYPES[z.dtype], ptr(z),
              z.size(0), z.size(1), z.stride(0), _ID_TYPES[y.dtype], ptr(y), ctx.temperature,
              ptr(entropy), ptr(stats), ptr(g), ptr(h), ptr(logits_grad))
        return logits_grad, None, None, None


def label_log_probs(logits: torch.Tensor, labels: torch.Tensor, top: int = 0,
                    temperature: float = 1.0) -> LabelLogProbs:
    """Log probabilities of labels under the softmax of ``logits / temperature``, with its
    entropy and the ``top`` (at most 64) best labels.

    logits [..., V]; labels [...].  log_prob [...] (0 where ``labels`` names none, -inf for
    a label masked out by a logit of -inf), entropy [...] (0 for a row of nothing but -inf),
    top_log_probs and top_labels (int64) [..., top], largest logit first, ties to the lowest
    label, -inf and -1 where fewer labels are above -inf.  Differentiable in ``logits``
    through log_prob and entropy."""
    temperature = _check_logits(logits, temperature)
    _id_type("labels", labels)
    _check_shape("labels", labels, logits.shape[:-1])
    top = int(top)
    if not 0 <= top <= MAX_TOP:
        raise RuntimeError(f"top must be from 0 to {MAX_TOP}")
    _no_tangent("label_log_probs", logits=logits)
    _check_devices("logits", logits, "labels", labels)
    if _wants_gradient(logits):
        return LabelLogProbs(*_LabelLogProbs.apply(logits, labels, top, temperature))
    return LabelLogProbs(*_answer(logits, labels, top, temperature))


__all__ = ["cell_rows", "cell_rows_backward", "distill_loss", "distill_loss_and_grad",
           "label_log_probs", "LabelLogProbs"]

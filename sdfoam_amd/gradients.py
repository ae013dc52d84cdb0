"""The norm of a training step's gradients, all tensors together, and clipping by it.

``gradient_norm`` gives the Euclidean norm over many tensors, ``clip_gradients`` scales them
in place (or into float32 copies for the optimizer) so that it is at most a given one.  Both
take tensors of any mix of float32, float16 and bfloat16 and run in a few launches whatever
their number; the norm stays on the device, nothing is read back.  Squares are added in
float64, in the same order on every run.  The reference has no counterpart.
"""

from __future__ import annotations

import ctypes as C
from typing import Iterable, Optional

import torch

from . import _lib
from .labels import _TYPES, _call, _element_type, _no_gradient, _no_tangent, _scratch


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one run of memory, each once, in any order of dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _gradients(call: str, gradients: Iterable[Optional[torch.Tensor]]):
    tensors = [gradients] if isinstance(gradients, torch.Tensor) else list(gradients)
    some = [g for g in tensors if g is not None]
    if not some:
        raise RuntimeError("gradients must hold at least one tensor")
    for g in some:
        _element_type("gradients", g)
        if not g.is_contiguous() and g.numel() > 0 and not _dense(g):
            raise RuntimeError("gradients must fill their memory without gaps or overlaps")
        if g.requires_grad:
            _no_gradient(call, gradients=g)
        _no_tangent(call, gradients=g)
    device = some[0].get_device()
    for g in some:
        if g.get_device() != device or device < 0:
            raise RuntimeError("gradients must be on CUDA device" if g.get_device() < 0
                               else "gradients must be on one device")
    return tensors, some[0].device


def _run(gradients, out, max_norm, scale, device) -> torch.Tensor:
    n = len(gradients)
    types = (C.c_int * n)(*[_TYPES[g.dtype] for g in gradients])
    at = (C.c_void_p * n)(*[g.data_ptr() for g in gradients])
    counts = (C.c_uint64 * n)(*[g.numel() for g in gradients])
    out_types = out_at = None
    if out is not None:
        out_types = (C.c_int * n)(*[_TYPES[o.dtype] for o in out])
        out_at = (C.c_void_p * n)(*[o.data_ptr() for o in out])
    norm = torch.empty((), dtype=torch.float32, device=device)
    L = _lib.lib()
    nbytes = L.sdf_clip_gradients_scratch_bytes(n)
    keep, base = _scratch(nbytes, device)
    _call(L.sdf_clip_gradients, norm, n, types, at, counts, out_types, out_at, max_norm, scale,
          norm.data_ptr(), base, nbytes)
    return norm


def _check_scale(scale) -> float:
    scale = float(scale)
    if not 0.0 < scale <= 3.0e38:
        raise RuntimeError("scale must be positive and finite")
    return scale


def gradient_norm(gradients: Iterable[Optional[torch.Tensor]], scale: float = 1.0) -> torch.Tensor:
    """``scale`` times the Euclidean norm of all gradients together (float32, on their
    device).  gradients: one tensor, or tensors of any shapes, empty ones and None (a
    parameter without a gradient) among them; one that is there twice counts twice."""
    scale = _check_scale(scale)
    tensors, device = _gradients("gradient_norm", gradients)
    return _run([g for g in tensors if g is not None], None, 0.0, scale, device)


def clip_gradients(gradients: Iterable[Optional[torch.Tensor]], max_norm: float,
                   scale: float = 1.0,
                   out: Optional[Iterable[Optional[torch.Tensor]]] = None) -> torch.Tensor:
    """Scales all gradients by ``scale * min(1, max_norm / (norm + 1e-6))`` and returns
    ``norm``, ``scale`` times their Euclidean norm before (float32, on their device).

    gradients: one tensor, or tensors of any shapes, for instance ``[p.grad for p in
    parameters]``; None among them is passed over.  scale undoes a loss scale or averages
    sums, before anything is rounded.  out (optional): as many tensors of the gradients'
    shapes, float32 or of their gradient's type, that the results are written to -- an
    optimizer's float32 copies --; default: the gradients themselves.  No result may lie on
    another, or on another gradient.

    The factor is that of the norm before it is rounded to float32: finite gradients whose
    norm passes float32's range are clipped all the same, and the norm returned for them is
    infinite.  Gradients that are not finite are not mended: with an infinite one among them
    each result is 0 times its gradient (NaN where max_norm is infinite too), with NaN each
    is NaN."""
    scale = _check_scale(scale)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise RuntimeError("max_norm must not be negative")
    tensors, device = _gradients("clip_gradients", gradients)
    if isinstance(gradients, torch.Tensor) and isinstance(out, torch.Tensor):
        out = [out]
    results = tensors if out is None else list(out)
    if out is not None:
        if len(results) != len(tensors):
            raise RuntimeError(f"out must hold as many tensors as gradients ({len(tensors)})")
        for g, o in zip(tensors, results):
            if g is None:
                continue
            if o is None or o.dtype not in (g.dtype, torch.float32):
                raise RuntimeError("out must be float32 or of the gradient's type")
            if o.shape != g.shape or (o.stride() != g.stride() and
                                      not (o.is_contiguous() and g.is_contiguous())):
                raise RuntimeError(f"out had shape {list(o.shape)} and strides "
                                   f"{list(o.stride())}, expected {list(g.shape)} and "
                                   f"{list(g.stride())}")
            if o.get_device() != g.get_device():
                raise RuntimeError("out must be on the device of the gradients")
            if o.requires_grad:
                _no_gradient("clip_gradients", out=o)
            _no_tangent("clip_gradients", out=o)
    keep = [k for k, g in enumerate(tensors) if g is not None]
    norm = _run([tensors[k] for k in keep], [results[k] for k in keep], max_norm, scale, device)
    # autograd, and whoever looks at versions, sees the write
    torch.autograd.graph.increment_version(
        [results[k] for k in keep if not results[k].is_inference()])
    return norm


__all__ = ["gradient_norm", "clip_gradients"]

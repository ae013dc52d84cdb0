"""What the heads' operators and the clipping refuse, without a GPU: the Python checks
(shapes and types come before devices, so CPU tensors reach them) and the C interface's,
before any HIP call."""

import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

import sdfoam_amd
from sdfoam_amd import _lib


def ids(*shape, dtype=torch.int64):
    return torch.zeros(shape, dtype=dtype)


def order(*shape, experts=3):
    return sdfoam_amd.ExpertOrder(ids(*shape, dtype=torch.int32),
                                  ids(experts + 1, dtype=torch.int32))


def refused(match):
    return pytest.raises(RuntimeError, match=match)


def test_expert_order_refuses():
    with refused("experts had dtype Float, expected uint32, int32 or int64"):
        sdfoam_amd.expert_order(torch.zeros(3, 2), 4)
    with refused("experts must have at least 1 dimension"):
        sdfoam_amd.expert_order(torch.tensor(1), 4)
    for bad in (-1, 2049):
        with refused("num_experts must be from 0 to 2048"):
            sdfoam_amd.expert_order(ids(3, 2), bad)
    with refused("experts must be on CUDA device"):
        sdfoam_amd.expert_order(ids(3, 2), 4)


def test_expert_rows_refuses():
    x = torch.zeros(3, 5)
    with refused("rows had dtype Double"):
        sdfoam_amd.expert_rows(x.double(), order(3, 2))
    with refused("order.places had dtype Long, expected int32"):
        sdfoam_amd.expert_rows(x, sdfoam_amd.ExpertOrder(ids(3, 2), ids(4)))
    with refused(r"rows had shape \[3, 5\], expected \[4\]"):
        sdfoam_amd.expert_rows(x, order(4, 2))
    with refused("rows of at most 2"):
        sdfoam_amd.expert_rows(torch.zeros(1, 1).expand(3, 2 ** 18 + 1), order(3, 2))
    with refused("rows must be on CUDA device"):
        sdfoam_amd.expert_rows(x, order(3, 2))


def test_expert_combine_refuses():
    y, g = torch.zeros(6, 5), torch.zeros(3, 5)
    with refused("rows must have 2 dimensions"):
        sdfoam_amd.expert_combine(torch.zeros(6), order(3, 2))
    with refused(r"rows had shape \[6, 5\], expected 8 rows"):
        sdfoam_amd.expert_combine(y, order(4, 2))
    with refused(r"weight had shape \[3\], expected \[3, 2\]"):
        sdfoam_amd.expert_combine(y, order(3, 2), torch.zeros(3))
    with refused("weight had dtype Half, expected float32"):
        sdfoam_amd.expert_combine(y, order(3, 2), torch.zeros(3, 2).half())
    with refused("rows must be on CUDA device"):
        sdfoam_amd.expert_combine(y, order(3, 2))
    with refused(r"out_grad had shape \[3, 5\], expected \[4\]"):
        sdfoam_amd.expert_combine_backward(g, None, order(4, 2))
    with refused("rows had dtype Half, expected Float as out_grad"):
        sdfoam_amd.expert_combine_backward(g, y.half(), order(3, 2))
    with refused(r"rows had shape \[6, 4\], expected \[6, 5\]"):
        sdfoam_amd.expert_combine_backward(g, y[:, :4], order(3, 2))
    with refused("out_grad must be on CUDA device"):
        sdfoam_amd.expert_combine_backward(g, y, order(3, 2))


def test_expert_linear_refuses():
    x, w, o, d = torch.zeros(6, 5), torch.zeros(3, 7, 5), ids(4, dtype=torch.int32), torch.zeros(6, 7)
    for call in (sdfoam_amd.expert_linear, lambda *a: sdfoam_amd.expert_linear_backward(d, *a)):
        with refused("rows had dtype Int"):
            call(x.int(), w, o)
        with refused("rows must have 2 dimensions"):
            call(x[0], w, o)
        with refused("weight must have 3 dimensions"):
            call(x, w[0], o)
        with refused("weight had dtype Half, expected Float as rows"):
            call(x, w.half(), o)
        with refused(r"weight had shape \[3, 7, 4\], expected a last dimension of 5"):
            call(x, w[..., :4], o)
        with refused("at most 2048 experts"):
            call(x, torch.zeros(2049, 1, 5), o)
        with refused("offsets had dtype Long, expected int32"):
            call(x, w, o.long())
        with refused(r"offsets had shape \[3\], expected \[4\]"):
            call(x, w, o[:3])
        with refused("rows must be on CUDA device|out_grad must be on CUDA device"):
            call(x, w, o)
    with refused(r"out_grad had shape \[6, 7\], expected \[6, 8\]"):
        sdfoam_amd.expert_linear_backward(d, x, torch.zeros(3, 8, 5), o)
    with refused("out_grad had dtype Half, expected Float as rows"):
        sdfoam_amd.expert_linear_backward(d.half(), x, w, o)


def test_adapter_linear_refuses():
    x, w, c = torch.zeros(6, 5), torch.zeros(7, 5), ids(6)
    a, b, d = torch.zeros(3, 2, 5), torch.zeros(3, 7, 2), torch.zeros(6, 7)
    for call in (sdfoam_amd.adapter_linear,
                 lambda *t: sdfoam_amd.adapter_linear_backward(d, *t)):
        with refused("rows had dtype Double"):
            call(x.double(), w, c, a, b)
        with refused("weight must have 2 dimensions"):
            call(x, w[0], c, a, b)
        with refused("down must have 3 dimensions"):
            call(x, w, c, a[0], b)
        for k in (1, 3, 4):
            t = [x, w, c, a, b]
            t[k] = t[k].half()
            with refused("had dtype Half, expected Float as rows"):
                call(*t)
        with refused(r"rows had shape \[6, 4\], expected a last dimension of 5"):
            call(x[:, :4], w, c, a, b)
        with refused(r"down had shape \[3, 2, 4\], expected \[3, 2, 5\]"):
            call(x, w, c, a[..., :4], b)
        with refused(r"up had shape \[3, 7, 1\], expected \[3, 7, 2\]"):
            call(x, w, c, a, b[..., :1])
        with refused("adapters had dtype Short"):
            call(x, w, c.short(), a, b)
        with refused(r"adapters had shape \[5\], expected \[6\]"):
            call(x, w, c[:5], a, b)
        with refused("at most 2048 adapters"):
            call(x, w, c, torch.zeros(2049, 1, 5), torch.zeros(2049, 7, 1))
        with refused("adapters of rank at most 256"):
            call(x, w, c, torch.zeros(1, 257, 5), torch.zeros(1, 7, 257))
        with refused("must be on CUDA device"):
            call(x, w, c, a, b)
    with refused(r"out_grad had shape \[6, 7\], expected \[5, 7\]"):
        sdfoam_amd.adapter_linear_backward(d, x[:5], w, c[:5], a, b)


def test_clip_gradients_refuses():
    t = torch.zeros(4)
    for call in (sdfoam_amd.gradient_norm, lambda g, **k: sdfoam_amd.clip_gradients(g, 1.0, **k)):
        with refused("gradients had dtype Double"):
            call([t.double()])
        with refused("must hold at least one tensor"):
            call([None])
        with refused("must hold at least one tensor"):
            call([])
        with refused("without gaps or overlaps"):
            call([torch.zeros(4, 4)[:, :2]])
        for bad in (0.0, -1.0, float("nan"), float("inf")):
            with refused("scale must be positive and finite"):
                call([t], scale=bad)
        with refused("has no gradient for gradients: detach it"):
            call([torch.zeros(4, requires_grad=True)])
        with refused("gradients must be on CUDA device"):
            call([t])
    for bad in (-1.0, float("nan")):
        with refused("max_norm must not be negative"):
            sdfoam_amd.clip_gradients([t], bad)


def test_forward_mode_is_refused():
    x = torch.zeros(6, 5)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with refused("expert_rows has no forward-mode derivative for rows"):
            sdfoam_amd.expert_rows(dual, order(6, 2))
        with refused("expert_combine has no forward-mode derivative for rows"):
            sdfoam_amd.expert_combine(dual, order(3, 2))
        with refused("expert_linear has no forward-mode derivative for rows"):
            sdfoam_amd.expert_linear(dual, torch.zeros(3, 7, 5), ids(4, dtype=torch.int32))
        with refused("adapter_linear has no forward-mode derivative for rows"):
            sdfoam_amd.adapter_linear(dual, torch.zeros(7, 5), ids(6), torch.zeros(1, 2, 5),
                                      torch.zeros(1, 7, 2))
        with refused("clip_gradients has no forward-mode derivative for gradients"):
            sdfoam_amd.clip_gradients([dual], 1.0)


def test_c_interface_refuses():
    L = _lib.lib()

    def says(rc, text):
        assert rc == _lib.SDF_E_INVALID and text in L.sdf_last_error().decode()

    p = 256  # an address that nothing reads
    says(L.sdf_expert_order(9, p, 4, 4, p, p, None, 0, None), "id_type")
    says(L.sdf_expert_order(0, p, 4, 2049, p, p, None, 0, None), "at most 2048 experts")
    says(L.sdf_expert_order(0, p, 2 ** 31, 4, p, p, None, 0, None), "fewer than 2^31")
    says(L.sdf_expert_order(0, p, 4, 4, p, None, None, 0, None), "NULL")
    assert L.sdf_expert_order_scratch_bytes(4096, 4) == 0
    need = L.sdf_expert_order_scratch_bytes(4097, 4)
    says(L.sdf_expert_order(0, p, 4097, 4, p, p, p, need - 1, None), "scratch must hold")
    says(L.sdf_expert_order(0, p, 4097, 4, p, p, p + 8, need, None), "256-byte aligned")

    says(L.sdf_expert_rows(7, p, 4, 1, 1, 4, p, p, None), "type must be")
    says(L.sdf_expert_rows(0, p, 4, 2 ** 30, 2, 4, p, p, None), "fewer than 2^31")
    says(L.sdf_expert_rows(0, p, 4, 1, 1, 2 ** 18 + 1, p, p, None), "2^18")
    says(L.sdf_expert_rows(0, p, 4, 1, 1, 4, None, p, None), "NULL")
    says(L.sdf_expert_combine(0, None, 4, 1, 1, 4, p, p, p, None), "NULL")
    says(L.sdf_expert_combine_backward(0, p, 4, None, 4, 1, 1, 4, p, None, p, p, None), "NULL")

    says(L.sdf_expert_linear(5, p, 4, 1, 1, 4, 4, p, p, p, None, 0, None), "type must be")
    says(L.sdf_expert_linear(0, p, 4, 1, 2049, 4, 4, p, p, p, None, 0, None), "2048 experts")
    says(L.sdf_expert_linear(0, p, 4, 2 ** 31, 1, 4, 4, p, p, p, None, 0, None), "2^31 rows")
    says(L.sdf_expert_linear(0, p, 4, 1, 1, 4, 4, None, p, p, None, 0, None), "NULL")
    says(L.sdf_expert_linear_backward(0, p, 4, None, 4, 1, 1, 4, 4, p, p, p, p, None, 0, None),
         "NULL")
    args = [p, 4, 1, 4, 4, p, 4, 0, p]
    says(L.sdf_adapter_linear(5, *args, 1, 1, p, p, 1.0, p, None, 0, None), "type must be")
    says(L.sdf_adapter_linear(0, *args, 2049, 1, p, p, 1.0, p, None, 0, None), "2048 adapters")
    says(L.sdf_adapter_linear(0, *args, 1, 257, p, p, 1.0, p, None, 0, None), "rank at most 256")
    need = L.sdf_adapter_linear_scratch_bytes(1, 4, 4, 1, 1)
    assert need > 0
    says(L.sdf_adapter_linear(0, *args, 1, 1, p, p, 1.0, p, p, need - 1, None), "scratch must hold")
    says(L.sdf_adapter_linear(0, *args, 1, 1, None, p, 1.0, p, p, need, None), "NULL")
    need = L.sdf_adapter_linear_backward_scratch_bytes(1, 4, 4, 1, 1)
    says(L.sdf_adapter_linear_backward(0, p, 4, *args, 1, 1, p, None, 1.0, p, p, p, p, p, need,
                                       None), "NULL")

    def arrays(n, at=(256, 512), size=4):
        return ((C.c_int * n)(*[0] * n), (C.c_void_p * n)(*at[:n]), (C.c_uint64 * n)(*[size] * n))

    types, at, counts = arrays(2)
    need = L.sdf_clip_gradients_scratch_bytes(2)
    clip = L.sdf_clip_gradients
    says(clip(2, types, at, counts, types, at, 1.0, 1.0, None, p, need, None), "NULL")
    says(clip(2, types, at, counts, types, at, -1.0, 1.0, p, p, need, None), "max_norm")
    says(clip(2, types, at, counts, types, at, 1.0, 0.0, p, p, need, None), "scale must be")
    says(clip(2, types, at, counts, types, at, 1.0, 1.0, p, p, need - 1, None), "scratch must")
    same = arrays(2, (256, 264))[1]
    says(clip(2, types, same, counts, types, same, 1.0, 1.0, p, p, need, None), "twice")
    says(clip(2, types, at, counts, types, arrays(2, (512, 1024))[1], 1.0, 1.0, p, p, need, None),
         "another gradient")
    says(clip(2, types, at, (C.c_uint64 * 2)(2 ** 39, 2 ** 39), None, None, 1.0, 1.0, p, p, need,
              None), "2^40")
    says(clip(2, types, arrays(2, (256, None))[1], counts, None, None, 1.0, 1.0, p, p, need, None),
         "NULL")
    halves = (C.c_int * 2)(1, 1)
    says(clip(2, types, at, counts, halves, at, 1.0, 1.0, p, p, need, None), "float32 or of")
    says(clip(2, halves, at, counts, types, at, 1.0, 1.0, p, p, need, None), "another type")


def test_scratch_of_no_experts():
    """Without experts the products of rows are zeros, and their plan may cut the inner
    dimension all the same: the size that a caller asks for is the one that the call needs."""
    L = _lib.lib()
    p = 256
    need = L.sdf_expert_linear_backward_scratch_bytes(300, 0, 6, 1024)
    assert need > 0 and need == L.sdf_expert_linear_scratch_bytes(300, 0, 1024, 6)
    for scratch, size in ((None, 0), (p, 0), (p, need - 1)):
        rc = L.sdf_expert_linear_backward(0, p, 1024, p, 6, 300, 0, 6, 1024, None, p, p, None,
                                          scratch, size, None)
        assert rc == _lib.SDF_E_INVALID and "scratch must hold" in L.sdf_last_error().decode()

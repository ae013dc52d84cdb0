"""What the label operators refuse, without a GPU: the Python checks (shapes and types come
before devices, so CPU tensors reach them) and the C interface's, before any HIP call."""

import ctypes as C

import pytest
import torch

import sdfoam_amd
from sdfoam_amd import _lib


def ids(*shape, dtype=torch.int64):
    return torch.zeros(shape, dtype=dtype)


def test_cell_rows_refuses():
    table = torch.zeros(5, 4)
    with pytest.raises(RuntimeError, match="table must have 2 dimensions"):
        sdfoam_amd.cell_rows(torch.zeros(5), ids(3))
    with pytest.raises(RuntimeError, match="table had dtype Double, expected float32, float16"):
        sdfoam_amd.cell_rows(table.double(), ids(3))
    with pytest.raises(RuntimeError, match="cells had dtype Float, expected uint32, int32 or int64"):
        sdfoam_amd.cell_rows(table, torch.zeros(3))
    with pytest.raises(RuntimeError, match=r"weight had shape \[4\], expected \[3\]"):
        sdfoam_amd.cell_rows(table, ids(3), torch.zeros(4))
    with pytest.raises(RuntimeError, match="weight had dtype Half, expected float32"):
        sdfoam_amd.cell_rows(table, ids(3), torch.zeros(3).half())
    with pytest.raises(RuntimeError, match="table must be on CUDA device"):
        sdfoam_amd.cell_rows(table, ids(3))


def test_cell_rows_backward_refuses():
    grad = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match=r"rows_grad had shape \[3, 4\], expected \[2\]"):
        sdfoam_amd.cell_rows_backward(grad, ids(2), 5)
    with pytest.raises(RuntimeError, match="num_cells must not be negative"):
        sdfoam_amd.cell_rows_backward(grad, ids(3), -1)
    with pytest.raises(RuntimeError, match="table and rows_grad must have the same dtype"):
        sdfoam_amd.cell_rows_backward(grad, ids(3), 5, table=torch.zeros(5, 4).half())
    with pytest.raises(RuntimeError, match=r"table had shape \[6, 4\], expected \[5, 4\]"):
        sdfoam_amd.cell_rows_backward(grad, ids(3), 5, table=torch.zeros(6, 4))
    with pytest.raises(RuntimeError, match="rows_grad must be on CUDA device"):
        sdfoam_amd.cell_rows_backward(grad, ids(3), 5)


@pytest.mark.parametrize("call", [sdfoam_amd.distill_loss, sdfoam_amd.distill_loss_and_grad])
def test_distill_refuses(call):
    z, j, t = torch.zeros(3, 7), ids(3, 2), torch.zeros(3, 2)
    with pytest.raises(RuntimeError, match="logits had dtype Long"):
        call(z.long(), j, t)
    with pytest.raises(RuntimeError, match="logits must have at least 1 dimension"):
        call(torch.tensor(1.0), j, t)
    with pytest.raises(RuntimeError, match="logits must have at least one label"):
        call(z[:, :0], j, t)
    with pytest.raises(RuntimeError, match="teacher_labels had dtype Short"):
        call(z, j.short(), t)
    with pytest.raises(RuntimeError, match=r"teacher_labels had shape \[2, 2\]"):
        call(z, j[:2], t)
    with pytest.raises(RuntimeError, match=r"teacher_logits had shape \[3, 1\], expected \[3, 2\]"):
        call(z, j, t[:, :1])
    with pytest.raises(RuntimeError, match="at most 1024 teacher logits"):
        call(z, ids(3, 1025), torch.zeros(3, 1025))
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="temperature must be positive and finite"):
            call(z, j, t, bad)
    with pytest.raises(RuntimeError, match=r"row_weight had shape \[2\], expected \[3\]"):
        call(z, j, t, 1.0, torch.zeros(2))
    with pytest.raises(RuntimeError, match="row_weight had dtype Double"):
        call(z, j, t, 1.0, torch.zeros(3).double())
    with pytest.raises(RuntimeError, match="reduction must be"):
        call(z, j, t, reduction="batchmean")
    with pytest.raises(RuntimeError, match="logits must be on CUDA device"):
        call(z, j, t)


def test_label_log_probs_refuses():
    z = torch.zeros(3, 7)
    with pytest.raises(RuntimeError, match="logits had dtype Int"):
        sdfoam_amd.label_log_probs(z.int(), ids(3))
    with pytest.raises(RuntimeError, match="labels had dtype Float"):
        sdfoam_amd.label_log_probs(z, torch.zeros(3))
    with pytest.raises(RuntimeError, match=r"labels had shape \[3, 1\], expected \[3\]"):
        sdfoam_amd.label_log_probs(z, ids(3, 1))
    for bad in (-1, 65):
        with pytest.raises(RuntimeError, match="top must be from 0 to 64"):
            sdfoam_amd.label_log_probs(z, ids(3), bad)
    with pytest.raises(RuntimeError, match="temperature must be positive"):
        sdfoam_amd.label_log_probs(z, ids(3), 0, 0.0)
    with pytest.raises(RuntimeError, match="logits must be on CUDA device"):
        sdfoam_amd.label_log_probs(z, ids(3))


def _memory():
    buf = (C.c_uint64 * 256)()
    base = (C.addressof(buf) + 255) & ~255
    return buf, base


def _refused(rc, text):
    assert rc == _lib.SDF_E_INVALID
    assert text in _lib.lib().sdf_last_error(), _lib.lib().sdf_last_error()


def test_c_cell_rows():
    L = _lib.lib()
    keep, p = _memory()

    def rows(type=0, table=p, cells=5, id_type=0, ids=p, count=3, out=p):
        return L.sdf_cell_rows(type, table, 4, cells, 4, id_type, ids, count, None, 1.0, out, None)

    _refused(rows(type=3), b"unknown element type 3")
    _refused(rows(id_type=-1), b"unknown id type -1")
    _refused(rows(cells=1 << 31), b"fewer than 2^31 cells")
    _refused(rows(count=1 << 31), b"fewer than 2^31 ids")
    _refused(rows(table=None), b"NULL pointer")
    _refused(rows(out=None), b"NULL pointer")
    _refused(rows(table=p + 2), b"aligned to their elements")
    assert rows(count=0, ids=None, out=None) == 0
    rc = L.sdf_cell_rows(0, p, 4, 5, (1 << 18) + 1, 0, p, 3, None, 1.0, p, None)
    _refused(rc, b"rows of at most 2^18 elements")

    def back(type=0, grad=p, table=None, cells=5, ids=p, count=3, tg=p, wg=None, scratch=p,
             nbytes=None):
        need = L.sdf_cell_rows_backward_scratch_bytes(cells, 4, count)
        return L.sdf_cell_rows_backward(type, grad, 4, table, 4, cells, 4, 0, ids, count, None,
                                        1.0, tg, wg, scratch, need if nbytes is None else nbytes,
                                        None)

    _refused(back(type=9), b"unknown element type 9")
    _refused(back(grad=None), b"NULL pointer")
    _refused(back(wg=p), b"NULL pointer")
    _refused(back(scratch=None), b"NULL pointer")
    _refused(back(nbytes=8), b"scratch must hold")
    _refused(back(scratch=p + 16), b"256-byte aligned")
    assert back(tg=None) == 0


def test_c_distill():
    L = _lib.lib()
    keep, p = _memory()

    def call(type=0, z=p, rows=3, labels=7, id_type=0, j=p, tt=0, t=p, top=2, temp=1.0, reduction=2,
             loss=p, scratch=p, nbytes=1 << 20):
        return L.sdf_distill(type, z, rows, labels, labels, id_type, j, tt, t, top, temp, None,
                             reduction, None, loss, None, None, scratch, nbytes, None)

    _refused(call(type=-1), b"unknown element type -1")
    _refused(call(tt=5), b"unknown element type 5")
    _refused(call(id_type=3), b"unknown id type 3")
    _refused(call(labels=0), b"1 to 2^31 - 1 labels")
    _refused(call(labels=1 << 31), b"1 to 2^31 - 1 labels")
    _refused(call(rows=1 << 31), b"fewer than 2^31 rows")
    _refused(call(top=1025), b"at most 1024 teacher logits")
    for bad in (0.0, float("nan"), float("inf")):
        _refused(call(temp=bad), b"temperature must be positive and finite")
    _refused(call(reduction=3), b"unknown reduction 3")
    _refused(call(z=None), b"NULL pointer")
    _refused(call(j=None), b"NULL pointer")
    _refused(call(loss=None), b"NULL pointer")
    _refused(call(z=p + 2), b"aligned to their elements")
    _refused(call(scratch=None), b"scratch must hold")
    _refused(call(nbytes=4), b"scratch must hold")
    _refused(call(scratch=p + 8), b"256-byte aligned")

    def back(grad=p, stats=p, out=p, rows=3, top=2):
        return L.sdf_distill_backward(0, p, rows, 7, 7, 0, p, 0, p, top, 1.0, None, 0, grad, stats,
                                      out, None)

    _refused(back(grad=None), b"NULL pointer")
    _refused(back(stats=None), b"NULL pointer")
    _refused(back(out=None), b"NULL pointer")
    _refused(back(top=2000), b"at most 1024 teacher logits")
    assert back(rows=0, out=None) == 0


def test_c_label_log_probs():
    L = _lib.lib()
    keep, p = _memory()

    def call(type=0, z=p, rows=3, labels=7, y=p, top=2, temp=1.0, lp=p, best=p, scratch=p,
             nbytes=1 << 20):
        return L.sdf_label_log_probs(type, z, rows, labels, labels, 0, y, top, temp, lp, p, best, p,
                                     None, scratch, nbytes, None)

    _refused(call(type=7), b"unknown element type 7")
    _refused(call(top=65), b"at most 64 best labels")
    _refused(call(temp=-1.0), b"temperature must be positive and finite")
    _refused(call(y=None), b"NULL pointer")
    _refused(call(lp=None), b"NULL pointer")
    _refused(call(best=None), b"NULL pointer")
    _refused(call(nbytes=0), b"scratch must hold")
    _refused(call(scratch=p + 8), b"256-byte aligned")
    assert call(rows=0) == 0

    def back(z=p, entropy=p, out=p):
        return L.sdf_label_log_probs_backward(0, z, 3, 7, 7, 0, p, 1.0, entropy, p, None, None, out,
                                              None)

    _refused(back(z=None), b"NULL pointer")
    _refused(back(entropy=None), b"NULL pointer")
    _refused(back(out=None), b"NULL pointer")


def test_temperature_without_a_reciprocal():
    z, j = torch.zeros(3, 7), ids(3, 2)
    for bad in (1e-39, 1e-60):
        with pytest.raises(RuntimeError, match="temperature must be positive and finite"):
            sdfoam_amd.distill_loss(z, j, torch.zeros(3, 2), bad)
        with pytest.raises(RuntimeError, match="temperature must be positive and finite"):
            sdfoam_amd.label_log_probs(z, ids(3), 0, bad)
    keep, p = _memory()
    _refused(_lib.lib().sdf_label_log_probs(0, p, 3, 7, 7, 0, p, 0, 1e-39, p, p, None, None, None, p,
                                            1024, None), b"temperature must be positive and finite")


def test_tangents_are_refused():
    """A dual tensor has requires_grad False; its tangent must not be lost without a word,
    with the recording of gradients on or off.  The same tensors pass outside of a level and
    as primals."""
    from torch.autograd import forward_ad

    table, z, j, t, w = torch.zeros(5, 4), torch.zeros(3, 7), ids(3, 2), torch.zeros(3, 2), torch.ones(3)
    calls = {  # arguments that derivatives reach, by name
        "cell_rows": (lambda x: sdfoam_amd.cell_rows(x["table"], ids(3), x["weight"]),
                      {"table": table, "weight": w}),
        "cell_rows_backward": (
            lambda x: sdfoam_amd.cell_rows_backward(x["rows_grad"], ids(3), 5, x["weight"],
                                                    table=x["table"]),
            {"rows_grad": torch.zeros(3, 4), "weight": w, "table": table}),
        "distill_loss": (
            lambda x: sdfoam_amd.distill_loss(x["logits"], j, x["teacher_logits"], 1.0,
                                              x["row_weight"]),
            {"logits": z, "teacher_logits": t, "row_weight": w}),
        "distill_loss_and_grad": (
            lambda x: sdfoam_amd.distill_loss_and_grad(x["logits"], j, x["teacher_logits"], 1.0,
                                                       x["row_weight"], "none", x["loss_grad"]),
            {"logits": z, "teacher_logits": t, "row_weight": w, "loss_grad": w.clone()}),
        "label_log_probs": (lambda x: sdfoam_amd.label_log_probs(x["logits"], ids(3)),
                            {"logits": z}),
    }
    for call, (f, plain) in calls.items():
        for name in plain:
            for enabled in (True, False):
                with forward_ad.dual_level(), torch.set_grad_enabled(enabled):
                    dual = forward_ad.make_dual(plain[name], torch.ones_like(plain[name]))
                    with pytest.raises(RuntimeError, match=f"{call} has no forward-mode "
                                                           f"derivative for {name}: detach it"):
                        f({**plain, name: dual})
                    with pytest.raises(RuntimeError, match="must be on CUDA device"):
                        f({**plain, name: dual.detach()})
        with pytest.raises(RuntimeError, match="must be on CUDA device"):
            f(plain)


@pytest.mark.parametrize("call", [sdfoam_amd.distill_loss, sdfoam_amd.distill_loss_and_grad])
def test_distill_refuses_what_it_has_no_gradient_for(call):
    z, j, t, w = torch.zeros(3, 7), ids(3, 2), torch.zeros(3, 2), torch.ones(3)
    for name, leaf in (("teacher_logits", t), ("row_weight", w)):
        args = {"teacher_logits": t, "row_weight": w, name: leaf.clone().requires_grad_()}
        with pytest.raises(RuntimeError, match=f"{call.__name__} has no gradient for {name}: detach it"):
            call(z, j, **args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="logits must be on CUDA device"):
            call(z, j, **args)
    with pytest.raises(RuntimeError, match="logits must be on CUDA device"):
        call(z.requires_grad_(), j, t, 1.0, w)


def test_c_weights_gradient_takes_no_scratch():
    L = _lib.lib()
    keep, p = _memory()

    def back(table_grad, scratch, nbytes):  # of no ids: nothing is launched for the weights
        return L.sdf_cell_rows_backward(0, p, 4, p, 4, 5, 4, 0, p, 0, None, 1.0, table_grad, p, scratch,
                                        nbytes, None)

    assert back(None, None, 0) != _lib.SDF_E_INVALID
    _refused(back(p, None, 1 << 20), b"NULL pointer")
    _refused(back(p, p, 0), b"scratch must hold")


@pytest.mark.parametrize("width", [(1 << 18) + 1, (1 << 32) + 4])
def test_rows_too_wide(width):
    """Also where the width's lower 32 bits alone would be a width."""
    wide = torch.zeros(1, 1).expand(1, width)
    with pytest.raises(RuntimeError, match=r"cell_rows takes rows of at most 2\^18 elements"):
        sdfoam_amd.cell_rows(wide, ids(1))
    with pytest.raises(RuntimeError, match=r"cell_rows_backward takes rows of at most 2\^18 elements"):
        sdfoam_amd.cell_rows_backward(wide, ids(1), 3)
    fits = wide[:, :1 << 18]
    with pytest.raises(RuntimeError, match="table must be on CUDA device"):
        sdfoam_amd.cell_rows(fits, ids(1))
    with pytest.raises(RuntimeError, match="rows_grad must be on CUDA device"):
        sdfoam_amd.cell_rows_backward(fits, ids(1), 3)

"""Root-mean-square norm with the residual's addition on the B200 kernels,
over the C ABI (``va_rms_norm_*``).

``h = x + residual``, ``y = h / sqrt(mean(h²) + eps) · w`` over the last
dimension, in one pass; ``y`` in the input's type (bf16, f16, f32) or in 8
bits with scales.  No CPU path.
"""
from __future__ import annotations

import torch

from . import _launch

_SFX = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
_FWD, _F8, _BWD = ({t: f"va_rms_norm_{kind}_{s}" for t, s in _SFX.items()} for kind in ("fwd", "fwd_f8", "bwd"))


def _rows(t):
    """(device index, rows, cols) of the tensor that the others are held to."""
    index, shape = t.get_device(), t.shape
    if index < 0 or t.dtype not in _SFX or not shape or not t.is_contiguous():
        raise ValueError("rows must be contiguous CUDA tensors of bf16, f16 or f32")
    cols = shape[-1]
    return index, (t.numel() // cols if cols else 0), cols


def _same(t, name, like, index):
    if t.dtype is not like.dtype or t.get_device() != index or t.shape != like.shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, with the shape, type and device of the other rows")
    return t.data_ptr()


def _weight(w, x, index, cols):
    f32 = w.dtype is torch.float32
    if not (f32 or w.dtype is x.dtype) or w.get_device() != index or w.shape != (cols,) or not w.is_contiguous():
        raise ValueError("w must be a contiguous CUDA [cols] tensor of the rows' type or f32")
    return w.data_ptr(), f32


def _apart(name, p, nbytes, *others):
    """Rows shifted against each other would be read and written by different blocks; exactly in place is fine."""
    for o in others:
        if o is not None and o != p and abs(o - p) < nbytes:
            raise ValueError(f"{name} overlaps another tensor of the call, and not exactly in place")
    return p


def _sum(x, residual, out_h, index):
    """Addresses of the residual and of the tensor for the sum, and that tensor (x itself without either)."""
    pr = None if residual is None else _same(residual, "residual", x, index)
    if out_h is not None:
        return pr, _apart("out_h", _same(out_h, "out_h", x, index), x.nbytes, x.data_ptr(), pr), out_h
    if residual is None:
        return None, None, x
    h = torch.empty_like(x)
    return pr, h.data_ptr(), h


def rms_norm_forward(x, w, residual=None, eps: float = 1e-6, out=None, out_h=None, stream=None):
    """``(y, h)``; without a residual ``h`` is ``x`` itself.  ``out_h`` may be
    ``x`` or ``residual`` (the sum is then updated in place), and ``out`` either
    that is not ``out_h``."""
    if stream is not None:
        with _launch.on(stream, x.get_device()):
            return rms_norm_forward(x, w, residual, eps, out, out_h)
    index, rows, cols = _rows(x)
    pw, w32 = _weight(w, x, index, cols)
    pr, ph, h = _sum(x, residual, out_h, index)
    px = x.data_ptr()
    if out is None:
        y = torch.empty_like(x)
        py = y.data_ptr()
    else:
        y, py = out, _apart("out", _same(out, "out", x, index), x.nbytes, px, pr, ph)
        if py == ph and rows:
            raise ValueError("out and out_h are one tensor")
    _launch.run(_FWD[x.dtype], index, px, pr, pw, w32, ph, py, rows, cols, eps)
    return y, h


def rms_norm_forward_f8(x, w, residual=None, eps: float = 1e-6, group: int = 0, out_h=None, stream=None):
    """``(q, scale, h)``: ``q`` float8_e4m3fn of x's shape and ``scale`` f32
    ``[..., cols/group]`` (``group`` 0: one for each row) with
    ``y ≈ q · scale`` and the largest magnitude of each group at 448."""
    if stream is not None:
        with _launch.on(stream, x.get_device()):
            return rms_norm_forward_f8(x, w, residual, eps, group, out_h)
    index, rows, cols = _rows(x)
    if group < 0 or (group and cols % group):
        raise ValueError(f"{cols} columns do not split into groups of {group}")
    pw, w32 = _weight(w, x, index, cols)
    pr, ph, h = _sum(x, residual, out_h, index)
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
    scale = x.new_empty((*x.shape[:-1], cols // group if group else 1), dtype=torch.float32)
    _launch.run(_F8[x.dtype], index, x.data_ptr(), pr, pw, w32, ph, q.data_ptr(), scale.data_ptr(), rows, cols, group,
                eps)
    return q, scale, h


def rms_norm_backward(grad_y, h, w, eps: float = 1e-6, grad_h=None, workspace=None, stream=None):
    """``(grad, grad_w)``: the gradient of ``x`` and of ``residual`` alike
    (with ``grad_h``, the gradient that reaches ``h`` itself, added), and
    f32 ``[cols]`` of the weight.  ``h`` is the sum that the forward returned.
    A ``workspace`` smaller than needed is not used."""
    if stream is not None:
        with _launch.on(stream, h.get_device()):
            return rms_norm_backward(grad_y, h, w, eps, grad_h, workspace)
    index, rows, cols = _rows(h)
    pw, w32 = _weight(w, h, index, cols)
    py = _same(grad_y, "grad_y", h, index)
    pg = None if grad_h is None else _same(grad_h, "grad_h", h, index)
    if workspace is not None and (workspace.get_device() != index or not workspace.is_contiguous()):
        raise ValueError("workspace must be a contiguous CUDA tensor on the rows' device")
    need = _launch.entry("va_rms_norm_bwd_workspace_bytes")(rows, cols)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = h.new_empty(need, dtype=torch.uint8)
    grad = torch.empty_like(h)
    grad_w = h.new_empty(cols, dtype=torch.float32)
    _launch.run(_BWD[h.dtype], index, py, h.data_ptr(), pw, w32, pg, grad.data_ptr(), grad_w.data_ptr(), rows, cols,
                eps, workspace.data_ptr(), need)
    return grad, grad_w

"""Root-mean-square norm with the residual's addition on the B200 kernels,
over the C ABI (``va_rms_norm_*``).

``h = x + residual``, ``y = h / sqrt(mean(h²) + eps) · w`` over the last
dimension, in one pass; ``y`` in the input's type (bf16, f16, f32) or in 8
bits with scales.  No CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .psa import _stream

_SFX = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}


def _check(t, name, like=None):
    if not t.is_cuda or t.dtype not in _SFX or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA tensor of bf16, f16 or f32")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the shape, type and device of the other rows")
    return t.data_ptr()


def _weight(w, x):
    if not w.is_cuda or w.device != x.device or w.dtype not in (x.dtype, torch.float32) or not w.is_contiguous() \
            or x.dim() == 0 or w.shape != x.shape[-1:]:
        raise ValueError("w must be a contiguous CUDA [cols] tensor of the rows' type or f32")
    return w.data_ptr(), int(w.dtype == torch.float32)


def _sizes(x):
    cols = x.shape[-1]
    return (x.numel() // cols if cols else 0), cols


def rms_norm_forward(x, w, residual=None, eps: float = 1e-6, out=None, out_h=None, stream=None):
    """``(y, h)``; without a residual ``h`` is ``x`` itself.  ``out_h`` may be
    ``x`` or ``residual`` (the sum is then updated in place)."""
    px, (pw, w32) = _check(x, "x"), _weight(w, x)
    pr = None if residual is None else _check(residual, "residual", x)
    y = torch.empty_like(x) if out is None else out
    h = out_h if out_h is not None else None if residual is None else torch.empty_like(x)
    rows, cols = _sizes(x)
    _lib.call("va_rms_norm_fwd_" + _SFX[x.dtype], px, pr, pw, w32, None if h is None else _check(h, "out_h", x),
              _check(y, "out", x), rows, cols, eps, _stream(stream))
    return y, x if h is None else h


def rms_norm_forward_f8(x, w, residual=None, eps: float = 1e-6, group: int = 0, out_h=None, stream=None):
    """``(q, scale, h)``: ``q`` float8_e4m3fn of x's shape and ``scale`` f32
    ``[..., cols/group]`` (``group`` 0: one for each row) with
    ``y ≈ q · scale`` and the largest magnitude of each group at 448."""
    px, (pw, w32) = _check(x, "x"), _weight(w, x)
    pr = None if residual is None else _check(residual, "residual", x)
    h = out_h if out_h is not None else None if residual is None else torch.empty_like(x)
    rows, cols = _sizes(x)
    if group < 0 or (group and cols % group):
        raise ValueError(f"{cols} columns do not split into groups of {group}")
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(*x.shape[:-1], cols // group if group else 1, dtype=torch.float32, device=x.device)
    _lib.call("va_rms_norm_fwd_f8_" + _SFX[x.dtype], px, pr, pw, w32, None if h is None else _check(h, "out_h", x),
              q.data_ptr(), scale.data_ptr(), rows, cols, group, eps, _stream(stream))
    return q, scale, x if h is None else h


def rms_norm_backward(grad_y, h, w, eps: float = 1e-6, grad_h=None, workspace=None, stream=None):
    """``(grad, grad_w)``: the gradient of ``x`` and of ``residual`` alike
    (with ``grad_h``, the gradient that reaches ``h`` itself, added), and
    f32 ``[cols]`` of the weight.  ``h`` is the sum that the forward returned."""
    ph, (pw, w32) = _check(h, "h"), _weight(w, h)
    pg = None if grad_h is None else _check(grad_h, "grad_h", h)
    rows, cols = _sizes(h)
    need = int(_lib.lib().va_rms_norm_bwd_workspace_bytes(rows, cols))
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=h.device)
    grad = torch.empty_like(h)
    grad_w = torch.empty(cols, dtype=torch.float32, device=h.device)
    _lib.call("va_rms_norm_bwd_" + _SFX[h.dtype], _check(grad_y, "grad_y", h), ph, pw, w32, pg, grad.data_ptr(),
              grad_w.data_ptr(), rows, cols, eps, workspace.data_ptr(), workspace.numel(), _stream(stream))
    return grad, grad_w

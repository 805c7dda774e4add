"""Attention over packed sequences of different lengths on the B200 kernels,
over the C ABI (``va_packed_*``): causal or full, grouped heads, whole prompts,
single tokens over cached keys, and the gradient.

The sequences' tokens lie one after another in ``q [total_q, heads, dim]`` and
``k, v [total_k, kv_heads, dim]`` (bf16 or f16; rows and heads may be strided,
e.g. slices of a packed QKV product); ``cu_seqlens`` (int32 ``[n + 1]`` on the
device) say where each begins.  A ``PackedPlan`` turns the offsets into the
kernels' work lists on the GPU; build it once a batch and share it between
layers.  No CPU path.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .psa import _stream

_SFX = {torch.bfloat16: "bf16", torch.float16: "f16"}
_Strides6 = C.c_int64 * 6
_Strides14 = C.c_int64 * 14


def cu_seqlens(lengths, device="cuda") -> torch.Tensor:
    """int32 ``[n + 1]`` offsets of sequences of the given lengths (host integers)."""
    off = [0]
    for n in lengths:
        if n < 0:
            raise ValueError(f"a length of {n}")
        off.append(off[-1] + int(n))
    return torch.tensor(off, dtype=torch.int32).to(device)


class PackedPlan:
    """Work lists of packed-sequence attention for one batch's sequences and
    one head layout (with the kernels' partial results: calls that share a
    plan must not overlap on the GPU).  ``cu_q`` and ``cu_k`` stay on the
    device and are read on ``stream``; ``check()`` raises if they were not
    ascending offsets from 0 to the totals."""

    def __init__(self, cu_q, cu_k, total_q: int, total_k: int, num_heads: int, num_kv_heads: int, head_dim: int,
                 causal: bool = False, training: bool = False, stream=None):
        for name, t in (("cu_q", cu_q), ("cu_k", cu_k)):
            if not t.is_cuda or t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] < 2 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous CUDA int32 [sequences + 1] tensor")
        if cu_q.shape != cu_k.shape or cu_q.device != cu_k.device:
            raise ValueError("cu_q and cu_k must have the same sequences and device")
        self.sizes = (cu_q.shape[0] - 1, total_q, total_k, num_heads, num_kv_heads, head_dim, int(causal),
                      int(training))
        need = _lib.lib().va_packed_plan_bytes(*self.sizes)
        if need == 0:
            raise _lib.VisionAttnError("va_packed_plan_bytes", 1,
                                       _lib.lib().va_get_last_error_string().decode(errors="replace"))
        self.buf = torch.empty(need, dtype=torch.uint8, device=cu_q.device)
        self.nbytes = need
        _lib.call("va_packed_plan_build", cu_q.data_ptr(), cu_k.data_ptr(), *self.sizes, self.buf.data_ptr(), need,
                  _stream(stream))

    def check(self, stream=None):
        """Raises if the offsets were out of order or range (synchronises)."""
        bad = C.c_int(0)
        _lib.call("va_packed_plan_status", self.buf.data_ptr(), self.sizes[7], C.byref(bad), _stream(stream))
        if bad.value:
            raise ValueError("cu_q or cu_k are not ascending offsets from 0 to the number of tokens")


def _heads(t, name, shape, like):
    if not t.is_cuda or t.dtype not in _SFX or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be a CUDA bf16 or f16 tensor of q's type and device")
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: a head's dimensions must be contiguous")
    return t.stride(0), t.stride(1)


def _dense(t, name, shape, dtype, device):
    if not t.is_cuda or t.dtype != dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA {dtype} tensor of {shape}")
    return t


def _inputs(q, k, v, plan):
    _, tq, tk, h, hk, d, _, _ = plan.sizes
    if plan.buf.device != q.device:
        raise ValueError("the plan is on another device")
    return _Strides6(*_heads(q, "q", (tq, h, d), q), *_heads(k, "k", (tk, hk, d), q), *_heads(v, "v", (tk, hk, d), q))


def packed_attention_forward(q, k, v, plan: PackedPlan, scale: float | None = None, out=None, lse=None, stream=None):
    """``(out [total_q, heads, dim], lse f32 [heads, total_q])``; ``scale``
    defaults to dim^-½.  A query that sees no key has out 0 and lse −∞."""
    st = _inputs(q, k, v, plan)
    _, tq, _, h, _, d, _, _ = plan.sizes
    out = torch.empty((tq, h, d), dtype=q.dtype, device=q.device) if out is None else \
        _dense(out, "out", (tq, h, d), q.dtype, q.device)
    lse = torch.empty((h, tq), dtype=torch.float32, device=q.device) if lse is None else \
        _dense(lse, "lse", (h, tq), torch.float32, q.device)
    _lib.call("va_packed_attention_fwd_" + _SFX[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
              lse.data_ptr(), st, *plan.sizes, d ** -0.5 if scale is None else scale, plan.buf.data_ptr(), plan.nbytes,
              _stream(stream))
    return out, lse


def packed_attention_backward(grad_out, q, k, v, out, lse, plan: PackedPlan, scale: float | None = None, grads=None,
                              stream=None):
    """``(grad_q, grad_k, grad_v)`` from the forward's inputs and results; the
    plan must be built with ``training=True``.  ``grads``: three tensors to
    write, which may be slices of one packed gradient."""
    st = _inputs(q, k, v, plan)
    _, tq, tk, h, hk, d, _, training = plan.sizes
    if not training:
        raise ValueError("the plan was not built with training=True")
    _dense(out, "out", (tq, h, d), q.dtype, q.device)
    _dense(lse, "lse", (h, tq), torch.float32, q.device)
    so = _heads(grad_out, "grad_out", (tq, h, d), q)
    if grads is None:
        grads = tuple(torch.empty(s, dtype=q.dtype, device=q.device) for s in ((tq, h, d), (tk, hk, d), (tk, hk, d)))
    gq, gk, gv = grads
    sg = (*_heads(gq, "grad_q", (tq, h, d), q), *_heads(gk, "grad_k", (tk, hk, d), q),
          *_heads(gv, "grad_v", (tk, hk, d), q))
    _lib.call("va_packed_attention_bwd_" + _SFX[q.dtype], grad_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
              out.data_ptr(), lse.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), _Strides14(*st, *so, *sg),
              *plan.sizes, d ** -0.5 if scale is None else scale, plan.buf.data_ptr(), plan.nbytes, _stream(stream))
    return gq, gk, gv

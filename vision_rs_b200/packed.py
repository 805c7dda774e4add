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
from functools import lru_cache

import torch

from . import _launch, _lib

_FWD = {torch.bfloat16: "va_packed_attention_fwd_bf16", torch.float16: "va_packed_attention_fwd_f16"}
_BWD = {torch.bfloat16: "va_packed_attention_bwd_bf16", torch.float16: "va_packed_attention_bwd_f16"}
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


@lru_cache(maxsize=256)
def _plan_bytes(*sizes) -> int:
    need = _lib.lib().va_packed_plan_bytes(*sizes)
    if need == 0:
        raise _lib.VisionAttnError("va_packed_plan_bytes", 1,
                                   _lib.lib().va_get_last_error_string().decode(errors="replace"))
    return need


class PackedPlan:
    """Work lists of packed-sequence attention for one batch's sequences and
    one head layout, with the kernels' partial results: calls that share a
    plan follow one another on the GPU.  A call on another stream than the
    last one's waits for that stream's work so far; within a capture the
    caller orders the streams (and a graph that holds a plan's calls must not
    overlap other calls with it).  With ``used_k`` (int32 ``[n]`` on the
    device) only that many of a sequence's key rows hold keys: a cache with
    room to grow.  The offsets stay on the device and are read on ``stream``; ``check()`` raises if they were not
    ascending offsets from 0 to the totals."""

    def __init__(self, cu_q, cu_k, total_q: int, total_k: int, num_heads: int, num_kv_heads: int, head_dim: int,
                 causal: bool = False, training: bool = False, used_k=None, stream=None):
        if stream is not None:
            with _launch.on(stream, cu_q.get_device()):
                return self.__init__(cu_q, cu_k, total_q, total_k, num_heads, num_kv_heads, head_dim, causal, training,
                                     used_k)
        index = cu_q.get_device()
        for t in (cu_q, cu_k):
            if t.dtype is not torch.int32 or t.dim() != 1 or t.get_device() != index or index < 0 \
                    or not t.is_contiguous():
                raise ValueError("cu_q and cu_k must be contiguous int32 [sequences + 1] tensors of one CUDA device")
        n = cu_q.shape[0] - 1
        if n < 1 or cu_k.shape[0] != n + 1:
            raise ValueError("cu_q and cu_k must have the same sequences, one at least")
        if used_k is not None and (used_k.dtype is not torch.int32 or used_k.get_device() != index
                                   or used_k.shape != (n,) or not used_k.is_contiguous() or training):
            raise ValueError("used_k must be a contiguous int32 [sequences] tensor beside cu_k, and not for training")
        self.sizes = sizes = (n, total_q, total_k, num_heads, num_kv_heads, head_dim, int(causal), int(training))
        self.nbytes = need = _plan_bytes(*sizes)
        self.index = index
        self.buf = cu_q.new_empty(need, dtype=torch.uint8)
        self.ptr = self.buf.data_ptr()
        self.stream = self.home = _launch.raw_stream(index)  # of the last call, and of the buffer
        _launch.run("va_packed_plan_build", index, cu_q.data_ptr(), cu_k.data_ptr(),
                    None if used_k is None else used_k.data_ptr(), *sizes, self.ptr, need)

    def check(self, stream=None):
        """Raises if the offsets were out of order or range (synchronises)."""
        if stream is not None:
            with _launch.on(stream, self.index):
                return self.check()
        if _launch.raw_stream(self.index) != self.stream:
            self._move()
        bad = C.c_int(0)
        _launch.run("va_packed_plan_status", self.index, self.ptr, self.sizes[7], C.byref(bad))
        if bad.value:
            raise ValueError("cu_q or cu_k are not ascending offsets from 0 to the number of tokens")

    def _move(self):
        """Before a call on another stream than the last one's."""
        now = torch.cuda.current_stream(self.index)
        if now.cuda_stream != self.home:
            self.buf.record_stream(now)  # the buffer must outlive the call
        with _launch.on(self.stream or torch.cuda.default_stream(self.index), self.index):
            last, captured = torch.cuda.current_stream(self.index), torch.cuda.is_current_stream_capturing()
        with torch.cuda.device(self.index):
            if captured or torch.cuda.is_current_stream_capturing():
                return
        now.wait_stream(last)
        self.stream = now.cuda_stream


def _heads(t, name, dtype, index, shape):
    if t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{name} must be a CUDA tensor of q's type on the plan's device")
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    row, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{name}: a head's dimensions must be contiguous")
    return row, head


def _dense(t, name, shape, dtype, index):
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA {dtype} tensor of {shape}")
    return t


def _refuse_overlap(written, read):
    """Results must not lie over what other blocks, or a later kernel, of the call still read.  Each: (tensor, shape,
    (row, head) strides), whose ends are compared first (small calls are paced by the host)."""
    lo, hi = 1 << 64, 0
    for t, (n, heads, d), (row, head) in written:
        if n:
            p = t.data_ptr()
            lo, hi = min(lo, p), max(hi, p + 2 * ((n - 1) * row + (heads - 1) * head + d))
    for t, (n, heads, d), (row, head) in read:
        p = t.data_ptr()
        if p < hi and lo < p + 2 * ((n - 1) * row + (heads - 1) * head + d) \
                and any(_launch.overlap(w, t) for w, _, _ in written):
            raise ValueError("a result overlaps an input of the call")


def packed_attention_forward(q, k, v, plan: PackedPlan, scale: float | None = None, out=None, lse=None, stream=None):
    """``(out [total_q, heads, dim], lse f32 [heads, total_q])``; ``scale``
    (positive) defaults to dim^-½.  A query that sees no key has out 0 and lse
    −∞.  ``out`` may be q itself where that is contiguous, but not overlap the
    inputs in another way."""
    if stream is not None:
        with _launch.on(stream, plan.index):
            return packed_attention_forward(q, k, v, plan, scale, out, lse)
    sizes, index, dtype = plan.sizes, plan.index, q.dtype
    name = _FWD.get(dtype)
    if name is None:
        raise ValueError("q must be bf16 or f16")
    _, tq, tk, h, hk, d, _, _ = sizes
    sq, sk = (tq, h, d), (tk, hk, d)
    qs, ks, vs = _heads(q, "q", dtype, index, sq), _heads(k, "k", dtype, index, sk), _heads(v, "v", dtype, index, sk)
    if out is None:
        out = q.new_empty_strided(sq, (h * d, d, 1))
    else:
        _dense(out, "out", sq, dtype, index)
        in_place = out.data_ptr() == q.data_ptr() and qs == (h * d, d)  # a tile's queries are read by its own unit alone
        _refuse_overlap([(out, sq, (h * d, d))], [(k, sk, ks), (v, sk, vs)] + ([] if in_place else [(q, sq, qs)]))
    lse = q.new_empty((h, tq), dtype=torch.float32) if lse is None else _dense(lse, "lse", (h, tq), torch.float32, index)
    if _launch.raw_stream(index) != plan.stream:
        plan._move()
    _launch.run(name, index, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                _Strides6(*qs, *ks, *vs), *sizes, d ** -0.5 if scale is None else scale,
                plan.ptr, plan.nbytes)
    return out, lse


def packed_attention_backward(grad_out, q, k, v, out, lse, plan: PackedPlan, scale: float | None = None, grads=None,
                              stream=None):
    """``(grad_q, grad_k, grad_v)`` from the forward's inputs and results; the
    plan must be built with ``training=True``.  ``grads``: three tensors to
    write, which may be slices of one packed gradient, but not lie over the
    inputs (dQ is written before dK's kernel reads q)."""
    if stream is not None:
        with _launch.on(stream, plan.index):
            return packed_attention_backward(grad_out, q, k, v, out, lse, plan, scale, grads)
    sizes, index, dtype = plan.sizes, plan.index, q.dtype
    name = _BWD.get(dtype)
    if name is None:
        raise ValueError("q must be bf16 or f16")
    _, tq, tk, h, hk, d, _, training = sizes
    if not training:
        raise ValueError("the plan was not built with training=True")
    sq, sk = (tq, h, d), (tk, hk, d)
    _dense(out, "out", sq, dtype, index)
    _dense(lse, "lse", (h, tq), torch.float32, index)
    gq, gk, gv = (q.new_empty(sq), k.new_empty(sk), v.new_empty(sk)) if grads is None else grads
    qs, ks, vs = _heads(q, "q", dtype, index, sq), _heads(k, "k", dtype, index, sk), _heads(v, "v", dtype, index, sk)
    gos, gqs = _heads(grad_out, "grad_out", dtype, index, sq), _heads(gq, "grad_q", dtype, index, sq)
    gks, gvs = _heads(gk, "grad_k", dtype, index, sk), _heads(gv, "grad_v", dtype, index, sk)
    if grads is not None:
        _refuse_overlap([(gq, sq, gqs), (gk, sk, gks), (gv, sk, gvs)],
                        [(grad_out, sq, gos), (q, sq, qs), (k, sk, ks), (v, sk, vs), (out, sq, (h * d, d))])
    strides = _Strides14(*qs, *ks, *vs, *gos, *gqs, *gks, *gvs)
    if _launch.raw_stream(index) != plan.stream:
        plan._move()
    _launch.run(name, index, grad_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                lse.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), strides, *sizes,
                d ** -0.5 if scale is None else scale, plan.ptr, plan.nbytes)
    return gq, gk, gv

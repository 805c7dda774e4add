"""Rotary positions on the B200 kernels, over the C ABI (``va_rotary_*``).

``rotary_forward`` turns the queries and keys of packed token sequences
(``[tokens, heads, head_dim]``, bf16, f16 or f32; rows and heads may be
strided, e.g. slices of a packed QKV product) by the angles
``positions[t] · inv_freq[i]``; ``rotary_backward`` turns gradients back.
``rotary_frequencies`` makes ``inv_freq``, for long contexts too.  No CPU path.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _launch

_ENTRY = {torch.bfloat16: "va_rotary_bf16", torch.float16: "va_rotary_f16", torch.float32: "va_rotary_f32"}
_POSITION = {torch.int32: 4, torch.int64: 8}  # bytes
_Strides = C.c_int64 * 8


def rotary_frequencies(rot_dim: int, base: float = 10000.0, stretch: float = 1.0, trained_length: int | None = None,
                       slow_turns: float = 1.0, fast_turns: float = 32.0, device="cuda") -> torch.Tensor:
    """f64 ``[rot_dim/2]`` radians per position: ``base^(-2i/rot_dim)``.

    ``stretch`` > 1 lets a model see contexts that many times longer than it
    was trained on.  Without ``trained_length`` every frequency is divided by
    it (positions interpolated).  With it, a pair that makes fewer than
    ``slow_turns`` turns over the trained length is divided, one with more
    than ``fast_turns`` is kept, and those between are blended linearly."""
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError(f"rot_dim must be positive and even, got {rot_dim}")
    if not base > 0 or not stretch > 0:
        raise ValueError("base and stretch must be positive")
    inv = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    if trained_length is None:
        inv = inv / stretch
    else:
        if not fast_turns > slow_turns:
            raise ValueError("fast_turns must be above slow_turns")
        turns = trained_length * inv / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / stretch)
    return inv.to(device)


def _heads(t, name, dtype, index):
    if t.dtype is not dtype or t.get_device() != index or t.dim() != 3:
        raise ValueError(f"{name} must be a CUDA [tokens, heads, head_dim] tensor of q's type and device")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"{name}: a head's dimensions must be contiguous")


def _apply(q, k, positions, inv_freq, interleaved, factor, backward, out, stream):
    if stream is not None:
        with _launch.on(stream):
            return _apply(q, k, positions, inv_freq, interleaved, factor, backward, out, None)
    dtype, index = q.dtype, q.get_device()
    name = _ENTRY.get(dtype)
    if name is None or index < 0:
        raise ValueError("q must be a CUDA tensor of bf16, f16 or f32")
    _heads(q, "q", dtype, index)
    tokens, hq, dim = shape = q.shape
    hk = 0
    if k is not None:
        _heads(k, "k", dtype, index)
        tk, hk, dk = k.shape
        if tk != tokens or dk != dim:
            raise ValueError("q and k must have the same tokens and head_dim")
    if positions.get_device() != index or positions.dtype not in _POSITION or positions.shape != (tokens,) \
            or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous CUDA int32 or int64 [tokens] tensor")
    if inv_freq.get_device() != index or inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 \
            or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous CUDA float64 [rot_dim/2] tensor")
    rot = 2 * inv_freq.shape[0]
    if rot > dim:
        raise ValueError(f"{rot} rotated dimensions in heads of {dim}")
    if out is None:
        qo = q.new_empty(shape)
        ko = None if k is None else k.new_empty(k.shape)
    else:
        qo, ko = out
        if (k is None) != (ko is None):
            raise ValueError("outputs must have the inputs' shapes")
        for o, x in ((qo, q), (ko, k)):
            if o is not None:
                _heads(o, "an output", dtype, index)
                if o.shape != x.shape:
                    raise ValueError("outputs must have the inputs' shapes")
    a, b, _ = q.stride()
    e, f, _ = qo.stride()
    if k is None:
        strides, pk, pko = _Strides(a, b, 0, 0, e, f, 0, 0), None, None
    else:
        c, d, _ = k.stride()
        g, h, _ = ko.stride()
        strides, pk, pko = _Strides(a, b, c, d, e, f, g, h), k.data_ptr(), ko.data_ptr()
    _launch.run(name, index, q.data_ptr(), pk, qo.data_ptr(), pko, strides, positions.data_ptr(),
                _POSITION[positions.dtype], inv_freq.data_ptr(), tokens, hq, hk, dim, rot, int(interleaved), backward,
                factor)
    return qo, ko


def rotary_forward(q, k, positions, inv_freq, interleaved: bool = False, factor: float = 1.0, out=None, stream=None):
    """Turned ``(q, k)``; ``k`` may be None.  ``factor`` multiplies the turned
    dimensions.  ``out``: a pair of tensors to write, which may be ``(q, k)``
    themselves."""
    return _apply(q, k, positions, inv_freq, interleaved, factor, 0, out, stream)


def rotary_backward(grad_q, grad_k, positions, inv_freq, interleaved: bool = False, factor: float = 1.0, out=None,
                    stream=None):
    """Gradients of ``rotary_forward``'s inputs from those of its outputs."""
    return _apply(grad_q, grad_k, positions, inv_freq, interleaved, factor, 1, out, stream)

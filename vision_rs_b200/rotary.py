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

from . import _lib
from .psa import _stream

_SFX = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
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


def _heads(t, name, ref=None):
    if not t.is_cuda or t.dim() != 3 or t.dtype not in _SFX:
        raise ValueError(f"{name} must be a CUDA [tokens, heads, head_dim] tensor of bf16, f16 or f32")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"{name}: a head's dimensions must be contiguous")
    if ref is not None and (t.dtype != ref.dtype or t.device != ref.device):
        raise ValueError(f"{name} must have q's type and device")
    return t


def _apply(q, k, positions, inv_freq, interleaved, factor, backward, out, stream):
    _heads(q, "q")
    tokens, hq, dim = q.shape
    if k is not None and (_heads(k, "k", q).shape[0] != tokens or k.shape[2] != dim):
        raise ValueError("q and k must have the same tokens and head_dim")
    if not positions.is_cuda or positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,) \
            or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous CUDA int32 or int64 [tokens] tensor")
    if not inv_freq.is_cuda or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous CUDA float64 [rot_dim/2] tensor")
    if 2 * inv_freq.shape[0] > dim:
        raise ValueError(f"{2 * inv_freq.shape[0]} rotated dimensions in heads of {dim}")
    if out is None:
        qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ko = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    else:
        qo, ko = out
        if _heads(qo, "q output", q).shape != q.shape or (k is None) != (ko is None) or \
                (k is not None and _heads(ko, "k output", q).shape != k.shape):
            raise ValueError("outputs must have the inputs' shapes")
    st = (q.stride(), (0, 0) if k is None else k.stride(), qo.stride(), (0, 0) if k is None else ko.stride())
    _lib.call("va_rotary_" + _SFX[q.dtype], q.data_ptr(), None if k is None else k.data_ptr(), qo.data_ptr(),
              None if k is None else ko.data_ptr(), _Strides(*(s for x in st for s in x[:2])), positions.data_ptr(),
              positions.element_size(), inv_freq.data_ptr(), tokens, hq, 0 if k is None else k.shape[1], dim,
              2 * inv_freq.shape[0], bool(interleaved), backward, factor, _stream(stream))
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

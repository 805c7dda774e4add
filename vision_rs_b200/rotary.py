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
    than ``fast_turns`` is kept, and those between are blended linearly in the
    number of turns.  (A blend that is linear in the pair's index instead,
    between the indices of the same two thresholds, gives the pairs between
    other frequencies: a model trained with that needs its own ``inv_freq``.)"""
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


def _refuse_overlap(q, k, qo, ko):
    """Other threads write a head's output while its input is read: only exactly in place is that the same element's."""
    outs, ins = [o for o in (qo, ko) if o is not None], [i for i in (q, k) if i is not None]
    if any(_launch.overlaps_itself(o) for o in outs):
        raise ValueError("an output's elements share memory")
    in_place = [o.data_ptr() == i.data_ptr() and o.stride() == i.stride() for o, i in zip(outs, ins)]
    if all(in_place):
        if len(outs) < 2 or not _launch.overlap(qo, ko):
            return
    elif not any(_launch.overlap(o, i) for n, o in enumerate(outs) for m, i in enumerate(ins) if n != m or not in_place[n]) \
            and not (len(outs) == 2 and _launch.overlap(qo, ko)):
        return
    raise ValueError("outputs may be the inputs exactly in place, but not overlap them or each other otherwise")


def _apply(q, k, positions, inv_freq, interleaved, factor, backward, out, stream):
    if stream is not None:
        with _launch.on(stream, q.get_device()):
            return _apply(q, k, positions, inv_freq, interleaved, factor, backward, out, None)
    dtype, index = q.dtype, q.get_device()
    name = _ENTRY.get(dtype)
    if name is None or index < 0 or q.dim() != 3:
        raise ValueError("q must be a CUDA [tokens, heads, head_dim] tensor of bf16, f16 or f32")
    shape = tokens, heads, dim = q.shape
    q_row, q_head, one = q.stride()
    pk = pko = ko = None
    kv_heads = k_row = k_head = ko_row = ko_head = 0
    if k is not None:
        if k.dtype is not dtype or k.get_device() != index or k.dim() != 3:
            raise ValueError("k must be a [tokens, heads, head_dim] tensor of q's type and device")
        k_tokens, kv_heads, k_dim = k_shape = k.shape
        k_row, k_head, k_one = k.stride()
        if k_tokens != tokens or k_dim != dim:
            raise ValueError("q and k must have the same tokens and head_dim")
        one = one if k_one == 1 else k_one
        pk = k.data_ptr()
    position_bytes = _POSITION.get(positions.dtype)
    if position_bytes is None or positions.get_device() != index or positions.shape != (tokens,) \
            or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous CUDA int32 or int64 [tokens] tensor")
    if inv_freq.dtype is not torch.float64 or inv_freq.get_device() != index or inv_freq.dim() != 1 \
            or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous CUDA float64 [rot_dim/2] tensor")
    rot = 2 * inv_freq.numel()
    if rot > dim:
        raise ValueError(f"{rot} rotated dimensions in heads of {dim}")
    if out is None:
        qo = torch.empty_like(q)  # dense
        if k is not None:
            ko = torch.empty_like(k)
    else:
        qo, ko = out
        if (k is None) != (ko is None) or qo.shape != shape or (ko is not None and ko.shape != k_shape):
            raise ValueError("outputs must have the inputs' shapes")
        for o in (qo, ko):
            if o is not None and (o.dtype is not dtype or o.get_device() != index):
                raise ValueError("outputs must have the inputs' type and device")
    qo_row, qo_head, o_one = qo.stride()
    one = one if o_one == 1 else o_one
    if ko is not None:
        ko_row, ko_head, o_one = ko.stride()
        one = one if o_one == 1 else o_one
        pko = ko.data_ptr()
    if one != 1 and dim > 1:
        raise ValueError("a head's dimensions must be contiguous")
    if out is not None:
        # (the usual case at once: slices of one packed product, in place; a token's heads in a row, q's beside k's)
        of_q, of_k = (heads - 1) * q_head + dim, (kv_heads - 1) * k_head + dim if kv_heads else 0
        apart = (pk - q.data_ptr()) // q.element_size() % max(q_row, 1) if kv_heads else of_q
        if not (qo is q and ko is k and q_head >= dim and (kv_heads == 0 or (k_row == q_row and k_head >= dim))
                and of_q <= apart <= q_row - of_k):
            _refuse_overlap(q, k, qo, ko)
    _launch.run(name, index, q.data_ptr(), pk, qo.data_ptr(), pko,
                _Strides(q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head), positions.data_ptr(),
                position_bytes, inv_freq.data_ptr(), tokens, heads, kv_heads, dim, rot, interleaved, backward, factor)
    return qo, ko


def rotary_forward(q, k, positions, inv_freq, interleaved: bool = False, factor: float = 1.0, out=None, stream=None):
    """Turned ``(q, k)``; ``k`` may be None.  ``factor`` multiplies the turned
    dimensions.  ``out``: a pair of tensors to write, which may be ``(q, k)``
    themselves, but not overlap them (or each other) in another way."""
    return _apply(q, k, positions, inv_freq, interleaved, factor, 0, out, stream)


def rotary_backward(grad_q, grad_k, positions, inv_freq, interleaved: bool = False, factor: float = 1.0, out=None,
                    stream=None):
    """Gradients of ``rotary_forward``'s inputs from those of its outputs."""
    return _apply(grad_q, grad_k, positions, inv_freq, interleaved, factor, 1, out, stream)

"""Launch helpers of the packed-sequence operators' Python side: bound C
entries, the raw stream of a device, and running a call on a given stream.

Small calls are paced by the host, so these avoid what costs microseconds a
call: looking an entry up by name, and building a stream object to read its
handle.
"""
from __future__ import annotations

import torch

from . import _lib

raw_stream = torch._C._cuda_getCurrentRawStream  # (device index) -> cudaStream_t of torch's current stream
_current_device = torch._C._cuda_getDevice
_entries: dict = {}


def entry(name: str):
    """The C entry ``name``, bound once."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.lib(), name)
    return fn


def run(name: str, index: int, *args) -> None:
    """Calls ``name(*args, stream)`` on torch's current stream of device ``index``; raises on a non-zero status."""
    fn = _entries.get(name) or entry(name)
    if index == _current_device():
        rc = fn(*args, raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, raw_stream(index))
    if rc:
        raise _lib.VisionAttnError(name, rc, _lib.lib().va_get_last_error_string().decode(errors="replace"))


def on(stream, index: int):
    """Context in which ``stream`` (a torch stream or a raw handle) of device
    ``index``, the tensors', is the current one, so that what a call allocates
    belongs to it as well."""
    if index < 0:
        raise ValueError("a stream was given, but the tensors are not on a CUDA device")
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream), device=index)
    elif stream.device.index != index:
        raise ValueError(f"a stream of {stream.device} was given for tensors on cuda:{index}")
    return torch.cuda.stream(stream)


def _starts(t):
    """Byte addresses of the heads' first elements of ``[tokens, heads, dim]``, sorted."""
    tokens, heads, _ = t.shape
    row, head, _ = t.stride()
    at = torch.arange(tokens)[:, None] * row + torch.arange(heads) * head
    return (at * t.element_size() + t.data_ptr()).flatten().sort().values


def span(t):
    """Addresses of the first byte of ``[tokens, heads, dim]`` and past the last."""
    tokens, heads, d = t.shape
    row, head, _ = t.stride()
    p = t.data_ptr()
    return p, p + ((tokens - 1) * row + (heads - 1) * head + d) * t.element_size() if tokens and heads and d else p


def overlap(a, b) -> bool:
    """Whether two tensors ``[tokens, heads, dim]`` of one type (dimensions
    contiguous, strides not negative) share an element."""
    (pa, end_a), (pb, end_b) = span(a), span(b)
    if pa == end_a or pb == end_b or end_a <= pb or end_b <= pa:
        return False
    (ta, ha, d), (tb, hb, e) = a.shape, b.shape
    (row_a, head_a, _), (row_b, head_b, _) = a.stride(), b.stride()
    size = a.element_size()
    # slices of one packed tensor: a period of the buffer holds both, one beside the other
    for period, other, of_a, of_b in ((row_a, row_b, (ha - 1) * head_a + d, (hb - 1) * head_b + e),
                                      (head_a, head_b, (ta - 1) * row_a + d, (tb - 1) * row_b + e)):
        if period == other and period >= max(of_a, of_b) and (pb - pa) % size == 0:
            apart = (pb - pa) // size % period
            if of_a <= apart <= period - of_b:
                return False
    starts, other = _starts(a), _starts(b)
    after = torch.searchsorted(other, starts).clamp(max=len(other) - 1)  # the nearest of b's at or behind each of a's
    before = (after - 1).clamp(min=0)
    gap = other[after] - starts
    near = ((gap >= 0) & (gap < d * size)) | (((starts - other[before]) >= 0) & ((starts - other[before]) < e * size))
    return bool((near | ((gap < 0) & (-gap < e * size))).any())


def overlaps_itself(t) -> bool:
    """Whether two elements of ``[tokens, heads, dim]`` are one in memory."""
    tokens, heads, d = t.shape
    row, head, _ = t.stride()
    (near, n), (far, m) = sorted(((row, tokens), (head, heads))) if tokens > 1 and heads > 1 else \
        ((0, 1), (row, tokens) if tokens > 1 else (head, heads))
    if (n == 1 or near >= d) and (m <= 1 or far >= (n - 1) * near + d):
        return False
    return bool((_starts(t).diff() < d * t.element_size()).any())

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

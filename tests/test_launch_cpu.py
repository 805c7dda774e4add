"""Which stream a call of the packed-sequence operators runs on, with stand-ins for torch's streams."""
import contextlib

import pytest
import torch

from vision_rs_b200 import _launch, packed, rmsnorm, rotary


class Stream:
    def __init__(self, index):
        self.device = torch.device("cuda", index)


class ExternalStream(Stream):
    def __init__(self, handle, device=0):
        super().__init__(device)
        self.handle = handle


@pytest.fixture
def entered(monkeypatch):
    seen = []
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", ExternalStream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: (seen.append(s), contextlib.nullcontext())[1])
    return seen


def test_a_raw_handle_belongs_to_the_tensors_device(entered):
    _launch.on(0x1234, 1)
    assert entered[0].handle == 0x1234 and entered[0].device.index == 1


def test_a_stream_of_another_device_is_refused(entered):
    own = Stream(1)
    _launch.on(own, 1)
    assert entered == [own]
    with pytest.raises(ValueError, match="cuda:0"):
        _launch.on(Stream(0), 1)
    assert entered == [own]


def test_host_tensors_with_a_stream_are_refused(entered):
    x, w = torch.zeros(3, 8), torch.zeros(8)
    q, cu = torch.zeros(3, 2, 8), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: rmsnorm.rms_norm_forward(x, w, stream=5), lambda: rmsnorm.rms_norm_forward_f8(x, w, stream=5),
                 lambda: rmsnorm.rms_norm_backward(x, x, w, stream=5),
                 lambda: rotary.rotary_forward(q, None, torch.zeros(3, dtype=torch.int32), torch.zeros(2), stream=5),
                 lambda: packed.PackedPlan(cu, cu, 0, 0, 1, 1, 8, stream=5)):
        with pytest.raises(ValueError):
            call()
    assert not entered

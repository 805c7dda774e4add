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


def _views():
    """Tensors [tokens, heads, dim] over one buffer of 4000 elements: slices of packed products, head-major ones, shifted
    and broadcast ones, empty ones."""
    base = torch.zeros(4000)
    v = lambda off, t, h, d, row, head: base.as_strided((t, h, d), (row, head, 1), off)
    return base, [v(0, 5, 4, 8, 64, 8), v(32, 5, 2, 8, 64, 8), v(48, 5, 2, 8, 64, 8), v(4, 5, 4, 8, 64, 8), v(28, 5, 4, 8, 64, 8),
                  v(0, 5, 4, 8, 8, 40), v(160, 5, 4, 8, 8, 40), v(0, 5, 4, 8, 8, 80), v(40, 5, 4, 8, 8, 80), v(36, 5, 4, 8, 8, 80),
                  v(0, 7, 3, 8, 24, 8), v(168, 7, 3, 8, 24, 8), v(167, 7, 3, 8, 24, 8), v(0, 6, 3, 5, 0, 9), v(5, 6, 3, 4, 0, 9),
                  v(0, 6, 3, 8, 50, 4), v(0, 0, 3, 8, 24, 8), v(3, 9, 1, 5, 11, 77), v(8, 9, 1, 5, 11, 3), v(0, 4, 5, 3, 7, 28),
                  v(3, 4, 5, 3, 7, 28), v(3, 4, 5, 3, 14, 56), v(4, 2, 2, 2, 1000, 3)]


def _elements(t):
    return (torch.arange(4000).as_strided(t.shape, t.stride(), t.storage_offset())).flatten().tolist()


def test_overlap_is_exact():
    _, views = _views()
    for a in views:
        own = _elements(a)
        assert _launch.overlaps_itself(a) == (len(set(own)) < len(own)), a.stride()
        for b in views:
            assert _launch.overlap(a, b) == bool(set(own) & set(_elements(b))), (a.stride(), b.stride())


def test_rotary_outputs_that_overlap_are_refused():
    qkv, new = torch.zeros(6, 12, 8), torch.zeros(6, 12, 8)
    q, k, v = qkv.split([6, 3, 3], dim=1)
    q2, k2, _ = new.split([6, 3, 3], dim=1)
    for good in ((q, k), (q2, k2), (q2, k), (q, k2), (q2, v)):
        rotary._refuse_overlap(q, k, *good)
    rotary._refuse_overlap(q, None, q, None)
    for bad in ((qkv[:, 1:7], k2), (q2, qkv[:, 5:8]), (k, q2[:, :3]), (q2, q2[:, :3]), (q, q[:, :3]), (q2[:1].expand(6, 6, 8), k2),
                (q2, k2[:, :1].expand(6, 3, 8)), (qkv.view(-1)[4:].as_strided(q.shape, q.stride()), k2)):
        with pytest.raises(ValueError):
            rotary._refuse_overlap(q, k, *bad)
    both = torch.zeros(6, 6, 8)
    with pytest.raises(ValueError):
        rotary._refuse_overlap(both, both[:, :3], both, both[:, :3])  # q and k in place over each other

"""The ways out of the packed-attention kernels after a bounded wait gave up,
read from their source: no GPU is made to hang for it.

A thread that leaves a loop by itself leaves its peers at an aligned barrier, a
vote or a warp-wide TMEM instruction that waits for it without a limit.  So the
warps that run the softmax or the scores go through their loops to the end, and
vote once before they store."""
import os
import re

import pytest

from conftest import ROOT


def _source(name):
    text = open(os.path.join(ROOT, "vision_rs_b200", "csrc", name)).read()
    return re.sub(r"//[^\n]*", "", text)  # without comments


def _roles(name):
    """Bodies of the warps that come last in each kernel's chain of roles: softmax (forward) or scores (backward)."""
    text = _source(name)
    starts = {"va_packed_attn.cu": [r"const int m = TILES == 2 \? warp >> 2 : 0, row"],
              "va_packed_attn_bwd.cu": [r"const int g = warp >> 2, key = ", r"const int g = warp >> 2, row = "]}[name]
    for start in starts:
        at = re.search(start, text).start()
        yield text[at:text.index("__syncthreads();", at)]


@pytest.mark.parametrize("name", ["va_packed_attn.cu", "va_packed_attn_bwd.cu"])
def test_no_thread_leaves_alone(name):
    assert "bar.arrive" not in _source(name)
    for body in _roles(name):
        assert "break;" not in body and "_leave" not in body
        assert not re.search(r"for \([^;]*;[^;]*\bok\b", body)  # no loop ends on one thread's wait
        assert not re.search(r"if \([^)]*\bok = ", body)        # nor is a step left out for it
        assert "__all_sync(0xffffffffu, ok" in body              # the warp agrees before it stores


@pytest.mark.parametrize("name,first", [("va_packed_attn.cu", "q_full"), ("va_packed_attn_bwd.cu", "a_full")])
def test_loads_in_flight_are_waited_for(name, first):
    """The producer waits (with a limit) for its last loads on every way out: a CTA that ends before they land lets them
    write into its successor's shared memory."""
    text = _source(name)
    issue = text.index("++issued;")
    drain = re.search(r"max\(0, issued - (C::kSlots|kStages)\)", text).start()
    between = text[issue:drain]
    assert issue < drain and not re.search(r"if \(!?ok\)", between)
    assert re.search(r"mbar_try_wait\(&sm\.%s, 0\) && clock64\(\)" % first, text[drain:drain + 600])


@pytest.mark.parametrize("name", ["va_packed_attn.cu", "va_packed_attn_bwd.cu"])
def test_every_part_arrives(name):
    """A part that gave up counts too: else the plan's counter is off by one and its next call joins the parts too early."""
    text = _source(name)
    arrive = text.index("sm.last = atomicAdd(cnt, 1)")
    leave = text.rindex("return;", 0, arrive)
    assert "if (it.slot < 0) return;" == text[text.rindex("if (", 0, leave):leave + len("return;")]

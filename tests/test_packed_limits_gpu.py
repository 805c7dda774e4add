"""Packed-sequence operators at the edges of what they accept."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,heads", [(1 << 20, 32), (1 << 21, 8)])
def test_plan_of_one_long_document(cuda, n, heads):
    """The dK/dV steps of all tiles add up to more than 2^31; the parts keep to the list (128 keys a tile, at most one
    part an SM more than tiles)."""
    from vision_rs_b200 import packed
    cu = packed.cu_seqlens([n])
    plan = packed.PackedPlan(cu, cu, n, n, heads, 1, 8, causal=True, training=True)
    plan.check()
    units = plan.buf[:12].view(torch.int32).tolist()
    assert n // 128 <= units[2] <= n // 128 + 148 and units[1] == n // 128

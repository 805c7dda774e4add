"""The plan's arithmetic of the packed-sequence attention, run on the host from
the header that the plan kernel uses: parts and partial results keep to the
lists' room, whatever the sizes.  The sums are checked against Python's exact
integers."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT
from vision_rs_b200 import _lib

HARNESS = r"""
#include "va_packed.h"
#include <cstdio>
#include <cstdlib>
using namespace va;
// one sequence: list ("f" forward, "b" dK/dV) lq lk heads kv_heads causal
int main(int, char** v) {
  const bool bwd = v[1][0] == 'b';
  const int lq = atoi(v[2]), lk = atoi(v[3]), heads = atoi(v[4]), kv = atoi(v[5]), causal = atoi(v[6]);
  const PackedShape s = packed_shape(1, lq, lk, heads, kv, 8, causal, bwd);
  const int tile = bwd ? kPackBlock : s.q_tile, tiles = ((bwd ? lk : lq) + tile - 1) / tile;
  const int budget = bwd ? s.dkv_budget : s.split_budget;
  auto blocks_of = [&](int t) {
    const int i0 = t * tile;
    return bwd ? query_steps(lq, lk, i0, causal, s.group) : key_blocks(lq, lk, i0, pk_min(tile, lq - i0), causal);
  };
  PackedSum blocks = 0;
  for (int t = 0; t < tiles; ++t) blocks += blocks_of(t);
  const int part = part_blocks(blocks, budget, bwd ? kMinQuerySteps : kMinKeyBlocks);
  long long items = 0, slots = 0;
  for (int t = 0; t < tiles; ++t) {
    const int p = part_count(blocks_of(t), part);
    items += p;
    slots += p > 1 ? p : 0;
  }
  printf("%d %lld %d %lld %d %lld %d %d %d\n", tiles, (long long)blocks, part, items,
         bwd ? s.max_dkv_items : s.max_items, slots, bwd ? 2 * s.dkv_budget : s.max_slots, tile, packed_sums_wide(s));
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++")
    cuda = next((d for d in (os.environ.get("CUDA_HOME", ""), "/usr/local/cuda")
                 if d and os.path.exists(os.path.join(d, "include", "cuda.h"))), None)
    if cxx is None or cuda is None:
        pytest.skip("needs g++ and the CUDA headers")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(HARNESS)
    subprocess.run([cxx, "-std=c++17", "-O1", "-I" + os.path.join(ROOT, "vision_rs_b200", "csrc"),
                    "-I" + os.path.join(cuda, "include"), str(d / "plan.cpp"), "-o", str(d / "plan")], check=True)
    return lambda *a: [int(x) for x in subprocess.run([str(d / "plan"), *map(str, a)], check=True, capture_output=True,
                                                      text=True).stdout.split()]


def _blocks(bwd, lq, lk, group, causal, tile):
    """The same sum in exact integers, from the definition: query i sees key j ≤ i + lk − lq."""
    if bwd:
        first = [max(0, j - (lk - lq)) // 64 if causal else 0 for j in range(0, lk, tile)]
        return sum(max(0, -(-lq // 64) - f) * group for f in first)
    ends = [min(lk, max(0, min(lq, i + tile) + lk - lq)) if causal else lk for i in range(0, lq, tile)]
    return sum(-(-e // 128) for e in ends)


@pytest.mark.parametrize("kind,lq,lk,heads,kv,causal", [
    ("b", 1 << 20, 1 << 20, 32, 1, 1), ("b", 1 << 20, 1 << 20, 16, 1, 0), ("b", 1 << 21, 1 << 21, 8, 1, 1),
    ("b", 1 << 24, 1 << 24, 128, 1, 0), ("b", 1 << 30, 77, 3, 1, 0), ("b", 5, 1 << 30, 128, 1, 1),
    ("b", 4095, 4095, 12, 3, 1), ("b", 0, 300, 2, 1, 0), ("b", 300, 1, 2, 2, 1), ("b", 700, 20, 4, 4, 1),
    ("f", 1, 8192, 32, 8, 1), ("f", 3000, 1 << 30, 12, 1, 0), ("f", 36000, 1 << 28, 1, 1, 1), ("f", 1, 0, 4, 1, 1),
    ("f", 64, 7 * 128, 8, 1, 0), ("f", 700, 20, 4, 4, 1), ("f", 1 << 30, 1 << 30, 1, 1, 1)])
def test_parts_keep_to_the_lists(plan, kind, lq, lk, heads, kv, causal):
    tiles, blocks, part, items, room, slots, slot_room, tile, wide = plan(kind, lq, lk, heads, kv, causal)
    assert wide or max(blocks, tiles) < 1 << 31  # the kernel sums in 32 bits then
    if tiles <= 1 << 20:
        assert blocks == _blocks(kind == "b", lq, lk, heads // kv, causal, tile)
    assert blocks >= 0 and tiles <= items <= room and slots <= slot_room
    assert part >= (32 if kind == "b" else 6)


def test_training_sizes_past_32_bits_are_refused():
    size = _lib.lib().va_packed_plan_bytes
    assert size(1, 1 << 20, 1 << 20, 32, 1, 8, 1, 1) > 0
    assert size(1, 1 << 26, 1 << 20, 64, 1, 8, 1, 0) > 0
    assert size(1, 1 << 26, 1 << 20, 64, 1, 8, 1, 1) == 0 and b"training" in _lib.lib().va_get_last_error_string()


def test_ordinary_sizes_sum_in_32_bits(plan):
    for args in (("b", 4095, 4095, 12, 3, 1), ("b", 1 << 17, 1 << 17, 32, 8, 1), ("f", 64, 1 << 20, 32, 8, 1)):
        assert plan(*args)[-1] == 0
    assert plan("b", 1 << 20, 1 << 20, 32, 1, 1)[-1] == 1

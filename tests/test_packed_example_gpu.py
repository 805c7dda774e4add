"""The example's cache at its end."""
import os
import sys

import pytest
import torch

from conftest import ROOT

sys.path.insert(0, os.path.join(ROOT, "examples"))
pytestmark = pytest.mark.gpu


def test_a_full_cache_refuses_a_token(cuda):
    """Its row would be the next sequence's, or past the tensor's end."""
    from packed_attention_layer import Cache, PackedAttentionLayer
    layer, n = PackedAttentionLayer(256, 4, causal=True), 3
    cache = Cache(layer, n, 2)
    x = torch.randn(n, 256, generator=torch.Generator().manual_seed(0)).to(cuda, torch.bfloat16)
    for _ in range(2):
        cache.token(layer, x, x)
    keys = cache.k.clone()
    with pytest.raises(ValueError):
        cache.token(layer, x, x)
    assert cache.used.tolist() == [2] * n and torch.equal(cache.k, keys)

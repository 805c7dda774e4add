"""The example layer (norm, QKV product, rotary positions, packed attention)
against the f64 restatement composed of the same steps, forward, backward and
token by token.

Tolerances: every step rounds its result to bf16 (2^-8 relative, half an ulp),
and four such steps follow one another, so a relative norm error of 4·2^-8/√3
(rounding errors are uniform) ≈ 1% is the size to expect; 2% is allowed, 4%
for the gradients, which run through the steps twice.  The 8-bit product adds
the rounding of both operands to 3 bits of fraction, 2^-4/√3 ≈ 3.6% each: 8%.
"""
import os
import sys

import pytest
import torch

from conftest import ROOT, rel_l2
from oracle import packed_oracle as po

sys.path.insert(0, os.path.join(ROOT, "examples"))
pytestmark = pytest.mark.gpu


def _reference(layer, x, r, pos, lengths):
    h, y = po.rms_norm(x, layer.w_norm, r, 1e-6)
    qkv = y @ layer.w_qkv.cpu().double().T + layer.b_qkv.cpu().double()
    q, k, v = qkv.view(-1, 3 * layer.heads, layer.dim).split(layer.heads, dim=1)
    q, k = (po.rotary(t, pos, layer.inv_freq, False) for t in (q, k))
    o, _ = po.attention_forward(q, k, v, lengths, lengths, layer.dim ** -0.5, layer.causal)
    return h, y, q, k, v, o


@pytest.mark.parametrize("causal", [False, True])
def test_layer_forward_and_backward(cuda, causal):
    from packed_attention_layer import PackedAttentionLayer
    lengths = [197, 65, 300]
    layer = PackedAttentionLayer(384, 6, causal)
    T = sum(lengths)
    gen = torch.Generator().manual_seed(0)
    x, r, g, gh = (torch.randn(T, 384, generator=gen).to(cuda, torch.bfloat16) for _ in range(4))
    pos = torch.cat([torch.arange(n) for n in lengths]).to(cuda)
    out, h, saved = layer.forward(x, r, pos, layer.plan(lengths, training=True))
    rh, ry, q, k, v, o = _reference(layer, x, r, pos, lengths)
    assert rel_l2(out.float().cpu(), o.view(T, -1)) < 0.02 and rel_l2(h.float().cpu(), rh) < 0.004
    gx, gw, gW, gb = layer.backward(g, gh, saved)
    grads = po.attention_backward(g.view_as(saved[3]), q, k, v, lengths, lengths, layer.dim ** -0.5, causal)
    gq, gk = (po.rotary(t, pos, layer.inv_freq, False, backward=True) for t in grads[:2])
    gqkv = torch.cat([gq, gk, grads[2]], dim=1).view(T, -1)
    rgx, rgw = po.rms_norm_backward(gqkv @ layer.w_qkv.cpu().double(), rh, layer.w_norm, 1e-6, gh)
    for got, ref in ((gx, rgx), (gw, rgw), (gW, gqkv.T @ ry), (gb, gqkv.sum(0))):
        assert rel_l2(got.float().cpu(), ref) < 0.04


@pytest.mark.parametrize("eight_bits", [False, True])
def test_token_by_token_is_the_whole_prompt(cuda, eight_bits):
    """The cache's answers, one token at a time, are the rows of one causal pass."""
    from packed_attention_layer import Cache, PackedAttentionLayer
    layer, n, steps = PackedAttentionLayer(256, 4, causal=True), 3, 20
    gen = torch.Generator().manual_seed(1)
    x, r = (torch.randn(n, steps, 256, generator=gen).to(cuda, torch.bfloat16) for _ in range(2))
    cache = Cache(layer, n, 32)
    got = torch.stack([cache.token(layer, x[:, i].contiguous(), r[:, i].contiguous(), eight_bits)[0]
                       for i in range(steps)], dim=1)
    pos = torch.arange(steps).repeat(n)
    *_, o = _reference(layer, x.view(-1, 256), r.view(-1, 256), pos, [steps] * n)
    assert rel_l2(got.float().cpu(), o.view(n, steps, -1)) < (0.08 if eight_bits else 0.02)


def test_training_step_in_a_cuda_graph(cuda):
    """Plan, forward and backward captured once and replayed on new data, new lengths included: the same bits as eager."""
    from vision_rs_b200 import packed, rmsnorm, rotary
    H, D, T = 4, 64, 500
    gen = torch.Generator().manual_seed(2)
    new = lambda: torch.randn(T, 3 * H, D, generator=gen).to(cuda, torch.bfloat16)
    qkv, gout, cu = new(), new()[:, :H], packed.cu_seqlens([200, 300])
    pos, inv, w = torch.arange(T, device=cuda), rotary.rotary_frequencies(D), torch.ones(H * D, device=cuda)

    def step():
        q, k, v = qkv.split(H, dim=1)
        q, k = rotary.rotary_forward(q, k, pos, inv)
        plan = packed.PackedPlan(cu, cu, T, T, H, H, D, causal=True, training=True)
        out, lse = packed.packed_attention_forward(q, k, v, plan)
        grads = packed.packed_attention_backward(gout, q, k, v, out, lse, plan)
        y, h = rmsnorm.rms_norm_forward(out.view(T, -1), w)
        return (out, lse, *grads, y, *rmsnorm.rms_norm_backward(y, h, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for lengths in ([200, 300], [499, 1], [37, 463]):
        qkv.copy_(new())
        cu.copy_(packed.cu_seqlens(lengths))
        graph.replay()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_example_runs(cuda, capsys):
    import packed_attention_layer
    packed_attention_layer.main()
    assert "us a step" in capsys.readouterr().out

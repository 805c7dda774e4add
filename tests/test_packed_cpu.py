"""The packed-sequence operators without a GPU: the restatement against
autograd, frequencies, plan sizes, and the C entries' refusals, which come
before any launch."""
import ctypes as C
import math

import pytest
import torch

from oracle import packed_oracle as po
from vision_rs_b200 import _lib, packed, rotary


@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradient_formula_is_autograd(causal):
    lq, lk = [5, 0, 9, 4], [7, 3, 9, 2]
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(n, h, 8, dtype=torch.float64, generator=g) for n, h in ((18, 4), (21, 2), (21, 2), (18, 4)))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    outs = []
    for sq, sk in po._sequences(lq, lk):
        for h in range(4):
            s = 0.3 * leaves[0][sq, h] @ leaves[1][sk, h // 2].T
            hide = po._mask(s.shape[0], s.shape[1], causal)
            seen = ~hide.all(1)  # rows that see a key
            p = torch.softmax(s[seen].masked_fill(hide[seen], -math.inf), 1)
            outs.append(((p @ leaves[2][sk, h // 2]) * do[sq, h][seen]).sum())
    sum(outs).backward()
    for got, leaf in zip(po.attention_backward(do, q, k, v, lq, lk, 0.3, causal), leaves):
        assert torch.allclose(got, leaf.grad, atol=1e-12)


def test_forward_restatement_is_torch_attention():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(6, 2, 8, dtype=torch.float64, generator=g) for _ in range(3))
    o, lse = po.attention_forward(q, k, v, [6], [6], 0.5, True)
    ref = torch.nn.functional.scaled_dot_product_attention(*(t.transpose(0, 1) for t in (q, k, v)), is_causal=True, scale=0.5)
    assert torch.allclose(o.transpose(0, 1), ref, atol=1e-12)
    assert torch.allclose(lse[:, 0], 0.5 * (q[0] * k[0]).sum(-1), atol=1e-12)


def test_norm_gradient_formula_is_autograd():
    g = torch.Generator().manual_seed(2)
    h, w, dy, gh = (torch.randn(*s, dtype=torch.float64, generator=g) for s in ((4, 6), (6,), (4, 6), (4, 6)))
    hl, wl = h.clone().requires_grad_(), w.clone().requires_grad_()
    y = hl / torch.sqrt((hl * hl).mean(-1, keepdim=True) + 1e-3) * wl
    ((y * dy).sum() + (hl * gh).sum()).backward()
    dh, dw = po.rms_norm_backward(dy, h, w, 1e-3, gh)
    assert torch.allclose(dh, hl.grad, atol=1e-12) and torch.allclose(dw, wl.grad, atol=1e-12)


def test_rotary_restatement_keeps_lengths_and_goes_back():
    x = torch.randn(5, 2, 10, dtype=torch.float64)
    pos, inv = torch.tensor([0, 1, 7, 100, -3]), torch.tensor([1.0, 0.1, 0.01], dtype=torch.float64)
    for inter in (False, True):
        y = po.rotary(x, pos, inv, inter)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.equal(y[0], x[0])
        assert torch.allclose(po.rotary(y, pos, inv, inter, backward=True), x, atol=1e-12)


def test_frequencies():
    inv = rotary.rotary_frequencies(8, base=100.0, device="cpu")
    assert inv.dtype == torch.float64 and torch.allclose(inv, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    assert torch.allclose(rotary.rotary_frequencies(8, 100.0, stretch=4.0, device="cpu"), inv / 4)
    long = rotary.rotary_frequencies(128, 10000.0, stretch=8.0, trained_length=4096, device="cpu")
    plain = rotary.rotary_frequencies(128, 10000.0, device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(long[turns >= 32], plain[turns >= 32]) and torch.allclose(long[turns <= 1], plain[turns <= 1] / 8)
    between = (turns > 1) & (turns < 32)
    assert ((long < plain) & (long > plain / 8))[between].all()
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, base=0.0), dict(rot_dim=8, stretch=0.0),
                dict(rot_dim=8, trained_length=64, fast_turns=1.0)):
        with pytest.raises(ValueError):
            rotary.rotary_frequencies(**{"device": "cpu", **bad})


def test_cu_seqlens():
    assert packed.cu_seqlens([3, 0, 2], device="cpu").tolist() == [0, 3, 3, 5]
    with pytest.raises(ValueError):
        packed.cu_seqlens([2, -1], device="cpu")


def test_plan_sizes_and_refusals():
    lib = _lib.lib()
    size = lib.va_packed_plan_bytes
    serving, training = size(4, 500, 500, 8, 2, 64, 1, 0), size(4, 500, 500, 8, 2, 64, 1, 1)
    assert 0 < serving < training
    # keys that fit the smallest part even as one sequence are never split: no room for partial results
    assert size(64, 64, 6 * 128, 32, 8, 128, 1, 0) < 1 << 17 < size(64, 64, 64 * 700, 32, 8, 128, 1, 0)
    for bad in ((0, 5, 5, 2, 1, 64), (2, -1, 5, 2, 1, 64), (2, 5, -1, 2, 1, 64), (2, 5, 5, 3, 2, 64), (2, 5, 5, 0, 1, 64),
                (2, 5, 5, 2, 1, 12), (2, 5, 5, 2, 1, 0), (2, 5, 5, 2, 1, 136), (2, 5, 5, 129, 1, 64), (2, (1 << 30) + 1, 5, 2, 1, 64)):
        assert size(*bad, 0, 0) == 0 and lib.va_get_last_error_string()
    st = (C.c_int64 * 14)(*[64] * 14)
    fwd = lambda **k: lib.va_packed_attention_fwd_bf16(
        256, 256, 256, k.get("out", 256), 256, (C.c_int64 * 6)(128, 64, 64, 64, 64, 64), 2, 5, 5, 2, 1, 64, 0, 0,
        k.get("scale", 0.1), k.get("plan", 256), k.get("bytes", 1 << 30), None)
    assert fwd(scale=-1.0) == 1 and b"scale" in lib.va_get_last_error_string()
    assert fwd(out=None) == 1
    assert fwd(plan=None, bytes=0) == 6 and fwd(bytes=10) == 6
    assert fwd(plan=257) == 4
    bwd = lambda training, n: lib.va_packed_attention_bwd_bf16(*[256] * 9, st, 2, 5, 5, 2, 1, 64, 0, training, 0.1, 256, n, None)
    assert bwd(0, 1 << 30) == 1 and b"training" in lib.va_get_last_error_string()
    assert bwd(1, 10) == 6
    build = lambda cu, used, training, plan, n: lib.va_packed_plan_build(cu, 256, used, 2, 5, 5, 2, 1, 64, 0, training, plan, n, None)
    assert build(None, None, 0, 256, 1 << 30) == 1 and build(256, 256, 1, 256, 1 << 30) == 1
    assert build(256, None, 0, None, 0) == 6 and build(256, None, 0, 8, 1 << 30) == 4


def test_rotary_and_norm_refusals():
    lib = _lib.lib()
    st = (C.c_int64 * 8)(128, 64, 128, 64, 128, 64, 128, 64)
    rot = lambda **k: lib.va_rotary_bf16(k.get("q", 256), 256, 256, 256, st, 256, k.get("pb", 4), 256, k.get("tokens", 3),
                                         k.get("heads", 2), 2, 64, k.get("rot", 64), 0, 0, 1.0, None)
    for bad in (dict(q=None), dict(pb=2), dict(tokens=-1), dict(heads=0), dict(rot=66), dict(rot=7), dict(rot=-2)):
        assert rot(**bad) == 1
    assert rot(tokens=0) == 0  # nothing to do, nothing launched
    assert lib.va_rotary_bf16(256, 256, 256, 256, None, 256, 4, 256, 3, 2, 2, 64, 64, 0, 0, 1.0, None) == 1
    fwd = lambda rows, cols, eps, x=256: lib.va_rms_norm_fwd_f32(x, None, 256, 1, None, 256, rows, cols, eps, None)
    assert fwd(-1, 8, 1e-6) == 1 and fwd(4, 0, 1e-6) == 1 and fwd(4, 8, -1.0) == 1 and fwd(4, 8, float("nan")) == 1
    assert fwd(4, 8, 1e-6, x=None) == 1 and fwd(0, 8, 1e-6) == 0
    assert lib.va_rms_norm_fwd_f8_f32(256, None, 256, 1, None, 256, 256, 4, 8, 3, 1e-6, None) == 1
    assert lib.va_rms_norm_fwd_f8_f32(256, None, 256, 1, None, 256, 256, 4, 8, -8, 1e-6, None) == 1
    need = lib.va_rms_norm_bwd_workspace_bytes(100, 384)
    assert need >= 384 * 4 and lib.va_rms_norm_bwd_workspace_bytes(-1, 384) == 0
    bwd = lambda ws, n: lib.va_rms_norm_bwd_f32(256, 256, 256, 1, None, 256, 256, 100, 384, 1e-6, ws, n, None)
    assert bwd(None, 0) == 6 and bwd(256, 16) == 6 and bwd(8, need) == 4

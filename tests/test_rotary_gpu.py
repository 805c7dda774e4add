"""Rotary positions on the B200 against the f64 restatement.

Bound for each element, derived from the arithmetic: the angle's remainder in
f32 turns and sincospif are good to 4e-7, and the two products and the sum
round by 2^-24 each, so the turned value is within 8e-7·factor·(|a| + |b|)
before it is rounded to its type (half an ulp: 2^-8, 2^-11, 2^-24 relative; a
16-bit result below the normal range adds its smallest step).
"""
import pytest
import torch

from oracle import packed_oracle as po

pytestmark = pytest.mark.gpu
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
STEP = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38}


def _close(got, ref, x, rot, interleaved, factor):
    got, x = got.cpu().double(), x.cpu().double()
    mate = x.clone()
    h = rot // 2
    if interleaved:
        mate[..., 0:rot:2], mate[..., 1:rot:2] = x[..., 1:rot:2], x[..., 0:rot:2]
    else:
        mate[..., :h], mate[..., h:rot] = x[..., h:rot], x[..., :h]
    return got, 8e-7 * factor * (x.abs() + mate.abs())


def _check(got, ref, x, rot, interleaved, factor):
    dt = got.dtype
    g, slack = _close(got, ref, x, rot, interleaved, factor)
    assert ((g - ref).abs() <= slack + HALF_ULP[dt] * (ref.abs() + slack) + STEP[dt]).all()
    assert torch.equal(got[..., rot:].cpu(), x[..., rot:].cpu())  # the rest of the head is copied


def _inputs(cuda, dt, tokens, hq, hk, dim, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, hq + 2 * hk, dim, generator=g).to(cuda, dt)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g).to(cuda)
    return qkv[:, :hq], qkv[:, hq:hq + hk], pos


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,dim,rot", [(1, 1, 1, 64, 64), (77, 6, 6, 64, 64), (33, 8, 2, 128, 64),
                                                  (5, 3, 1, 80, 36), (9, 2, 1, 40, 10), (3, 5, 5, 96, 2),
                                                  (700, 4, 1, 128, 128), (2, 1, 1, 512, 512), (4, 2, 1, 7, 6),
                                                  (2400, 2, 1, 32, 32), (4, 2, 2, 16, 0)])
def test_rotary_matches_f64(cuda, dt, interleaved, tokens, hq, hk, dim, rot):
    from vision_rs_b200 import rotary
    q, k, pos = _inputs(cuda, dt, tokens, hq, hk, dim, seed=tokens)
    inv = rotary.rotary_frequencies(rot, device=cuda) if rot else torch.empty(0, dtype=torch.float64, device=cuda)
    for turn, back in ((rotary.rotary_forward, False), (rotary.rotary_backward, True)):
        qo, ko = turn(q, k, pos.int() if back else pos, inv, interleaved=interleaved, factor=1.25)
        for got, x in ((qo, q), (ko, k)):
            _check(got, po.rotary(x, pos, inv, interleaved, 1.25, back), x, rot, interleaved, 1.25)


def test_long_and_negative_positions(cuda):
    """Positions up to 2^31 and below zero: the angle is reduced in 64 bits."""
    from vision_rs_b200 import rotary
    q, k, _ = _inputs(cuda, torch.float32, 6, 2, 1, 64)
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 123456789], device=cuda)
    inv = rotary.rotary_frequencies(64, base=500000.0, stretch=8.0, trained_length=8192, device=cuda)
    qo, ko = rotary.rotary_forward(q, k, pos, inv)
    # 2^31 rad in f64 is itself rounded by 2^-22 rad: that much more than the usual bound
    ref = po.rotary(q, pos, inv, False)
    assert ((qo.cpu().double() - ref).abs() <= 2e-6 * (1 + q.abs().max().item())).all()
    assert torch.equal(qo[0], q[0])


def test_in_place_without_keys_and_other_stream(cuda):
    from vision_rs_b200 import rotary
    q, k, pos = _inputs(cuda, torch.bfloat16, 50, 4, 2, 64)
    inv = rotary.rotary_frequencies(64, device=cuda)
    want_q, want_k = rotary.rotary_forward(q, k, pos, inv)
    only_q, none = rotary.rotary_forward(q, None, pos, inv)
    assert none is None and torch.equal(only_q, want_q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    rotary.rotary_forward(q, k, pos, inv, out=(q, k), stream=side)  # q and k are slices of one buffer
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)


def test_no_tokens(cuda):
    from vision_rs_b200 import rotary
    q, k, pos = _inputs(cuda, torch.bfloat16, 0, 4, 2, 64)
    qo, ko = rotary.rotary_forward(q, k, pos, rotary.rotary_frequencies(64, device=cuda))
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)


def test_backward_is_the_transpose(cuda):
    """⟨R x, y⟩ = ⟨x, Rᵀ y⟩, and the difference quotient of ⟨R x, y⟩ along a direction (the map is linear)."""
    from vision_rs_b200 import rotary
    q, k, pos = _inputs(cuda, torch.float32, 40, 3, 1, 64)
    y = torch.randn_like(q)
    inv = rotary.rotary_frequencies(48, device=cuda)
    fwd = lambda x: rotary.rotary_forward(x, None, pos, inv, interleaved=True, factor=0.7)[0].double()
    grad = rotary.rotary_backward(y, None, pos, inv, interleaved=True, factor=0.7)[0].double()
    d = torch.randn_like(q)
    # a linear map: the central difference has no truncation, only rounding: n products of O(1), each to 1e-6
    quotient = ((fwd(q + d) - fwd(q - d)) / 2 * y.double()).sum()
    n = y.numel()
    assert abs(quotient - (grad * d.double()).sum()) <= 1e-6 * 8 * n
    assert abs((fwd(q) * y.double()).sum() - (q.double() * grad).sum()) <= 1e-6 * 8 * n


def test_refusals(cuda):
    from vision_rs_b200 import _lib, rotary
    q, k, pos = _inputs(cuda, torch.bfloat16, 4, 2, 1, 64)
    inv = rotary.rotary_frequencies(64, device=cuda)
    for bad in (lambda: rotary.rotary_forward(q.cpu(), k, pos, inv), lambda: rotary.rotary_forward(q, k[:3], pos, inv),
                lambda: rotary.rotary_forward(q, k.float(), pos, inv), lambda: rotary.rotary_forward(q, k, pos[:3], inv),
                lambda: rotary.rotary_forward(q, k, pos.float(), inv), lambda: rotary.rotary_forward(q, k, pos, inv.float()),
                lambda: rotary.rotary_forward(q, k, pos, torch.cat([inv, inv])),
                lambda: rotary.rotary_forward(q.transpose(1, 2), None, pos, inv),
                lambda: rotary.rotary_forward(q, k, pos, inv, out=(q, None)),
                lambda: rotary.rotary_forward(q.double(), None, pos, inv)):
        with pytest.raises(ValueError):
            bad()
    big = torch.zeros(1, 1, 1024, device=cuda)
    with pytest.raises(_lib.VisionAttnError):  # more rotated dimensions than the kernel's table holds
        rotary.rotary_forward(big, None, pos[:1], rotary.rotary_frequencies(1024, device=cuda))

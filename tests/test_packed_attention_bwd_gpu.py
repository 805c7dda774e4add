"""Gradient of the packed-sequence attention on the B200 against the f64 formula
and against differences of the f64 forward.

Bounds for each element (u = half an ulp of the 16-bit type; e_s: the scores'
f32 error, see the forward's tests): P and dS are rounded to the type for
their products, Δ carries the rounding of the stored output, and the result
is rounded once more:

    e(dS) = u |dS| + P·Σ_d |dO| u (Σ P|v| + |O|) + (2 e_s + 2e-5) P (Σ_d |dO||v| + Σ_d |dO||O|)
    |err dQ| ≤ scale Σ_j e(dS) |k| + u |dQ|      |err dK| ≤ scale Σ_i e(dS) |q| + u |dK|
    |err dV| ≤ (u + 2 e_s + 2e-5) Σ_i P |dO| + u |dV|

and an f16 result below the normal range adds its smallest step.
"""
import pytest
import torch

from oracle import packed_oracle as po
from test_packed_attention_gpu import HALF_ULP, TYPES, _plan, _qkv, _score_error

pytestmark = pytest.mark.gpu


def _bounds(do, q, k, v, lq, lk, scale, causal, u, es):
    do, q, k, v = (t.cpu().double() for t in (do, q, k, v))
    bq, bk, bv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    group, soft = q.shape[1] // k.shape[1], 2 * es + 2e-5
    for sq, sk in po._sequences(lq, lk):
        for h in range(q.shape[1]):
            g = h // group
            K, V, Q, D = k[sk, g], v[sk, g], q[sq, h], do[sq, h]
            p, o, _ = po.attention_one(Q, K, V, scale, causal)
            ds = p * (D @ V.T - (D * o).sum(1, keepdim=True))
            delta = (D.abs() * (u * (p @ V.abs() + o.abs()))).sum(1, keepdim=True)
            e = u * ds.abs() + p * delta + soft * p * (D.abs() @ V.abs().T + (D.abs() * o.abs()).sum(1, keepdim=True))
            bq[sq, h] = scale * e @ K.abs()
            bk[sk, g] += scale * e.T @ Q.abs()
            bv[sk, g] += (u + soft) * p.T @ D.abs()
    return bq, bk, bv


def _grads(q, k, v, do, lq, lk, causal, scale=None):
    from vision_rs_b200 import packed
    plan = _plan(lq, lk, q.shape[1], k.shape[1], q.shape[2], causal, training=True)
    o, lse = packed.packed_attention_forward(q, k, v, plan, scale)
    return packed.packed_attention_backward(do, q, k, v, o, lse, plan, scale)


def _check(got, do, q, k, v, lq, lk, scale, causal):
    u, es = HALF_ULP[q.dtype], _score_error(q, k, scale)
    ref = po.attention_backward(do, q, k, v, lq, lk, scale, causal)
    step = 2.0 ** -24 if q.dtype == torch.float16 else 1e-30
    for name, g, r, b in zip("qkv", got, ref, _bounds(do, q, k, v, lq, lk, scale, causal, u, es)):
        err, tol = (g.cpu().double() - r).abs(), b * (1 + u) + u * r.abs() + step
        assert (err <= tol).all(), (name, (err - tol).max().item(), (err / tol).max().item())


def _run(cuda, dt, lq, lk, H, Hk, D, causal, seed=0, amp=1.0):
    q, k, v = _qkv(cuda, dt, lq, lk, H, Hk, D, seed)
    do = (amp * torch.randn(q.shape, generator=torch.Generator().manual_seed(seed + 1))).to(cuda, dt)
    _check(_grads(q, k, v, do, lq, lk, causal), do, q, k, v, lq, lk, D ** -0.5, causal)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,H,Hk,D", [
    ([1], 1, 1, 64), ([2, 1, 1], 2, 2, 8), ([63, 64, 65], 3, 3, 64), ([127, 128, 129], 2, 1, 128), ([255, 1, 257], 4, 2, 128),
    ([16, 17, 15, 0, 31, 33], 4, 2, 80), ([300, 0, 190], 6, 6, 64), ([513], 7, 1, 96), ([40] * 30, 3, 3, 32),
    ([700, 400, 1000], 6, 2, 64), ([1100, 30], 8, 4, 128)])
def test_gradient(cuda, dt, causal, lens, H, Hk, D):
    _run(cuda, dt, lens, lens, H, Hk, D, causal, seed=len(lens))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [([5, 300, 1], [200, 1000, 129]), ([300, 10, 7, 128], [100, 0, 7, 127]),
                                   ([0, 3, 0], [5, 0, 9]), ([0], [40])])
def test_unequal_lengths(cuda, causal, lq, lk):
    """Keys before the queries, rows that see no key, keys that no row sees: zeros there."""
    _run(cuda, torch.bfloat16, lq, lk, 4, 2, 64, causal, seed=5)


@pytest.mark.parametrize("amp", [1e-3, 1.0, 300.0])
def test_f16_gradients_of_any_size(cuda, amp):
    """Small and large gradients in f16: dS keeps its bits whatever the loss is scaled by."""
    _run(cuda, torch.float16, [400, 130], [400, 130], 4, 2, 64, True, seed=2, amp=amp)


def test_f16_large_values(cuda):
    """Values in the hundreds beside large gradients stay inside f16's range."""
    lens = [300]
    q, k, v = _qkv(cuda, torch.float16, lens, lens, 2, 2, 64)
    do = 20 * torch.randn(q.shape, generator=torch.Generator().manual_seed(4))
    v, do = (v.float() * 100).half(), do.to(cuda, torch.float16)
    q = (q.float() * 0.02).half()  # keeps the gradients of q and k below 65504
    k = (k.float() * 0.02).half()
    got = _grads(q, k, v, do, lens, lens, False)
    assert all(torch.isfinite(g).all() for g in got)
    _check(got, do, q, k, v, lens, lens, 0.125, False)


def test_differences(cuda):
    """Central differences of L = Σ dO ⊙ O (f64 forward) along a direction of each input.  Step 1e-3: truncation of the
    third derivative ~1e-6 of the sum of |dO||O| sizes; the kernel's error is at most Σ bound·|direction|."""
    lens, H, Hk, D, causal = [50, 81], 4, 2, 64, True
    for dt in TYPES:
        q, k, v = _qkv(cuda, dt, lens, lens, H, Hk, D, seed=9)
        do = torch.randn(q.shape, generator=torch.Generator().manual_seed(10)).to(cuda, dt)
        got = _grads(q, k, v, do, lens, lens, causal)
        u, es = HALF_ULP[dt], _score_error(q, k, 0.125)
        bounds = _bounds(do, q, k, v, lens, lens, 0.125, causal, u, es)
        x = [t.cpu().double() for t in (q, k, v)]
        dd = do.cpu().double()
        loss = lambda *z: (po.attention_forward(*z, lens, lens, 0.125, causal)[0] * dd).sum()
        for i in range(3):
            d = torch.randn(x[i].shape, generator=torch.Generator().manual_seed(20 + i), dtype=torch.float64)
            e = 1e-3
            hi, lo = list(x), list(x)
            hi[i], lo[i] = x[i] + e * d, x[i] - e * d
            quot = (loss(*hi) - loss(*lo)) / (2 * e)
            g = got[i].cpu().double()
            tol = ((bounds[i] * (1 + u) + u * g.abs() + 2.0 ** -24) * d.abs()).sum() + 1e-5 * dd.abs().sum()
            assert abs(quot - (g * d).sum()) <= tol


def test_strided_gradients_and_repeats(cuda):
    """Inputs and gradients as slices of packed products; the same bits each time and on another stream."""
    from vision_rs_b200 import packed
    lens, H, Hk, D = [500, 333, 77], 6, 2, 128
    T = sum(lens)
    qkv = torch.randn(T, H + 2 * Hk, D, generator=torch.Generator().manual_seed(1)).to(cuda, torch.bfloat16)
    q, k, v = qkv.split([H, Hk, Hk], dim=1)
    big = torch.randn(T, 2 * H, D, generator=torch.Generator().manual_seed(2)).to(cuda, torch.bfloat16)
    do = big[:, H:]
    want = _grads(q, k, v, do, lens, lens, True)
    _check(want, do, q, k, v, lens, lens, D ** -0.5, True)
    plan = _plan(lens, lens, H, Hk, D, True, training=True)
    o, lse = packed.packed_attention_forward(q, k, v, plan)
    gqkv = torch.full_like(qkv, float("nan"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    packed.packed_attention_backward(do, q, k, v, o, lse, plan, grads=gqkv.split([H, Hk, Hk], dim=1), stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(gqkv.split([H, Hk, Hk], dim=1), want))


def test_other_sequences_stay_out(cuda):
    lens, H, Hk, D = [130, 65, 200], 4, 2, 64
    for dt in TYPES:
        q, k, v = _qkv(cuda, dt, lens, lens, H, Hk, D)
        do = torch.randn(q.shape, generator=torch.Generator().manual_seed(3)).to(cuda, dt)
        want = _grads(q, k, v, do, lens, lens, True)
        keep = torch.ones(sum(lens), dtype=torch.bool)
        keep[130:195] = False
        for bad in (float("nan"), float("inf")):
            q2, k2, v2, do2 = q.clone(), k.clone(), v.clone(), do.clone()
            for t in (q2, k2, v2, do2):
                t[130:195] = bad
            for a, b in zip(_grads(q2, k2, v2, do2, lens, lens, True), want):
                assert torch.equal(a[keep], b[keep])


def test_refusals(cuda):
    from vision_rs_b200 import _lib, packed
    lens = [30, 20]
    q, k, v = _qkv(cuda, torch.bfloat16, lens, lens, 4, 2, 64)
    bwd = packed.packed_attention_backward
    plan = _plan(lens, lens, 4, 2, 64, True, training=True)
    o, lse = packed.packed_attention_forward(q, k, v, plan)
    serving = _plan(lens, lens, 4, 2, 64, True)
    for bad in (lambda: bwd(o, q, k, v, o, lse, serving), lambda: bwd(o.half(), q, k, v, o, lse, plan),
                lambda: bwd(o, q, k, v, o, lse.double(), plan), lambda: bwd(o[:9], q, k, v, o, lse, plan),
                lambda: bwd(o, q, k, v, o, lse, plan, grads=(q, k, v[:3]))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.VisionAttnError):
        bwd(o, q, k, v, o, lse, plan, scale=-1.0)
    odd = torch.empty(50, 4, 68, dtype=torch.bfloat16, device=cuda)[..., :64]
    with pytest.raises(_lib.VisionAttnError) as e:
        bwd(o, q, k, v, o, lse, plan, grads=(odd, torch.empty_like(k), torch.empty_like(v)))
    assert e.value.code == 4

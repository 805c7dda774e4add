"""Attention over packed sequences on the B200 against the f64 restatement.

Bounds for each element, from the arithmetic (u = half an ulp of the type,
2^-8 or 2^-11): P is rounded to the type (u·Σ P|v|), the output too (u·|o|);
scores are f32 sums of D products, e_s = 2^-23·(16 + D)·scale·max‖q‖·max‖k‖,
which moves lse by e_s and P by twice that relatively; 2^x and the sums add
2e-5; an f16 P below the normal range is off by up to 2^-25 of the largest,
for each key.
"""
import pytest
import torch

from oracle import packed_oracle as po

pytestmark = pytest.mark.gpu
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16]


def _qkv(cuda, dt, lq, lk, H, Hk, D, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (scale * torch.randn(*s, generator=g)).to(cuda, dt)
    return r(sum(lq), H, D), r(sum(lk), Hk, D), r(sum(lk), Hk, D)


def _plan(lq, lk, H, Hk, D, causal, training=False, **kw):
    from vision_rs_b200 import packed
    return packed.PackedPlan(packed.cu_seqlens(lq), packed.cu_seqlens(lk), sum(lq), sum(lk), H, Hk, D, causal=causal,
                             training=training, **kw)


def _score_error(q, k, scale):
    if q.numel() == 0 or k.numel() == 0:
        return 0.0
    n = lambda t: t.float().norm(dim=-1).max().item()
    return 2.0 ** -23 * (16 + q.shape[-1]) * scale * n(q) * n(k)


def _check(o, lse, q, k, v, lq, lk, scale, causal):
    ro, rl = po.attention_forward(q, k, v, lq, lk, scale, causal)
    ra, _ = po.attention_forward(q, k, v.abs(), lq, lk, scale, causal)
    es, u = _score_error(q, k, scale), HALF_ULP[o.dtype]
    finite = torch.isfinite(rl)
    lse = lse.cpu().double()
    assert torch.equal(torch.isfinite(lse), finite) and (lse[~finite] == -float("inf")).all()
    assert ((lse - rl).abs()[finite] <= es + 1e-6 * (1 + rl.abs()[finite])).all()
    small = 2.0 ** -25 * max(lk, default=0) * v.abs().max().item() if o.dtype == torch.float16 and v.numel() else 0.0
    tol = (u + 2 * es + 2e-5) * ra + u * (ro.abs() + u * ra) + small + 2.0 ** -25
    err = (o.cpu().double() - ro).abs()
    assert (err <= tol).all(), (err - tol).max().item()


def _run(cuda, dt, lq, lk, H, Hk, D, causal, seed=0):
    from vision_rs_b200 import packed
    q, k, v = _qkv(cuda, dt, lq, lk, H, Hk, D, seed)
    plan = _plan(lq, lk, H, Hk, D, causal)
    o, lse = packed.packed_attention_forward(q, k, v, plan)
    plan.check()
    _check(o, lse, q, k, v, lq, lk, D ** -0.5, causal)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,H,Hk,D", [
    ([1], 1, 1, 64), ([2, 1, 1], 2, 2, 8), ([127, 128, 129], 3, 3, 64), ([255, 256, 257], 2, 1, 128),
    ([16, 17, 15, 0, 31, 33], 4, 2, 80), ([600, 1, 300], 6, 6, 64), ([513], 7, 1, 96), ([0, 0, 70], 12, 4, 40),
    ([1601, 257, 1000], 6, 6, 64), ([2000, 700, 3], 8, 1, 128), ([40] * 40, 3, 3, 32), ([300, 200, 100] * 12, 12, 4, 128),
    ([900] * 20, 8, 8, 64)])
def test_whole_prompts(cuda, dt, causal, lens, H, Hk, D):
    _run(cuda, dt, lens, lens, H, Hk, D, causal, seed=len(lens))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lk,H,Hk,D", [([1], 1, 1, 64), ([1, 2, 3, 0, 500], 8, 2, 128), ([4096, 17, 1000], 32, 8, 128),
                                       ([20000], 4, 4, 64), ([333] * 70, 14, 2, 64), ([129, 128, 127], 12, 4, 80),
                                       ([5000, 1, 1, 1], 128, 1, 64), ([700, 30], 6, 2, 96)])
def test_single_tokens(cuda, dt, lk, H, Hk, D):
    _run(cuda, dt, [1] * len(lk), lk, H, Hk, D, True, seed=sum(lk))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk,H,Hk,D", [
    ([5, 300, 1], [2000, 1000, 129], 8, 2, 128),       # prompts behind a cache
    ([300, 10, 7, 128], [100, 0, 7, 127], 4, 4, 64),   # more queries than keys: rows that see nothing
    ([1000, 700], [20, 3000], 6, 3, 64), ([0, 3, 0], [5, 0, 9], 2, 1, 64), ([4] * 30, [900] * 30, 16, 2, 64)])
def test_unequal_lengths(cuda, causal, lq, lk, H, Hk, D):
    _run(cuda, torch.bfloat16, lq, lk, H, Hk, D, causal, seed=7)


def test_large_scores(cuda):
    """Scores in the hundreds: the running maximum moves, P keeps to one or two keys."""
    from vision_rs_b200 import packed
    for dt in TYPES:
        lens = [700, 300]
        q, k, v = _qkv(cuda, dt, lens, lens, 4, 2, 64, scale=6.0)
        v = (v / 6).to(dt)
        o, lse = packed.packed_attention_forward(q, k, v, _plan(lens, lens, 4, 2, 64, True))
        _check(o, lse, q, k, v, lens, lens, 0.125, True)


@pytest.mark.parametrize("few", [False, True])
def test_strided_inputs(cuda, few):
    """Slices of one packed product, and head-major tensors."""
    from vision_rs_b200 import packed
    lens, H, Hk, D = ([30, 60] if few else [900, 700, 1100, 800]), 16, 8, 64
    T = sum(lens)
    qkv = torch.randn(T, H + 2 * Hk, D, generator=torch.Generator().manual_seed(3)).to(cuda, torch.bfloat16)
    q, k, v = qkv.split([H, Hk, Hk], dim=1)
    plan = _plan(lens, lens, H, Hk, D, True)
    o, lse = packed.packed_attention_forward(q, k, v, plan)
    _check(o, lse, q, k, v, lens, lens, D ** -0.5, True)
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    o2, lse2 = packed.packed_attention_forward(*major, plan)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [130, 3, 200]), ([700, 650, 900, 31], [700, 650, 900, 31])])
def test_other_sequences_stay_out(cuda, lq, lk):
    """NaN and infinity in one sequence reach no other, though their tiles overlap its rows."""
    from vision_rs_b200 import packed
    H, Hk, D = 8, 4, 128
    q, k, v = _qkv(cuda, torch.bfloat16, lq, lk, H, Hk, D)
    plan = _plan(lq, lk, H, Hk, D, True)
    o, lse = packed.packed_attention_forward(q, k, v, plan)
    a, b, c, d = lq[0], lq[0] + lq[1], lk[0], lk[0] + lk[1]
    for bad in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).min):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        q2[a:b], k2[c:d], v2[c:d] = bad, bad, bad
        o2, lse2 = packed.packed_attention_forward(q2, k2, v2, plan)
        keep = torch.ones(sum(lq), dtype=torch.bool)
        keep[a:b] = False
        assert torch.equal(o2[keep], o[keep]) and torch.equal(lse2[:, keep], lse[:, keep])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lq,lk,H,Hk,D", [([300], [300], 2, 2, 64), ([700, 800, 900], [700, 800, 900], 8, 4, 128),
                                          ([40], [1500], 4, 1, 64), ([9, 300], [9, 400], 2, 1, 80)])
def test_later_keys_may_hold_anything(cuda, dt, lq, lk, H, Hk, D):
    """Causal: NaN or infinity in a key or value of each sequence reaches the rows that see it and no earlier one."""
    from vision_rs_b200 import packed
    q, k, v = _qkv(cuda, dt, lq, lk, H, Hk, D, seed=1)
    plan = _plan(lq, lk, H, Hk, D, True)
    o, lse = packed.packed_attention_forward(q, k, v, plan)
    for bad in (float("nan"), float("inf")):
        for which in "kv":
            k2, v2, sees, at = k.clone(), v.clone(), [], 0
            for a, b in zip(lq, lk):
                j = b - min(a, 37) + 3 if a > 3 else b - 1  # a key that the last rows see
                (k2 if which == "k" else v2)[at + j, :, 5] = bad
                sees += [i >= j - (b - a) for i in range(a)]
                at += b
            sees = torch.tensor(sees)
            o2, lse2 = packed.packed_attention_forward(q, k2, v2, plan)
            assert torch.equal(o2[~sees], o[~sees]) and torch.equal(lse2[:, ~sees], lse[:, ~sees])
            if which == "v":
                rest = [c for c in range(D) if c != 5]
                assert torch.equal(lse2, lse) and torch.equal(o2[..., rest], o[..., rest])
                got = o2[sees][..., 5]
                assert (got.isnan() if bad != bad else got == bad).all()
            elif bad != bad:
                assert o2[sees].isnan().all() and lse2[:, sees].isnan().all()


def test_plan_is_shared_and_results_repeat(cuda):
    """Layer after layer over one plan, on another stream too; the same bits each time."""
    from vision_rs_b200 import packed
    for lq, lk in (([1] * 5, [3000, 40, 900, 1, 0]), ([800, 900, 700], [800, 900, 700])):
        plan = _plan(lq, lk, 8, 2, 64, True)
        ins = [_qkv(cuda, torch.bfloat16, lq, lk, 8, 2, 64, seed=s) for s in range(3)]
        outs = [packed.packed_attention_forward(*x, plan) for x in ins]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for x, (o, lse) in zip(ins, outs):
            o2, lse2 = torch.empty_like(o), torch.empty_like(lse)
            packed.packed_attention_forward(*x, plan, out=o2, lse=lse2, stream=side)
            side.synchronize()
            assert torch.equal(o, o2) and torch.equal(lse, lse2)
            _check(o, lse, *x, lq, lk, 0.125, True)


def test_nothing_to_do(cuda):
    from vision_rs_b200 import packed
    q, k, v = _qkv(cuda, torch.bfloat16, [0], [5], 2, 1, 64)
    o, lse = packed.packed_attention_forward(q, k, v, _plan([0], [5], 2, 1, 64, False))
    assert o.shape == (0, 2, 64) and lse.shape == (2, 0)
    q, k, v = _qkv(cuda, torch.bfloat16, [3, 4], [0, 0], 2, 1, 64)
    o, lse = packed.packed_attention_forward(q, k, v, _plan([3, 4], [0, 0], 2, 1, 64, False))
    assert (o == 0).all() and (lse == -float("inf")).all()


def test_cache_of_more_than_2_31_elements(cuda):
    """The second sequence's keys begin past 2^31 elements of the cache."""
    from vision_rs_b200 import packed
    Hk, D, far, n = 16, 128, 1_100_000, 500
    kv = torch.zeros(far + n, Hk, D, dtype=torch.bfloat16, device=cuda)
    assert far * Hk * D > 2 ** 31
    g = torch.Generator().manual_seed(0)
    kv[far:] = torch.randn(n, Hk, D, generator=g).to(cuda, torch.bfloat16)
    q = torch.randn(3, 32, D, generator=g).to(cuda, torch.bfloat16)
    plan = packed.PackedPlan(packed.cu_seqlens([0, 3]), packed.cu_seqlens([far, n]), 3, far + n, 32, Hk, D, causal=True)
    o, lse = packed.packed_attention_forward(q, kv, kv, plan)
    _check(o, lse, q, kv[far:], kv[far:], [3], [n], D ** -0.5, True)


@pytest.mark.parametrize("lq", [[1, 1, 1, 1], [3, 0, 300, 40]])
def test_cache_with_room_to_grow(cuda, lq):
    """Key rows past the used length hold anything (NaN here) and are never seen."""
    from vision_rs_b200 import packed
    room, used, H, Hk, D = [200, 64, 1000, 300], [130, 0, 1000, 77], 8, 2, 64
    q, k, v = _qkv(cuda, torch.bfloat16, lq, used, H, Hk, D)
    kc = torch.full((sum(room), Hk, D), float("nan"), dtype=torch.bfloat16, device=cuda)
    vc, at, a = kc.clone(), 0, 0
    for r, u in zip(room, used):
        kc[at:at + u], vc[at:at + u] = k[a:a + u], v[a:a + u]
        at, a = at + r, a + u
    plan = packed.PackedPlan(packed.cu_seqlens(lq), packed.cu_seqlens(room), sum(lq), sum(room), H, Hk, D, causal=True,
                             used_k=torch.tensor(used, dtype=torch.int32, device=cuda))
    o, lse = packed.packed_attention_forward(q, kc, vc, plan)
    plan.check()
    _check(o, lse, q, k, v, lq, used, D ** -0.5, True)
    over = packed.PackedPlan(packed.cu_seqlens(lq), packed.cu_seqlens(room), sum(lq), sum(room), H, Hk, D, causal=True,
                             used_k=torch.tensor([201, 0, 5, 5], dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError):
        over.check()
    with pytest.raises(ValueError):
        packed.PackedPlan(packed.cu_seqlens(lq), packed.cu_seqlens(room), sum(lq), sum(room), H, Hk, D, training=True,
                          used_k=torch.tensor(used, dtype=torch.int32, device=cuda))


def test_offsets_out_of_order_are_reported(cuda):
    from vision_rs_b200 import packed
    q, k, v = _qkv(cuda, torch.bfloat16, [64], [64], 2, 1, 64)
    good = packed.cu_seqlens([20, 44])
    for cu in ([0, 50, 20], [0, 20, 9999], [-5, 20, 64], [3, 20, 64], [0, 20, 60]):
        plan = packed.PackedPlan(torch.tensor(cu, dtype=torch.int32, device=cuda), good, 64, 64, 2, 1, 64)
        packed.packed_attention_forward(q, k, v, plan)  # clamped: stays inside the tensors
        torch.cuda.synchronize()
        with pytest.raises(ValueError):
            plan.check()
    plan = packed.PackedPlan(good, good, 64, 64, 2, 1, 64)
    plan.check()


def test_many_sequences(cuda):
    """More sequences than the plan kernel's shared memory holds, most of them empty or tiny."""
    lens = [(i * 7) % 5 for i in range(3000)]
    _run(cuda, torch.bfloat16, lens, lens, 2, 2, 64, True)


def test_refusals(cuda):
    from vision_rs_b200 import _lib, packed
    lens = [30, 20]
    q, k, v = _qkv(cuda, torch.bfloat16, lens, lens, 4, 2, 64)
    cu = packed.cu_seqlens(lens)
    plan = packed.PackedPlan(cu, cu, 50, 50, 4, 2, 64)
    fwd = packed.packed_attention_forward
    for bad in (lambda: fwd(q.float(), k, v, plan), lambda: fwd(q, k.half(), v, plan), lambda: fwd(q[:40], k, v, plan),
                lambda: fwd(q, k.cpu(), v, plan), lambda: fwd(q, k[:, :1], v, plan), lambda: fwd(q, k, v, plan, out=q.half()),
                lambda: fwd(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, plan),
                lambda: packed.PackedPlan(cu.cpu(), cu, 50, 50, 4, 2, 64), lambda: packed.PackedPlan(cu.long(), cu, 50, 50, 4, 2, 64),
                lambda: packed.PackedPlan(cu[:2], cu, 50, 50, 4, 2, 64), lambda: packed.cu_seqlens([3, -1])):
        with pytest.raises(ValueError):
            bad()
    for sizes in ((50, 50, 4, 3, 64), (50, 50, 4, 2, 60), (50, 50, 4, 2, 136), (-1, 50, 4, 2, 64), (50, 50, 0, 2, 64),
                  (50, 50, 256, 1, 64)):
        with pytest.raises(_lib.VisionAttnError):
            packed.PackedPlan(cu, cu, *sizes)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(_lib.VisionAttnError):
            fwd(q, k, v, plan, scale=scale)
    wide = torch.empty(50, 4, 68, dtype=torch.bfloat16, device=cuda)[..., :64]  # rows of 136 bytes: no 16-byte stride
    with pytest.raises(_lib.VisionAttnError) as e:
        fwd(wide, k, v, plan)
    assert e.value.code == 4
    lib = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    assert lib.va_packed_plan_build(cu.data_ptr(), cu.data_ptr(), None, *plan.sizes, plan.buf.data_ptr(), 16, st) == 6
    assert lib.va_packed_plan_build(cu.data_ptr(), cu.data_ptr(), None, *plan.sizes, None, 0, st) == 6

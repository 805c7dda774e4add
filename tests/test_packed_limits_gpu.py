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


def test_a_unit_of_more_than_a_second(cuda):
    """256 queries a head over 200 million keys: each unit works for longer than a wait's limit (2·10^9 cycles), with a
    last V block that is checked.  Keys of zeros: every weight is 1/n.  One value in 256 is one and the others zero: their
    sum stays below 2^20, where the product's f32 sums (which drop what lies 2^-25 below the running sum) are exact."""
    import math
    from vision_rs_b200 import packed
    n, H, D = 200_000_005, 76, 8
    q = torch.randn(256, H, D, device=cuda).bfloat16()
    k, v = (torch.zeros(n, 1, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    v[::256] = 1
    plan = packed.PackedPlan(packed.cu_seqlens([256]), packed.cu_seqlens([n]), 256, n, H, 1, D)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    o, lse = packed.packed_attention_forward(q, k, v, plan)
    b.record()
    b.synchronize()
    assert a.elapsed_time(b) > 1100.0  # or this test shows nothing
    # the weights' sum: steps of 64 stay exact in 32 bits, the last keys are rounded to 16 in 2·10^8
    mean = (n + 255) // 256 / n
    assert ((o.double() - mean).abs() <= 2.0 ** -8 * mean).all() and ((lse - math.log(n)).abs() <= 1e-6 * math.log(n)).all()


def test_rotary_in_place_and_overlapping(cuda):
    """In place (slices of one product, head-major, one alone) gives the bits of a separate output; other overlaps are refused."""
    from vision_rs_b200 import rotary
    T, H, Hk, D = 37, 6, 2, 64
    qkv = torch.randn(T, H + 2 * Hk, D, generator=torch.Generator().manual_seed(0)).to(cuda, torch.bfloat16)
    pos, inv = torch.arange(T, device=cuda), rotary.rotary_frequencies(D)
    split = lambda t: t.split([H, Hk, Hk], dim=1)
    q, k, v = split(qkv)
    ref = rotary.rotary_forward(q, k, pos, inv)
    for which in ((0, 1), (0,), (1,)):
        buf = qkv.clone()
        a, b, c = split(buf)
        out = (a if 0 in which else torch.empty_like(a), b if 1 in which else torch.empty_like(b))
        got = rotary.rotary_forward(a, b, pos, inv, out=out)
        assert all(torch.equal(x, y) for x, y in zip(got, ref)) and torch.equal(c, v)
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k)]
    assert all(torch.equal(x, y) for x, y in zip(rotary.rotary_forward(*major, pos, inv, out=tuple(major)), ref))
    for bad in ((qkv[:, 1:H + 1], torch.empty_like(k)), (k, k), (q, q[:, :Hk]), (q[:1].expand(T, H, D), k)):
        with pytest.raises(ValueError):
            rotary.rotary_forward(q, k, pos, inv, out=bad)
    assert torch.equal(qkv[:, :H], q)


def test_calls_that_share_a_plan_follow_one_another(cuda):
    """A call on a second stream waits for the first stream's call, and the first stream's next one for it."""
    from vision_rs_b200 import packed
    lk, H, Hk, D = [3000, 40, 900], 8, 2, 64
    g = torch.Generator().manual_seed(0)
    new = lambda n, h: torch.randn(n, h, D, generator=g).to(cuda, torch.bfloat16)
    k, v, qs = new(sum(lk), Hk), new(sum(lk), Hk), [new(3, H) for _ in range(3)]
    make = lambda: packed.PackedPlan(packed.cu_seqlens([1] * 3), packed.cu_seqlens(lk), 3, sum(lk), H, Hk, D, causal=True)
    refs = [packed.packed_attention_forward(q, k, v, make())[0] for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    plan = make()
    torch.cuda.synchronize()
    for first, second in (streams, streams[::-1], (torch.cuda.current_stream(), streams[0]), (streams[0].cuda_stream, streams[1])):
        done, outs = [], []
        for n, s in enumerate((first, second, first)):
            ext = s if isinstance(s, torch.cuda.Stream) else torch.cuda.ExternalStream(s)
            with torch.cuda.stream(ext):
                if n == 0:
                    torch.cuda._sleep(40_000_000)  # ~20 ms
                outs.append(packed.packed_attention_forward(qs[n], k, v, plan, stream=s)[0])
                done.append(torch.cuda.Event())
                done[-1].record()
        done[1].synchronize()
        assert done[0].query()
        done[2].synchronize()
        assert done[1].query() and all(torch.equal(a, b) for a, b in zip(outs, refs))
    plan.check()


@pytest.mark.parametrize("lens", [[30, 60], [900, 700, 1100, 800]])
def test_results_over_inputs(cuda, lens):
    """out over a contiguous q gives the bits of a separate out; results over other inputs are refused."""
    from vision_rs_b200 import packed
    H, Hk, D, T = 16, 8, 64, sum(lens)
    g = torch.Generator().manual_seed(0)
    new = lambda h: torch.randn(T, h, D, generator=g).to(cuda, torch.bfloat16)
    q, k, v, do, qkv = new(H), new(Hk), new(Hk), new(H), new(H + 2 * Hk)
    cu = packed.cu_seqlens(lens)
    plan = packed.PackedPlan(cu, cu, T, T, H, Hk, D, causal=True, training=True)
    out, lse = packed.packed_attention_forward(q, k, v, plan)
    q2 = q.clone()
    o2, lse2 = packed.packed_attention_forward(q2, k, v, plan, out=q2)
    assert o2 is q2 and torch.equal(o2, out) and torch.equal(lse2, lse)
    sq, sk, sv = qkv.split([H, Hk, Hk], dim=1)
    flat = qkv.view(-1)
    for bad in (flat[:T * H * D].view(T, H, D), flat[-T * H * D:].view(T, H, D)):
        with pytest.raises(ValueError):
            packed.packed_attention_forward(sq, sk, sv, plan, out=bad)
    grads = packed.packed_attention_backward(do, q, k, v, out, lse, plan)
    buf = torch.empty_like(qkv)
    got = packed.packed_attention_backward(do, q, k, v, out, lse, plan, grads=buf.split([H, Hk, Hk], dim=1))
    assert all(torch.equal(a, b) for a, b in zip(grads, got))
    for bad in ((q, k, v), (do, grads[1], grads[2]), (out, grads[1], grads[2]), (grads[0], grads[1], k)):
        with pytest.raises(ValueError):
            packed.packed_attention_backward(do, q, k, v, out, lse, plan, grads=bad)

"""The root-mean-square norm with the residual's addition on the B200 against
the f64 restatement.

Bounds, derived from the arithmetic in f32: the sum of squares of n terms in
partial sums of at most 64 terms a thread and a tree is good to ~80·2^-24, so
y carries a relative error of at most 80·2^-25 + a few roundings < 4e-6
before it is rounded to its type (half an ulp: 2^-8, 2^-11, 2^-24).  Gradients
add the terms of a difference: 4e-6 of each term's size.  The 8-bit values are
within one step of e4m3 (2^-3 relative), and equal but for near ties.
"""
import pytest
import torch

from oracle import packed_oracle as po

pytestmark = pytest.mark.gpu
EPS = 1e-6
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
STEP = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows(cuda, dt, rows, cols, seed=0, w_f32=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    x, res = r(rows, cols).to(cuda, dt), (2 * r(rows, cols)).to(cuda, dt)
    w = (1 + 0.2 * r(cols)).to(cuda, torch.float32 if w_f32 else dt)
    return x, res, w, r(rows, cols).to(cuda, dt), r(rows, cols).to(cuda, dt)


def _within(got, ref, size):
    """|got − ref| ≤ 4e-6·size and then the rounding to got's type."""
    dt, slack = got.dtype, 4e-6 * size
    return bool(((got.cpu().double() - ref).abs() <= slack + HALF_ULP[dt] * (ref.abs() + slack) + STEP[dt]).all())


SHAPES = [(1, 1), (3, 7), (2, 64), (5, 384), (300, 384), (77, 768), (9, 1000), (1, 4096), (300, 4096), (6, 4104),
          (300, 8192), (4, 16384), (300, 16384), (2, 16392), (2, 40000)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(cuda, dt, rows, cols):
    from vision_rs_b200 import rmsnorm
    x, res, w, *_ = _rows(cuda, dt, rows, cols, w_f32=rows % 2 == 1)
    y, h = rmsnorm.rms_norm_forward(x, w, res, eps=EPS)
    rh, ry = po.rms_norm(x, w, res, EPS)
    assert _within(h, rh, rh.abs()) and _within(y, ry, ry.abs())
    y1, h1 = rmsnorm.rms_norm_forward(x, w, eps=EPS)
    _, ry1 = po.rms_norm(x, w, None, EPS)
    assert h1 is x and _within(y1, ry1, ry1.abs())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,cols,group", [(5, 384, 0), (300, 384, 128), (64, 4096, 128), (300, 4096, 0), (3, 1000, 0),
                                             (3, 1000, 8), (2, 4096, 64), (300, 512, 32), (2, 63, 21), (7, 16384, 0),
                                             (300, 2048, 256), (2, 40000, 0), (1, 1, 1)])
def test_forward_8_bits(cuda, dt, rows, cols, group):
    from vision_rs_b200 import rmsnorm
    x, res, w, *_ = _rows(cuda, dt, rows, cols, seed=1)
    q, scale, h = rmsnorm.rms_norm_forward_f8(x, w, res, eps=EPS, group=group)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows, cols // group if group else 1)
    rh, ry = po.rms_norm(x, w, res, EPS)
    assert _within(h, rh, rh.abs())
    blocks = ry.reshape(rows, -1, group or cols)
    rs = blocks.abs().amax(-1).clamp_min(2.0 ** -100) / 448
    assert ((scale.cpu().double() - rs).abs() <= 5e-6 * rs).all()
    want = blocks / rs[..., None]
    got = q.cpu().double().reshape(blocks.shape)
    # 3 bits of fraction: half a step is 2^-4 relative, and 2^-10 below the normal range
    assert ((got - want).abs() <= 2.0 ** -4 * want.abs() * (1 + 1e-4) + 2.0 ** -10 * (1 + 1e-4)).all()
    # equal to the rounded values but where those lie within 1e-5 of a tie
    same = got == want.float().to(torch.float8_e4m3fn).double()
    lo, hi = want * (1 - 1e-5), want * (1 + 1e-5)
    tie = lo.float().to(torch.float8_e4m3fn).double() != hi.float().to(torch.float8_e4m3fn).double()
    assert (same | tie).all()
    assert (got.abs().amax(-1) == 448).all()


def test_zero_rows_and_non_finite_rows_stay_apart(cuda):
    """A row of zeros gives zeros and a finite scale; NaN or infinity in one row reaches no other."""
    from vision_rs_b200 import rmsnorm
    for cols, dt in ((384, torch.bfloat16), (1001, torch.float32)):
        x, _, w, *_ = _rows(cuda, dt, 9, cols, seed=2)
        x[1] = 0
        x[3, 5] = float("nan")
        x[6, 2] = float("inf")
        clean = x.clone()
        clean[3], clean[6] = 1, 1
        y, _ = rmsnorm.rms_norm_forward(x, w, eps=EPS)
        yc, _ = rmsnorm.rms_norm_forward(clean, w, eps=EPS)
        keep = [0, 1, 2, 4, 5, 7, 8]
        assert torch.equal(y[keep], yc[keep]) and (y[1] == 0).all() and y[3].isnan().all() and y[6, 2].isnan()
        q, s, _ = rmsnorm.rms_norm_forward_f8(x, w, eps=EPS)
        qc, sc, _ = rmsnorm.rms_norm_forward_f8(clean, w, eps=EPS)
        assert torch.equal(q.float()[keep], qc.float()[keep]) and torch.equal(s[keep], sc[keep])
        assert (q[1].float() == 0).all() and 0 < s[1] < 1e-30 and s[3].isnan() and q[3].float().isnan().all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + [(0, 384), (5000, 384), (1200, 2048)])
def test_backward(cuda, dt, rows, cols):
    from vision_rs_b200 import rmsnorm
    h, _, w, dy, gh = _rows(cuda, dt, rows, cols, seed=3, w_f32=rows % 2 == 1)
    for grad_h in (gh, None):
        dh, dw = rmsnorm.rms_norm_backward(dy, h, w, eps=EPS, grad_h=grad_h)
        rdh, rdw = po.rms_norm_backward(dy, h, w, EPS, grad_h)
        hd, g = h.cpu().double(), (dy.cpu().double() * w.cpu().double())
        r = 1 / torch.sqrt((hd * hd).mean(-1, keepdim=True) + EPS)
        size = r * (g.abs() + hd.abs() * r * r * (g * hd).abs().mean(-1, keepdim=True)) + \
            (0 if grad_h is None else grad_h.cpu().double().abs())
        assert _within(dh, rdh, size)
        terms = (dy.cpu().double() * hd * r).abs().sum(0)
        assert ((dw.cpu().double() - rdw).abs() <= 4e-6 * terms).all()
        assert torch.equal(dw, rmsnorm.rms_norm_backward(dy, h, w, eps=EPS, grad_h=grad_h)[1])


def test_gradient_is_the_difference_quotient(cuda):
    """Central differences of L = Σ dy ⊙ y in f64 along directions of x and w, against the kernel's f32 gradients.
    Step 1e-4 in f64: truncation ~1e-8, rounding ~1e-12; the gradients' own error is 4e-6 of n O(1) terms."""
    from vision_rs_b200 import rmsnorm
    h, d, w, dy, _ = _rows(cuda, torch.float32, 12, 96, seed=4)
    dh, dw = rmsnorm.rms_norm_backward(dy, h, w, eps=EPS)
    loss = lambda hh, ww: (po.rms_norm(hh, ww, None, EPS)[1] * dy.cpu().double()).sum()
    e, hd, wd, dd = 1e-4, h.cpu().double(), w.cpu().double(), d.cpu().double()
    n = h.numel()
    quot = (loss(hd + e * dd, wd) - loss(hd - e * dd, wd)) / (2 * e)
    assert abs(quot - (dh.cpu().double() * dd).sum()) <= 4e-6 * 4 * n + 1e-5
    dirw = dd[0]
    quot = (loss(hd, wd + e * dirw) - loss(hd, wd - e * dirw)) / (2 * e)
    assert abs(quot - (dw.cpu().double() * dirw).sum()) <= 4e-6 * 4 * n + 1e-5


def test_in_place_sum_unaligned_rows_and_other_stream(cuda):
    from vision_rs_b200 import rmsnorm
    x, res, w, *_ = _rows(cuda, torch.bfloat16, 40, 384, seed=5)
    y, h = rmsnorm.rms_norm_forward(x, w, res, eps=EPS)
    buf = torch.empty(40 * 384 + 1, dtype=torch.bfloat16, device=cuda)
    odd = buf[1:].view(40, 384)  # 2-byte aligned: the any-width kernel
    odd.copy_(x)
    y2, h2 = rmsnorm.rms_norm_forward(odd, w, res, eps=EPS)
    assert torch.equal(h2, h) and (y2.double() - y.double()).abs().max() <= 2 ** -7 * y.double().abs().max()
    r2 = res.clone()
    rmsnorm.rms_norm_forward(odd, w, r2, eps=EPS, out_h=r2)
    assert torch.equal(r2, h)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(x)
    rmsnorm.rms_norm_forward(x, w, res, eps=EPS, out=out, out_h=res, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(res, h) and torch.equal(out, y)


def test_refusals(cuda):
    from vision_rs_b200 import _lib, rmsnorm
    x, res, w, dy, _ = _rows(cuda, torch.bfloat16, 4, 384)
    for bad in (lambda: rmsnorm.rms_norm_forward(x.cpu(), w), lambda: rmsnorm.rms_norm_forward(x.t(), w),
                lambda: rmsnorm.rms_norm_forward(x, w[:5]), lambda: rmsnorm.rms_norm_forward(x, w.half()),
                lambda: rmsnorm.rms_norm_forward(x, w, res[:2]), lambda: rmsnorm.rms_norm_forward(x, w, res.float()),
                lambda: rmsnorm.rms_norm_forward_f8(x, w, group=100), lambda: rmsnorm.rms_norm_forward_f8(x, w, group=-1),
                lambda: rmsnorm.rms_norm_backward(dy.float(), x, w), lambda: rmsnorm.rms_norm_forward(x.double(), w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.VisionAttnError):
        rmsnorm.rms_norm_forward(x, w, eps=-1.0)
    dw = torch.empty(384, device=cuda)
    lib = _lib.lib()
    rc = lib.va_rms_norm_bwd_bf16(dy.data_ptr(), x.data_ptr(), w.data_ptr(), 0, None, dy.data_ptr(), dw.data_ptr(), 4,
                                  384, EPS, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 6 and b"workspace" in lib.va_get_last_error_string()

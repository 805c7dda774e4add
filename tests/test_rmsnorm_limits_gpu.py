"""RMS norm at the edges of what its entries accept."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sfx,cols", [("bf16", 384), ("f16", 8192), ("f32", 7), ("f32", 512)])
def test_backward_of_no_rows_reads_nothing(cuda, sfx, cols):
    """Rows, gradients and weight may all be null then; the weight's gradient is zero."""
    from vision_rs_b200 import _lib
    lib = _lib.lib()
    dw = torch.full((cols,), 5.0, device=cuda)
    need = lib.va_rms_norm_bwd_workspace_bytes(0, cols)
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    _lib.call(f"va_rms_norm_bwd_{sfx}", None, None, None, 0, None, None, dw.data_ptr(), 0, cols, 1e-6, ws.data_ptr(), need,
              torch.cuda.current_stream().cuda_stream)
    assert (dw == 0).all()


def test_backward_workspace(cuda):
    """A host tensor, or one whose elements are not where its size says, never reaches a kernel; a smaller one is not used."""
    from vision_rs_b200 import _lib, rmsnorm
    g = torch.Generator().manual_seed(0)
    dy, h, w = (torch.randn(*s, generator=g).to(cuda) for s in ((40, 96), (40, 96), (96,)))
    need = _lib.lib().va_rms_norm_bwd_workspace_bytes(40, 96)
    ref = rmsnorm.rms_norm_backward(dy, h, w)
    for bad in (torch.empty(need, dtype=torch.uint8), torch.empty(1, dtype=torch.uint8, device=cuda).expand(need),
                torch.empty(2 * need, dtype=torch.uint8, device=cuda)[::2]):
        with pytest.raises(ValueError):
            rmsnorm.rms_norm_backward(dy, h, w, workspace=bad)
    for ws in (torch.empty(need, dtype=torch.uint8, device=cuda), torch.empty(need // 4 + 8, device=cuda),
               torch.empty(16, dtype=torch.uint8, device=cuda)):
        assert all(torch.equal(a, b) for a, b in zip(ref, rmsnorm.rms_norm_backward(dy, h, w, workspace=ws)))


@pytest.mark.parametrize("cols", [384, 50])
def test_outputs_in_place_and_overlapping(cuda, cols):
    """Exactly in place gives the bits of separate outputs; rows shifted against their inputs are refused."""
    from vision_rs_b200 import rmsnorm
    g = torch.Generator().manual_seed(1)
    R = 30
    big = torch.randn(R + 8, cols, generator=g).to(cuda)
    res, w = torch.randn(R, cols, generator=g).to(cuda), torch.randn(cols, generator=g).to(cuda)
    x = big[:R]
    y, h = rmsnorm.rms_norm_forward(x.clone(), w, res)
    for pick in ((0, None), (None, 0), (1, 0), (0, 1), (None, 1)):
        a, b = x.clone(), res.clone()
        out, out_h = (None if i is None else (a, b)[i] for i in pick)
        got = rmsnorm.rms_norm_forward(a, w, b, out=out, out_h=out_h)
        assert torch.equal(got[0], y) and torch.equal(got[1], h)
    q, s, h8 = rmsnorm.rms_norm_forward_f8(x.clone(), w, res)
    b = res.clone()
    got = rmsnorm.rms_norm_forward_f8(x.clone(), w, b, out_h=b)
    assert torch.equal(got[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(got[1], s) and torch.equal(got[2], h8)
    one = torch.empty_like(x)
    for bad in (dict(out=big[2:R + 2]), dict(out_h=big[1:R + 1]), dict(out=one, out_h=one),
                dict(out=big[8:], out_h=x)):
        with pytest.raises(ValueError):
            rmsnorm.rms_norm_forward(x, w, res, **bad)
    with pytest.raises(ValueError):
        rmsnorm.rms_norm_forward_f8(x, w, res, out_h=big[3:R + 3])

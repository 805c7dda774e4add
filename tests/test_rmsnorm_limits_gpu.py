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

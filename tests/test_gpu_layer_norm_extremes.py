"""Layer norm's gradient of rows whose mean times 1 / deviation leaves the fp32 range, against its formula."""

import pytest
import torch

import apexw_amd
from test_gpu_layer_norm import E, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 2, 4, 16, 64, 256, 1024, 4096, 8192])
def test_constant_rows_far_from_zero(width, dtype):
    """Rows of one number (widths whose reciprocal is exact, so their mean is that number) with a tiny eps:
    xh = 0 at every element that exists, and dx = rstd (g - mean(g))."""
    g = torch.Generator().manual_seed(width)
    x = torch.tensor([2.0 ** 65, -2.0 ** 70, 1.0])[:, None].expand(3, width).contiguous().to(dtype).cuda()
    dy = torch.randn(3, width, generator=g).to(dtype).cuda()
    w, b = (torch.randn(width, generator=g).to(dtype).cuda() for _ in range(2))
    _, mean, rstd = apexw_amd.layer_norm_forward(x, w, b, 1e-38)
    assert torch.equal(mean, x[:, 0].float()) and float(rstd.min()) > 2.0 ** 62
    dx, dw, db = apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b)
    d = dy.double()
    gw, r = d * w.double(), rstd.double()[:, None]
    close(dx, r * (gw - gw.mean(1, keepdim=True)), E * r * (gw.abs() + gw.abs().mean(1, keepdim=True)))
    assert (dw == 0).all()
    close(db, d.sum(0), E * d.abs().sum(0))

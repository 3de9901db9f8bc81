"""scale_grads refuses a norm that lies in what it writes, before anything is written."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


def test_norm_among_the_gradients():
    base = torch.rand(9000, device="cuda") + 1
    before = base.clone()
    with pytest.raises(ValueError, match="total_norm"):
        apexw_amd.scale_grads([base[:5000], base[5000:]], 0.5, base[7000])
    torch.cuda.synchronize()
    assert torch.equal(base, before)
    apexw_amd.scale_grads([base[:5000], base[5001:]], 0.5, base[5000])
    c = 0.5 / (float(before[5000]) + 1e-6)
    assert float((base[:5000] - before[:5000] * c).abs().max()) <= 1e-6 and float(base[5000]) == float(before[5000])

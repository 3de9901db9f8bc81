"""expert_combine_backward without the combined rows: only where the weights' gradient is not wanted."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


def test_without_rows():
    order = apexw_amd.expert_order(torch.tensor([[0, 1], [1, 2], [2, 0]], device="cuda"), 3)
    dout, y, w = torch.randn(3, 16, device="cuda"), torch.randn(6, 16, device="cuda"), torch.rand(3, 2, device="cuda")
    dy, none = apexw_amd.expert_combine_backward(dout, None, order, w, need=(True, False))
    assert none is None and torch.equal(dy, apexw_amd.expert_combine_backward(dout, y, order, w)[0])
    for need in ((True, True), (False, True)):
        with pytest.raises(ValueError, match="takes y"):
            apexw_amd.expert_combine_backward(dout, None, order, w, need=need)

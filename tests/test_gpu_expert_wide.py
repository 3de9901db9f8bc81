"""The weights' gradient of rows whose 32-bit byte offsets would wrap: 64 rows of 36 million elements."""

import pytest
import torch

import apexw_amd
from test_gpu_experts import close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("swap", [False, True])
def test_rows_of_36_million_elements(swap):
    rows, n, k = 64, 36_000_001, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    thin = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    ends = torch.tensor([rows], dtype=torch.int32, device="cuda")
    got = apexw_amd.expert_matmul_weight_grad(*((thin, wide) if swap else (wide, thin)), ends)[0]
    got = got if swap else got.t()
    for at in (0, 17_000_000, 33_554_000, 35_999_000):
        part = wide[:, at:at + 1001].double()
        close(got[:, at:at + 1001], thin.double().t() @ part, thin.double().abs().t() @ part.abs(), rows)

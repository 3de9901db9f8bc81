"""The most rows that the linear cross entropy takes, few of which count: the join's workgroups go along two dimensions of a
grid, since 2^22 of them with 1024 threads each are more than one holds."""

import pytest
import torch

import apexw_amd
from test_gpu_linear_cross_entropy import Exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2 ** 26 - 16, 2 ** 26 - 15, 2 ** 26 - 1])
def test_most_rows(rows):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 8, generator=g).bfloat16().cuda().expand(rows, 8)
    w = torch.randn(16, 8, generator=g).bfloat16().cuda()
    target = torch.full((rows,), -100, dtype=torch.int32, device="cuda")
    at = torch.cat([torch.arange(0, 40), torch.tensor([rows // 2]), torch.arange(rows - 40, rows)]).cuda()
    target[at] = torch.randint(0, 16, (len(at),), generator=g).int().cuda()
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    exact = Exact(x[at], w, target[at])
    exact.check_forward(loss[at], lse[at])
    total = apexw_amd.linear_cross_entropy(x, w, target, reduction="sum")
    assert int((loss != 0).sum()) == len(at) and int((lse != 0).sum()) == len(at)
    assert float(total) == pytest.approx(float(loss[at].double().sum()), rel=2.0 ** -23)
    d = torch.full((), 1.0 / len(at), device="cuda").expand(rows)
    dx, dw = apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse)
    exact.check_backward(d[at], lse[at], dx[at], dw)
    assert int((dx != 0).any(1).sum()) == len(at)


def test_all_of_them_refused_beyond():
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda").expand(2 ** 26, 8)
    with pytest.raises(RuntimeError):
        apexw_amd.linear_cross_entropy_forward(x, x[:16].contiguous(), torch.zeros(2 ** 26, dtype=torch.int32, device="cuda"))

"""Expert products of operands whose rows overlap in memory (a row broadcast over all rows, sliding windows),
against float64 with the bars of test_gpu_experts.

Such rows follow each other at less than their width, so the memory of an expert's own rows also holds what
would be its next rows: those must not be summed."""

import pytest
import torch

import apexw_amd
from test_gpu_experts import check, close, exact, make

pytestmark = pytest.mark.gpu
SIZES = {"one": [20], "ragged": [1, 0, 37, 64, 65, 100, 63], "long": [5000], "many": [(7 * i) % 23 for i in range(80)]}


def windows(rows, width, step, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    flat = torch.randn((rows - 1) * step + width, generator=g).to(dtype).cuda()
    return flat.as_strided((rows, width), (step, 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [0, 8, 24])
@pytest.mark.parametrize("name", list(SIZES))
def test_both_operands_overlap(name, step, dtype):
    sizes = SIZES[name]
    for inner, outer in ((64, 96), (200, 136), (64, 90)):
        _, _, w, ends = make(sizes, inner, outer, dtype)
        rows = sum(sizes) + 3
        x, dy = windows(rows, inner, step, dtype, inner), windows(rows, outer, step, dtype, outer + 1)
        assert x.stride() == (step, 1) and dy.stride() == (step, 1)
        check(sizes, x, dy, w, ends)


@pytest.mark.parametrize("which", ["x", "dy"])
def test_one_operand_overlaps(which):
    """The last element of expert 0's last row is infinite; row 20's would be in other columns."""
    sizes, inner, outer = [20, 44], 64, 96
    x, dy, w, ends = make(sizes, inner, outer, torch.bfloat16)
    if which == "x":
        x = windows(64, inner, 8, torch.bfloat16, 1)
        x[19, inner - 1] = float("inf")
    else:
        dy = windows(64, outer, 8, torch.bfloat16, 1)
        dy[19, outer - 1] = float("inf")
    (_, _, dw), (_, _, mag) = exact(sizes, x, dy, w)
    got = apexw_amd.expert_matmul_weight_grad(dy, x, ends)
    assert torch.equal(torch.isfinite(got), torch.isfinite(dw))
    fine = torch.isfinite(dw)
    close(got[fine], dw[fine], mag[fine], 64)


@pytest.mark.parametrize("transposed", [False, True])
def test_overlapping_weights(transposed):
    """Weights whose rows along k overlap; their last element is infinite."""
    k, n, sizes = 40, 64, [30, 7]
    g = torch.Generator().manual_seed(5)
    flat = torch.randn(4096, generator=g).bfloat16().cuda()
    w = flat.as_strided((2, k, n), (2048, 8, 1))
    w[:, k - 1, n - 1] = float("inf")
    a = torch.randn(37, k, generator=g).bfloat16().cuda()
    ends = torch.tensor([30, 37], dtype=torch.int32, device="cuda")
    got = (apexw_amd.expert_matmul_forward(a, w.transpose(1, 2), ends) if transposed
           else apexw_amd.expert_matmul_rows_grad(a, w, ends))
    want, mag = (torch.cat([f(a[:30]).double() @ f(w[0]).double(), f(a[30:]).double() @ f(w[1]).double()])
                 for f in (lambda t: t, torch.abs))
    fine = torch.isfinite(want)
    assert not fine.all() and torch.equal(torch.isfinite(got), fine)
    close(got[fine], want[fine], mag[fine], k)


def test_broadcast_rows_through_autograd():
    """One row for all of an expert layer's inputs, and the gradient of a sum over its rows."""
    sizes = [20, 0, 70, 5]
    _, _, w, ends = make(sizes, 64, 96, torch.bfloat16)
    u, v = torch.randn(64, device="cuda").bfloat16(), torch.randn(96, device="cuda").bfloat16()
    leaf = w.clone().requires_grad_()
    apexw_amd.expert_matmul(u.expand(95, 64), leaf, ends).sum(0).backward(v)
    outer = v.double()[:, None] * u.double()
    want = torch.stack([n * outer for n in sizes])
    close(leaf.grad, want, want.abs(), 70)

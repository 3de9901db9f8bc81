"""The norm of gradients whose squares leave the normal fp32 range downwards, against float64 with the bars of
test_gpu_clip_grads."""

import pytest
import torch

import apexw_amd
from test_gpu_clip_grads import E, check, exact_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-14, 1e-17, 1e-19, 1e-20, 1e-22, 1e-25, 1e-30, 1e-34])
def test_scales(scale, dtype):
    g = torch.Generator().manual_seed(int(-torch.tensor(scale).log10()))
    for sizes in ([1], [7, 9000], [40000, 0, 3]):
        grads = [(torch.randn(n, generator=g).double() * scale).to(dtype).cuda() for n in sizes]
        if scale >= 1e-30:                   # (smaller copies are subnormal numbers, which lose more than the bars)
            check(grads, 1e-6 * 0.25, 2.0)   # the coefficient is about a quarter
        for p in (1.0, 2.0, float("inf")):
            norm, want = float(apexw_amd.grad_norm(grads, p)), exact_norm(grads, p)
            assert want > 0 and abs(norm - want) <= E * want


def test_subnormal_gradients():
    """The norm itself may be subnormal: half of the smallest number is lost at most."""
    for value, n in ((1e-40, 1), (3e-45, 5000), (1e-38, 9000)):
        grads = [torch.full((n,), value, device="cuda")]
        want = exact_norm(grads, 2.0)
        assert want > 0 and abs(float(apexw_amd.grad_norm(grads)) - want) <= E * want + 2.0 ** -150


def test_among_larger_and_zero_ones():
    """Small elements next to zeros, and next to larger ones that decide the norm."""
    z = torch.zeros(20000, device="cuda")
    z[12345] = 1e-25
    assert abs(float(apexw_amd.grad_norm([z])) - float(z.double().norm())) <= E * 1e-25
    check([z, torch.full((9000,), 1e-24, device="cuda")], 1e-7)
    check([z, torch.full((100,), 2.0, device="cuda")], 1.0)
    zeros = [torch.zeros(70000, device="cuda"), torch.zeros(5, device="cuda").bfloat16()]
    assert float(apexw_amd.clip_grads(zeros, 1.0)) == 0.0

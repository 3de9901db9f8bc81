"""Tensors that share memory are refused by each form of the clip before anything is written."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [2, 60])
def test_refused(count):
    base = torch.randn(count * 100, device="cuda")
    grads = [base[100 * i:100 * i + 100] for i in range(count)]
    before = base.clone()
    for bad in (grads + [grads[1]], grads + [base[150:160]], [base] + grads):
        with pytest.raises(ValueError, match="share memory"):
            apexw_amd.clip_grads(bad, 1e-3)
        with pytest.raises(ValueError, match="share memory"):
            apexw_amd.scale_grads(bad, 1e-3, torch.ones((), device="cuda"))
    with pytest.raises(ValueError, match="share memory"):
        apexw_amd.clip_grads(grads[:2], 1e-3, out=[grads[1], torch.empty_like(grads[0])])
    p = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    p.grad = grads[0]
    with pytest.raises(ValueError, match="share memory"):
        apexw_amd.clip_grad_norm_([p, p], 1e-3)
    torch.cuda.synchronize()
    assert torch.equal(base, before)
    want = float((2 * base.double().square().sum()).sqrt())
    assert abs(float(apexw_amd.grad_norm(grads + [base])) - want) <= 2.0 ** -18 * want      # reading them twice is fine
    out = [torch.empty(100, device="cuda") for _ in range(2)]
    apexw_amd.clip_grads([grads[0], grads[0]], 1e9, out=out)
    assert torch.equal(out[0], grads[0]) and torch.equal(out[1], grads[0])

"""Autograd notices gradients that a clip has changed."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("clip", [lambda g: apexw_amd.clip_grads(g, 0.1), lambda g: apexw_amd.scale_grads(g, 0.1, torch.ones((), device="cuda")),
                                  lambda g: apexw_amd.clip_grads(g + [torch.ones(3, device="cuda") for _ in range(60)], 0.1)])
def test_saved_gradients(clip):
    g = [torch.randn(100, device="cuda")]
    w = torch.randn(100, device="cuda", requires_grad=True)
    loss = (w * g[0]).sum()                   # saves g[0]
    clip(g)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    loss = (w * g[0]).sum()
    apexw_amd.grad_norm(g)                    # only reads
    apexw_amd.clip_grads(g, 0.01, out=[torch.empty(100, device="cuda")])
    loss.backward()
    assert torch.equal(w.grad, g[0])


def test_inference_tensors():
    with torch.inference_mode():
        g = torch.ones(100, device="cuda")
        apexw_amd.clip_grads([g], 1.0)
    apexw_amd.clip_grads([g], 0.5)
    assert abs(float(g.norm()) - 0.5) <= 1e-5

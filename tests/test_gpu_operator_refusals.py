"""What the operators around the step refuse for tensors on the GPU: they raise, and write nothing."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


def test_layer_norm():
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(ValueError, match="shape"):
        apexw_amd.layer_norm_forward(x, w[:7], None)
    with pytest.raises(TypeError, match="bfloat16"):
        apexw_amd.layer_norm_forward(x, w.bfloat16(), None)
    with pytest.raises(TypeError, match="bias"):
        apexw_amd.layer_norm_forward(x.bfloat16(), w, w.bfloat16())
    with pytest.raises(ValueError, match="GPU"):
        apexw_amd.layer_norm_forward(x, w.cpu(), None)
    with pytest.raises(ValueError, match="eps"):
        apexw_amd.layer_norm_forward(x, w, None, -1.0)
    _, mean, rstd = apexw_amd.layer_norm_forward(x, w, w)
    with pytest.raises(ValueError, match="dy"):
        apexw_amd.layer_norm_backward(x[:3], x, mean, rstd, w, w)
    with pytest.raises(ValueError, match="mean"):
        apexw_amd.layer_norm_backward(x, x, mean[:3], rstd, w, w)
    with pytest.raises(ValueError, match="rstd"):
        apexw_amd.layer_norm_backward(x, x, mean, rstd.double(), w, w)


def test_expert_matmul():
    x = torch.randn(10, 16, device="cuda").bfloat16()
    w = torch.randn(3, 24, 16, device="cuda").bfloat16()
    ends = torch.tensor([2, 5, 10], dtype=torch.int32, device="cuda")
    for call in (lambda: apexw_amd.expert_matmul_forward(x[:, :8], w, ends),
                 lambda: apexw_amd.expert_matmul_forward(x, w, ends[:2]),
                 lambda: apexw_amd.expert_matmul_forward(x, w, ends.float()),
                 lambda: apexw_amd.expert_matmul_forward(x, w, ends.cpu()),
                 lambda: apexw_amd.expert_matmul_forward(x, w[0], ends),
                 lambda: apexw_amd.expert_matmul_rows_grad(x, w, ends),
                 lambda: apexw_amd.expert_matmul_weight_grad(x[:9], x, ends)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        apexw_amd.expert_matmul_forward(x, w.half(), ends)
    with pytest.raises(TypeError):
        apexw_amd.expert_matmul_weight_grad(x, x, ends, torch.float16)


def test_clip():
    g = [torch.randn(100, device="cuda"), torch.randn(20, 30, device="cuda")]
    before = [t.clone() for t in g]
    for bad, match in ((g + [torch.randn(4)], "device"), (g + [torch.randn(4, device="cuda").double()], "float32"),
                       (g + [torch.randn(40, 8, device="cuda")[:, :4]], "dense"),
                       (g + [torch.zeros(3, device="cuda").to_sparse()], "sparse")):
        with pytest.raises((ValueError, TypeError), match=match):
            apexw_amd.clip_grads(bad, 1e-3)
    with pytest.raises(ValueError, match="layout"):
        apexw_amd.clip_grads(g, 1e-3, out=[g[0], torch.empty(30, 20, device="cuda").t()])
    with pytest.raises(ValueError, match="shape"):
        apexw_amd.clip_grads(g, 1e-3, out=[g[0], torch.empty(600, device="cuda")])
    with pytest.raises(TypeError):
        apexw_amd.clip_grads(g + [1.0], 1e-3)
    with pytest.raises(ValueError, match="total_norm"):
        apexw_amd.scale_grads(g, 1.0, torch.ones(2, device="cuda"))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, g))

"""The operators around the step used together: the example's block against plain torch, and its training."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


def test_block_and_gradients_against_float64():
    """Output and gradients against the same block in float64 with the routing that the bf16 block took.  bf16
    results of each of the four operators and of the two products' inputs add up to a few units of 2^-8 of
    the largest value: 2^-4 of it bounds them."""
    from train_experts import ExpertBlock
    torch.manual_seed(3)
    block = ExpertBlock(64, 96, 5).cuda().bfloat16()
    x = torch.randn(333, 64, device="cuda").bfloat16()
    c = torch.randn(333, 64, device="cuda").bfloat16()
    y = block(x)
    params = dict(block.named_parameters())
    grads = torch.autograd.grad((y * c).sum(), list(params.values()))

    p = {k: v.detach().double().requires_grad_() for k, v in params.items()}
    x64 = x.double()
    h = torch.nn.functional.layer_norm(x64, (64,), p["norm_weight"], p["norm_bias"])
    import apexw_amd
    with torch.no_grad():
        taken = torch.softmax((apexw_amd.layer_norm(x, block.norm_weight, block.norm_bias) @ block.router.t()).float(), -1).max(-1)[1]
    weight = torch.softmax(h @ p["router"].t(), -1).gather(1, taken[:, None])
    up = (p["up"][taken] @ h[:, :, None])[:, :, 0]
    out = x64 + (p["down"][taken] @ torch.nn.functional.gelu(up)[:, :, None])[:, :, 0] * weight
    want = torch.autograd.grad((out * c.double()).sum(), list(p.values()))
    for got, ref in zip((y, *grads), (out, *want)):
        assert float((got.double() - ref).abs().max()) <= 2.0 ** -4 * float(ref.abs().max())


def test_training_lowers_the_loss_and_clips():
    from train_experts import train
    losses, norms = train(steps=60)
    assert all(n > 0 for n in norms)
    assert sum(losses[-5:]) < 0.75 * sum(losses[:5])
    again, _ = train(steps=3)
    assert again == pytest.approx(losses[:3], rel=1e-3)

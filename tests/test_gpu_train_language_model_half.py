"""The example's language model in fp16 against float64: losses and every parameter's gradient, in the norm.

Bars.  About two dozen fp16 results lie on the way of a gradient, each off by half a step, 2^-11, at most and by 2^-11 / sqrt(3)
of itself on average: together 2^-9.5 of the norm where they are independent.  Logits of up to 10 that are off by that part
change a probability by ten times as much, 2^-6, so 2^-5 of the norm; a term that is a tenth too large fails."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

from test_gpu_train_language_model import plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", [3, 4])
def test_gradients_in_the_norm(seed):
    import apexw_amd
    from train_language_model import LanguageModel, batch
    torch.manual_seed(seed)
    vocab, layers = 150, 2
    model = LanguageModel(vocab, 32, 48, 5, layers=layers).cuda().half()
    ids, target = batch(torch.randperm(vocab, device="cuda"), 5, 12, torch.Generator(device="cuda").manual_seed(seed))
    chosen, real = [], apexw_amd.expert_order
    try:
        apexw_amd.expert_order = lambda e, n: (chosen.append(e.clamp(min=0)), real(e, n))[1]
        losses = model(ids, target, reduction="none")
    finally:
        apexw_amd.expert_order = real
    params = dict(model.named_parameters())
    c = torch.rand(losses.shape, device="cuda")
    grads = torch.autograd.grad((losses * c).sum(), list(params.values()))
    p = {k: v.detach().double().requires_grad_() for k, v in params.items()}
    want = plain(p, ids, target, layers, chosen)
    ref = torch.autograd.grad((want * c.double()).sum(), list(p.values()))
    for name, got, exact in zip(("losses", *params), (losses, *grads), (want, *ref)):
        part = float((got.double() - exact).norm() / exact.norm())
        assert part <= 2.0 ** -5, (name, part)

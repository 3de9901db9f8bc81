"""The operators used together: the example's language model against plain torch in float64, and its training loop."""

import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


def plain(p, ids, target, layers, chosen):
    """The model in elementary operations, with the experts that the bf16 model chose."""
    width, padding = p["table"].shape[1], ids.flatten() < 0

    def embed(table, i):
        return torch.where((i >= 0)[..., None], table[i.clamp(min=0)], 0) * width ** 0.5

    before = torch.nn.functional.pad(ids[:, :-1], (1, 0), value=-1)
    x = (embed(p["table"], ids) + embed(p["before"], before)).flatten(0, 1)
    for n in range(layers):
        q = {k.split(".")[2]: v for k, v in p.items() if k.startswith(f"blocks.{n}.")}
        h = torch.nn.functional.layer_norm(x, (width,), q["norm_weight"], q["norm_bias"])
        weight = torch.softmax((h @ q["router"].t()).gather(1, chosen[n]), -1)
        out = 0
        for j in range(chosen[n].shape[1]):
            e = chosen[n][:, j]
            up = torch.stack([q["up"][i] @ v for i, v in zip(e.tolist(), h)])
            y = torch.stack([q["down"][i] @ v for i, v in zip(e.tolist(), torch.nn.functional.gelu(up))])
            out = out + torch.where(padding[:, None], 0, y * weight[:, j:j + 1])
        x = x + out
    h = torch.nn.functional.layer_norm(x, (width,), p["norm_weight"], p["norm_bias"])
    return torch.nn.functional.cross_entropy(h @ p["table"].t(), target.flatten(), ignore_index=-1, reduction="none")


def test_model_and_gradients_against_float64():
    """Losses and gradients against the same model in float64 with the routing that the bf16 model took.  About a dozen
    bf16 results lie between the parameters and a loss, each off by 2^-8 of its value at most, and as many on the way
    back; the residual stream and the norms keep their scale, so a few units of 2^-5 of the largest value bound
    the loss's terms (logits of up to 10) and the gradients."""
    import apexw_amd
    from train_language_model import LanguageModel, batch
    torch.manual_seed(3)
    vocab, layers = 150, 2
    model = LanguageModel(vocab, 32, 48, 5, layers=layers).cuda().bfloat16()
    ids, target = batch(torch.randperm(vocab, device="cuda"), 5, 12, torch.Generator(device="cuda").manual_seed(1))
    assert (ids < 0).any() and (target < 0).any()
    chosen = []
    real = apexw_amd.expert_order
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
    assert ((losses == 0) == (target.flatten() < 0)).all()
    for got, exact in zip((losses, *grads), (want, *ref)):
        assert float((got.double() - exact).abs().max()) <= 2.0 ** -3 * float(exact.abs().max())


def test_mean_is_over_the_tokens_that_count():
    from train_language_model import LanguageModel, batch
    torch.manual_seed(5)
    model = LanguageModel(100, 32, 32, 4).cuda().bfloat16()
    ids, target = batch(torch.randperm(100, device="cuda"), 4, 10, torch.Generator(device="cuda").manual_seed(1))
    each, mean = model(ids, target, reduction="none"), model(ids, target)
    assert float(mean.detach()) == pytest.approx(float(each.detach().double().sum() / (target >= 0).sum()), rel=1e-6)


def test_training_runs():
    from train_language_model import train
    losses, norms = train(steps=4, vocab=500, width=64, hidden=96, sequences=8, length=32)
    assert all(math.isfinite(x) and x > 0 for x in losses + norms)
    again, _ = train(steps=2, vocab=500, width=64, hidden=96, sequences=8, length=32)
    assert again == pytest.approx(losses[:2], rel=1e-3)

"""The backward half of the fp16 cross entropy where G is small: probabilities far below fp16's normal range, and rows whose
dloss is small beside another's.

Bars.  As in test_gpu_linear_cross_entropy: a probability is formed with the part e of itself and G rounds by half a
step, 2^-11 of itself, but G is kept with 2^14 for the largest |dloss|, so a step below the normal range, 2^-24 there, is
2^-38 of the largest |dloss|, and t is half of it.  A result below fp16's own normal range is off by 2^-25 at most."""

import pytest
import torch

import apexw_amd
from test_gpu_linear_cross_entropy import make

pytestmark = pytest.mark.gpu
HALF, LEAST = 2.0 ** -11, 2.0 ** -39


def graded(rows, width, vocab, ignored=0.0):
    """Rows and weights whose logits fall by up to 16 over the vocabulary: probabilities down to some 2^-35."""
    x, w, target = make(rows, width, vocab, torch.float16, ignored)
    x[:, 0] = 4.0
    w[:, 0] = -torch.linspace(0, 4, vocab).cuda()
    return x, w, target


def check(x, w, target, d, dx, dw, lse):
    kept = target >= 0
    x64, w64 = torch.where(kept[:, None], x, 0).double(), w.double()
    d = torch.where(kept, d.double(), 0)
    l = x64 @ w64.t()
    p = torch.exp(l - torch.where(kept, lse.double(), torch.logsumexp(l, 1))[:, None])
    a = x.shape[1] * 2.0 ** -23 * (x64.abs() @ w64.abs().t()).max(1)[0]
    constant = 1.5 * lse.double().abs() + torch.where(d == 0, 1.0, d.abs()).log2().abs()
    e = a + (3 * (l.max(1)[0] - l.min(1)[0]) + 8) * 2.0 ** -24 + 2.0 ** -22 * (25 + constant)
    err = e[:, None] * p * d.abs()[:, None]
    p[torch.arange(len(p), device="cuda"), target.clamp(min=0)] -= 1
    G = p * d[:, None]
    err += HALF * G.abs() + LEAST * float(d.abs().max()) * (d != 0)[:, None]
    for got, want, slack in ((dx, G @ w64, (err + w.shape[0] * 2.0 ** -23 * G.abs()) @ w64.abs()),
                             (dw, G.t() @ x64, (err + len(p) * 2.0 ** -23 * G.abs()).t() @ x64.abs())):
        over = (got.double() - want).abs() - (slack * (1 + HALF) + HALF * want.abs() + 2.0 ** -25)
        assert float(over.max()) <= 0, f"over the bar by {float(over.max())} at {int(over.argmax())}"
    return G


# (few tiles, 64 x 128, 128 x 256, and 256 x 256 with the targets' elements apart; parts of both products)
SIZES = [(40, 64, 700), (150, 136, 700), (900, 264, 5003), (2500, 264, 1203), (4800, 320, 16500)]


@pytest.mark.parametrize("rows,width,vocab", SIZES)
def test_small_probabilities(rows, width, vocab):
    """A loss scaled by 2^17, so that the gradients of improbable words are well within fp16."""
    x, w, target = graded(rows, width, vocab, 0.2)
    lse = apexw_amd.linear_cross_entropy_forward(x, w, target)[1]
    for sign in (1.0, -1.0):
        d = torch.full((rows,), sign * 2.0 ** 17 / rows, device="cuda")
        dx, dw = apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse)
        G = check(x, w, target, d, dx, dw, lse)
    # (the inputs are what this is about: an eighth of G and more lies below half of fp16's least value times dloss)
    assert float((G[target >= 0].abs() < 2.0 ** -25 * float(d.abs().max())).double().mean()) > 0.125


@pytest.mark.parametrize("rows,width,vocab", SIZES)
def test_small_dloss(rows, width, vocab):
    """Every second row's dloss is 2^-12 of the others'."""
    x, w, target = make(rows, width, vocab, torch.float16, 0.2)
    lse = apexw_amd.linear_cross_entropy_forward(x, w, target)[1]
    d = torch.where(torch.arange(rows, device="cuda") % 2 == 0, 2.0 ** 9, 2.0 ** -3)
    dx, dw = apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse)
    check(x, w, target, d, dx, dw, lse)


@pytest.mark.parametrize("power", [-126, -124, -112, -100, 100, 112, 119, 121, 126])
def test_dloss_of_any_size(power):
    """The largest |dloss| at the ends of fp32: what fp16 holds of the gradients is the rounded product."""
    x, w, target = make(100, 64, 300, torch.float16)
    lse = apexw_amd.linear_cross_entropy_forward(x, w, target)[1]
    d = torch.full((100,), 2.0 ** power, device="cuda")
    dx, dw = apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse)
    if power < 0:      # far below fp16's 2^-24
        assert not dx.any() and not dw.any()
    else:              # far above its 65504 wherever G is not tiny
        l = x.double() @ w.double().t()
        G = torch.exp(l - lse.double()[:, None])
        G[torch.arange(100), target] -= 1
        want = G @ w.double()
        assert (dx[want.abs() > 1e-4].abs() == float("inf")).all() and (torch.sign(dx.double()) == torch.sign(want))[want.abs() > 1e-4].all()

"""The gradients of the cross entropy of a linear head against differences of the definition in float64, along the gradient
itself, where the derivative is the gradient's whole norm.

Bars.  (f(+s v) - f(-s v)) / 2 s differs from the derivative by s^2 / 6 of the third one.  Along v a row's logits move at a
rate of at most r = max |x| |v| (or |v| |w|), and the third cumulant of a bounded variable of range 2 r is below r^3.  An element of the gradient
is off by what test_gpu_linear_cross_entropy gives it: the part e of each probability and half a step of G, times the
other operand, the sum's roundings, and half a step of itself.  All of it is below a tenth of the derivative, so that a
gradient of zeros or of the other sign fails."""

import pytest
import torch

import apexw_amd
from test_gpu_linear_cross_entropy import HALF, Exact, make

pytestmark = pytest.mark.gpu
STEP = 1e-3


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rows,width,vocab", [(1, 16, 50), (80, 48, 200), (300, 130, 1003), (1030, 1021, 2050), (2049, 264, 9003)])
def test_along_the_gradient(rows, width, vocab, dtype):
    x, w, target = make(rows, width, vocab, dtype, ignored=0.2 if rows > 1 else 0.0)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    apexw_amd.linear_cross_entropy(*leaves, target).backward()

    def f(a, b):
        return torch.nn.functional.cross_entropy(a @ b.t(), target)

    x64, w64 = x.double(), w.double()
    exact64 = [t.clone().requires_grad_() for t in (x64, w64)]
    f(*exact64).backward()

    exact = Exact(x, w, target)
    count = int(exact.kept.sum())
    p = torch.exp(exact.l - exact.lse[:, None]) * exact.kept[:, None] / count
    # (the gradient's lse is the forward pass's, off by b)
    e = exact.a + exact.b + (3 * exact.R + 8) * 2.0 ** -24 + 2.0 ** -22 * (25 + 1.5 * exact.lse.abs() + 20)
    err = e[:, None] * p
    G = p.clone()
    G[torch.arange(rows), exact.at] -= exact.kept.double() / count
    half = HALF[dtype]
    err += half * G.abs() + 2.0 ** -39 / count
    for k, (slack, reach) in enumerate((((err + vocab * 2.0 ** -23 * G.abs()) @ w64.abs(), w64),
                                        ((err + rows * 2.0 ** -23 * G.abs()).t() @ exact.x64.abs(), exact.x64))):
        g = exact64[k].grad
        v = g / g.norm()
        ends = [f(x64 + t * v, w64) if k == 0 else f(x64, w64 + t * v) for t in (STEP, -STEP)]
        difference = float(ends[0] - ends[1]) / (2 * STEP)
        rate = float(reach.norm(dim=1).max() * v.norm(dim=1).max())
        bar = float((v.abs() * (slack * (1 + half) + half * g.abs() + 2.0 ** -25)).sum())
        bar += STEP ** 2 / 6 * rate ** 3 + 1e-10 / STEP
        assert bar < 0.1 * difference
        assert abs(float((leaves[k].grad.double() * v).sum()) - difference) <= bar

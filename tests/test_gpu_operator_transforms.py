"""What the differentiable operators do not take: a second derivative, forward mode and vmap raise, as a compiled
graph without breaks does; a compiled program with breaks runs them."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


def calls():
    x = torch.randn(6, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    a, m = torch.randn(6, 16, device="cuda").bfloat16(), torch.randn(2, 8, 16, device="cuda").bfloat16()
    ends = torch.tensor([2, 6], dtype=torch.int32, device="cuda")
    return [(x, lambda t: apexw_amd.layer_norm(t, w, w)), (a, lambda t: apexw_amd.expert_matmul(t, m, ends))]


@pytest.mark.parametrize("which", [0, 1])
def test_refused(which):
    x, f = calls()[which]
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(leaf).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(torch.stack([x, x]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: f(t).float().sum())(x)
    with pytest.raises(torch._dynamo.exc.Unsupported):
        torch.compile(f, backend="eager", fullgraph=True)(x)


@pytest.mark.parametrize("which", [0, 1])
def test_compiled_with_breaks(which):
    x, f = calls()[which]
    want = f(x * 2) + 1
    compiled = torch.compile(lambda t: f(t * 2) + 1, backend="eager")
    assert torch.equal(compiled(x), want)
    grads = []
    for g in (compiled, lambda t: f(t * 2) + 1):
        leaf = x.clone().requires_grad_()
        g(leaf).float().square().sum().backward()
        grads.append(leaf.grad)
    assert torch.equal(*grads)

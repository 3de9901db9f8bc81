"""What the tokens' operators, the embedding and the linear cross entropy refuse for tensors on the GPU, and which
derivatives and transforms."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


def order():
    return apexw_amd.expert_order(torch.tensor([[0, 1], [1, 2], [2, 0]], device="cuda"), 3)


def refused(error, match, *calls):
    for call in calls:
        with pytest.raises(error, match=match):
            call()


def test_expert_order():
    e = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    refused(ValueError, "tokens", lambda: apexw_amd.expert_order(e[None], 3), lambda: apexw_amd.expert_order(e[0, 0], 3),
            lambda: apexw_amd.expert_order(e[:, :0], 3))
    refused(ValueError, "expert", lambda: apexw_amd.expert_order(e, 0), lambda: apexw_amd.expert_order(e, -1),
            lambda: apexw_amd.expert_order(e, 2 ** 31 - 1))
    refused(TypeError, "int32 or int64", lambda: apexw_amd.expert_order(e.short(), 3), lambda: apexw_amd.expert_order(e.float(), 3))


def test_dispatch_and_combine():
    o = order()
    x, y, w = torch.randn(3, 16, device="cuda"), torch.randn(6, 16, device="cuda"), torch.ones(3, 2, device="cuda")
    refused(ValueError, "3 tokens", lambda: apexw_amd.expert_dispatch_forward(y, o))
    refused(ValueError, "choices", lambda: apexw_amd.expert_combine_forward(x, o), lambda: apexw_amd.expert_dispatch_backward(x, o))
    refused(ValueError, "weight", lambda: apexw_amd.expert_combine_forward(y, o, w[:, :1]),
            lambda: apexw_amd.expert_combine_backward(x, y, o, w.view(-1)))
    refused(TypeError, "weights", lambda: apexw_amd.expert_combine_forward(y, o, w.half()),
            lambda: apexw_amd.expert_combine_forward(y.half(), o, w.bfloat16()))
    refused(ValueError, "tokens", lambda: apexw_amd.expert_combine_backward(y, y, o, w))
    refused(ValueError, "y", lambda: apexw_amd.expert_combine_backward(x, y[:, :8], o, w), lambda: apexw_amd.expert_combine_backward(x, x, o, w))
    refused(TypeError, "float16", lambda: apexw_amd.expert_combine_backward(x, y.half(), o, w))
    refused(ValueError, "GPU", lambda: apexw_amd.expert_combine_forward(y, o, w.cpu()))
    cpu = apexw_amd.ExpertOrder(*(t.cpu() for t in o))
    refused(ValueError, "GPU", lambda: apexw_amd.expert_dispatch_forward(x, cpu), lambda: apexw_amd.expert_combine_forward(y, cpu, w))
    refused(TypeError, "int32", lambda: apexw_amd.expert_dispatch_forward(x, o._replace(source=o.source.long())),
            lambda: apexw_amd.expert_dispatch_forward(x, o._replace(place=o.place.t())))
    refused(ValueError, "order", lambda: apexw_amd.expert_dispatch_forward(x, o._replace(source=o.source[:5])),
            lambda: apexw_amd.expert_dispatch_forward(x, o._replace(place=o.place[None])))


def test_embedding():
    ids, w = torch.tensor([[1, 2]], device="cuda"), torch.randn(5, 8, device="cuda")
    dy = torch.randn(1, 2, 8, device="cuda")
    refused(TypeError, "int32 or int64", lambda: apexw_amd.embedding_forward(ids.float(), w))
    refused(ValueError, "shape", lambda: apexw_amd.embedding_forward(ids, w[0]), lambda: apexw_amd.embedding_forward(ids, w[:, :0]))
    refused(ValueError, "row", lambda: apexw_amd.embedding_forward(ids, w[:0]), lambda: apexw_amd.embedding_weight_grad(dy, ids, 0))
    refused(ValueError, "GPU", lambda: apexw_amd.embedding_forward(ids, w.cpu()), lambda: apexw_amd.embedding_weight_grad(dy, ids.cpu(), 5))
    refused(ValueError, "scale", lambda: apexw_amd.embedding_forward(ids, w, float("inf")),
            lambda: apexw_amd.embedding_weight_grad(dy, ids, 5, float("nan")))
    refused(ValueError, "gradients", lambda: apexw_amd.embedding_weight_grad(dy[0], ids, 5), lambda: apexw_amd.embedding_weight_grad(dy[:, :1], ids, 5),
            lambda: apexw_amd.embedding_weight_grad(dy[..., :0], ids, 5))
    refused(TypeError, "gradient", lambda: apexw_amd.embedding_weight_grad(dy, ids, 5, dtype=torch.bfloat16),
            lambda: apexw_amd.embedding_weight_grad(dy.double(), ids, 5))


def test_linear_cross_entropy():
    x, w = torch.randn(4, 8, device="cuda").bfloat16(), torch.randn(6, 8, device="cuda").bfloat16()
    t, lse, d = torch.tensor([0, 1, 2, 5], device="cuda"), torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    f, g = apexw_amd.linear_cross_entropy_forward, apexw_amd.linear_cross_entropy_backward
    refused(TypeError, "bfloat16 or float16", lambda: f(x.float(), w.float(), t), lambda: f(x, w.half(), t))
    refused(ValueError, "width", lambda: f(x, w[:, :4], t), lambda: f(x, w[None], t), lambda: f(x, w[:0], t), lambda: f(x[:, :0], w[:, :0], t))
    refused(ValueError, "target", lambda: f(x, w, t[:3]), lambda: f(x[None], w, t))
    refused(TypeError, "int32 or int64", lambda: f(x, w, t.float()))
    refused(ValueError, "GPU", lambda: f(x, w.cpu(), t), lambda: f(x, w, t.cpu()), lambda: g(d, x, w, t, lse.cpu()))
    refused(ValueError, "lse", lambda: g(d, x, w, t, lse[:3]), lambda: g(d, x, w, t, lse.half()))
    refused(ValueError, "dloss", lambda: g(d[:1], x, w, t, lse), lambda: g(d.double(), x, w, t, lse))
    refused(ValueError, "reduction", lambda: apexw_amd.linear_cross_entropy(x, w, t, reduction="max"))


def calls():
    o = order()
    x, y = torch.randn(3, 16, device="cuda"), torch.randn(6, 16, device="cuda")
    ids, table = torch.tensor([0, 3, 3], device="cuda"), torch.randn(5, 16, device="cuda")
    rows, w = torch.randn(3, 16, device="cuda").bfloat16(), torch.randn(7, 16, device="cuda").bfloat16()
    return {"dispatch": (x, lambda t: apexw_amd.expert_dispatch(t, o)), "combine": (y, lambda t: apexw_amd.expert_combine(t, o)),
            "embedding": (table, lambda t: apexw_amd.embedding(ids, t)),
            "head": (rows, lambda t: apexw_amd.linear_cross_entropy(t, w, ids, reduction="none"))}


@pytest.mark.parametrize("which", ["dispatch", "combine", "embedding", "head"])
def test_derivatives_and_transforms(which):
    """A second derivative, forward mode, vmap and torch.func raise; a compiled program with breaks runs them."""
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
    compiled = torch.compile(lambda t: f(t * 2) + 1, backend="eager")
    assert torch.equal(compiled(x), f(x * 2) + 1)

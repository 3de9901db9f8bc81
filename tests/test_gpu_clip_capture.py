"""The clip of a list of gradients in a captured graph: every replay clips the captured tensors.

Between the replays other lists of the same length are clipped eagerly and the streams are synchronized, and
every replay is checked against the eager call on the same values, bit for bit."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


def make(count, seed):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(1 + (977 * i) % 12000, generator=g) * (1 + i % 3)).to((torch.float32, torch.bfloat16)[i % 2]).cuda()
            for i in range(count)]


def captured(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def replays(graph, grads, check):
    """Four replays over new values, with other lists clipped in between."""
    for k in range(4):
        values = make(len(grads), 100 + k)
        others = make(len(grads), 200 + k)
        apexw_amd.clip_grads(others, 1.0)
        apexw_amd.scale_grads(others, 0.5, apexw_amd.grad_norm(others))
        for g, v in zip(grads, values):
            g.copy_(v)
        torch.cuda.synchronize()
        kept = [o.clone() for o in others]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, others))
        check(values)


@pytest.mark.parametrize("p", [1.0, 2.0, float("inf")])
@pytest.mark.parametrize("count", [3, 48, 49, 97, 500])
def test_clip_grads(count, p):
    grads = make(count, 1)
    graph, norm = captured(lambda: apexw_amd.clip_grads(grads, 7.0, p))

    def check(values):
        want = apexw_amd.clip_grads(values, 7.0, p)
        assert torch.equal(norm, want)
        assert all(torch.equal(a, b) for a, b in zip(grads, values))

    replays(graph, grads, check)


@pytest.mark.parametrize("count", [1, 60, 300])
def test_copies(count):
    grads = make(count, 2)
    out = [torch.empty_like(g, dtype=torch.bfloat16) for g in grads]
    graph, norm = captured(lambda: apexw_amd.clip_grads(grads, 3.0, out=out))

    def check(values):
        copies = [torch.empty_like(o) for o in out]
        assert torch.equal(norm, apexw_amd.clip_grads(values, 3.0, out=copies))
        assert all(torch.equal(a, b) for a, b in zip(out, copies))
        assert all(torch.equal(a, b) for a, b in zip(grads, values))

    replays(graph, grads, check)


@pytest.mark.parametrize("count", [1, 5, 130])
def test_halves(count):
    grads = make(count, 3)

    def call():
        norm = apexw_amd.grad_norm(grads)
        apexw_amd.scale_grads(grads, 2.0, norm)
        return norm

    graph, norm = captured(call)

    def check(values):
        want = apexw_amd.grad_norm(values)
        apexw_amd.scale_grads(values, 2.0, want)
        assert torch.equal(norm, want)
        assert all(torch.equal(a, b) for a, b in zip(grads, values))

    replays(graph, grads, check)


def test_parameters():
    params = [torch.nn.Parameter(torch.zeros(30 + i, device="cuda")) for i in range(70)]
    for i, q in enumerate(params):
        q.grad = torch.full_like(q, 1.0 + i)
    graph, norm = captured(lambda: apexw_amd.clip_grad_norm_(params, 1.0))
    for k in range(3):
        for i, q in enumerate(params):
            q.grad.fill_(k + i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = sum((k + i) ** 2 * (30 + i) for i in range(70)) ** 0.5
        assert abs(float(norm) - want) <= 2.0 ** -18 * want
        after = sum(float(q.grad.double().square().sum()) for q in params) ** 0.5
        assert abs(after - want / (want + 1e-6)) <= 1e-6

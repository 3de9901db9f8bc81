"""The tokens' operators, the embedding and the linear cross entropy in a captured graph: every replay against the
eager call on the same values, bit for bit, with eager calls on other tensors in between; on another stream; two calls
at a time on two streams."""

import pytest
import torch

import apexw_amd
from test_gpu_clip_capture import captured
from test_gpu_operator_capture import replays

pytestmark = pytest.mark.gpu


def tokens(n, k, experts, width):
    def make(seed):
        g = torch.Generator().manual_seed(seed)
        e = torch.randint(-1, experts, (n, k), generator=g).cuda()
        return [e] + [torch.randn(s, generator=g).bfloat16().cuda() for s in ((n, width), (n * k, width))] + [torch.rand(n, k, generator=g).cuda()]

    def call(e, x, y, w):
        order = apexw_amd.expert_order(e, experts)
        rows = apexw_amd.expert_dispatch_forward(x, order)
        return [*order, rows, apexw_amd.expert_dispatch_backward(y, order), apexw_amd.expert_combine_forward(y, order, w),
                *apexw_amd.expert_combine_backward(x, y, order, w)]
    return make, call


def embedding(n, vocab, width):
    def make(seed):
        g = torch.Generator().manual_seed(seed)
        ids = (torch.rand(n, generator=g) ** 3 * (vocab + 1)).long().cuda()
        return [ids] + [torch.randn(s, generator=g).bfloat16().cuda() for s in ((vocab, width), (n, width))]

    def call(ids, w, dy):
        return [apexw_amd.embedding_forward(ids, w, 2.0), apexw_amd.embedding_weight_grad(dy, ids, vocab),
                apexw_amd.embedding_weight_grad(dy, ids, vocab, 0.5, torch.float32)]
    return make, call


def head(n, width, vocab):
    def make(seed):
        g = torch.Generator().manual_seed(seed)
        target = torch.randint(-5, vocab, (n,), generator=g).cuda()
        x, w = torch.randn(n, width, generator=g).bfloat16().cuda(), (torch.randn(vocab, width, generator=g) / 8).bfloat16().cuda()
        return [target, x, w, torch.randn(n, generator=g).cuda()]

    def call(target, x, w, d):
        loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
        return [loss, lse, *apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse),
                apexw_amd.linear_cross_entropy(x, w, target), apexw_amd.linear_cross_entropy(x, w, target, reduction="sum")]
    return make, call


# one workgroup's sort and more, one and two passes; few tokens, one sort workgroup, more; tiles of each shape
CASES = {"tokens": tokens(50, 2, 6, 72), "tokens_large": tokens(3000, 4, 700, 264), "embedding_few": embedding(100, 900, 40),
         "embedding": embedding(3000, 700, 264), "embedding_large": embedding(9000, 3000, 72),
         "head": head(9, 64, 300), "head_odd": head(300, 101, 2003), "head_large": head(2100, 264, 9000)}


@pytest.mark.parametrize("name", list(CASES))
def test_replays(name):
    make, call = CASES[name]
    inputs = make(1)
    graph, outs = captured(lambda: call(*inputs))
    replays(graph, outs, inputs, call, make)


@pytest.mark.parametrize("name", list(CASES))
def test_streams(name):
    """On a stream of its own, and two different calls at once: each has its own workspace."""
    make, call = CASES[name]
    one, two = make(2), make(3)
    want = call(*one), call(*two)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(a):
            first = call(*one)
        with torch.cuda.stream(b):
            second = call(*two)
        a.synchronize(), b.synchronize()
        for got, ref in ((first, want[0]), (second, want[1])):
            assert all(torch.equal(p, q) for p, q in zip(got, ref))


def test_two_graphs():
    """Two captured calls replayed in turn and at once share nothing."""
    make, call = CASES["head_odd"]
    one, two = make(4), make(5)
    graphs = [captured(lambda: call(*one)), captured(lambda: call(*two))]
    want = call(*one), call(*two)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(a):
            graphs[0][0].replay()
        with torch.cuda.stream(b):
            graphs[1][0].replay()
        a.synchronize(), b.synchronize()
        for (_, got), ref in zip(graphs, want):
            assert all(torch.equal(p, q) for p, q in zip(got, ref))

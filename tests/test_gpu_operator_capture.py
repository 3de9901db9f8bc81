"""Layer norm and the expert products in a captured graph: every replay against the eager call on the same
values, bit for bit, with eager calls on other tensors in between."""

import pytest
import torch

import apexw_amd
from test_gpu_clip_capture import captured

pytestmark = pytest.mark.gpu


def replays(graph, outs, inputs, call, make):
    for k in range(3):
        for t, v in zip(inputs, make(10 + k)):
            t.copy_(v)
        call(*make(20 + k))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, call(*[t.clone() for t in inputs])):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,width", [(5, 70), (3000, 768), (7, 20000)])
def test_layer_norm(rows, width):
    def make(seed):
        g = torch.Generator().manual_seed(seed)
        return [torch.randn(s, generator=g).bfloat16().cuda() for s in ((rows, width), (width,), (width,), (rows, width))]

    def call(x, w, b, dy):
        y, mean, rstd = apexw_amd.layer_norm_forward(x, w, b)
        return [y, mean, rstd, *apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b)]

    inputs = make(1)
    graph, outs = captured(lambda: call(*inputs))
    replays(graph, outs, inputs, call, make)


# decode, uneven, widths copied to whole chunks, a long sum in parts, more than 64 experts
@pytest.mark.parametrize("experts,rows,inner,outer", [(8, 16, 256, 128), (5, 700, 512, 320), (2, 1000, 1501, 203),
                                                      (1, 6000, 64, 128), (90, 200, 64, 72)])
def test_expert_products(experts, rows, inner, outer):
    def make(seed):
        g = torch.Generator().manual_seed(seed)
        cuts = torch.randint(0, rows + 1, (experts,), generator=g).sort()[0].to(torch.int32).cuda()
        return [torch.randn(s, generator=g).bfloat16().cuda() for s in ((rows, inner), (rows, outer), (experts, outer, inner))] + [cuts]

    def call(x, dy, w, ends):
        return [apexw_amd.expert_matmul_forward(x, w, ends), apexw_amd.expert_matmul_rows_grad(dy, w, ends),
                apexw_amd.expert_matmul_weight_grad(dy, x, ends), apexw_amd.expert_matmul_weight_grad(dy, x, ends, torch.float32)]

    inputs = make(1)
    graph, outs = captured(lambda: call(*inputs))
    replays(graph, outs, inputs, call, make)

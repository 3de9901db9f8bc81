"""Many tokens: sorts of so many workgroups that a launch adds up their counts, more workgroups than go along one
dimension of a grid, more rows than the cross entropy's packing takes at once.  Bars as in the modules whose checks are
used."""

import pytest
import torch

import apexw_amd
from test_gpu_linear_cross_entropy import check as check_head
from test_gpu_linear_cross_entropy import make
from test_gpu_tokens import check_embedding, words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("choices,experts", [(524288, 8), (524289, 8), (600001, 300), (1000000, 1), (1000003, 3), (700000, 5000),
                                             (3000000, 64)])
def test_order_of_many(choices, experts):
    g = torch.Generator().manual_seed(choices)
    e = (torch.rand(choices, generator=g) ** 2 * experts).long().clamp(max=experts - 1)
    e[torch.rand(choices, generator=g) < 0.1] = -1
    key = torch.where(e < 0, experts, e)
    item = torch.sort(key, stable=True)[1]
    rows = int((e >= 0).sum())
    source = torch.where(torch.arange(choices) < rows, item, -1)
    place = torch.full((choices,), -1)
    place[item[:rows]] = torch.arange(rows)
    ends = torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)
    for got, want in zip(apexw_amd.expert_order(e.cuda(), experts), (source, place, ends)):
        assert torch.equal(got.cpu().long(), want)


@pytest.mark.parametrize("tokens,vocab", [(530000, 300), (700001, 40000), (1100000, 5)])
def test_embedding_of_many(tokens, vocab):
    check_embedding(words((tokens,), vocab) - int(vocab > 5), vocab, 24, torch.bfloat16, 1.0, (torch.float32,))


def test_more_workgroups_than_one_dimension_takes():
    """1.1 million tokens of a workgroup each, 2^20 of which go along the first dimension."""
    tokens, width = 1100000, 2048
    x = torch.empty(tokens, width, dtype=torch.bfloat16, device="cuda").normal_()
    expert = torch.randint(0, 5, (tokens,), device="cuda")
    order = apexw_amd.expert_order(expert, 5)
    rows = apexw_amd.expert_dispatch_forward(x, order)
    assert torch.equal(rows, x[order.source.long()])
    weight = torch.randint(0, 2, (tokens,), device="cuda").float()
    assert torch.equal(apexw_amd.expert_combine_forward(rows, order, weight), x * weight[:, None].bfloat16())
    ones = torch.ones_like(rows)
    dy, dw = apexw_amd.expert_combine_backward(x, ones, order, weight)
    assert torch.equal(dy, rows * weight[order.source.long(), None].bfloat16())
    # sums of 2048 products with 1, as of any other sum: a half of 2^-23 of the magnitudes each
    some = slice(tokens - 60000, tokens)
    exact = x[some].double()
    assert ((dw[some].double() - exact.sum(1)).abs() <= 2050 * 2.0 ** -24 * exact.abs().sum(1)).all()
    del ones, dy, rows, x, exact
    ids = torch.randint(-1, 3, (tokens,), device="cuda")
    table = torch.randn(3, width, device="cuda").bfloat16()
    assert torch.equal(apexw_amd.embedding_forward(ids, table), torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)], 0))


@pytest.mark.parametrize("rows", [262144, 300001])
def test_linear_cross_entropy_of_many_rows(rows):
    x, w, target = make(rows, 16, 40, torch.bfloat16, ignored=0.3)
    check_head(x, w, target)
    target[:] = -100
    target[-1] = 3
    check_head(x, w, target)


def test_scale_beyond_fp32():
    ids, w = torch.tensor([0, 5], device="cuda"), torch.randn(3, 8, device="cuda")
    for scale in (1e39, float("inf"), float("nan"), -1e300):
        with pytest.raises(ValueError, match="scale"):
            apexw_amd.embedding(ids, w, scale)
        with pytest.raises(ValueError, match="scale"):
            apexw_amd.embedding_weight_grad(torch.randn(2, 8, device="cuda"), ids, 3, scale)
    assert torch.equal(apexw_amd.embedding(ids, w, 2.0 ** 127)[1], torch.zeros(8, device="cuda"))

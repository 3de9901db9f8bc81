"""Orders by the most experts there may be: sorts of four passes, and the ends of nearly 2^31 experts."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 2


@pytest.mark.parametrize("choices", [1, 3000, 70000])
@pytest.mark.parametrize("experts", [2 ** 27 + 1, 2 ** 30, MOST - 255, MOST])
def test_order(choices, experts):
    g = torch.Generator().manual_seed(choices)
    e = torch.randint(0, experts, (choices,), generator=g)
    e[::3] = e[0]                       # an expert of many
    e[1::7] = experts - 1
    e[2::11] = experts                  # no expert
    e[3::13] = -1
    valid = (e >= 0) & (e < experts)
    key = torch.where(valid, e, experts)
    item = torch.sort(key, stable=True)[1]
    rows = int(valid.sum())
    source = torch.where(torch.arange(choices) < rows, item, -1)
    place = torch.full((choices,), -1)
    place[item[:rows]] = torch.arange(rows)
    order = apexw_amd.expert_order(e.cuda(), experts)
    assert torch.equal(order.source.cpu().long(), source) and torch.equal(order.place.cpu().long(), place)
    # an end rises at the experts that have rows, by as many, and nowhere else
    ids, counts = torch.unique(key[valid], return_counts=True)
    ends = order.ends
    assert ends.shape == (experts,) and int(ends[-1]) == rows
    assert torch.equal(ends[ids.cuda()].cpu().long(), counts.cumsum(0))
    before = torch.where(ids > 0, ends[(ids - 1).clamp(min=0).cuda()].cpu().long(), 0)
    assert torch.equal(before, counts.cumsum(0) - counts)
    step, last = 2 ** 28, 0
    for a in range(0, experts, step):   # never falls
        part = ends[a:a + step]
        assert int(part[0]) >= last and not (part[1:] < part[:-1]).any()
        last = int(part[-1])

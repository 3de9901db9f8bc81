"""Each way that the cross entropy of a linear head may take -- few rows as they stand, the four tile shapes of the logits, forward and
backward, the shapes and parts of the two products with the probabilities, one piece of the vocabulary and more,
weights copied to whole chunks -- at a size that takes it, against
float64 with the bars of test_gpu_linear_cross_entropy.  The kernels that ran are read from a profile, so a size that a
changed rule sends elsewhere fails here."""

import re

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

import apexw_amd
from test_gpu_linear_cross_entropy import Exact, make

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SHAPES = {"256, 256": "Large", "128, 256": "Wide", "64, 128": "Mid", "32, 128": "Small"}


def taken(call):
    """The call's result, and what ran: the shape of each product, whether parts or pieces were joined."""
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        out = call()
        torch.cuda.synchronize()
    ways = set()
    for name in (e.name for e in p.events() if "head_" in e.name):
        shape = re.search(r"Shape<(\d+, \d+)", name)
        for kernel, what in (("logits", "logits"), ("rows", "dx"), ("weight_kernel", "dw")):
            if f"head_{kernel}" in name and shape:
                ways.add(f"{what}:{SHAPES[shape[1]]}")
        if "head_rows" in name and "true>" in name:
            ways.add("added")
        if "join_weight" in name:
            ways.add("dw:parts")
        if "head_few" in name:
            ways.add("few")
        if "head_targets" in name:
            ways.add("targets")
    return out, ways


def check(what, rows, width, vocab, dtype, ignored):
    x, w, target = make(rows, width, vocab, dtype, ignored)
    exact = Exact(x, w, target)
    dloss = torch.full((rows,), 1.0 / max(1, int(exact.kept.sum())), device="cuda")
    lse = exact.lse.float()
    if "forward" in what:
        (loss, got), ways = taken(lambda: apexw_amd.linear_cross_entropy_forward(x, w, target))
        exact.check_forward(loss, got)
        assert ways == what - {"forward"}
        return
    (dx, dw), ways = taken(lambda: apexw_amd.linear_cross_entropy_backward(dloss, x, w, target, lse))
    exact.check_backward(dloss, lse, dx, dw)
    assert what <= ways, (what, ways)


# rows with remainders modulo 256 of 1, 128, 129 and others, widths that end inside a stage, a chunk and a tile
CASES = [
    ("forward logits:Large", 2049, 520, 16500, BF16, 0.1), ("forward logits:Large", 2176, 264, 20011, FP16, 0.0),
    ("forward logits:Wide", 582, 701, 7374, BF16, 0.2), ("forward logits:Wide", 641, 264, 9003, FP16, 0.0),
    ("forward logits:Mid", 1500, 101, 2003, BF16, 0.1), ("forward logits:Mid", 4605, 1569, 416, FP16, 0.3),
    ("forward logits:Small", 31, 765, 5003, BF16, 0.1), ("forward few", 31, 768, 5003, BF16, 0.1),
    ("forward few", 1, 64, 129, FP16, 0.0), ("forward few", 32, 1024, 70001, BF16, 0.3), ("forward few", 16, 4096, 300, FP16, 0.0),
    ("forward logits:Small", 640, 1021, 1500, FP16, 0.0),
    ("logits:Large targets dx:Large dw:Large", 4800, 768, 16500, BF16, 0.1),
    ("logits:Large targets dx:Large dw:Wide", 5798, 325, 14144, FP16, 0.0),
    ("logits:Large targets dx:Mid dw:Large dw:parts", 6677, 24, 18997, BF16, 0.1),
    ("logits:Wide dx:Large dw:Wide dw:parts", 7274, 1599, 698, BF16, 0.0),
    ("logits:Wide dx:Wide", 2227, 131, 10340, FP16, 0.1), ("logits:Wide dx:Mid dw:Wide", 900, 264, 5003, BF16, 0.2),
    ("logits:Mid dx:Wide", 4605, 1569, 416, FP16, 0.1), ("logits:Mid dx:Small dw:parts", 2500, 264, 1203, BF16, 0.1),
    ("logits:Small dx:Wide dw:parts", 7899, 1792, 212, BF16, 0.4), ("logits:Small dx:Small dw:Wide", 513, 300, 2100, FP16, 0.1),
    ("logits:Small dx:Small", 20, 520, 3000, BF16, 0.0), ("dw:parts", 9000, 72, 130, FP16, 0.0),
]


@pytest.mark.parametrize("what,rows,width,vocab,dtype,ignored", CASES,
                         ids=[f"{c[0].replace(' ', '-')}-{c[1]}x{c[2]}x{c[3]}-{str(c[4])[6:]}" for c in CASES])
def test_way(what, rows, width, vocab, dtype, ignored):
    check(set(what.split()), rows, width, vocab, dtype, ignored)


@pytest.mark.parametrize("rows,width,vocab", [(60000, 64, 20011), (100000, 1024, 30010)])
def test_pieces(rows, width, vocab):
    """Several pieces, each of whose sums of dx is added to the ones before."""
    x, w, target = make(rows, width, vocab, BF16, 0.3)
    dloss = torch.full((rows,), 1.0 / rows, device="cuda")
    _, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    (dx, dw), ways = taken(lambda: apexw_amd.linear_cross_entropy_backward(dloss, x, w, target, lse))
    assert "added" in ways
    # against the formula over some of the rows and of the vocabulary, with the bars of `check_backward`
    some = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:500].cuda()
    words = torch.cat([torch.arange(0, 300), torch.arange(vocab - 300, vocab)]).cuda()
    part = Exact(x[some], w, target[some])
    given = torch.where(part.kept, lse[some], 0)
    part.check_backward(dloss[some], given, dx[some], None)
    kept = target >= 0
    p = torch.exp(x.double() @ w[words].double().t() - lse.double()[:, None])
    p = (p - (target[:, None] == words[None, :]).double()) * dloss.double()[:, None] * kept[:, None]
    want, mag = p.t() @ x.double(), p.abs().t() @ x.double().abs()
    # a probability is off by its part e and G by half a step: 2^-8 and the logits' error, below 2^-14 here
    bar = (2.0 ** -8 + 2.0 ** -12 + rows * 2.0 ** -23) * mag + 2.0 ** -8 * want.abs()
    assert float(((dw[words].double() - want).abs() - bar).max()) <= 0


@pytest.mark.parametrize("rows", [1, 15, 17, 32])
def test_few_rows(rows):
    """Rows as they stand: other targets that do not count, distances between rows, logits far apart, what stands in rows
    that do not count, the mean."""
    x, w, target = make(rows, 136, 1000, BF16, lean=40.0)
    wide = torch.randn(rows, 144, device="cuda").bfloat16()
    wide[:, 8:] = x
    target[::3], ignored = 7, 7
    if rows > 3:
        target[1], target[2] = 1000, -1
    exact = Exact(x, w, target, ignored)
    for t in (target, target.int()):
        for rows_of in (x, wide[:, 8:]):
            loss, lse = apexw_amd.linear_cross_entropy_forward(rows_of, w, t, ignored)
            exact.check_forward(loss, lse)
    bad = x.clone()
    bad[~exact.kept] = float("nan")
    loss, lse = apexw_amd.linear_cross_entropy_forward(bad, w, target, ignored)
    exact.check_forward(loss, lse)
    mean = apexw_amd.linear_cross_entropy(bad, w, target, ignored)
    kept = int(exact.kept.sum())
    assert mean.isnan() if kept == 0 else float(mean) == pytest.approx(float(loss.double().sum()) / kept, rel=1e-6)
    assert float(apexw_amd.linear_cross_entropy(bad, w, target, ignored, "sum")) == pytest.approx(float(loss.double().sum()), rel=1e-6)


def test_few_rows_of_infinite_logits():
    """A row whose logits overflow to infinity or are not numbers makes its own results alone so."""
    x, w, target = make(9, 64, 500, BF16)
    x[2], x[5] = 1e38, float("nan")
    w[3] = w[3].abs() * 100
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    others = torch.tensor([0, 1, 3, 4, 6, 7, 8], device="cuda")
    assert not loss[2].isfinite() and loss[5].isnan() and lse[5].isnan()
    part = Exact(x[others], w, target[others])
    part.check_forward(loss[others], lse[others])

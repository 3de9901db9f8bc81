"""Losses of rows that are nearly certain of their target, whose logits are large.

Bars.  The loss is log(1 + sum of exp(l_v - l_t) over the other words).  Where the target's term in the sum and its logit
are one number, what is off in the logits (at most a = width 2^-23 of the sum of the magnitudes each, and 3 R 2^-24 for
the difference's rounding, R their range) reaches the loss by the other words alone, whose part is 1 - p.  To that come
250 additions and products of 2^-24 of a sum that is about 1, the instructions' 2^-20, and roundings of the loss itself,
2^-21 of it."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


def make(rows, width, vocab, dtype, scale):
    """Every second row certain of its target by thousands of units of the logits' last place, the others less so."""
    g = torch.Generator().manual_seed(rows + width + vocab)
    w = torch.randn(vocab, width, generator=g) * width ** -0.5
    target = torch.randint(0, vocab, (rows,), generator=g)
    lean = torch.where(torch.arange(rows) % 2 == 0, 1.0, torch.rand(rows, generator=g))[:, None]
    x = torch.randn(rows, width, generator=g) + scale * lean * w[target]
    return x.to(dtype).cuda(), w.to(dtype).cuda(), target.cuda()


def check(rows, width, vocab, dtype, scale=400.0):
    x, w, target = make(rows, width, vocab, dtype, scale)
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    x64, w64 = x.double(), w.double()
    l = x64 @ w64.t()
    want = torch.logsumexp(l, 1) - l.gather(1, target[:, None])[:, 0]
    others = -torch.expm1(-want)
    a = width * 2.0 ** -23 * (x64.abs() @ w64.abs().t()).max(1)[0]
    R = l.max(1)[0] - l.min(1)[0]
    bar = others * (2 * a + 3 * R * 2.0 ** -24) + 250 * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -21 * want
    assert float(l.max()) > scale / 2 and float(want.min()) < 1e-12
    assert (loss >= 0).all(), f"a loss of {float(loss.min())}"
    over = (loss.double() - want).abs() - bar
    assert float(over.max()) <= 0, f"over the bar by {float(over.max())}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width,vocab", [(33, 4096, 300), (40, 1021, 5003), (200, 4096, 2000), (582, 701, 7374),
                                              (1500, 1029, 2003), (2049, 520, 16500)])
def test_packed_rows(rows, width, vocab, dtype):
    check(rows, width, vocab, dtype)


@pytest.mark.parametrize("rows,width,vocab", [(300, 264, 2003), (70, 4096, 300), (2049, 520, 16500)])
def test_logits_of_any_size(rows, width, vocab):
    """Logits up to some 10^9, of both signs: the exponents' range is left wherever a target is not the largest."""
    for scale in (1e-30, 1e-3, 1e5, 1e9):
        x, w, target = make(rows, width, vocab, torch.bfloat16, 40.0)
        for y in (x * scale, x * -scale):
            loss, lse = apexw_amd.linear_cross_entropy_forward(y, w, target)
            l = y.double() @ w.double().t()
            at = l.gather(1, target[:, None])[:, 0]
            want = torch.logsumexp(l, 1)
            # b and 2 b of test_gpu_linear_cross_entropy
            a = width * 2.0 ** -23 * (y.double().abs() @ w.double().abs().t()).max(1)[0]
            bar = a + (3 * (l.max(1)[0] - l.min(1)[0]) + 250) * 2.0 ** -24 + 2.0 ** -22 * (want.abs() + 20)
            assert (loss >= 0).all() and loss.isfinite().all() and lse.isfinite().all()
            assert float(((lse.double() - want).abs() - bar).max()) <= 0
            assert float(((loss.double() - (want - at)).abs() - 2 * bar).max()) <= 0


def test_vocabulary_beyond_the_places():
    """More than 2^18 words: several words share a place in a row's shift."""
    x, w, target = make(70, 64, 300001, torch.bfloat16, 100.0)
    target[:8] = torch.tensor([0, 131072, 131071, 262144, 300000, 31, 131103, 262175])
    x[:8] = (60.0 * w[target[:8]].float()).bfloat16()
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    l = x.double() @ w.double().t()
    want = torch.logsumexp(l, 1)
    # b and 2 b of test_gpu_linear_cross_entropy; its 250 additions are 64 in a wave, 4700 waves' sums over 64 threads and 20
    a = 64 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).max(1)[0]
    bar = a + (3 * (l.max(1)[0] - l.min(1)[0]) + 250) * 2.0 ** -24 + 2.0 ** -22 * (want.abs() + 20)
    assert float(((lse.double() - want).abs() - bar).max()) <= 0
    assert float(((loss.double() - (want - l.gather(1, target[:, None])[:, 0])).abs() - 2 * bar).max()) <= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width,vocab", [(1, 64, 129), (8, 768, 5003), (16, 4096, 300), (32, 1024, 40001)])
def test_few_rows(rows, width, vocab, dtype):
    """Rows as they stand, without a packing."""
    for scale in (400.0, 100.0):
        check(rows, width, vocab, dtype, scale)


@pytest.mark.parametrize("rows,width,vocab", [(5, 264, 2003), (32, 4096, 300)])
def test_few_rows_of_any_size(rows, width, vocab):
    test_logits_of_any_size(rows, width, vocab)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0.0, 30.0, 1000.0, -1000.0])
@pytest.mark.parametrize("rows", [1, 20, 32, 33, 300, 2049])
def test_offset(rows, offset, dtype):
    """A number that all logits of a row share changes nothing.  Logits are sums that fp32 holds exactly here, so a is 0."""
    g = torch.Generator().manual_seed(rows)
    w = torch.zeros(5003, 8)
    w[:, 0], w[:, 1:4] = 1.0, torch.randint(-32, 33, (5003, 3), generator=g) / 32.0
    x = torch.zeros(rows, 8)
    x[:, 0], x[:, 1:4] = offset, torch.randint(-8, 9, (rows, 3), generator=g) / 2.0
    target = torch.randint(0, 5003, (rows,), generator=g).cuda()
    x, w = x.to(dtype).cuda(), w.to(dtype).cuda()
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    l = x.double() @ w.double().t()
    full = torch.logsumexp(l, 1)
    want = full - l.gather(1, target[:, None])[:, 0]
    bar = (3 * (l.max(1)[0] - l.min(1)[0]) + 250) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -21 * want
    over = (loss.double() - want).abs() - bar
    assert float(over.max()) <= 0, f"over the bar by {float(over.max())}"
    assert float(((lse.double() - full).abs() - bar - 2.0 ** -22 * full.abs()).max()) <= 0

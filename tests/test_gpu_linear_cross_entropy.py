"""The cross entropy of a linear head against float64.

Bars.  A logit is a sum of `width` exact products in fp32, of which each addition loses at most 2^-23 of what it has added
up (the matrix cores may truncate): it is off by at most a = width 2^-23 of the sum of the magnitudes.  exp(l - m) of a
logit R below the largest rounds the difference and its product with log2 e and takes a constant of 25 bits, 3 R 2^-24,
and 2^-22 for the instruction; fewer than 250 additions and products bring a row's sum together.  So
    lse is off by   b = a + (3 R + 250) 2^-24 + 2^-22 (|lse| + 20)      (logarithm and last additions)
and the loss by 2 b.  With an lse that is given, a probability times dloss is formed as one power of 2, whose exponent's
constant part is held in fp32 but for its lowest bit (2^-22 of it, with the roundings of its three terms), so it is off by
the part e = a + (3 R + 8) 2^-24 + 2^-22 (1 + 1.5 |lse| + |log2 dloss| + 24) of itself, and G rounds by half a step of its type (in fp16 by 2^-25 of the largest |dloss| at least), so
    dx is off by    sum_v |W| (h |G| + e p |dloss| + t) + vocabulary 2^-23 sum_v |G W|
before it rounds by half a step itself, and dW likewise over the rows.  Below 2^-126, the normal range of fp32 and
bf16, the exponential's instruction and the matrix cores may give 0: t is 2^-126 times |dloss|'s largest or one at least,
and so is what a result may be off by."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(rows, width, vocab, dtype, ignored=0.0, seed=0, lean=6.0):
    g = torch.Generator().manual_seed(seed + rows * 7 + width * 3 + vocab)
    w = torch.randn(vocab, width, generator=g) * width ** -0.5
    target = torch.randint(0, vocab, (rows,), generator=g)
    x = torch.randn(rows, width, generator=g) + lean * torch.rand(rows, 1, generator=g) * w[target]
    if ignored:
        target[torch.rand(rows, generator=g) < ignored] = -100
    return x.to(dtype).cuda(), w.to(dtype).cuda(), target.cuda()


class Exact:
    """The definition in float64, with the bars."""

    def __init__(self, x, w, target, ignore_index=-100):
        rows, vocab = target.numel(), w.shape[0]
        self.x, self.w, self.target = x.reshape(rows, -1), w, target.reshape(rows)
        self.kept = (self.target != ignore_index) & (self.target >= 0) & (self.target < vocab)
        self.x64 = torch.where(self.kept[:, None], self.x, 0).double()
        self.w64, self.at = w.double(), self.target.long().clamp(0, vocab - 1)
        self.l = self.x64 @ self.w64.t()
        self.lse = torch.logsumexp(self.l, 1)
        self.loss = torch.where(self.kept, self.lse - self.l.gather(1, self.at[:, None])[:, 0], 0)
        self.a = x.shape[-1] * 2.0 ** -23 * (self.x64.abs() @ self.w64.abs().t()).max(1)[0]
        self.R = self.l.max(1)[0] - self.l.min(1)[0]
        self.b = self.a + (3 * self.R + 250) * 2.0 ** -24 + 2.0 ** -22 * (self.lse.abs() + 20)

    def check_forward(self, loss, lse):
        assert loss.dtype == lse.dtype == torch.float32
        for got, want, bar in ((lse, torch.where(self.kept, self.lse, 0), self.b), (loss, self.loss, 2 * self.b)):
            assert (got.reshape(-1)[~self.kept] == 0).all()
            over = ((got.reshape(-1).double() - want).abs() - bar)[self.kept]
            assert over.numel() == 0 or float(over.max()) <= 0, f"over the bar by {float(over.max())}"

    def check_backward(self, dloss, lse, dx, dw):
        d = torch.where(self.kept, dloss.reshape(-1).double(), 0)
        p = torch.exp(self.l - torch.where(self.kept, lse.reshape(-1).double(), self.lse)[:, None])
        constant = 1.5 * self.lse.abs() + torch.where(d == 0, 1.0, d.abs()).log2().abs()
        e = (self.a + (3 * self.R + 8) * 2.0 ** -24 + 2.0 ** -22 * (25 + constant))[:, None]
        err = e * p * d.abs()[:, None]
        p[torch.arange(len(p), device=p.device), self.at] -= 1
        G, half = p * d[:, None], HALF[self.w.dtype]
        least = 2.0 ** -126 * max(1.0, float(d.abs().max()))
        t = max(least, 2.0 ** -25 * float(d.abs().max())) if self.w.dtype == torch.float16 else least
        err += half * G.abs() + t * (d != 0)[:, None]
        for got, want, slack in ((dx, G @ self.w64, (err + self.w.shape[0] * 2.0 ** -23 * G.abs()) @ self.w64.abs()),
                                 (dw, G.t() @ self.x64, (err + len(p) * 2.0 ** -23 * G.abs()).t() @ self.x64.abs())):
            if got is None:
                continue
            assert got.dtype == self.w.dtype
            got = got.reshape(want.shape).double()
            slack = slack * (1 + half) + half * want.abs() + (2.0 ** -25 if self.w.dtype == torch.float16 else least)
            over = (got - want).abs() - slack
            assert float(over.max()) <= 0, f"over the bar by {float(over.max())}"
        if dx is not None:
            assert (dx.reshape(self.x.shape)[~self.kept] == 0).all()


def check(x, w, target, dloss=None, ignore_index=-100):
    exact = Exact(x, w, target, ignore_index)
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target, ignore_index)
    exact.check_forward(loss, lse)
    if dloss is None:
        dloss = torch.full(target.shape, 1.0 / max(int(exact.kept.sum()), 1), device="cuda")
    given = exact.lse.float().view(target.shape)
    dx, dw = apexw_amd.linear_cross_entropy_backward(dloss, x, w, target, given, ignore_index)
    exact.check_backward(dloss, given, dx, dw)
    return exact, (loss, lse, dx, dw)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rows,width,vocab", [(1, 8, 1), (1, 1, 2), (2, 64, 100), (5, 72, 129), (33, 100, 257), (31, 33, 255),
                                              (70, 264, 1000), (130, 500, 1003), (257, 127, 640), (300, 768, 5003),
                                              (700, 96, 4099), (1030, 1021, 2050)])
def test_sizes(rows, width, vocab, dtype):
    check(*make(rows, width, vocab, dtype, ignored=0.2 if rows > 4 else 0.0))


@pytest.mark.parametrize("rows", [1, 8, 32, 64, 65, 200, 600, 2100])
def test_rows(rows):
    """From a few scored tokens to a batch: every tile shape, sums in parts."""
    check(*make(rows, 512, 16385, torch.bfloat16))


@pytest.mark.parametrize("rows,width,vocab", [(6000, 64, 300), (20000, 64, 9000), (3000, 2048, 70), (9000, 40, 33000)])
def test_long_sums_and_pieces(rows, width, vocab):
    """Many rows of a small head (the weights' gradient in parts), and vocabularies in more than one piece."""
    check(*make(rows, width, vocab, torch.bfloat16, ignored=0.1))


def test_dloss():
    """One for each row, of both signs and very different sizes, zeros; one number for all rows."""
    for dtype in HALF:
        x, w, target = make(150, 136, 700, dtype, ignored=0.2)
        d = torch.randn(150, device="cuda") * torch.exp(3 * torch.randn(150, device="cuda"))
        d[::9] = 0
        check(x, w, target, d)
        check(x, w, target, d * 2.0 ** -40)
        check(x, w, target, torch.full((), -0.37, device="cuda").expand(150))
        check(x, w, target, torch.zeros(150, device="cuda"))
        check(x, w, target, torch.stack([d, d], 1)[:, 1])


def test_ignored_rows():
    """All, none, the first, the last; another ignore_index, targets outside the vocabulary, int32."""
    x, w, target = make(100, 64, 300, torch.bfloat16)
    for change in (slice(0, 100), slice(0, 1), slice(99, 100), slice(0, 99), slice(1, 100), slice(30, 95)):
        t = target.clone()
        t[change] = -100
        check(x, w, t)
    target[::3] = 7
    check(x, w, target, ignore_index=7)
    target[1::5], target[2::5], target[3::7] = 300, -1, 2 ** 40
    check(x, w, target, ignore_index=7)
    check(x, w, target.int())


def test_what_does_not_count_reaches_nothing():
    x, w, target = make(400, 200, 900, torch.float16, ignored=0.4)
    _, clean = check(x, w, target)
    x[target < 0] = float("nan")
    x[(target < 0) & (torch.arange(400, device="cuda") % 2 == 0)] = float("inf")
    _, dirty = check(x, w, target)
    assert all(torch.equal(a, b) for a, b in zip(clean, dirty))
    # a row of NaN that counts stays with its row, and reaches every row of dw
    at = int(torch.nonzero(target >= 0)[3])
    x[at] = float("nan")
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    assert torch.isnan(loss[at]) and torch.isnan(loss).sum() == 1 and torch.isnan(lse).sum() == 1
    dx, dw = apexw_amd.linear_cross_entropy_backward(torch.ones(400, device="cuda"), x, w, target, lse)
    assert torch.isnan(dx[at]).all() and torch.isnan(dx).any(1).sum() == 1 and torch.isnan(dw).all()


def test_extreme_logits():
    """Logits of hundreds, all equal ones, -inf from weights (a word that cannot be), a certain target."""
    x, w, target = make(60, 64, 500, torch.bfloat16)
    check(x * 40, w, target)
    check(x * 0, w, target)
    x = x.abs()
    w[3] = float("-inf")
    target[target == 3] = 4
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    keep = torch.arange(500, device="cuda") != 3
    exact = Exact(x, w[keep], torch.where(target > 3, target - 1, target))
    exact.check_forward(loss, lse)
    dx, dw = apexw_amd.linear_cross_entropy_backward(torch.ones(60, device="cuda"), x, w, target, lse, need=(False, True))
    assert dx is None and torch.isfinite(dw).all() and (dw[3] == 0).all()


def test_views():
    x, w, target = make(90, 160, 600, torch.bfloat16)
    check(x[:, 8:136], w[:, 16:144], target)
    check(x[:, 1:64], w[:, 3:66], target)
    check(x.t().contiguous().t(), w.t().contiguous().t(), target)
    check(x[:1].expand(90, 160), w, target)
    check(x.view(9, 10, 160), w, target.view(9, 10))
    check(x.view(9, 10, 160).transpose(0, 1), w, target.view(9, 10).t())
    check(x[0], w, target[0])
    check(x, w[:1].expand(600, 160), target)


def test_no_rows():
    w = torch.randn(50, 24, device="cuda").bfloat16()
    x, target = w[:0], torch.empty(0, dtype=torch.int64, device="cuda")
    loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
    assert loss.shape == lse.shape == (0,)
    dx, dw = apexw_amd.linear_cross_entropy_backward(loss, x, w, target, lse)
    assert dx.shape == (0, 24) and dw.shape == w.shape and (dw == 0).all()
    assert torch.isnan(apexw_amd.linear_cross_entropy(x, w, target))
    assert apexw_amd.linear_cross_entropy(x, w, target, reduction="sum") == 0


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd(reduction):
    """The reductions and their gradients; the mean is over the rows that count."""
    for dtype in HALF:
        x, w, target = make(220, 72, 333, dtype, ignored=0.3)
        exact = Exact(x, w, target)
        leaves = [t.clone().requires_grad_() for t in (x, w)]
        loss = apexw_amd.linear_cross_entropy(*leaves, target, reduction=reduction)
        count = int(exact.kept.sum())
        if reduction == "none":
            exact.check_forward(loss, apexw_amd.linear_cross_entropy_forward(x, w, target)[1])
            c = torch.randn(220, device="cuda")
            loss.backward(c)
            d = c
        else:
            want = float(exact.loss.sum()) / (count if reduction == "mean" else 1)
            bar = float(2 * exact.b.sum()) / (count if reduction == "mean" else 1) + 2.0 ** -23 * abs(want)
            assert loss.shape == () and abs(float(loss) - want) <= bar
            (loss * 3.0).backward()
            d = torch.full((220,), 3.0 / (count if reduction == "mean" else 1), device="cuda")
        # (the gradient's lse is the forward pass's: off by b, which its probabilities multiply)
        exact.a = exact.a + exact.b
        exact.check_backward(d, exact.lse.float(), leaves[0].grad, leaves[1].grad)
    only = w.clone().requires_grad_()
    apexw_amd.linear_cross_entropy(x, only, target).backward()
    assert only.grad is not None


def test_all_ignored():
    x, w, _ = make(40, 64, 100, torch.bfloat16)
    target = torch.full((40,), -100, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    loss = apexw_amd.linear_cross_entropy(*leaves, target)
    loss.backward()
    assert torch.isnan(loss) and (leaves[0].grad == 0).all() and (leaves[1].grad == 0).all()
    assert apexw_amd.linear_cross_entropy(x, w, target, reduction="sum") == 0


def test_gradient_against_differences():
    """Along random directions: (f(+s v) - f(-s v)) / 2 s of the definition in float64 differs from the derivative by
    s^2 / 6 of the third one, here below 1e-6; the gradient's own bars are its rounding, 2^-8 of each element."""
    x, w, target = make(80, 48, 200, torch.bfloat16, ignored=0.2)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    apexw_amd.linear_cross_entropy(*leaves, target).backward()
    f = lambda a, b: float(torch.nn.functional.cross_entropy(a @ b.t(), target))   # noqa: E731
    x64, w64, s = x.double(), w.double(), 1e-3
    for leaf, g in ((leaves[0], lambda v: (f(x64 + s * v, w64), f(x64 - s * v, w64))),
                    (leaves[1], lambda v: (f(x64, w64 + s * v), f(x64, w64 - s * v)))):
        v = torch.randn(leaf.shape, device="cuda", dtype=torch.float64)
        v /= v.norm()
        up, down = g(v)
        exact = Exact(x, w, target)
        # each element: rounding of G (2^-8 of |p - 1| + p <= 2 times the largest operand, over the mean) and its own
        bar = float((2.0 ** -8 * leaf.grad.double().abs() * v.abs()).sum()) + 1e-6
        bar += 2.0 ** -8 * 2 * float(w64.abs().max() if leaf is leaves[0] else x64.abs().max() / int(exact.kept.sum()) * 80)
        assert abs(float((leaf.grad.double() * v).sum()) - (up - down) / (2 * s)) <= bar


def test_offsets_beyond_32_bits():
    """Weights and their gradient that reach more than 2^32 bytes from their start."""
    vocab = 1100000
    w = torch.zeros(vocab, 2048, dtype=torch.bfloat16, device="cuda")          # 4.5 GB
    at = torch.tensor([0, 7, 1050000, vocab - 1], device="cuda")
    g = torch.Generator().manual_seed(1)
    some = (torch.randn(4, 2048, generator=g) / 45).bfloat16().cuda()
    w[at] = some
    x = torch.randn(4, 2048, generator=g).bfloat16().cuda()
    l = x.double() @ some.double().t()                                       # the others are 0
    lse = torch.log(torch.exp(l).sum(1) + (vocab - 4))
    loss, got = apexw_amd.linear_cross_entropy_forward(x, w, at)
    # b of above with the 8600 tiles' joins
    bar = 2048 * 2.0 ** -23 * float((x.double().abs() @ some.double().abs().t()).max()) + 3000 * 2.0 ** -24 + 2.0 ** -22 * 40
    assert float((got.double() - lse).abs().max()) <= bar and float((loss.double() - (lse - l.diag())).abs().max()) <= 2 * bar
    dx, dw = apexw_amd.linear_cross_entropy_backward(torch.ones(4, device="cuda"), x, w, at, lse.float())
    G = torch.exp(l - lse[:, None]) - torch.eye(4, device="cuda")
    want = G.t() @ x.double()
    assert float((dw[at].double() - want).abs().max()) <= 2.0 ** -6 * float(want.abs().max())
    other = torch.exp(-lse) @ x.double()
    dw[at] = other.bfloat16()
    assert float((dw.float() - other.float()).abs().max()) <= 2.0 ** -6 * float(other.abs().max())
    want = G @ some.double()
    assert float((dx.double() - want).abs().max()) <= 2.0 ** -6 * float(want.abs().max())


def test_equal_calls_give_equal_bits():
    x, w, target = make(1500, 256, 7000, torch.bfloat16, ignored=0.3)
    _, first = check(x, w, target)
    for _ in range(3):
        loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
        d = torch.full((1500,), 1.0 / int((target >= 0).sum()), device="cuda")
        assert torch.equal(loss, first[0]) and torch.equal(lse, first[1])
        dx, dw = apexw_amd.linear_cross_entropy_backward(d, x, w, target, Exact(x, w, target).lse.float())
        assert torch.equal(dx, first[2]) and torch.equal(dw, first[3])


def test_need():
    x, w, target = make(300, 64, 500, torch.bfloat16)
    lse, d = apexw_amd.linear_cross_entropy_forward(x, w, target)[1], torch.ones(300, device="cuda")
    dx, dw = apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse)
    one = apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse, need=(True, False))
    two = apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse, need=(False, True))
    assert torch.equal(one[0], dx) and one[1] is None and two[0] is None and torch.equal(two[1], dw)
    assert apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse, need=(False, False)) == (None, None)

"""Tokens by expert and back, and the embedding, against plain computations in float64.

Bars.  Rows that are only moved have to be equal.  A sum of n products in fp32 (a fused multiply-add each, half a unit
of 2^-23 of what it has added up) is off by at most n 2^-24 of the sum of the magnitudes; partial sums joined add no
more.  Scaling rounds once more (2^-24), and the result rounds to its type by half a step: 2^-24, 2^-8 or 2^-11 of
the value, 2^-25 below fp16's normal range."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(got, want, mag, n):
    assert got.shape == want.shape
    slack = (n + 2) * 2.0 ** -24 * mag + HALF[got.dtype] * want.abs() * (1 + 2.0 ** -8)
    slack = slack + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    over = (got.double() - want).abs() - slack
    assert got.numel() == 0 or float(over.max()) <= 0, f"over the bar by {float(over.max())}"


def plain_order(expert, experts):
    flat = expert.reshape(-1).cpu().tolist()
    rows = sorted((e, c) for c, e in enumerate(flat) if 0 <= e < experts)
    source, place, ends = [-1] * len(flat), [-1] * len(flat), [0] * experts
    for r, (e, c) in enumerate(rows):
        source[r], place[c] = c, r
        ends[e] = r + 1
    for e in range(1, experts):
        ends[e] = max(ends[e], ends[e - 1])
    return (torch.tensor(source, dtype=torch.int32), torch.tensor(place, dtype=torch.int32).view(expert.shape),
            torch.tensor(ends, dtype=torch.int32))


def check_order(expert, experts):
    order = apexw_amd.expert_order(expert, experts)
    for got, want in zip(order, plain_order(expert, experts)):
        assert got.dtype == torch.int32 and got.is_cuda and torch.equal(got.cpu(), want)
    return order


def choose(tokens, k, experts, seed=0, dropped=0.0, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed + 31 * tokens + experts)
    e = (torch.rand(tokens, k, generator=g) ** 2 * experts).to(dtype).clamp(max=experts - 1)
    if dropped:
        e[torch.rand(tokens, k, generator=g) < dropped] = -1
    return e.cuda()


# one workgroup up to 4096 choices, two launches behind; experts of one, two and three passes of the sort
@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (1, 8, 3), (7, 2, 64), (63, 3, 5), (64, 1, 511), (65, 1, 512), (512, 8, 8),
                                              (513, 8, 8), (4096, 1, 1), (4097, 1, 300), (3000, 6, 17), (20000, 2, 8),
                                              (9000, 4, 511), (9000, 4, 512), (9001, 3, 5000), (700, 2, 300000),
                                              (70000, 8, 256), (5000, 1, 2 ** 30)])
def test_order(tokens, k, experts):
    for dropped, dtype in ((0.0, torch.int64), (0.3, torch.int32)):
        if experts >= 2 ** 30:   # the ends alone are checked at the rows' ids
            expert = choose(tokens, k, experts, dropped=dropped, dtype=dtype)
            order = apexw_amd.expert_order(expert, 2 ** 20)
            expert = torch.where(expert < 2 ** 20, expert, -1)
            want = plain_order(expert, 2 ** 20)
            assert all(torch.equal(a.cpu(), b) for a, b in zip(order, want))
            continue
        check_order(choose(tokens, k, experts, dropped=dropped, dtype=dtype), experts)


@pytest.mark.parametrize("tokens", [5, 6000])
def test_order_of_strange_ids(tokens):
    """All one expert, none at all, ids far outside, one dimension, another stride."""
    check_order(torch.full((tokens, 2), 3, device="cuda"), 8)
    check_order(torch.full((tokens, 2), -1, device="cuda"), 8)
    check_order(torch.full((tokens,), 8, device="cuda"), 8)
    e = choose(tokens, 2, 8)
    e[::3, 0], e[1::3, 1], e[2::5, 0], e[3::5, 1] = 2 ** 40 + 1, -2 ** 62, 2 ** 32 + 2, 2 ** 31
    check_order(e, 8)
    check_order(e.int(), 8)
    check_order(choose(tokens, 4, 8)[:, 1], 8)
    check_order(choose(2, tokens, 8).t(), 8)


def test_no_tokens():
    for shape in ((0,), (0, 4)):
        order = apexw_amd.expert_order(torch.empty(shape, dtype=torch.int64, device="cuda"), 700)
        assert order.source.shape == (0,) and order.place.shape == shape and (order.ends == 0).all()
        x = torch.randn(0, 16, device="cuda")
        assert apexw_amd.expert_dispatch_forward(x, order).shape == (0, 16)
        assert apexw_amd.expert_combine_forward(x, order, torch.ones(shape, device="cuda")).shape == (0, 16)
        dy, dw = apexw_amd.expert_combine_backward(x, x, order, torch.ones(shape, device="cuda"))
        assert dy.shape == (0, 16) and dw.shape == shape
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    w = torch.randn(9, 24, device="cuda")
    assert apexw_amd.embedding_forward(ids, w).shape == (0, 24)
    assert (apexw_amd.embedding_weight_grad(w[:0], ids, 9) == 0).all()


def check_rows(expert, experts, width, dtype, w_dtype, x=None, y=None, dout=None, w=None):
    tokens, k = expert.shape
    g = torch.Generator().manual_seed(width + tokens)

    def normal(*shape):
        return torch.randn(shape, generator=g).to(dtype).cuda()

    order = apexw_amd.expert_order(expert, experts)
    source, place, ends = (t.cpu().long() for t in order)
    used = int(ends[-1])
    x = normal(tokens, width) if x is None else x
    y = normal(tokens * k, width) if y is None else y
    dout = normal(tokens, width) if dout is None else dout
    w = torch.rand(tokens, k, generator=g).to(w_dtype).cuda() if w is None else w
    of = (source[:used] // k).cuda()

    rows = apexw_amd.expert_dispatch_forward(x, order)
    assert rows.dtype == dtype and torch.equal(rows[:used], x[of]) and (rows[used:] == 0).all()

    drows = apexw_amd.expert_dispatch_backward(y, order)
    wf = w.reshape(-1).double()[source[:used].cuda()][:, None]
    zero = torch.zeros(tokens, width, dtype=torch.float64, device="cuda")
    y64 = y[:used].double()
    close(drows, zero.index_add(0, of, y64), zero.index_add(0, of, y64.abs()), k)
    out = apexw_amd.expert_combine_forward(y, order, w)
    close(out, zero.index_add(0, of, y64 * wf), zero.index_add(0, of, (y64 * wf).abs()), k)

    dy, dw = apexw_amd.expert_combine_backward(dout, y, order, w)
    want = dout[of].double() * wf
    close(dy[:used], want, 0 * want, 0)
    assert (dy[used:] == 0).all() and dw.dtype == w_dtype
    products = dout[of].double() * y64
    for got, f in ((dw, lambda t: t),):
        value, mag = torch.zeros(2, tokens * k, dtype=torch.float64, device="cuda")
        value[source[:used].cuda()], mag[source[:used].cuda()] = products.sum(1), products.abs().sum(1)
        close(got.reshape(-1), value, mag, width)
        assert (got.reshape(-1)[place.reshape(-1).cuda() < 0] == 0).all()
    only = apexw_amd.expert_combine_backward(dout, None, order, w, need=(True, False))
    assert torch.equal(only[0], dy) and only[1] is None
    only = apexw_amd.expert_combine_backward(dout, y, order, w, need=(False, True))
    assert only[0] is None and torch.equal(only[1], dw)
    alone, none = apexw_amd.expert_combine_backward(dout, y, order)
    assert none is None and torch.equal(alone[:used], dout[of]) and (alone[used:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 3, 7, 8, 9, 64, 127, 130, 255, 500, 512, 1021, 2048, 2056, 5003])
def test_widths(width, dtype):
    check_rows(choose(37, 3, 5, dropped=0.2), 5, width, dtype, dtype)
    check_rows(choose(11, 2, 5), 5, width, dtype, torch.float32)


@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (2, 9, 4), (300, 1, 7), (65, 17, 64), (1000, 8, 128), (2500, 6, 256)])
def test_choices(tokens, k, experts):
    for dtype in TYPES:
        check_rows(choose(tokens, k, experts, dropped=0.1), experts, 264, dtype, torch.float32)
    check_rows(torch.full((tokens, k), -1, device="cuda"), experts, 72, torch.bfloat16, torch.bfloat16)


def test_views():
    """Rows of a wider buffer, at odd addresses, a transposed one, one row for all; weights of another stride."""
    e = choose(50, 2, 6, dropped=0.1)
    big = torch.randn(100, 400, device="cuda").bfloat16()
    check_rows(e, 6, 96, torch.bfloat16, torch.float32, x=big[:50, 3:99], y=big[:, 5:101], dout=big[:50, 7:103])
    check_rows(e, 6, 96, torch.bfloat16, torch.bfloat16, x=big[:50, :96].t().contiguous().t(), y=big[:1, :96].expand(100, 96),
               dout=big[:, :96][::2])
    check_rows(e, 6, 96, torch.bfloat16, torch.float32, w=torch.rand(2, 50, device="cuda").t())


def test_what_no_expert_takes_reaches_nothing():
    """NaN and infinity in rows behind the last end, and in weights of choices without a row."""
    e = choose(200, 3, 5, dropped=0.3)
    order = apexw_amd.expert_order(e, 5)
    used, none = int(order.ends[-1]), order.place < 0
    y, w = torch.randn(600, 136, device="cuda"), torch.rand(200, 3, device="cuda")
    dout = torch.randn(200, 136, device="cuda")
    bad_y, bad_w = y.clone(), w.clone()
    bad_y[used:], bad_w[none] = float("nan"), float("inf")
    for a, b in zip((apexw_amd.expert_combine_forward(y, order, w), apexw_amd.expert_dispatch_backward(y, order),
                     *apexw_amd.expert_combine_backward(dout, y, order, w)),
                    (apexw_amd.expert_combine_forward(bad_y, order, bad_w), apexw_amd.expert_dispatch_backward(bad_y, order),
                     *apexw_amd.expert_combine_backward(dout, bad_y, order, bad_w))):
        assert torch.equal(a, b) and torch.isfinite(b).all()


def test_places_that_are_no_rows():
    """A place outside the rows counts as none: nothing outside the buffers is read or written."""
    order = apexw_amd.expert_order(choose(9, 2, 3), 3)
    place = order.place.clone()
    place[0, 0], place[3, 1], place[8, 0] = 18, 2 ** 31 - 1, -2 ** 31
    bad = apexw_amd.ExpertOrder(order.source, place, order.ends)
    y, w = torch.randn(18, 40, device="cuda"), torch.ones(9, 2, device="cuda")
    got = apexw_amd.expert_combine_forward(y, bad, w)
    keep = ((place >= 0) & (place < 18))[..., None]
    assert torch.equal(got, (y[place.clamp(0, 17).long()] * keep).sum(1))
    dy, dw = apexw_amd.expert_combine_backward(got, y, bad, w)
    assert (dw[place != order.place] == 0).all()


def test_gradients_through_autograd():
    """dispatch, an expert product and combine as a program runs them, against float64 autograd.  Two roundings to
    bf16 lie between input and output (2^-8 each, of rows and of products), so a few units of 2^-7 of the largest
    value bound every result; the operators' own bars are above."""
    tokens, k, experts, width = 120, 2, 4, 64
    e = choose(tokens, k, experts, dropped=0.1)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(tokens, width, generator=g).bfloat16().cuda()
    m = (torch.randn(experts, width, width, generator=g) / 8).bfloat16().cuda()
    w = torch.rand(tokens, k, generator=g).cuda()
    c = torch.randn(tokens, width, generator=g).bfloat16().cuda()
    leaves = [t.clone().requires_grad_() for t in (x, m, w)]
    order = apexw_amd.expert_order(e, experts)
    rows = apexw_amd.expert_dispatch(leaves[0], order)
    out = apexw_amd.expert_combine(apexw_amd.expert_matmul(rows, leaves[1], order.ends), order, leaves[2])
    out.backward(c)
    l64 = [t.double().requires_grad_() for t in (x, m, w)]
    mats = l64[1][e.clamp(min=0)]                                     # [tokens, k, width, width]
    y = (mats @ l64[0][:, None, :, None])[..., 0] * (e >= 0)[..., None] * l64[2][..., None]
    y.sum(1).backward(c.double())
    for got, want in zip((out, *(t.grad for t in leaves)), (y.sum(1), *(t.grad for t in l64))):
        assert float((got.double() - want).abs().max()) <= 2.0 ** -5 * float(want.abs().max())


def test_combine_against_differences():
    """Combine is linear in each argument: a difference over a step of one is exact up to its roundings, three a term
    and one of the step, and up to 33 in the gradients: 40 half units of each term's magnitude."""
    e = choose(30, 3, 4, dropped=0.1)
    order = apexw_amd.expert_order(e, 4)
    y, w = torch.randn(90, 33, device="cuda"), torch.rand(30, 3, device="cuda")
    c = torch.randn(30, 33, device="cuda")
    yl, wl = y.clone().requires_grad_(), w.clone().requires_grad_()
    apexw_amd.expert_combine(yl, order, wl).backward(c)
    f = lambda y, w: float((apexw_amd.expert_combine_forward(y, order, w).double() * c).sum())   # noqa: E731
    v, u = torch.randn_like(y), torch.randn_like(w)
    bar = 40 * 2.0 ** -24 * float((apexw_amd.expert_combine_forward(y.abs() + v.abs(), order, w + u.abs()) * c.abs()).sum())
    assert abs(float((yl.grad.double() * v).sum()) - (f(y + v, w) - f(y - v, w)) / 2) <= bar
    assert abs(float((wl.grad.double() * u).sum()) - (f(y, w + u) - f(y, w - u)) / 2) <= bar
    broad = y.clone().requires_grad_()
    apexw_amd.expert_combine(broad, order).sum().backward()           # a broadcast gradient, no weights
    assert torch.equal(broad.grad, apexw_amd.expert_dispatch_forward(torch.ones(30, 33, device="cuda"), order))


# ---------------------------------------------------------------------------- embedding
def words(shape, vocab, seed=0):
    g = torch.Generator().manual_seed(seed + vocab)
    return torch.exp(torch.rand(shape, generator=g).double() * torch.log(torch.tensor(vocab + 1.0).double())).long().sub(1).clamp(0, vocab - 1).cuda()


def check_embedding(ids, vocab, width, dtype, scale=1.0, grads=(None,), w=None, dy=None):
    g = torch.Generator().manual_seed(width)
    w = torch.randn(vocab, width, generator=g).to(dtype).cuda() if w is None else w
    dy = torch.randn(*ids.shape, width, generator=g).to(dtype).cuda() if dy is None else dy
    has = (ids >= 0) & (ids < vocab)
    y = apexw_amd.embedding_forward(ids, w, scale)
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    want = w[ids.long().clamp(0, vocab - 1)].double() * s32 * has[..., None]
    assert y.dtype == dtype
    close(y, want, 0 * want, 0)
    flat, rows = ids.reshape(-1).long()[has.reshape(-1)], dy.reshape(-1, width)[has.reshape(-1)].double() * s32
    zero = torch.zeros(vocab, width, dtype=torch.float64, device="cuda")
    most = int(torch.bincount(flat, minlength=1).max()) if len(flat) else 0
    value, mag = zero.index_add(0, flat, rows), zero.index_add(0, flat, rows.abs())
    for d in grads:
        got = apexw_amd.embedding_weight_grad(dy, ids, vocab, scale, d)
        assert got.dtype == (d or dtype)
        close(got, value, mag, most)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 5, 8, 63, 72, 500, 513, 768, 1021, 4104])
def test_embedding_widths(width, dtype):
    check_embedding(words((40,), 101), 101, width, dtype, 27.7, (None, torch.float32))
    check_embedding(words((4, 1300), 300), 300, width, dtype, 1.0, (None, torch.float32))


@pytest.mark.parametrize("tokens,vocab", [(1, 1), (1, 50257), (17, 3), (4096, 2000), (4097, 2000), (5000, 511), (5000, 512),
                                          (8192, 128256), (33000, 300000), (40000, 1), (40000, 70), (270000, 9)])
def test_embedding_tokens(tokens, vocab):
    for dtype in (torch.bfloat16, torch.float32):
        check_embedding(words((tokens,), vocab), vocab, 40, dtype, 0.5)


@pytest.mark.parametrize("tokens", [300, 10000])
def test_embedding_strange_ids(tokens):
    """Ids outside the table, one id for all, evenly spread ones, int32."""
    ids = words((tokens,), 500)
    ids[::7], ids[1::7], ids[2::7] = -1, 500, 2 ** 33
    check_embedding(ids, 500, 136, torch.bfloat16)
    check_embedding(ids.int(), 500, 136, torch.float32)
    check_embedding(torch.full((tokens,), 499, device="cuda"), 500, 136, torch.bfloat16, 2.0)
    check_embedding(torch.full((tokens,), -100, device="cuda"), 500, 136, torch.bfloat16)
    check_embedding(torch.arange(tokens, device="cuda") % 500, 500, 136, torch.float16)
    # NaN in the gradients of tokens outside the table reaches nothing
    dy = torch.randn(tokens, 24, device="cuda")
    dy[(ids < 0) | (ids >= 500)] = float("nan")
    assert torch.isfinite(apexw_amd.embedding_weight_grad(dy, ids, 500)).all()


def test_embedding_views():
    ids = words((6, 900), 700)[:, ::2]
    big = torch.randn(700, 200, device="cuda").half()
    check_embedding(ids, 700, 65, torch.float16, 3.0, w=big[:, 7:72], dy=torch.randn(6, 450, 90, device="cuda").half()[..., 3:68])
    check_embedding(ids, 700, 64, torch.float16, w=big.t()[:64].t(), dy=torch.randn(1, 1, 64, device="cuda").half().expand(6, 450, 64))


def test_embedding_autograd_and_differences():
    ids = words((3, 50), 20)
    w = torch.randn(20, 24, device="cuda")
    c = torch.randn(3, 50, 24, device="cuda")
    wl = w.clone().requires_grad_()
    apexw_amd.embedding(ids, wl, 4.0).backward(c)
    v = torch.randn_like(w)
    up, down = (float((apexw_amd.embedding_forward(ids, w + s * v, 4.0).double() * c).sum()) for s in (1, -1))
    # a gradient sums up to 150 products, each product and difference rounds three times more
    bar = 160 * 2.0 ** -24 * 4.0 * float(((w.abs() + v.abs())[ids] * c.abs()).sum())
    assert abs(float((wl.grad.double() * v).sum()) - (up - down) / 2) <= bar


def test_offsets_beyond_32_bits():
    """Tables, rows and results that reach more than 2^32 bytes from their start."""
    w = torch.zeros(1100000, 2048, dtype=torch.bfloat16, device="cuda")          # 4.5 GB
    ids = torch.tensor([0, 1099999, 5, 1050000], device="cuda")
    w[ids] = torch.randn(4, 2048, device="cuda").bfloat16()
    assert torch.equal(apexw_amd.embedding_forward(ids, w), w[ids])
    dy = torch.randn(4, 2048, device="cuda").bfloat16()
    dw = apexw_amd.embedding_weight_grad(dy, ids, 1100000)
    assert torch.equal(dw[ids], dy)
    dw[ids] = 0
    assert not dw.any()
    del dw
    expert = torch.arange(1100000, device="cuda") % 7
    order = apexw_amd.expert_order(expert, 7)
    rows = apexw_amd.expert_dispatch_forward(w, order)
    for t in ids.tolist():
        assert torch.equal(rows[order.place[t].long()], w[t])
    back = apexw_amd.expert_combine_forward(rows, order, torch.ones(1100000, device="cuda"))
    assert torch.equal(back, w)


def test_equal_calls_give_equal_bits():
    ids, dy = words((20000,), 3000), torch.randn(20000, 264, device="cuda").bfloat16()
    first = apexw_amd.embedding_weight_grad(dy, ids, 3000, dtype=torch.float32)
    e = choose(8000, 2, 16)
    order = apexw_amd.expert_order(e, 16)
    for _ in range(4):
        assert torch.equal(first, apexw_amd.embedding_weight_grad(dy, ids, 3000, dtype=torch.float32))
        assert all(torch.equal(a, b) for a, b in zip(order, apexw_amd.expert_order(e, 16)))


# up to 1024 tokens each id that occurs is summed by itself, beside a cleared gradient of any number of bytes
@pytest.mark.parametrize("dtype,grad", [(torch.bfloat16, None), (torch.float16, torch.float32), (torch.float32, None)])
@pytest.mark.parametrize("tokens", [1, 255, 257, 1024, 1025])
def test_embedding_gradient_of_few(tokens, dtype, grad):
    for vocab, width in ((1, 1), (3, 1), (7, 1), (2, 3), (5, 9), (1000, 8), (300, 513), (50257, 24)):
        ids = words((tokens,), vocab) - int(tokens % 2)
        check_embedding(ids, vocab, width, dtype, 1.5, (grad,))
        check_embedding(torch.full((tokens,), vocab - 1, device="cuda"), vocab, width, dtype, 1.0, (grad,))
    dy = torch.full((tokens, 8), float("nan"), device="cuda", dtype=dtype)
    assert (apexw_amd.embedding_weight_grad(dy, torch.full((tokens,), -1, device="cuda"), 9, dtype=grad) == 0).all()

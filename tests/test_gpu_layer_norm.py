"""Layer norm, forward and backward, against float64.

Bars, with u = 2^-24.  A row's sums are taken by each thread over at most 64 of its elements and then by
halves, so a sum of n terms is off by at most 2^-17 of the sum of their magnitudes; the mean is then off by
2^-17 (|mean| + 1/rstd), xh by 2^-17 (|xh| + |mean| rstd + 1), and what is formed from them by the same
share of the magnitudes that it adds.  A column's sums join at most 2^6 terms in a row, and as many partial
sums.  A 16-bit result adds half a unit of its last place: 2^-8 (bf16), 2^-11 (fp16) of itself."""

import itertools

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E = 2.0 ** -17
WIDTHS = [1, 2, 7, 8, 64, 65, 500, 511, 768, 1021, 1024, 1999, 2048, 4096, 4097, 8192, 8200, 12345, 16384, 16385,
          32768, 40001]
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
         (torch.float16, torch.float16), (torch.float16, torch.float32)]


def inputs(rows, width, dtype, w_dtype, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed + 31 * rows + width)
    x = torch.randn(rows, width, generator=g) * torch.exp(torch.randn(rows, 1, generator=g)) + shift
    return (x.to(dtype).cuda(), (1 + 0.2 * torch.randn(width, generator=g)).to(w_dtype).cuda(),
            (0.3 * torch.randn(width, generator=g)).to(w_dtype).cuda(),
            torch.randn(rows, width, generator=g).to(dtype).cuda())


def exact(x, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    return mean, rstd, (x - mean) * rstd


def close(got, want, slack):
    assert got.shape == want.shape
    over = (got.double() - want).abs() - (HALF[got.dtype] * want.abs() + slack + (2.0 ** -25 if got.dtype == torch.float16 else 0))
    assert float(over.max()) <= 0, f"over the bar by {float(over.max())}"


def check_forward(x, w, b, eps=1e-5):
    y, mean, rstd = apexw_amd.layer_norm_forward(x, w, b, eps)
    m, r, xh = exact(x, eps)
    mag = xh.abs() + m.abs() * r + 1
    w64 = torch.ones(x.shape[-1], device=x.device).double() if w is None else w.double()
    b64 = torch.zeros_like(w64) if b is None else b.double()
    close(y, xh * w64 + b64, E * (mag * w64.abs() + b64.abs()))
    close(mean, m[..., 0], E * (m.abs() + 1 / r)[..., 0])
    close(rstd, r[..., 0], (E * r * (1 + m.abs() * r))[..., 0])


def check_backward(dy, x, w, b, eps=1e-5):
    _, mean, rstd = apexw_amd.layer_norm_forward(x, w, b, eps)
    dx, dw, db = apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b)
    # from the statistics that the forward pass gave: their own error is the forward's
    m, r, d = mean.double()[..., None], rstd.double()[..., None], dy.double()
    xh = (x.double() - m) * r
    g = d if w is None else d * w.double()
    close(dx, r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)),
          E * r * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)))
    d, xh = d.reshape(-1, x.shape[-1]), xh.reshape(-1, x.shape[-1])
    if w is not None:
        close(dw, (d * xh).sum(0), E * (d * xh).abs().sum(0))
    if b is not None:
        close(db, d.sum(0), E * d.abs().sum(0))
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    return dx, dw, db


@pytest.mark.parametrize("dtype,w_dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(width, dtype, w_dtype):
    for rows in (1, 5, 67):
        x, w, b, dy = inputs(rows, width, dtype, w_dtype)
        check_forward(x, w, b)
        check_backward(dy, x, w, b)


@pytest.mark.parametrize("rows", [2, 255, 4099, 20000])
def test_many_rows(rows):
    for width, (dtype, w_dtype) in itertools.product((24, 200), TYPES[:3]):
        x, w, b, dy = inputs(rows, width, dtype, w_dtype)
        check_forward(x, w, b)
        check_backward(dy, x, w, b)


@pytest.mark.parametrize("width", [96, 1021, 4096, 40001])
def test_without_weight_or_bias(width):
    x, w, b, dy = inputs(33, width, torch.bfloat16, torch.bfloat16)
    for ww, bb in ((None, None), (w, None), (None, b)):
        check_forward(x, ww, bb)
        check_backward(dy, x, ww, bb)


@pytest.mark.parametrize("need", list(itertools.product((True, False), repeat=3)))
def test_gradients_left_out(need):
    for width in (100, 2049, 40001):
        x, w, b, dy = inputs(40, width, torch.float32, torch.float32)
        _, mean, rstd = apexw_amd.layer_norm_forward(x, w, b)
        whole = apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b)
        some = apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b, need)
        for a, s, n in zip(whole, some, need):
            assert (s is not None) == n
            assert not n or torch.equal(a, s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_far_from_zero(dtype):
    """A mean of 1000 deviations: the deviations are taken from the mean before they are squared."""
    x, w, b, _ = inputs(50, 777, torch.float32, torch.float32)
    x = (x / x.std(1, keepdim=True) + 1000.0).to(dtype)
    if dtype == torch.bfloat16:
        w, b = w.to(dtype), b.to(dtype)
    check_forward(x, w, b)


def test_views_and_orders():
    """Rows of a wider buffer, rows at odd addresses, a transposed tensor, a broadcast gradient, more dimensions."""
    x, w, b, dy = inputs(64, 600, torch.bfloat16, torch.bfloat16)
    for v, ww, bb in ((x[:, 100:356], w[100:356], b[100:356]), (x[::3, 1:78], w[1:78], b[1:78]),
                      (x[:, 3:4], w[3:4], b[3:4]), (x.t(), w[:64], b[:64]), (x.view(4, 16, 600)[:, 5], w, b),
                      (x.view(4, 16, 600).transpose(0, 1), w, b), (x.view(2, 2, 16, 600)[:, 1], w, b),
                      (x[7], w, b), (x.view(4, 16, 600)[:, :, 10:40], w[:30], b[:30])):
        check_forward(v, ww, bb)
        check_backward(torch.randn(v.shape, device="cuda").to(v.dtype), v, ww, bb)
    one = torch.ones((), device="cuda", dtype=torch.bfloat16)
    check_backward(one.expand(64, 600), x, w, b)
    check_backward(dy[:1].expand(64, 600), x, w, b)
    check_backward(dy[:, :1].expand(64, 600), x, w, b)
    check_forward(x, w[::1].flip(0), torch.stack([b, b], 1)[:, 0])


def test_rows_keep_to_themselves():
    """NaN and infinity make their own row NaN, and the columns' sums, and nothing else."""
    x, w, b, dy = inputs(70, 300, torch.float32, torch.float32)
    want = apexw_amd.layer_norm_forward(x, w, b)[0]
    x[3, 5], x[10, 0], x[69, 299] = float("nan"), float("inf"), -float("inf")
    y, mean, rstd = apexw_amd.layer_norm_forward(x, w, b)
    bad = torch.zeros(70, dtype=torch.bool, device="cuda")
    bad[[3, 10, 69]] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], want[~bad])
    dx, dw, db = apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b)
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    assert torch.isnan(dw).all() and torch.isfinite(db).all()


def test_constant_rows_and_eps():
    x = torch.full((6, 130), 3.0, device="cuda")
    w, b = torch.rand(130, device="cuda"), torch.rand(130, device="cuda")
    y, mean, rstd = apexw_amd.layer_norm_forward(x, w, b, 1e-5)
    assert torch.equal(y, b.expand(6, 130)) and (mean == 3).all()
    close(rstd, torch.full_like(rstd, 1e-5).double() ** -0.5, E * 400)
    y, _, rstd = apexw_amd.layer_norm_forward(x, w, b, 0.0)
    assert torch.isinf(rstd).all() and torch.isnan(y).all()       # 0 * inf, as the formula has it
    check_forward(x * torch.rand(6, 130, device="cuda"), w, b, 0.5)


def test_empty():
    w = torch.ones(9, device="cuda")
    y, mean, rstd = apexw_amd.layer_norm_forward(torch.empty(0, 9, device="cuda"), w, w)
    assert y.shape == (0, 9) and mean.shape == rstd.shape == (0,)
    dx, dw, db = apexw_amd.layer_norm_backward(y, y, mean, rstd, w, w)
    assert dx.shape == (0, 9) and (dw == 0).all() and (db == 0).all()


def test_equal_calls_give_equal_bits():
    x, w, b, dy = inputs(5000, 321, torch.bfloat16, torch.float32)
    _, mean, rstd = apexw_amd.layer_norm_forward(x, w, b)
    first = apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b)
    for _ in range(5):
        for a, c in zip(first, apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b)):
            assert torch.equal(a, c)


def test_gradient_against_differences():
    """dx, dw and db along random directions against central differences of the float64 definition."""
    x, w, b, c = inputs(7, 45, torch.float32, torch.float32)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad((apexw_amd.layer_norm(*leaves) * c).sum(), leaves)

    def f(x, w, b):
        _, _, xh = exact(x, 1e-5)
        return float(((xh * w + b) * c.double()).sum())

    point = [t.double() for t in (x, w, b)]
    for i in range(3):
        v = torch.randn_like(point[i])
        h = 1e-5
        ends = [[p + s * h * v if j == i else p for j, p in enumerate(point)] for s in (1, -1)]
        want = (f(*ends[0]) - f(*ends[1])) / (2 * h)
        got = float((grads[i].double() * v).sum())
        # an element's gradient is off by at most 2^-15 of the row's largest, the difference by 1e-8
        assert abs(got - want) <= 2.0 ** -15 * float(grads[i].abs().max()) * float(v.abs().sum()) + 1e-6


def test_autograd_takes_what_is_asked():
    x, w, b, _ = inputs(9, 33, torch.float32, torch.float32)
    w.requires_grad_()
    apexw_amd.layer_norm(x, w, b).sum().backward()
    assert w.grad is not None
    x.requires_grad_()
    y = apexw_amd.layer_norm(x)
    y.square().sum().backward()
    assert x.grad is not None


def test_another_stream():
    x, w, b, _ = inputs(3000, 512, torch.float32, torch.float32)
    want = apexw_amd.layer_norm_forward(x, w, b)[0]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        z = x * 1.0
        y = apexw_amd.layer_norm_forward(z, w, b)[0]
    s.synchronize()
    assert torch.equal(y, want)

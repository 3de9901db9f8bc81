"""The products of a mixture of experts against float64.

Bar: a product of two 16-bit numbers is exact in fp32, and each of the k additions of a sum loses at most
2^-23 of what it has added up (the matrix cores may truncate), so a sum is off by at most k 2^-23 of the sum
of its magnitudes; rounding the result adds half a unit of its last place."""

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def close(got, want, mag, k):
    assert got.shape == want.shape
    slack = k * 2.0 ** -23 * mag + HALF[got.dtype] * want.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    over = (got.double() - want).abs() - slack
    assert got.numel() == 0 or float(over.max()) <= 0, f"over the bar by {float(over.max())}"


def make(sizes, inner, outer, dtype, spare=0, seed=0):
    g = torch.Generator().manual_seed(seed + inner * 7 + outer)
    rows = sum(sizes) + spare
    x = torch.randn(rows, inner, generator=g).to(dtype).cuda()
    dy = torch.randn(rows, outer, generator=g).to(dtype).cuda()
    w = (torch.randn(len(sizes), outer, inner, generator=g) * inner ** -0.5).to(dtype).cuda()
    ends = torch.tensor(sizes).cumsum(0).to(torch.int32).cuda()
    return x, dy, w, ends


def exact(sizes, x, dy, w):
    """(y, dx, dW) and the sums of the magnitudes that each adds."""
    x, dy, w = x.double(), dy.double(), w.double()
    out = []
    for f in (lambda t: t, torch.abs):
        xs, ds, ws = f(x), f(dy), f(w)
        y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        a = 0
        for e, n in enumerate(sizes):
            b = a + n
            y[a:b] = xs[a:b] @ ws[e].t()
            dx[a:b] = ds[a:b] @ ws[e]
            dw[e] = ds[a:b].t() @ xs[a:b]
            a = b
        out.append((y, dx, dw))
    return out


def check(sizes, x, dy, w, ends, dw_dtypes=(None, torch.float32)):
    (y, dx, dw), (ym, dxm, dwm) = exact(sizes, x, dy, w)
    inner, outer, most = w.shape[2], w.shape[1], max(max(sizes), 1)
    close(apexw_amd.expert_matmul_forward(x, w, ends), y, ym, inner)
    close(apexw_amd.expert_matmul_rows_grad(dy, w, ends), dx, dxm, outer)
    for d in dw_dtypes:
        got = apexw_amd.expert_matmul_weight_grad(dy, x, ends, d)
        assert got.dtype == (d or dy.dtype)
        close(got, dw, dwm, most)


SIZES = {"one row": [1], "one expert": [300], "empty ones": [0, 5, 0, 0, 130, 0], "all empty": [0, 0, 0],
         "ragged": [1, 127, 128, 129, 0, 255, 257, 31], "many": [(7 * i) % 11 for i in range(150)],
         "last only": [0, 0, 0, 64], "first only": [200, 0]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", list(SIZES))
def test_sizes(name, dtype):
    sizes = SIZES[name]
    for inner, outer in ((64, 96), (40, 264)):
        check(sizes, *make(sizes, inner, outer, dtype))


WIDTHS = [(1, 1), (1, 70), (70, 1), (7, 9), (8, 8), (31, 33), (129, 127), (500, 386), (513, 200), (256, 1024),
          (1000, 264), (768, 512), (2048, 520)]


@pytest.mark.parametrize("inner,outer", WIDTHS)
def test_widths(inner, outer):
    sizes = [3, 0, 140, 61, 16, 1]
    for dtype in (torch.bfloat16, torch.float16):
        check(sizes, *make(sizes, inner, outer, dtype, spare=5))


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 65, 600, 5000])
def test_rows_per_expert(rows):
    """From a decode step to a training batch, spread over the experts by chance."""
    g = torch.Generator().manual_seed(rows)
    for experts in (1, 8, 40):
        sizes = torch.bincount(torch.randint(0, experts, (rows,), generator=g), minlength=experts).tolist()
        check(sizes, *make(sizes, 328, 256, torch.bfloat16, spare=rows % 3))


@pytest.mark.parametrize("inner,outer", [(2311, 387), (387, 2311), (4097, 131), (5, 1030), (1531, 134), (135, 777)])
def test_few_rows_of_odd_widths(inner, outer):
    """Decode steps that no whole chunks serve: long sums in parts, and columns that end inside a chunk."""
    for sizes, spare in (([1], 0), ([0, 0, 2, 0, 1, 0], 2), ([3] * 9, 1), ([40], 3)):
        for dtype in (torch.bfloat16, torch.float16):
            check(sizes, *make(sizes, inner, outer, dtype, spare=spare))


def test_large():
    sizes = [900, 0, 1500, 33, 2048, 600]
    check(sizes, *make(sizes, 1536, 2048, torch.bfloat16, spare=70))


def test_rows_of_no_expert_are_zero():
    sizes = [3, 4]
    x, dy, w, ends = make(sizes, 64, 80, torch.bfloat16, spare=300)
    x[7:], dy[7:] = float("nan"), float("inf")
    y, dx = apexw_amd.expert_matmul_forward(x, w, ends), apexw_amd.expert_matmul_rows_grad(dy, w, ends)
    assert (y[7:] == 0).all() and (dx[7:] == 0).all()
    assert torch.isfinite(y).all() and torch.isfinite(dx).all()
    dw = apexw_amd.expert_matmul_weight_grad(dy, x, ends)
    assert torch.isfinite(dw).all()


@pytest.mark.parametrize("inner,outer", [(64, 80), (50, 70), (520, 264)])
def test_rows_and_experts_keep_to_themselves(inner, outer):
    """NaN in one expert's rows or weights stays with that expert, also next to ragged ends and odd widths."""
    sizes = [37, 130, 1, 64]
    x, dy, w, ends = make(sizes, inner, outer, torch.float16)
    y, dx = apexw_amd.expert_matmul_forward(x, w, ends), apexw_amd.expert_matmul_rows_grad(dy, w, ends)
    dw = apexw_amd.expert_matmul_weight_grad(dy, x, ends)
    xb, db, wb = x.clone(), dy.clone(), w.clone()
    xb[37:167], db[37:167], wb[2] = float("nan"), float("inf"), float("nan")
    yb, dxb = apexw_amd.expert_matmul_forward(xb, wb, ends), apexw_amd.expert_matmul_rows_grad(db, wb, ends)
    dwb = apexw_amd.expert_matmul_weight_grad(db, xb, ends)
    for a, b in ((y, yb), (dx, dxb)):
        assert torch.equal(a[:37], b[:37]) and torch.equal(a[168:], b[168:]) and not torch.isfinite(b[37:168]).any()
    assert torch.equal(dw[0], dwb[0]) and torch.equal(dw[2:], dwb[2:]) and torch.isnan(dwb[1]).all()


def test_views_and_orders():
    """Rows of a wider buffer, at odd addresses, transposed rows; weights stored (experts, inner, outer), a
    slice of wider ones, in neither order; shared weights."""
    sizes = [20, 0, 77, 5]
    x, dy, w, ends = make(sizes, 128, 192, torch.bfloat16)
    check(sizes, x[:, 8:72], dy[:, 16:112], w[:, 16:112, 8:72], ends)
    check(sizes, x[:, 1:64], dy[:, 3:40], w[:, 3:40, 1:64], ends)
    check(sizes, x[:, 1:2], dy[:, 3:4], w[:, 3:4, 1:2], ends)
    check(sizes, x, dy, w.transpose(1, 2).contiguous().transpose(1, 2), ends)
    check(sizes, x, dy, w.permute(1, 2, 0).contiguous().permute(2, 0, 1), ends)
    check(sizes, x, dy, w[:1].expand(4, 192, 128), ends)
    check(sizes, x.t().contiguous().t(), dy.t().contiguous().t(), w, ends)
    check(sizes, x[:1].expand(102, 128), dy[:, :1].expand(102, 192), w, ends.long())


def test_ends_out_of_range():
    """Ends that decrease, are negative or pass the buffer count as clamped."""
    x, dy, w, _ = make([10, 20, 5, 15], 64, 72, torch.bfloat16)
    ends = torch.tensor([-3, 30, 12, 1000], dtype=torch.int32, device="cuda")
    check([0, 30, 0, 20], x, dy, w, ends)
    check([50, 0, 0, 0], x, dy, w, torch.tensor([2 ** 31 - 1, -2 ** 31, 7, 50], dtype=torch.int32, device="cuda"))


def test_no_rows():
    w = torch.randn(3, 16, 24, device="cuda").bfloat16()
    ends = torch.zeros(3, dtype=torch.int32, device="cuda")
    x, dy = w.new_empty(0, 24), w.new_empty(0, 16)
    assert apexw_amd.expert_matmul_forward(x, w, ends).shape == (0, 16)
    assert apexw_amd.expert_matmul_rows_grad(dy, w, ends).shape == (0, 24)
    assert (apexw_amd.expert_matmul_weight_grad(dy, x, ends) == 0).all()


def test_offsets_beyond_32_bits():
    """Rows and weights that lie more than 2^32 bytes from their buffer's start."""
    x = torch.zeros(300, 2 ** 23, dtype=torch.bfloat16, device="cuda")[:, :64]      # rows 16 MiB apart
    big = torch.zeros(3, 2 ** 30, dtype=torch.bfloat16, device="cuda")               # experts 2 GiB apart
    w = big[:, : 96 * 64].view(3, 96, 64)
    x.copy_(torch.randn(300, 64))
    w.copy_(torch.randn(3, 96, 64) / 8)
    dy = torch.randn(300, 96, device="cuda").bfloat16()
    sizes = [100, 60, 140]
    check(sizes, x, dy, w, torch.tensor(sizes).cumsum(0).to(torch.int32).cuda())


def test_equal_calls_give_equal_bits():
    sizes = [700, 3, 0, 450]
    x, dy, w, ends = make(sizes, 512, 384, torch.bfloat16)
    calls = (lambda: apexw_amd.expert_matmul_forward(x, w, ends), lambda: apexw_amd.expert_matmul_rows_grad(dy, w, ends),
             lambda: apexw_amd.expert_matmul_weight_grad(dy, x, ends, torch.float32))
    first = [c() for c in calls]
    for _ in range(4):
        assert all(torch.equal(a, c()) for a, c in zip(first, calls))


def test_gradient_through_autograd_and_differences():
    """Against differences of the definition along random directions: the products are bilinear, so a
    difference over a step of one is exact; the bars are the products' own."""
    sizes = [9, 0, 40, 3]
    x, c, w, ends = make(sizes, 48, 56, torch.bfloat16, spare=2)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    apexw_amd.expert_matmul(xl, wl, ends).backward(c)

    def f(x, w):
        a, s = 0, 0.0
        for e, n in enumerate(sizes):
            s += float(((x[a:a + n] @ w[e].t()) * c[a:a + n].double()).sum())
            a += n
        return s

    x64, w64 = x.double(), w.double()
    for leaf, ends_ in ((xl, lambda v: (f(x64 + v, w64), f(x64 - v, w64))), (wl, lambda v: (f(x64, w64 + v), f(x64, w64 - v)))):
        v = torch.randn(leaf.shape, device="cuda", dtype=torch.float64)
        up, down = ends_(v)
        g = leaf.grad.double()
        bar = float(((2.0 ** -8 * g.abs() + 2.0 ** -12) * v.abs()).sum())
        assert abs(float((g * v).sum()) - (up - down) / 2) <= bar
    only = w.clone().requires_grad_()
    apexw_amd.expert_matmul(x, only, ends).sum().backward()      # a broadcast gradient, rows without one
    assert only.grad is not None


def test_another_stream():
    sizes = [500, 200, 300]
    x, dy, w, ends = make(sizes, 512, 512, torch.bfloat16)
    want = apexw_amd.expert_matmul_forward(x, w, ends)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = apexw_amd.expert_matmul_forward(x * 1, w, ends * 1)
    s.synchronize()
    assert torch.equal(y, want)

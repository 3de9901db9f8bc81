"""The clip of a list of gradients by their global norm against float64.

Bars: a thread adds at most 64 squares in fp32 before they join in float64, so the norm is off by less than
2^-18 of itself and so is the coefficient; a clipped element adds half a unit of its last place."""

import math

import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E = 2.0 ** -18


def make(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * (1 + i % 5)).to(dtypes[i % len(dtypes)]).cuda()
            for i, n in enumerate(sizes)]


def exact_norm(grads, p):
    if not grads or not sum(g.numel() for g in grads):
        return 0.0
    return float(torch.linalg.vector_norm(torch.cat([g.double().reshape(-1) for g in grads]), p))


def check(grads, max_norm, p=2.0, out=None):
    before = [g.double().clone() for g in grads]
    want = exact_norm(grads, p)
    norm = apexw_amd.clip_grads(grads, max_norm, p, out)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= E * want
    c = min(max_norm / (want + 1e-6), 1.0)
    for b, g, o in zip(before, grads, grads if out is None else out):
        if out is not None:
            assert torch.equal(g.double(), b)
        r = b * c
        slack = (HALF[o.dtype] + E) * r.abs() + (2.0 ** -25 if o.dtype == torch.float16 else 0)
        assert o.numel() == 0 or float(((o.double() - r).abs() - slack).max()) <= 0
    return norm


LISTS = {"one element": [1], "one": [5000], "unit edges": [8191, 8192, 8193, 16384, 1], "empty ones": [0, 3, 0, 0, 9000, 0],
         "only empty": [0, 0], "small": [3, 1, 2, 7, 100, 8, 9] * 10, "ragged": [17, 300000, 1, 70001, 8192, 5, 123456],
         "many": [(37 * i) % 2000 for i in range(3000)]}


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("name", list(LISTS))
def test_lists(name, p):
    for dtypes in ([torch.float32], [torch.bfloat16], [torch.float16, torch.float32, torch.bfloat16]):
        want = exact_norm(make(LISTS[name], dtypes), p)
        check(make(LISTS[name], dtypes), 0.25 * want, p)
        check(make(LISTS[name], dtypes), 2.0 * want + 1.0, p)


@pytest.mark.parametrize("to", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_copies(dtype, to):
    for f in (0.3, 3.0):       # clipped, and a plain copy
        grads = make([1, 8195, 33, 100000, 0, 4096], [dtype])
        out = [torch.full_like(g, float("nan"), dtype=to) for g in grads]
        check(grads, f * exact_norm(grads, 2), 2.0, out)


def test_under_the_bound_in_place_is_untouched():
    grads = make([100, 9000], [torch.bfloat16, torch.float32])
    before = [g.clone() for g in grads]
    apexw_amd.clip_grads(grads, 1e9)
    assert all(torch.equal(a, b) for a, b in zip(before, grads))


def test_layouts_and_addresses():
    """Transposed and channels-last gradients, slices that start at odd addresses."""
    base = torch.randn(70000, device="cuda")
    half = torch.randn(70000, device="cuda").bfloat16()
    grads = [base[1:8200], base[8201:8208], half[1:20002], half[20003:20004], base[30000:30000 + 600].view(20, 30).t(),
             torch.randn(4, 6, 5, 7, device="cuda").to(memory_format=torch.channels_last),
             torch.randn((), device="cuda")]
    out = [torch.empty_like(g, dtype=torch.bfloat16) for g in grads]
    assert out[4].stride() == grads[4].stride()
    check(grads, 3.0, 2.0, out)
    check(grads, 3.0)


def test_against_torch():
    params = [torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in ((300, 40), (7,), (64, 3, 3, 3), (5,))]
    g = [torch.randn_like(p) for p in params[:3]]
    for p in (1.0, 2.0, math.inf):
        for q, x in zip(params, g):
            q.grad = x.clone()
        want = torch.nn.utils.clip_grad_norm_(params, 0.7, p)
        theirs = [q.grad for q in params[:3]]
        for q, x in zip(params, g):
            q.grad = x.clone()
        got = apexw_amd.clip_grad_norm_(params, 0.7, p)
        torch.testing.assert_close(got, want, rtol=2.0 ** -17, atol=0)
        for a, q in zip(theirs, params):
            torch.testing.assert_close(q.grad, a, rtol=2.0 ** -17, atol=1e-12)
    assert params[3].grad is None


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_not_finite(p, value):
    """torch's arithmetic: a NaN everywhere, or coefficient 0 (NaN where 0 meets infinity)."""
    grads = make([10, 9000, 4], [torch.float32])
    grads[1][8500] = value
    norm = apexw_amd.clip_grads(grads, 1.0, p)
    if math.isnan(value):
        assert torch.isnan(norm) and all(torch.isnan(g).all() for g in grads)
    else:
        assert float(norm) == math.inf
        assert torch.isnan(grads[1][8500]) and (grads[0] == 0).all() and (grads[2] == 0).all()
    params = [torch.nn.Parameter(torch.zeros(3, device="cuda"))]
    params[0].grad = torch.tensor([1.0, value, 2.0], device="cuda")
    with pytest.raises(RuntimeError, match="non-finite"):
        apexw_amd.clip_grad_norm_(params, 1.0, p, error_if_nonfinite=True)
    assert float(params[0].grad[2]) == 2.0
    params[0].grad = torch.tensor([3.0, 0.0, 4.0], device="cuda")
    assert float(apexw_amd.clip_grad_norm_(params, 1.0, 2.0, error_if_nonfinite=True)) == 5.0
    assert float(params[0].grad[0]) < 0.6001


def test_large_and_small_magnitudes():
    """Squares beyond the fp32 range do not make the norm infinite."""
    grads = [torch.full((100,), 1e25, device="cuda"), torch.full((20000,), -3e25, device="cuda")]
    check(grads, 1e24)
    check([torch.full((5000,), 1e-15, device="cuda")], 1e-14)
    check([torch.zeros(10, device="cuda"), torch.zeros(9000, device="cuda")], 1.0)


def test_bounds():
    grads = make([5000], [torch.float32])
    check(grads, 0.0)
    assert (grads[0] == 0).all()
    grads = make([5000], [torch.float32])
    check(grads, math.inf)


def test_parts():
    """The norm over two lists put together, then each list scaled with it, as over two processes."""
    a, b = make([8193, 5], [torch.float32]), make([100, 70000], [torch.bfloat16], seed=1)
    want = exact_norm(a + b, 2)
    total = (apexw_amd.grad_norm(a).square() + apexw_amd.grad_norm(b).square()).sqrt()
    assert abs(float(total) - want) <= 2 * E * want
    whole = [g.clone() for g in a + b]
    apexw_amd.clip_grads(whole, 0.5)
    apexw_amd.scale_grads(a, 0.5, total)
    apexw_amd.scale_grads(b, 0.5, total)
    for x, y in zip(whole, a + b):
        assert float((x.double() - y.double()).abs().max()) <= 2 * (HALF[x.dtype] + E) * float(x.double().abs().max())


def test_equal_calls_give_equal_bits():
    grads = make([123457, 9, 400000, 77], [torch.bfloat16, torch.float32])
    norms = [apexw_amd.grad_norm(grads) for _ in range(5)]
    assert all(torch.equal(n, norms[0]) for n in norms)


def test_no_gradients():
    assert float(apexw_amd.clip_grads([], 1.0)) == 0.0
    assert float(apexw_amd.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3, device="cuda"))], 1.0)) == 0.0


def test_another_stream():
    grads = make([200000, 30], [torch.float32])
    want = exact_norm(grads, 2)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        mine = [g * 1 for g in grads]
        norm = apexw_amd.clip_grads(mine, 0.5 * want)
    s.synchronize()
    assert abs(float(norm) - want) <= E * want
    assert abs(exact_norm(mine, 2) - 0.5 * want) <= 1e-5 * want

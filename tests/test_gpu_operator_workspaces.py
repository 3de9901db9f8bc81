"""Workspaces of exactly the bytes that the _workspace calls answer, full of NaN, and outputs of exactly their size at any
element's address, with patterns around all of them: the C entries write nothing beside them, and give the bits that the
calls of the package give."""

import pytest
import torch

import apexw_amd
from apexw_amd import _lib
from test_gpu_linear_cross_entropy import make

pytestmark = pytest.mark.gpu
CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
EDGE = 512          # bytes of pattern on either side


class Place:
    """`size` bytes full of 0xFF (NaN in every type) at `shift` bytes past a multiple of 256, patterns around them."""
    every = []

    def __init__(self, size, shift=0):
        self.size, self.begin = size, EDGE + shift
        self.all = torch.full((size + 2 * EDGE + 256,), 0x5A, dtype=torch.uint8, device="cuda")
        assert self.all.data_ptr() % 256 == 0
        self.all[self.begin:self.begin + size] = 0xFF
        self.ptr = self.all.data_ptr() + self.begin if size else None
        Place.every.append(self)

    def tensor(self, dtype, shape):
        return self.all[self.begin:self.begin + self.size].clone().view(dtype).view(shape)   # (a clone is aligned)

    @classmethod
    def check(cls):
        for p in cls.every:
            around = torch.cat([p.all[:p.begin], p.all[p.begin + p.size:]])
            assert (around == 0x5A).all(), f"written beside {p.size} bytes"
        cls.every.clear()


def out_like(t):
    """Room for t's elements, at an address that is no multiple of more than an element's size."""
    return Place(t.numel() * t.element_size(), t.element_size())


def same(place, t):
    got = place.tensor(t.dtype, t.shape)
    assert torch.equal(got, t) and not (got.is_floating_point() and got.isnan().any())


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.fixture(autouse=True)
def nothing_beside():
    Place.every.clear()
    yield
    Place.check()


# ---------------------------------------------------------------------------- cross entropy of a linear head
FORWARD = [(1, 64, 129), (20, 768, 5003), (32, 1024, 300), (31, 765, 5003), (33, 100, 257), (640, 1021, 1500), (1500, 101, 2003),
           (582, 701, 7374), (641, 264, 9003), (2049, 520, 16500), (2176, 264, 20011)]


@pytest.mark.parametrize("reduction", [0, 2])
@pytest.mark.parametrize("rows,width,vocab", FORWARD)
def test_head_forward(rows, width, vocab, reduction):
    lib = _lib.load()
    for dtype, ignored in ((torch.bfloat16, 0.0), (torch.float16, 0.7)):
        x, w, target = make(rows, width, vocab, dtype, ignored)
        loss, lse = apexw_amd.linear_cross_entropy_forward(x, w, target)
        space = Place(lib.apexw_linear_cross_entropy_workspace(w.data_ptr(), width, rows, width, vocab, 0))
        to, to_lse, total = out_like(loss), out_like(lse), Place(4, 4)
        _lib.check(lib.apexw_linear_cross_entropy_forward(
            x.data_ptr(), width, rows, width, w.data_ptr(), width, vocab, CODE[dtype], target.data_ptr(), 8, -100, to.ptr,
            to_lse.ptr, reduction, total.ptr if reduction else None, space.ptr, stream()), "forward")
        same(to, loss), same(to_lse, lse)
        if reduction and (target >= 0).any():
            same(total, apexw_amd.linear_cross_entropy(x, w, target))
        Place.check()


# (every shape of the three products, parts of dw and dx, several pieces)
BACKWARD = [(1, 8, 1), (20, 520, 3000), (33, 33, 255), (513, 300, 2100), (900, 264, 5003), (2500, 264, 1203), (2227, 131, 10340),
            (4800, 768, 16500), (5798, 325, 14144), (6677, 24, 18997), (7274, 1599, 698), (7899, 1792, 212), (9000, 72, 130),
            (60000, 64, 20011)]


@pytest.mark.parametrize("rows,width,vocab", BACKWARD)
def test_head_backward(rows, width, vocab):
    lib = _lib.load()
    for dtype, ignored, need in ((torch.bfloat16, 0.1, 3), (torch.float16, 0.9, 3), (torch.bfloat16, 1.1, 3), (torch.float16, 0.3, 1),
                                 (torch.bfloat16, 0.3, 2)):
        x, w, target = make(rows, width, vocab, dtype, ignored)
        lse = apexw_amd.linear_cross_entropy_forward(x, w, target)[1]
        d = torch.rand(rows, generator=torch.Generator().manual_seed(3)).cuda() - 0.5
        dx, dw = apexw_amd.linear_cross_entropy_backward(d, x, w, target, lse, need=(bool(need & 1), bool(need & 2)))
        space = Place(lib.apexw_linear_cross_entropy_workspace(w.data_ptr(), width, rows, width, vocab, need))
        outs = [None if t is None else out_like(t) for t in (dx, dw)]
        _lib.check(lib.apexw_linear_cross_entropy_backward(
            d.data_ptr(), 1, 0, x.data_ptr(), width, rows, width, w.data_ptr(), width, vocab, CODE[dtype], target.data_ptr(), 8, -100,
            lse.data_ptr(), *(None if o is None else o.ptr for o in outs), space.ptr, stream()), "backward")
        for o, t in zip(outs, (dx, dw)):
            if t is not None:
                same(o, t)
        Place.check()


# ---------------------------------------------------------------------------- tokens by expert
def choices_of(tokens, k, experts, seed=0):
    g = torch.Generator().manual_seed(seed + tokens * 3 + experts)
    e = (torch.rand(tokens, k, generator=g) ** 2 * experts).long().clamp(max=experts - 1)
    e[torch.rand(tokens, k, generator=g) < 0.2] = -1
    return e.cuda()


@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (37, 3, 5), (2048, 2, 600), (4096, 1, 511), (2500, 2, 8), (70001, 1, 3),
                                              (35000, 2, 5000), (17500, 4, 300000), (300001, 2, 300)])
def test_order(tokens, k, experts):
    lib, e = _lib.load(), choices_of(tokens, k, experts)
    for ids in (e, e.int()):
        order = apexw_amd.expert_order(ids, experts)
        space = Place(lib.apexw_expert_order_workspace(tokens * k, experts))
        outs = [out_like(t) for t in order]
        _lib.check(lib.apexw_expert_order(ids.data_ptr(), ids.element_size(), tokens * k, experts, *(o.ptr for o in outs), space.ptr,
                                          stream()), "order")
        for o, t in zip(outs, order):
            same(o, t)
        Place.check()


@pytest.mark.parametrize("dtype", list(CODE))
@pytest.mark.parametrize("width", [1, 3, 7, 8, 9, 130, 513, 1021, 2056])
def test_rows(width, dtype):
    lib, tokens, k, code = _lib.load(), 37, 3, CODE[dtype]
    order = apexw_amd.expert_order(choices_of(tokens, k, 5), 5)
    source, place = order.source.data_ptr(), order.place.data_ptr()
    g = torch.Generator().manual_seed(width)
    x, y, dout = (torch.randn(n, width, generator=g).to(dtype).cuda() for n in (tokens, tokens * k, tokens))
    rows = apexw_amd.expert_dispatch_forward(x, order)
    to = out_like(rows)
    _lib.check(lib.apexw_expert_dispatch(x.data_ptr(), width, tokens, k, width, code, source, place, to.ptr, stream()), "dispatch")
    same(to, rows)
    for w_dtype in {dtype, torch.float32}:
        weight = torch.rand(tokens, k, generator=g).to(w_dtype).cuda()
        out = apexw_amd.expert_combine_forward(y, order, weight)
        to = out_like(out)
        _lib.check(lib.apexw_expert_combine(y.data_ptr(), width, tokens, k, width, code, place, weight.data_ptr(), CODE[w_dtype], to.ptr,
                                            stream()), "combine")
        same(to, out)
        dy, dw = apexw_amd.expert_combine_backward(dout, y, order, weight)
        to, to_w = out_like(dy), out_like(dw)
        _lib.check(lib.apexw_expert_combine_backward(dout.data_ptr(), width, y.data_ptr(), width, tokens, k, width, code, source, place,
                                                     weight.data_ptr(), CODE[w_dtype], to.ptr, to_w.ptr, stream()), "backward")
        same(to, dy), same(to_w, dw)


# ---------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", list(CODE))
@pytest.mark.parametrize("tokens,width,vocab", [(1, 1, 1), (5, 7, 3), (300, 9, 40), (1000, 1021, 70), (1024, 24, 5003), (1025, 24, 5003),
                                                (3000, 130, 17), (5000, 2056, 300), (20000, 33, 50021), (140000, 24, 3001),
                                                (530001, 8, 700001)])
def test_embedding(tokens, width, vocab, dtype):
    lib, g = _lib.load(), torch.Generator().manual_seed(tokens + width)
    ids = (torch.rand(tokens, generator=g) ** 3 * (vocab + 1)).long().cuda() - 1         # some outside the table
    table, dy = (torch.randn(n, width, generator=g).to(dtype).cuda() for n in (vocab, tokens))
    out = apexw_amd.embedding_forward(ids, table, 3.0)
    to = out_like(out)
    _lib.check(lib.apexw_embedding_forward(ids.data_ptr(), 8, tokens, table.data_ptr(), width, vocab, width, CODE[dtype], 3.0, to.ptr,
                                           stream()), "forward")
    same(to, out)
    for kind in {dtype, torch.float32}:
        dw = apexw_amd.embedding_weight_grad(dy, ids, vocab, 3.0, kind)
        space, to = Place(lib.apexw_embedding_weight_grad_workspace(tokens, vocab, width)), out_like(dw)
        _lib.check(lib.apexw_embedding_weight_grad(dy.data_ptr(), width, ids.data_ptr(), 8, tokens, vocab, width, CODE[dtype], 3.0,
                                                   to.ptr, CODE[kind], space.ptr, stream()), "gradient")
        same(to, dw)

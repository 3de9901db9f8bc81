"""Each way that an expert product may take -- the four tile shapes in both orders of the weights, whole and in
parts, operands copied to whole chunks, the general kernel -- at a size that takes it, against float64 with the
bars of test_gpu_experts.  The kernels that ran are read from a profile, so a size that a changed rule sends
elsewhere fails here."""

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

import apexw_amd
from test_gpu_experts import close, exact, make

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SHAPES = {"Large": "Shape<256, 256", "Wide": "Shape<128, 256", "Mid": "Shape<64, 128", "Small": "Shape<32, 128"}


def taken(call):
    """The call's result, and how it was formed: copied or not, tile shapes, parts joined or not."""
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        out = call()
        torch.cuda.synchronize()
    names = [e.name for e in p.events() if "expert_" in e.name or "pad_kernel" in e.name or "join_" in e.name]
    what = {s for s, text in SHAPES.items() if any(text in n for n in names)}
    what |= {"general" for n in names if "expert_rows_kernel" in n or "expert_weight_kernel" in n}
    what |= {"copied" for n in names if "pad_kernel" in n}
    what |= {"parts" for n in names if "join_" in n}
    return out, what


def uneven(rows, experts):
    """Sizes of one to three parts, an empty expert and a single row among them."""
    if experts == 1:
        return [rows]
    if experts == 2:
        return [rows // 3, rows - rows // 3]
    parts = [1 + (5 * e) % 3 for e in range(experts - 2)]
    sizes = [(rows - 1) * p // sum(parts) for p in parts]
    sizes[0] += rows - 1 - sum(sizes)
    return sizes[:1] + [0] + sizes[1:] + [1]


# remainders modulo 256 of 0, 0 (no rows), 1, 128, 129, 255 and others
LAST_TILES = [1024, 0, 769, 896, 1153, 1023, 300, 1500, 335]

# what, rows, experts or their sizes, rows behind the last end, inner, outer, types
FORWARD = [
    ("Large Wide", 7000, LAST_TILES, 0, 256, 6144, (BF16, FP16)),
    ("Large Wide", 7040, LAST_TILES, 40, 264, 6200, (BF16,)),                  # a last stage, column and chunk in part
    ("Large Wide", 4500, [1280, 512, 0, 2707, 1], 0, 520, 4104, (FP16,)),
    ("Large Wide", 30001, 2, 1, 72, 264, (BF16,)),
    ("Wide", 4000, 5, 11, 264, 2056, (BF16, FP16)),
    ("Mid", 2048, 8, 5, 1024, 1024, (BF16, FP16)),
    ("Small", 300, 6, 0, 320, 200, (BF16, FP16)),
    ("Mid parts", 256, 2, 9, 4096, 1024, (BF16, FP16)),
    ("Small parts", 40, 1, 2, 2048, 2048, (BF16, FP16)),
    ("copied Large Wide", 9000, 2, 0, 501, 2001, (BF16, FP16)),
    ("copied Wide", 16574, 5, 30, 19, 140, (BF16,)),
    ("copied Mid", 17150, 5, 0, 9, 7, (FP16,)),
    ("copied Small", 6251, 2, 0, 9, 10, (BF16,)),
    ("copied Mid parts", 1052, 2, 0, 2924, 163, (BF16,)),
    ("copied Small parts", 400, 1, 4, 4097, 130, (BF16, FP16)),
    ("general", 800, 2, 6, 1003, 2000, (BF16, FP16)),
    ("general parts", 1000, 1, 0, 1001, 130, (BF16, FP16)),
]
ROWS_GRAD = [
    ("Large Wide", 7000, LAST_TILES, 0, 6144, 256, (BF16, FP16)),
    ("Large Wide", 7040, LAST_TILES, 40, 6200, 264, (BF16,)),
    ("Wide", 4000, 5, 11, 2056, 264, (BF16, FP16)),
    ("Mid", 2048, 8, 5, 1024, 1024, (BF16, FP16)),
    ("Small", 300, 6, 0, 200, 320, (BF16, FP16)),
    ("Mid parts", 256, 2, 9, 1024, 4096, (BF16, FP16)),
    ("Small parts", 40, 1, 2, 2048, 2048, (BF16, FP16)),
    ("copied Large Wide", 9000, 2, 0, 2001, 501, (BF16, FP16)),
    ("copied Wide", 9000, 2, 7, 504, 2001, (BF16,)),                           # the rows alone
    ("copied Wide", 9000, 2, 0, 501, 2000, (FP16,)),                           # the weights alone
    ("copied Mid", 16720, 8, 0, 8, 9, (BF16,)),
    ("copied Small", 192, 2, 0, 8, 11, (BF16,)),
    ("copied Mid parts", 254, 2, 0, 1054, 3898, (BF16,)),
    ("copied Small parts", 400, 1, 4, 130, 4097, (BF16, FP16)),
    ("general", 60, 50, 0, 300, 203, (BF16, FP16)),
    ("general parts", 30, 3, 1, 2000, 1001, (BF16, FP16)),
]
WEIGHT_GRAD = [
    ("Large", 7040, LAST_TILES, 40, 520, 6200, (BF16, FP16)),
    ("Large", 4500, 5, 0, 520, 4104, (BF16,)),
    ("Wide", 4000, 5, 11, 264, 2056, (BF16, FP16)),
    ("Large parts", 3397, 3, 0, 16, 1720, (BF16, FP16)),
    ("Wide parts", 9000, 1, 7, 512, 512, (BF16, FP16)),
    ("Wide parts", 20000, 14, 0, 288, 104, (BF16,)),
    ("copied Large", 7, 12, 0, 1303, 2174, (BF16,)),
    ("copied Wide", 800, 2, 5, 1003, 2001, (BF16, FP16)),
    ("copied Wide", 800, 2, 0, 1003, 2000, (BF16,)),                          # x alone
    ("copied Wide", 900, 2, 0, 1032, 333, (FP16,)),                           # dy alone
    ("copied Large parts", 3728, 3, 1, 16, 1689, (BF16,)),
    ("copied Wide parts", 9000, 1, 3, 510, 511, (BF16, FP16)),
    ("general", 60, 50, 2, 300, 203, (BF16, FP16)),
]


def cases(table):
    for what, total, experts, spare, inner, outer, dtypes in table:
        sizes = experts if isinstance(experts, list) else uneven(total - spare, experts)
        assert sum(sizes) + spare == total
        for dtype in dtypes:
            yield pytest.param(set(what.split()), sizes, spare, inner, outer, dtype,
                               id=f"{what.replace(' ', '-')}-{total}x{inner}x{outer}-{str(dtype)[6:]}")


@pytest.mark.parametrize("what,sizes,spare,inner,outer,dtype", cases(FORWARD))
def test_forward(what, sizes, spare, inner, outer, dtype):
    x, dy, w, ends = make(sizes, inner, outer, dtype, spare)
    (want, _, _), (mag, _, _) = exact(sizes, x, dy, w)
    got, ways = taken(lambda: apexw_amd.expert_matmul_forward(x, w, ends))
    close(got, want, mag, inner)
    assert ways == what


@pytest.mark.parametrize("what,sizes,spare,inner,outer,dtype", cases(ROWS_GRAD))
def test_rows_grad(what, sizes, spare, inner, outer, dtype):
    x, dy, w, ends = make(sizes, inner, outer, dtype, spare)
    (_, want, _), (_, mag, _) = exact(sizes, x, dy, w)
    got, ways = taken(lambda: apexw_amd.expert_matmul_rows_grad(dy, w, ends))
    close(got, want, mag, outer)
    assert ways == what


@pytest.mark.parametrize("what,sizes,spare,inner,outer,dtype", cases(WEIGHT_GRAD))
def test_weight_grad(what, sizes, spare, inner, outer, dtype):
    x, dy, w, ends = make(sizes, inner, outer, dtype, spare)
    (_, _, want), (_, _, mag) = exact(sizes, x, dy, w)
    for to in (dtype, torch.float32):
        got, ways = taken(lambda: apexw_amd.expert_matmul_weight_grad(dy, x, ends, to))
        close(got, want, mag, max(sizes))
        assert ways == what


def test_one_operand_copied():
    """An operand at an odd address beside one that needs no copy."""
    sizes = [700, 0, 1301]
    x, dy, w, ends = make(sizes, 2056, 520, BF16)
    for xs, ws in ((x[:, 1:2049], w[:, :, :2048]), (x[:, :2048], w[:, :, 1:2049])):
        (want, _, _), (mag, _, _) = exact(sizes, xs, dy, ws)
        got, ways = taken(lambda: apexw_amd.expert_matmul_forward(xs, ws, ends))
        close(got, want, mag, 2048)
        assert "copied" in ways


def test_parts_of_nothing():
    """Sums cut into more parts than some experts have rows, and experts without any."""
    sizes = [0, 9000, 0, 1, 63]
    x, dy, w, ends = make(sizes, 128, 64, BF16, 20)
    (_, _, want), (_, _, mag) = exact(sizes, x, dy, w)
    got, ways = taken(lambda: apexw_amd.expert_matmul_weight_grad(dy, x, ends, torch.float32))
    close(got, want, mag, 9000)
    assert "parts" in ways and (got[0] == 0).all() and (got[2] == 0).all()

"""The softmax cross entropy of a linear head over a large vocabulary, on the kernels of libapexw_hip.so.

``linear_cross_entropy(x, weight, target)`` is ``cross_entropy(x @ weight.T, target)`` without the logits in memory:
the forward pass keeps one number a row, the backward pass computes them again a piece of the vocabulary at a time.

The tensors are CUDA (ROCm) ones; calls run on the current stream of their device, with nothing read back on the
host, and equal calls give equal bits.  What is not supported raises before anything is launched.
"""

import torch

from . import _lib
from .ops import _CODE, _current, _done, _Launch, _native, _on_device, _ptr, _raw_stream, _rows
from .tokens import _ID_BYTES, _space

_REDUCTION = {"none": 0, "sum": 1, "mean": 2}


def _check(x, weight, target):
    if x.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != x.dtype:
        raise TypeError(f"linear_cross_entropy: expected rows and weights of bfloat16 or float16, got {x.dtype} and "
                        f"{weight.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0 or weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"linear_cross_entropy: expected rows of shape (..., width) and weights of (vocabulary, width), "
                         f"got {tuple(x.shape)} and {tuple(weight.shape)}")
    if target.dtype not in _ID_BYTES:
        raise TypeError(f"linear_cross_entropy: expected targets of int32 or int64, got {target.dtype}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: expected a target for each row {tuple(x.shape[:-1])}, got "
                         f"{tuple(target.shape)}")
    _on_device(x, "linear_cross_entropy: x")
    _on_device(weight, "linear_cross_entropy: weight", x.device)
    _on_device(target, "linear_cross_entropy: target", x.device)
    src, n, stride = _rows(x, x.shape[-1])
    weight = weight if weight.stride(1) == 1 or weight.shape[1] == 1 else weight.contiguous()
    return src, n, stride, weight, target.contiguous()


def _forward(x, weight, target, ignore_index, reduction):
    native = _native(x)
    if native is not None:
        dev = _current()
        out = native.head_forward(x, weight, target, ignore_index, reduction, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_linear_cross_entropy_forward")
    src, n, stride, weight, target = _check(x, weight, target)
    (vocab, width), lib = weight.shape, _lib.load()
    with _Launch(x.device) as stream:
        loss = torch.empty(target.shape, dtype=torch.float32, device=x.device)
        lse = torch.empty(target.shape, dtype=torch.float32, device=x.device)
        total = torch.empty((), dtype=torch.float32, device=x.device) if reduction else None
        space = _space(lib.apexw_linear_cross_entropy_workspace(weight.data_ptr(), weight.stride(0), n, width, vocab, 0),
                       x.device, "apexw_linear_cross_entropy_forward")
        _lib.check(lib.apexw_linear_cross_entropy_forward(
            _ptr(src), stride, n, width, weight.data_ptr(), weight.stride(0), vocab, _CODE[x.dtype], _ptr(target),
            _ID_BYTES[target.dtype], ignore_index, _ptr(loss), _ptr(lse), reduction, _ptr(total), _ptr(space), stream),
            "apexw_linear_cross_entropy_forward")
    return loss, lse, total


def _backward(dloss, stride_d, mean, x, weight, target, lse, ignore_index, need):
    native = _native(x)
    if native is not None:
        dev = _current()
        out = native.head_backward(dloss, stride_d, mean, x, weight, target, lse, ignore_index, need[0], need[1],
                                   _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_linear_cross_entropy_backward")
    src, n, stride, weight, target = _check(x, weight, target)
    (vocab, width), lib = weight.shape, _lib.load()
    if not need[0] and not need[1]:
        return None, None
    with _Launch(x.device) as stream:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        dw = torch.empty((vocab, width), dtype=x.dtype, device=x.device) if need[1] else None
        ways = (1 if need[0] else 0) | (2 if need[1] else 0)
        space = _space(lib.apexw_linear_cross_entropy_workspace(weight.data_ptr(), weight.stride(0), n, width, vocab, ways),
                       x.device, "apexw_linear_cross_entropy_backward")
        _lib.check(lib.apexw_linear_cross_entropy_backward(
            _ptr(dloss), stride_d, mean, _ptr(src), stride, n, width, weight.data_ptr(), weight.stride(0), vocab,
            _CODE[x.dtype], _ptr(target), _ID_BYTES[target.dtype], ignore_index, _ptr(lse), _ptr(dx), _ptr(dw),
            _ptr(space), stream), "apexw_linear_cross_entropy_backward")
    return dx, dw


def linear_cross_entropy_forward(x, weight, target, ignore_index=-100):
    """(loss, lse) of each row: lse = log(sum(exp(weight @ x))), loss = lse - (weight @ x)[target], in fp32.

    x: (..., width) of bfloat16 or float16; weight: (vocabulary, width) of the same type; target: int32 or int64,
    x's shape without its last dimension.  Rows whose target is ignore_index or outside the vocabulary count for
    nothing: both results are 0 there, whatever the row holds.  lse is what the backward half takes."""
    return _forward(x, weight, target, ignore_index, 0)[:2]


def linear_cross_entropy_backward(dloss, x, weight, target, lse, ignore_index=-100, need=(True, True)):
    """(dx, dweight) from the gradient dloss (float32) of each row's loss and the lse that the forward half gave.

    Rows that count for nothing get zeros in dx and give nothing to dweight, whatever they hold; ``need`` leaves out
    gradients nobody wants (None).  The softmax minus the target's one, times dloss, is rounded to x's type (scaled
    so that the largest |dloss| is 2^14) before the two products, which are summed in fp32 and rounded once."""
    for t, name in ((dloss, "dloss"), (lse, "lse")):
        if t.dtype != torch.float32 or t.shape != target.shape:
            raise ValueError(f"linear_cross_entropy: expected {name} as one float32 for each row {tuple(target.shape)}, got "
                             f"{tuple(t.shape)} of {t.dtype}")
    for t, name in ((dloss, "dloss"), (lse, "lse")):
        _on_device(t, f"linear_cross_entropy: {name}", x.device)
    one = all(s == 0 or n == 1 for n, s in zip(dloss.shape, dloss.stride()))   # one number for all rows
    return _backward(dloss if one else dloss.contiguous(), 0 if one else 1, 0, x, weight, target, lse.contiguous(),
                     ignore_index, need)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        loss, lse, total = _forward(x, weight, target, ignore_index, reduction)
        ctx.save_for_backward(x, weight, target, lse)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return total if reduction else loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, weight, target, lse = ctx.saved_tensors
        need = ctx.needs_input_grad[:2]
        if not ctx.reduction:
            grads = linear_cross_entropy_backward(dloss, x, weight, target, lse, ctx.ignore_index, need)
        else:
            grads = _backward(dloss, 0, int(ctx.reduction == 2), x, weight, target, lse, ctx.ignore_index, need)
        return (*grads, None, None, None)


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean"):
    """torch.nn.functional.cross_entropy(x @ weight.T, target) in fp32, differentiable in x and weight.

    reduction: "mean" over the rows that count (NaN where none does), "sum", or "none": one loss a row."""
    code = _REDUCTION.get(reduction)
    if code is None:
        raise ValueError(f'linear_cross_entropy: reduction is "mean", "sum" or "none", not {reduction!r}')
    return _LinearCrossEntropy.apply(x, weight, target, ignore_index, code)

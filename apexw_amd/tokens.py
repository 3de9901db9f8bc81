"""Tokens sorted by expert and back, and the embedding, on the kernels of libapexw_hip.so.

* ``expert_order``, ``expert_dispatch`` and ``expert_combine``: the rows of a mixture of experts in the order that
  ``expert_matmul`` takes, and its products brought back to their tokens with the router's weights;
* ``embedding``: rows of a table by token id, scaled, with the gradient summed over the sorted tokens.

They take CUDA (ROCm) tensors, run on the current stream of the tensors' device and allocate their outputs
there; nothing is read back on the host.  Sums are taken in fp32 in a fixed order, so equal calls give equal bits.
What they do not support raises before anything is launched.
"""

from typing import NamedTuple

import torch

from . import _lib
from .ops import _CODE, _current, _done, _Launch, _native, _on_device, _ptr, _raw_stream, _rows

_ID_BYTES = {torch.int32: 4, torch.int64: 8}


class ExpertOrder(NamedTuple):
    """Where each choice of an expert lies among the rows sorted by expert, as ``expert_order`` makes it.

    source: the choice (its flat index) that each row belongs to, -1 in rows behind the last expert's;
    place: the row of each choice, -1 for one that no expert takes; ends: one past each expert's last row.
    All int32.  source and place are each other's inverse; the operators trust that they are."""
    source: torch.Tensor
    place: torch.Tensor
    ends: torch.Tensor


def _check_ids(t, name):
    if t.dtype not in _ID_BYTES:
        raise TypeError(f"{name}: expected int32 or int64, got {t.dtype}")
    _on_device(t, name)
    return t.contiguous()


def _space(size, device, what):
    if size < 0:
        _lib.check(-size, what)
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _check_matrix(t, name, rows=None, width=None):
    """Rows for the kernels: the tensor or a copy, and the elements from row to row."""
    if t.dtype not in _CODE:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != 2 or t.shape[1] == 0 or rows not in (None, t.shape[0]) or width not in (None, t.shape[1]):
        raise ValueError(f"{name}: expected shape ({'rows' if rows is None else rows}, {width or 'width'}), got "
                         f"{tuple(t.shape)}")
    _on_device(t, name)
    t = t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()
    return t, t.stride(0)


def _check_order(order, name, device):
    """(tokens, choices a token) of an order whose tensors lie on `device`."""
    source, place = order.source, order.place
    for t, what in ((source, "source"), (place, "place")):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise TypeError(f"{name}: expected the order's {what} as contiguous int32, got {t.dtype}")
        _on_device(t, f"{name}: {what}", device)
    if place.dim() not in (1, 2) or source.dim() != 1 or source.shape[0] != place.numel() or 0 in place.shape[1:]:
        raise ValueError(f"{name}: expected an order of (tokens,) or (tokens, choices), got places of shape "
                         f"{tuple(place.shape)} and {tuple(source.shape)} rows")
    return place.shape[0], place.shape[1] if place.dim() == 2 else 1


def _check_weight(weight, order, dtype, name, device):
    if weight is None:
        return None, dtype
    if weight.dtype not in (dtype, torch.float32):
        raise TypeError(f"{name}: weights are {dtype} or float32 for rows of {dtype}, got {weight.dtype}")
    if weight.shape != order.place.shape:
        raise ValueError(f"{name}: expected a weight for each of the choices {tuple(order.place.shape)}, got "
                         f"{tuple(weight.shape)}")
    _on_device(weight, f"{name}: weight", device)
    return weight.contiguous(), weight.dtype


# ---------------------------------------------------------------------------- tokens by expert
def expert_order(expert, experts):
    """The order of the tokens' choices by expert, an ``ExpertOrder``.

    expert: the experts that each token chose, (tokens,) or (tokens, choices), int32 or int64.  An id outside
    [0, experts) belongs to no expert: such choices (padding, or what exceeds an expert's capacity) get no row.
    Rows of one expert keep the order of their choices.  ``order.ends`` is what ``expert_matmul`` takes."""
    native = _native(expert)
    if native is not None:
        dev = _current()
        out = native.expert_order(expert, experts, _raw_stream(dev), dev)
        if out is not None:
            return ExpertOrder._make(_done(out, "apexw_expert_order"))
    expert = _check_ids(expert, "expert_order: expert")
    if expert.dim() not in (1, 2) or 0 in expert.shape[1:]:
        raise ValueError(f"expert_order: expected (tokens,) or (tokens, choices), got {tuple(expert.shape)}")
    if not 0 < experts < 2 ** 31 - 1:
        raise ValueError(f"expert_order: expected at least one expert, got {experts}")
    lib, n = _lib.load(), expert.numel()
    with _Launch(expert.device) as stream:
        space = _space(lib.apexw_expert_order_workspace(n, experts), expert.device, "apexw_expert_order")
        source = torch.empty(n, dtype=torch.int32, device=expert.device)
        place = torch.empty(expert.shape, dtype=torch.int32, device=expert.device)
        ends = torch.empty(experts, dtype=torch.int32, device=expert.device)
        _lib.check(lib.apexw_expert_order(expert.data_ptr(), _ID_BYTES[expert.dtype], n, experts, source.data_ptr(),
                                          place.data_ptr(), ends.data_ptr(), _ptr(space), stream), "apexw_expert_order")
    return ExpertOrder(source, place, ends)


def expert_dispatch_forward(x, order):
    """rows[r] = x[t] for the token t whose choice row r belongs to; zeros in rows that belong to none.

    x: (tokens, width) of float32, bfloat16 or float16; the result has a row for each choice."""
    native = _native(x)
    if native is not None:
        dev = _current()
        out = native.expert_dispatch(x, order[0], order[1], _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_expert_dispatch")
    x, stride = _check_matrix(x, "expert_dispatch: x")
    tokens, k = _check_order(order, "expert_dispatch", x.device)
    if x.shape[0] != tokens:
        raise ValueError(f"expert_dispatch: {x.shape[0]} rows for an order of {tokens} tokens")
    with _Launch(x.device) as stream:
        rows = torch.empty((tokens * k, x.shape[1]), dtype=x.dtype, device=x.device)
        _lib.check(_lib.load().apexw_expert_dispatch(x.data_ptr(), stride, tokens, k, x.shape[1], _CODE[x.dtype],
                                                     order.source.data_ptr(), order.place.data_ptr(), rows.data_ptr(),
                                                     stream), "apexw_expert_dispatch")
    return rows


def expert_combine_forward(y, order, weight=None):
    """out[t] = sum over token t's choices j of weight[t, j] * y[row of the choice], without those that have no row.

    y: a row for each choice; weight: (tokens,) or (tokens, choices) as the order's, of y's type or float32, None
    for ones."""
    native = _native(y)
    if native is not None:
        dev = _current()
        out = native.expert_combine(y, order[0], order[1], weight, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_expert_combine")
    y, stride = _check_matrix(y, "expert_combine: y")
    tokens, k = _check_order(order, "expert_combine", y.device)
    if y.shape[0] != tokens * k:
        raise ValueError(f"expert_combine: {y.shape[0]} rows for an order of {tokens * k} choices")
    weight, w_dtype = _check_weight(weight, order, y.dtype, "expert_combine", y.device)
    with _Launch(y.device) as stream:
        out = torch.empty((tokens, y.shape[1]), dtype=y.dtype, device=y.device)
        _lib.check(_lib.load().apexw_expert_combine(y.data_ptr(), stride, tokens, k, y.shape[1], _CODE[y.dtype],
                                                    order.place.data_ptr(), _ptr(weight), _CODE[w_dtype],
                                                    out.data_ptr(), stream), "apexw_expert_combine")
    return out


def expert_dispatch_backward(drows, order):
    """The gradient of expert_dispatch's x: each token's rows added up."""
    return expert_combine_forward(drows, order)


def expert_combine_backward(dout, y, order, weight=None, need=(True, True)):
    """(dy, dweight) of expert_combine: dy[r] = weight * dout[t] of the choice that row r belongs to, zeros in rows that
    belong to none; dweight = <dout[t], y[row]>, 0 for a choice without a row (None without weights).

    ``need`` leaves out gradients nobody wants (None); y may be None where dweight is not wanted."""
    if weight is None:
        return expert_dispatch_forward(dout, order) if need[0] else None, None
    native = _native(dout)
    if native is not None:
        dev = _current()
        out = native.expert_combine_backward(dout, y, order[0], order[1], weight, need[0], need[1], _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_expert_combine_backward")
    dout, dout_stride = _check_matrix(dout, "expert_combine: dout")
    tokens, k = _check_order(order, "expert_combine", dout.device)
    if dout.shape[0] != tokens:
        raise ValueError(f"expert_combine: {dout.shape[0]} rows of gradients for an order of {tokens} tokens")
    weight, w_dtype = _check_weight(weight, order, dout.dtype, "expert_combine", dout.device)
    y_stride = 0
    if need[1]:
        if y is None:
            raise ValueError("expert_combine: the weights' gradient takes y, got None")
        if y.dtype != dout.dtype:
            raise TypeError(f"expert_combine: rows of {y.dtype} and gradients of {dout.dtype}")
        y, y_stride = _check_matrix(y, "expert_combine: y", tokens * k, dout.shape[1])
        _on_device(y, "expert_combine: y", dout.device)
    with _Launch(dout.device) as stream:
        dy = torch.empty((tokens * k, dout.shape[1]), dtype=dout.dtype, device=dout.device) if need[0] else None
        dw = torch.empty(weight.shape, dtype=w_dtype, device=dout.device) if need[1] else None
        _lib.check(_lib.load().apexw_expert_combine_backward(
            dout.data_ptr(), dout_stride, _ptr(y) if need[1] else None, y_stride, tokens, k, dout.shape[1],
            _CODE[dout.dtype], order.source.data_ptr(), order.place.data_ptr(), weight.data_ptr(), _CODE[w_dtype],
            _ptr(dy), _ptr(dw), stream), "apexw_expert_combine_backward")
    return dy, dw


class _ExpertDispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, source, place, ends):
        ctx.save_for_backward(source, place, ends)
        return expert_dispatch_forward(x, ExpertOrder(source, place, ends))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows):
        return expert_dispatch_backward(drows, ExpertOrder(*ctx.saved_tensors)), None, None, None


class _ExpertCombine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weight, source, place, ends):
        # (the rows are kept for the weights' gradient alone)
        ctx.save_for_backward(y if ctx.needs_input_grad[1] else None, weight, source, place, ends)
        return expert_combine_forward(y, ExpertOrder(source, place, ends), weight)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, weight, *order = ctx.saved_tensors
        return (*expert_combine_backward(dout, y, ExpertOrder(*order), weight, ctx.needs_input_grad[:2]), None, None, None)


def expert_dispatch(x, order):
    """expert_dispatch_forward, differentiable in x."""
    return _ExpertDispatch.apply(x, *order)


def expert_combine(y, order, weight=None):
    """expert_combine_forward, differentiable in y and weight."""
    return _ExpertCombine.apply(y, weight, *order)


# ---------------------------------------------------------------------------- embedding
def _check_scale(scale):
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"embedding: expected a scale that float32 holds, got {scale}")


def embedding_forward(ids, weight, scale=1.0):
    """out[...] = scale * weight[ids[...]], rounded once; zeros for an id outside the table.

    ids: int32 or int64 of any shape; weight: (vocabulary, width) of float32, bfloat16 or float16."""
    native = _native(ids)
    if native is not None:
        dev = _current()
        out = native.embedding_forward(ids, weight, scale, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_embedding_forward")
    ids = _check_ids(ids, "embedding: ids")
    weight, stride = _check_matrix(weight, "embedding: weight")
    _on_device(weight, "embedding: weight", ids.device)
    _check_scale(scale)
    if weight.shape[0] == 0:
        raise ValueError("embedding: expected a table of at least one row")
    with _Launch(ids.device) as stream:
        out = torch.empty((*ids.shape, weight.shape[1]), dtype=weight.dtype, device=ids.device)
        _lib.check(_lib.load().apexw_embedding_forward(ids.data_ptr(), _ID_BYTES[ids.dtype], ids.numel(), weight.data_ptr(),
                                                       stride, *weight.shape, _CODE[weight.dtype], scale, out.data_ptr(),
                                                       stream), "apexw_embedding_forward")
    return out


def embedding_weight_grad(dy, ids, vocab, scale=1.0, dtype=None):
    """dW[v] = scale * the sum of dy over the tokens whose id is v, (vocab, width): the gradient of embedding's
    weight, zero for an id that no token has; tokens whose id is outside the table count for nothing.

    dtype: dy's (the default) or float32.  Summed in fp32, in an order that the ids alone set."""
    native = _native(dy)
    if native is not None and dtype in (None, dy.dtype, torch.float32):
        dev = _current()
        out = native.embedding_weight_grad(dy, ids, vocab, scale, dtype is torch.float32, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_embedding_weight_grad")
    ids = _check_ids(ids, "embedding: ids")
    if dy.dtype not in _CODE:
        raise TypeError(f"embedding: expected float32, bfloat16 or float16 gradients, got {dy.dtype}")
    if dy.dim() != ids.dim() + 1 or dy.shape[:-1] != ids.shape or dy.shape[-1] == 0:
        raise ValueError(f"embedding: expected gradients of shape {(*ids.shape, 'width')}, got {tuple(dy.shape)}")
    _on_device(dy, "embedding: dy", ids.device)
    _check_scale(scale)
    dtype = dtype or dy.dtype
    if dtype not in (dy.dtype, torch.float32):
        raise TypeError(f"embedding: the weight's gradient is {dy.dtype} or float32, not {dtype}")
    if not 0 < vocab < 2 ** 31 - 1:
        raise ValueError(f"embedding: expected a table of at least one row, got {vocab}")
    width, n, lib = dy.shape[-1], ids.numel(), _lib.load()
    src, _, stride = _rows(dy, width)
    with _Launch(ids.device) as stream:
        dw = torch.empty((vocab, width), dtype=dtype, device=ids.device)
        space = _space(lib.apexw_embedding_weight_grad_workspace(n, vocab, width), ids.device, "apexw_embedding_weight_grad")
        _lib.check(lib.apexw_embedding_weight_grad(_ptr(src), stride, _ptr(ids), _ID_BYTES[ids.dtype], n, vocab, width,
                                                   _CODE[dy.dtype], scale, dw.data_ptr(), _CODE[dtype], _ptr(space), stream),
                   "apexw_embedding_weight_grad")
    return dw


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.scale = weight.shape[0], scale
        return embedding_forward(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        return None, embedding_weight_grad(dy, ids, ctx.vocab, ctx.scale), None


def embedding(ids, weight, scale=1.0):
    """embedding_forward, differentiable in weight (a dense gradient of the weight's type)."""
    return _Embedding.apply(ids, weight, scale)

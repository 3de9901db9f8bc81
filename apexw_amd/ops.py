"""Operators that a training program runs around the optimizer step, on the kernels of libapexw_hip.so.

* ``layer_norm`` with its forward and backward halves;
* ``expert_matmul``: the products of a mixture of experts whose rows are sorted by expert, with the gradients
  of the rows and of the weights;
* ``clip_grads`` / ``clip_grad_norm_``: the clip of a list of gradients by their global norm.

They take CUDA (ROCm) tensors, run on the current stream of the tensors' device and allocate their outputs
there; nothing is read back on the host.  What they do not support raises before anything is launched.
"""

import ctypes

import torch

from . import _lib
from ._plan import _host

_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_ORDER = {1.0: 1, 2.0: 2, float("inf"): 0}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # (None in a torch without GPU functions)
_current = getattr(torch._C, "_cuda_getDevice", None)
_NATIVE = None
_ENTRIES = ("apexw_layer_norm_forward", "apexw_layer_norm_backward", "apexw_layer_norm_workspace", "apexw_expert_rows",
            "apexw_expert_rows_workspace", "apexw_expert_weight_grad", "apexw_expert_weight_grad_workspace",
            "apexw_clip_layout", "apexw_clip_grads", "apexw_clip_grads_small")


def _native(t):
    """The host module with the library's entry points, for a call on the GPU tensor t (else None)."""
    global _NATIVE
    if _NATIVE is None:
        if not (isinstance(t, torch.Tensor) and t.is_cuda):
            return None
        lib, mod = _lib.load(), _host()
        mod.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _ENTRIES))
        _NATIVE = mod
    return _NATIVE if isinstance(t, torch.Tensor) and t.is_cuda else None


def _done(out, what):
    """A native call's result; raises for a status."""
    if type(out) is int:
        _lib.check(out, what)
    return out


def _on_device(t, name, device=None):
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a tensor on the GPU, got one on {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


class _Launch:
    """`with _Launch(device) as stream`: the device made current, its current stream's handle."""

    def __init__(self, device):
        self.index = device.index
        self.before = torch.cuda.current_device()

    def __enter__(self):
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------- layer norm
def _rows(t, width):
    """A tensor as rows of `width` consecutive elements at one distance: (the tensor or a copy, rows, distance)."""
    if t.dim() == 1:
        return (t, 1, width) if t.stride(0) == 1 or width == 1 else (t.contiguous(), 1, width)
    if t.is_contiguous():
        return t, t.numel() // width, width
    if t.stride(-1) == 1 or width == 1:
        shape, strides = t.shape[:-1], t.stride()[:-1]
        dims = [(n, s) for n, s in zip(shape, strides) if n != 1]
        if not dims:
            return t, 1, width
        if all(a[1] == b[0] * b[1] for a, b in zip(dims, dims[1:])):
            return t, t.numel() // width, dims[-1][1]
    return t.contiguous(), t.numel() // width, width


def _check_norm(x, weight, bias):
    if x.dtype not in _CODE:
        raise TypeError(f"layer_norm: expected float32, bfloat16 or float16 rows, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: expected rows of at least one element, got a tensor of shape {tuple(x.shape)}")
    _on_device(x, "layer_norm: x")
    width, w_dtype = x.shape[-1], None
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        _on_device(t, f"layer_norm: {name}", x.device)
        if t.dim() != 1 or t.shape[0] != width:
            raise ValueError(f"layer_norm: expected a {name} of shape ({width},), got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32) or w_dtype not in (None, t.dtype):
            raise TypeError(f"layer_norm: weight and bias are both {x.dtype} or both float32 for rows of {x.dtype}, "
                            f"got a {name} of {t.dtype}")
        w_dtype = t.dtype
    return width, w_dtype or x.dtype


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd) of the layer norm of x over its last dimension.

    ``y = (x - mean) * rstd * weight + bias`` has x's shape and type, contiguous; ``mean`` and
    ``rstd = 1 / sqrt(var + eps)`` (float32, x's shape without its last dimension) are what
    ``layer_norm_backward`` takes.  weight and bias are of x's type, or float32 with 16-bit rows."""
    native = _native(x)
    if native is not None:
        dev = _current()
        out = native.layer_norm_forward(x, weight, bias, eps, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_layer_norm_forward")
    width, w_dtype = _check_norm(x, weight, bias)
    if not eps >= 0:
        raise ValueError(f"layer_norm: expected eps >= 0, got {eps}")
    src, rows, stride = _rows(x, width)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    lib = _lib.load()
    with _Launch(x.device) as stream:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        if rows:
            _lib.check(lib.apexw_layer_norm_forward(src.data_ptr(), rows, width, stride, _CODE[x.dtype], _ptr(weight),
                                                    _ptr(bias), _CODE[w_dtype], eps, y.data_ptr(), mean.data_ptr(),
                                                    rstd.data_ptr(), stream), "apexw_layer_norm_forward")
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias=None, need=(True, True, True)):
    """(dx, dw, db) of a layer norm from the gradient dy of its output and what its forward pass kept.

    dw and db are None without a weight or a bias; ``need`` leaves out gradients nobody wants (None).  The
    sums over rows are taken in a fixed order, so equal calls give equal bits."""
    native = _native(x)
    if native is not None:
        dev = _current()
        out = native.layer_norm_backward(dy, x, mean, rstd, weight, bias, *need, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_layer_norm_backward")
    width, w_dtype = _check_norm(x, weight, bias)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"layer_norm: expected dy of shape {tuple(x.shape)} and {x.dtype}, got {tuple(dy.shape)} "
                         f"and {dy.dtype}")
    _on_device(dy, "layer_norm: dy", x.device)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype != torch.float32 or t.numel() * width != x.numel():
            raise ValueError(f"layer_norm: expected {name} as one float32 per row, got {tuple(t.shape)} of {t.dtype}")
        _on_device(t, f"layer_norm: {name}", x.device)
    src, rows, stride = _rows(x, width)
    grad, _, grad_stride = _rows(dy, width)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    w = None if weight is None else weight.contiguous()
    lib = _lib.load()
    with _Launch(x.device) as stream:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        dw = torch.empty(width, dtype=w_dtype, device=x.device) if weight is not None and need[1] else None
        db = torch.empty(width, dtype=w_dtype, device=x.device) if bias is not None and need[2] else None
        ws = None
        if dw is not None or db is not None:
            floats = lib.apexw_layer_norm_workspace(rows, width)
            if floats < 0:
                _lib.check(-floats, "apexw_layer_norm_workspace")
            ws = torch.empty(max(floats, 1), dtype=torch.float32, device=x.device)
        if ws is not None or (dx is not None and rows):
            _lib.check(lib.apexw_layer_norm_backward(
                grad.data_ptr() or _ptr(ws), grad_stride, src.data_ptr() or _ptr(ws), stride,
                mean.data_ptr() or _ptr(ws), rstd.data_ptr() or _ptr(ws), _ptr(w), rows, width, _CODE[x.dtype],
                _CODE[w_dtype], _ptr(dx) or None, _ptr(dw), _ptr(db), _ptr(ws), stream), "apexw_layer_norm_backward")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight, bias)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight, bias = ctx.saved_tensors
        return (*layer_norm_backward(dy, x, mean, rstd, weight, bias, ctx.needs_input_grad[:3]), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """The layer norm of x over its last dimension, differentiable in x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ---------------------------------------------------------------------------- expert products
def _check_rows(t, name, width=None):
    if t.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"expert_matmul: expected bfloat16 or float16 operands, got {name} of {t.dtype}")
    if t.dim() != 2 or t.shape[1] == 0 or width not in (None, t.shape[1]):
        raise ValueError(f"expert_matmul: expected {name} of shape (rows, {width or 'width'}), got {tuple(t.shape)}")
    _on_device(t, f"expert_matmul: {name}")
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check_ends(ends, device, experts=None):
    if ends.dtype not in (torch.int32, torch.int64) or ends.dim() != 1 or ends.shape[0] == 0:
        raise ValueError(f"expert_matmul: expected ends as a vector of int32, one per expert, got {tuple(ends.shape)} "
                         f"of {ends.dtype}")
    if experts not in (None, ends.shape[0]):
        raise ValueError(f"expert_matmul: {ends.shape[0]} ends for the weights of {experts} experts")
    _on_device(ends, "expert_matmul: ends", device)
    return ends.to(torch.int32).contiguous()


def _check_weight(weight, like):
    if weight.dtype != like.dtype:
        raise TypeError(f"expert_matmul: rows of {like.dtype} and weights of {weight.dtype}")
    if weight.dim() != 3 or 0 in weight.shape:
        raise ValueError(f"expert_matmul: expected weights of shape (experts, outer, inner), got {tuple(weight.shape)}")
    _on_device(weight, "expert_matmul: weight", like.device)


def _workspace(size, device):
    if size < 0:
        _lib.check(-size, "expert_matmul")
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _row_products(a, weight, ends, outer_first):
    """out[i] = W_e a[i] with W_e = weight[e] (outer_first) or its transpose."""
    w = weight if outer_first else weight.transpose(1, 2)      # [experts, n, k]
    if w.stride(2) == 1 or w.shape[2] == 1:
        order, ldw = _lib.EXPERT_NK, w.stride(1)
    elif w.stride(1) == 1 or w.shape[1] == 1:
        order, ldw = _lib.EXPERT_KN, w.stride(2)
    else:
        w = w.contiguous()
        order, ldw = _lib.EXPERT_NK, w.stride(1)
    lib = _lib.load()
    with _Launch(a.device) as stream:
        out = torch.empty((a.shape[0], w.shape[1]), dtype=a.dtype, device=a.device)
        if a.shape[0]:
            operands = (a.data_ptr(), a.stride(0), w.data_ptr(), ldw, w.stride(0), order)
            sizes = (ends.shape[0], a.shape[0], a.shape[1], w.shape[1])
            ws = _workspace(lib.apexw_expert_rows_workspace(*operands, *sizes), a.device)
            _lib.check(lib.apexw_expert_rows(*operands, ends.data_ptr(), *sizes, _CODE[a.dtype], out.data_ptr(),
                                             out.shape[1], _ptr(ws), stream), "apexw_expert_rows")
    return out


def expert_matmul_forward(x, weight, ends):
    """y[i] = weight[e] @ x[i] for the rows i of expert e; zeros in rows behind the last end.

    x: (rows, inner), sorted by expert; weight: (experts, outer, inner), contiguous in either of its last two
    dimensions; ends: int32, ends[e] one past expert e's last row (int64 is converted).  bfloat16 or float16,
    summed in fp32."""
    native = _native(x)
    if native is not None:
        dev = _current()
        out = native.expert_rows(x, weight, ends, False, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_expert_rows")
    x = _check_rows(x, "x")
    _check_weight(weight, x)
    if weight.shape[2] != x.shape[1]:
        raise ValueError(f"expert_matmul: rows of {x.shape[1]} elements for weights of shape {tuple(weight.shape)}")
    return _row_products(x, weight, _check_ends(ends, x.device, weight.shape[0]), True)


def expert_matmul_rows_grad(dy, weight, ends):
    """dx[i] = weight[e]^T @ dy[i]: the gradient of expert_matmul's rows; zeros behind the last end."""
    native = _native(dy)
    if native is not None:
        dev = _current()
        out = native.expert_rows(dy, weight, ends, True, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_expert_rows")
    dy = _check_rows(dy, "dy")
    _check_weight(weight, dy)
    if weight.shape[1] != dy.shape[1]:
        raise ValueError(f"expert_matmul: gradients of {dy.shape[1]} elements for weights of shape {tuple(weight.shape)}")
    return _row_products(dy, weight, _check_ends(ends, dy.device, weight.shape[0]), False)


def expert_matmul_weight_grad(dy, x, ends, dtype=None):
    """dW[e] = sum over expert e's rows of dy[i] x[i]^T, (experts, outer, inner): the gradient of
    expert_matmul's weights, zero for an expert without rows; dtype: dy's (the default) or float32."""
    native = _native(dy)
    if native is not None and dtype in (None, dy.dtype, torch.float32):
        dev = _current()
        out = native.expert_weight_grad(dy, x, ends, dtype is torch.float32, _raw_stream(dev), dev)
        if out is not None:
            return _done(out, "apexw_expert_weight_grad")
    dy, x = _check_rows(dy, "dy"), _check_rows(x, "x")
    if x.dtype != dy.dtype or x.device != dy.device or x.shape[0] != dy.shape[0]:
        raise ValueError(f"expert_matmul: dy {tuple(dy.shape)} of {dy.dtype} on {dy.device} and x {tuple(x.shape)} of "
                         f"{x.dtype} on {x.device} do not belong together")
    dtype = dtype or dy.dtype
    if dtype not in (dy.dtype, torch.float32):
        raise TypeError(f"expert_matmul: the weights' gradient is {dy.dtype} or float32, not {dtype}")
    ends = _check_ends(ends, dy.device)
    lib = _lib.load()
    with _Launch(dy.device) as stream:
        dw = torch.empty((ends.shape[0], dy.shape[1], x.shape[1]), dtype=dtype, device=dy.device)
        operands = (_ptr(dy), dy.stride(0), _ptr(x), x.stride(0))
        sizes = (ends.shape[0], dy.shape[0], dy.shape[1], x.shape[1])
        ws = _workspace(lib.apexw_expert_weight_grad_workspace(*operands, *sizes), dy.device)
        _lib.check(lib.apexw_expert_weight_grad(*operands, ends.data_ptr(), *sizes, _CODE[dy.dtype], dw.data_ptr(),
                                                _CODE[dtype], _ptr(ws), stream), "apexw_expert_weight_grad")
    return dw


class _ExpertMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ends):
        ctx.save_for_backward(x, weight, ends)
        return expert_matmul_forward(x, weight, ends)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, ends = ctx.saved_tensors
        dx = expert_matmul_rows_grad(dy, weight, ends) if ctx.needs_input_grad[0] else None
        dw = expert_matmul_weight_grad(dy, x, ends) if ctx.needs_input_grad[1] else None
        return dx, dw, None


def expert_matmul(x, weight, ends):
    """expert_matmul_forward, differentiable in x and weight."""
    return _ExpertMatmul.apply(x, weight, ends)


# ---------------------------------------------------------------------------- clip by the global norm
def _clip_lists(grads, out, name):
    """The lists of a clip, the same one twice in place, and their device (None: nothing to clip)."""
    grads = grads if type(grads) is list else list(grads)
    to = grads if out is None else out if type(out) is list else list(out)
    if len(to) != len(grads):
        raise ValueError(f"{name}: {len(grads)} gradients and {len(to)} tensors for their copies")
    if not grads:
        return grads, to, None
    if not isinstance(grads[0], torch.Tensor):
        raise TypeError(f"{name}: expected a list of tensors")
    _on_device(grads[0], name)
    return grads, to, grads[0].device


def _clip_table(grads, to, device, stream, name, writes=True, total=0):
    """The launch table on the device (made the current one): (table, entries, units); writes: `to` is written;
    total: the address of the norm that it is scaled by.

    A captured call puts the entries into the graph: it may not allocate pinned memory, nor copy from a block
    that is given back when the call returns."""
    lib, capturing = _lib.load(), torch.cuda.is_current_stream_capturing()
    host = torch.empty(len(grads) * _lib.CLIP_TENSOR_DTYPE.itemsize, dtype=torch.uint8, pin_memory=not capturing)
    _host().clip_table(grads, to, host.data_ptr(), name, writes, total)
    units = lib.apexw_clip_layout(host.data_ptr(), len(grads))
    if units < 0:
        _lib.check(-units, "apexw_clip_layout")
    if not capturing:
        return host.to(device, non_blocking=True), len(grads), units
    table = torch.empty_like(host, device=device)
    _lib.check(lib.apexw_clip_upload(host.data_ptr(), len(grads), table.data_ptr(), stream), "apexw_clip_upload")
    return table, len(grads), units


def _order(norm_type, name):
    order = _ORDER.get(float(norm_type))
    if order is None:
        raise ValueError(f"{name}: norm_type is 1, 2 or infinity, not {norm_type}")
    return order


def grad_norm(grads, norm_type=2.0):
    """The norm of all elements of a list of gradients, as a float32 scalar on their device (p = 1, 2, inf)."""
    order = _order(norm_type, "grad_norm")
    grads, to, device = _clip_lists(grads, None, "grad_norm")
    if device is None:
        return torch.tensor(0.0)
    with _Launch(device) as stream:
        table, n, units = _clip_table(grads, to, device, stream, "grad_norm", False)
        ws = torch.empty(_lib.CLIP_PARTIALS, dtype=torch.float64, device=device)
        norm = torch.empty((), dtype=torch.float32, device=device)
        _lib.check(_lib.load().apexw_grad_norm(table.data_ptr(), n, units, order, ws.data_ptr(), norm.data_ptr(), stream),
                   "apexw_grad_norm")
    return norm


def scale_grads(grads, max_norm, total_norm, out=None):
    """The second half of clip_grads with a norm that the caller formed (a float32 scalar on the gradients'
    device), for instance over the gradients of all processes."""
    if not max_norm >= 0:
        raise ValueError(f"scale_grads: expected max_norm >= 0, got {max_norm}")
    grads, to, device = _clip_lists(grads, out, "scale_grads")
    if device is None:
        return
    if total_norm.dtype != torch.float32 or total_norm.numel() != 1:
        raise ValueError("scale_grads: expected total_norm as one float32")
    _on_device(total_norm, "scale_grads: total_norm", device)
    with _Launch(device) as stream:
        table, n, units = _clip_table(grads, to, device, stream, "scale_grads", total=total_norm.data_ptr())
        _lib.check(_lib.load().apexw_grad_scale(table.data_ptr(), n, units, total_norm.data_ptr(), max_norm, stream),
                   "apexw_grad_scale")


def clip_grads(grads, max_norm, norm_type=2.0, out=None):
    """Clip a list of gradients by the norm of all their elements; returns that norm (float32 scalar on the
    device), as torch.nn.utils.clip_grad_norm_ computes and applies it:
    ``g * min(max_norm / (norm + 1e-6), 1)``, rounded once.

    out: tensors for the clipped copies, shaped and laid out like the gradients, of float32, bfloat16 or
    float16 each (fp32 accumulated gradients clipped into the parameters' type); None clips in place.  The
    gradients may mix types; each is dense, of any layout.  What is written shares memory with no other tensor
    of the lists (a tensor listed twice in place is refused)."""
    order = _order(norm_type, "clip_grads")
    if not max_norm >= 0:
        raise ValueError(f"clip_grads: expected max_norm >= 0, got {max_norm}")
    grads, to, device = _clip_lists(grads, out, "clip_grads")
    if device is None:
        return torch.tensor(0.0)
    native = _native(grads[0])
    if len(grads) <= _lib.CLIP_SMALL or not torch.cuda.is_current_stream_capturing():
        dev = _current()
        norm = native.clip_grads(grads, to, max_norm, order, _raw_stream(dev), dev)
        if norm is not None:
            return _done(norm, "apexw_clip_grads")
    with _Launch(device) as stream:
        table, n, units = _clip_table(grads, to, device, stream, "clip_grads")
        ws = torch.empty(_lib.CLIP_PARTIALS, dtype=torch.float64, device=device)
        norm = torch.empty((), dtype=torch.float32, device=device)
        _lib.check(_lib.load().apexw_clip_grads(table.data_ptr(), n, units, order, max_norm, ws.data_ptr(),
                                                norm.data_ptr(), stream), "apexw_clip_grads")
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ over the parameters that have a gradient (error_if_nonfinite reads the
    norm on the host, before the gradients are touched)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not error_if_nonfinite:
        return clip_grads(grads, max_norm, norm_type)
    if not max_norm >= 0:
        raise ValueError(f"clip_grad_norm_: expected max_norm >= 0, got {max_norm}")
    norm = grad_norm(grads, norm_type)
    if not torch.isfinite(norm):
        raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it "
                           "cannot be clipped.")
    scale_grads(grads, max_norm, norm)
    return norm

"""Layer norm over the last axes, forward and backward, with the sum of a residual stream in the same pass.

`layer_norm` is torch.nn.functional.layer_norm on this library's kernels (float32, bfloat16 or float16 on CUDA; statistics
and sums in fp32); with `residual` it first forms h = x + residual, as the blocks of a residual network do, and returns the norm of h
together with h.  `FusedLayerNorm` is the nn.LayerNorm around it, beside `batchnorm.FusedBatchNorm2d`, which normalises channels over
the batch where this normalises each row (or, with a shape of (C, H, W), each image) by itself.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn

from . import _lib, _native, adder_cuda


def _row_stride(shape, strides, d: int) -> Optional[int]:
    """Elements from row to row of a tensor whose last axes make rows of d consecutive elements; None where it is no such tensor.  Asked of the
    strides: a view that is refused while a torch.jit trace is made leaves an operation without a result in it, which ended the process."""
    i, inner = len(shape), 1
    while inner < d:
        i -= 1
        if shape[i] != 1 and strides[i] != inner:
            return None
        inner *= shape[i]
    stride = want = None
    for size, step in zip(reversed(shape[:i]), reversed(strides[:i])):
        if size == 1:
            continue
        if stride is None:
            stride = want = step
        elif step != want:
            return None
        want *= size
    return d if stride is None else stride


def _rows(t: torch.Tensor, rows: int, d: int):
    """(tensor, elements from row to row) of t as `rows` rows of d consecutive elements; a copy only where it has no such rows."""
    t = t.resolve_neg()
    if t.is_contiguous():
        return t, d
    stride = _row_stride(t.shape, t.stride(), d)
    return (t.contiguous(), d) if stride is None else (t, stride)


def _whole(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t as its memory stands: contiguous, and no lazy negation (which a view of a conjugate's imaginary part is)."""
    return None if t is None else t.resolve_neg().contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _form(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.dtype, t.device)


def _save(ctx, *tensors) -> None:
    ctx.forms = tuple(_form(t) for t in tensors)
    ctx.save_for_backward(*tensors)


def _saved(ctx):
    """The saved tensors.  What a saved-tensor hook hands back need not be what it was given, and the kernels go by the sizes of the
    forward call."""
    tensors = ctx.saved_tensors
    if tuple(_form(t) for t in tensors) != ctx.forms:
        raise RuntimeError("the saved tensors came back in another form: the shapes, types and device of the forward are needed")
    return tensors


def _sizes(x: torch.Tensor, normalized_shape) -> Tuple[int, int]:
    d = math.prod(normalized_shape)
    return (x.numel() // d if d else 0), d


class _Once(torch.autograd.Function):
    """Hands on a gradient as what follows from `sources`, and raises where it is differentiated."""

    @staticmethod
    def forward(ctx, name, grad, *sources):
        ctx.name = name
        return grad.detach()

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"{ctx.name} is differentiable once")


def _once(name: str, grad: Optional[torch.Tensor], *sources) -> Optional[torch.Tensor]:
    """`grad` of an operator that is differentiable once, computed from `sources`.  Where the backward pass is itself recorded
    (create_graph) it must not count as a constant, so differentiating it raises."""
    sources = [t for t in sources if t is not None and t.requires_grad]
    if grad is None or not sources or not torch.is_grad_enabled():
        return grad
    return _Once.apply(name, grad, *sources)


class _Recorded(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, *args):
        state = torch._C._get_tracing_state()
        torch._C._set_tracing_state(None)      # what `call` allocates and copies is no part of the trace
        try:
            return call(*args)
        finally:
            torch._C._set_tracing_state(state)


def _recorded(call, *args):
    """call(*args) of an operator without a gradient: in a torch.jit trace as one operation, where otherwise the allocation of its outputs would be
    all that is recorded."""
    return _Recorded.apply(call, *args) if torch.jit.is_tracing() else call(*args)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, normalized_shape, eps, needs_grad):
        rows, d = _sizes(x, normalized_shape)
        dev = x.device
        x2, xs = _rows(x, rows, d)
        r2, rs = _rows(residual, rows, d) if residual is not None else (None, 0)
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        h = torch.empty_like(y) if residual is not None else None
        mean = torch.empty(rows, device=dev) if needs_grad else None
        rstd = torch.empty(rows, device=dev) if needs_grad else None
        w, b = _whole(weight), _whole(bias)
        wtype = w if w is not None else b if b is not None else x
        with torch.cuda.device(dev):
            _lib.check(_lib.load().adder_b200_layernorm_forward(
                x2.data_ptr(), _ptr(r2), _ptr(w), _ptr(b), y.data_ptr(), _ptr(h), _ptr(mean), _ptr(rstd), rows, d, xs, rs,
                _lib.TYPE_CODES[x.dtype], _lib.TYPE_CODES[wtype.dtype], eps, adder_cuda._stream(dev)), "adder_b200_layernorm_forward")
        ctx.sizes = (rows, d, _lib.TYPE_CODES[wtype.dtype])
        ctx.has_residual = residual is not None
        ctx.shape = normalized_shape
        ctx.bias_type = bias.dtype if bias is not None else None
        ctx.set_materialize_grads(False)
        if needs_grad:
            _save(ctx, h if residual is not None else x, w, mean, rstd)
        if residual is None:
            return y
        return y, h

    @staticmethod
    def backward(ctx, dy, dh=None):
        if dy is None and dh is None:
            return (None,) * 7
        saved = _saved(ctx)
        with torch.no_grad():
            dx, dw, db = _LayerNorm.gradients(ctx, saved, dy, dh)
        need_x, need_r = ctx.needs_input_grad[0], ctx.has_residual and ctx.needs_input_grad[1]
        h = saved[0] if need_x or need_r else None      # it is an output as well, and asks for gradients whatever the inputs do
        dx = _once("layer_norm", dx, dy, dh, h, saved[1])
        return (dx if need_x else None, dx if need_r else None, _once("layer_norm", dw, dy, h), _once("layer_norm", db, dy),
                None, None, None)

    @staticmethod
    def gradients(ctx, saved, dy, dh):
        h, (w, mean, rstd) = saved[0], map(_whole, saved[1:])
        rows, d, wcode = ctx.sizes
        need_x = ctx.needs_input_grad[0] or (ctx.has_residual and ctx.needs_input_grad[1])
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if w is not None and ctx.needs_input_grad[2] else None
        db = torch.empty(ctx.shape, dtype=ctx.bias_type, device=h.device) if ctx.bias_type is not None and ctx.needs_input_grad[3] else None
        dy = _whole(dy) if dy is not None else torch.zeros(h.shape, dtype=h.dtype, device=h.device)
        dh = _whole(dh)
        h2, hs = _rows(h, rows, d)
        dx = torch.empty(h.shape, dtype=h.dtype, device=h.device) if need_x else None
        lib = _lib.load()
        with torch.cuda.device(h.device):
            nbytes = lib.adder_b200_layernorm_backward_workspace_bytes(rows, d) if dw is not None or db is not None else 0
            ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device) if nbytes else None
            _lib.check(lib.adder_b200_layernorm_backward(
                dy.data_ptr(), _ptr(dh), h2.data_ptr(), _ptr(w), mean.data_ptr(), rstd.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db),
                _ptr(ws), nbytes, rows, d, hs, _lib.TYPE_CODES[h.dtype], wcode, adder_cuda._stream(h.device)),
                "adder_b200_layernorm_backward")
        return dx, dw, db


def _check_input(t, name: str, dev=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if dev is not None and t.device != dev:
        raise RuntimeError(f"tensors are on different devices ({dev} and {t.device})")
    if t.dtype not in _lib.TYPE_CODES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")


def layer_norm(x: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """y = (h - mean) / sqrt(var + eps) * weight + bias over the last axes, which are `normalized_shape`.

    Without `residual` h is x, and y is returned.  With it h = x + residual, rounded to the type of both, and (y, h) is returned.
    `weight` and `bias` have the shape `normalized_shape` and x's type or float32 (both the same).  x and residual may be
    any views; those whose rows are not consecutive are copied.  Differentiable once, with respect to x, residual, weight and bias: a
    gradient of create_graph=True raises where it is differentiated.  At most 2^28 - 1 rows of at most 2^30 - 2^16 elements."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    out = _native.layer_norm(x, residual, weight, bias, shape, eps)
    if out is not None:
        return out
    _check_input(x, "x")
    if not shape or x.dim() < len(shape) or tuple(x.shape[x.dim() - len(shape):]) != shape or math.prod(shape) == 0:
        raise ValueError(f"x has shape {tuple(x.shape)}, whose last axes are not {shape}")
    if residual is not None:
        _check_input(residual, "residual", x.device)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual must have the shape and type of x: {tuple(residual.shape)} {residual.dtype}, "
                             f"expected {tuple(x.shape)} {x.dtype}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        _check_input(t, name, x.device)
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be {x.dtype} or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    needs_grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias))
    return _LayerNorm.apply(x, residual, weight, bias, shape, float(eps), needs_grad)


class FusedLayerNorm(nn.LayerNorm):
    """nn.LayerNorm with `forward(x, residual=None)`: with a residual it returns (norm of x + residual, x + residual).  Same parameters
    and state-dict keys.  CPU tensors go through torch."""

    def forward(self, x, residual=None):
        if x.is_cuda:
            return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps, residual=residual)
        if residual is None:
            return super().forward(x)
        h = x + residual
        return super().forward(h), h

"""RMS norm over the last axes, forward and backward, with the sum of a residual stream in the same pass, and its output in 8 bits.

`rms_norm` is torch.nn.functional.rms_norm on this library's kernels (float32, bfloat16 or float16 on CUDA; sums in fp32); with
`residual` it first forms h = x + residual and returns the norm of h together with h, as `layernorm.layer_norm` does.
`rms_norm_8bit` gives the norm as e4m3 codes with a scale for each 128 columns of a row, as `linear8.linear_8bit` takes them, so that
it is never written in 16 bits.  `FusedRMSNorm` is the nn.RMSNorm around both.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch
import torch.nn as nn

from . import _lib, _native, adder_cuda
from .layernorm import _check_input, _once, _ptr, _recorded, _rows, _save, _saved, _sizes, _whole
from .linear8 import Rows8, _empty_rows, _refuse_gradient


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, normalized_shape, eps, needs_grad):
        rows, d = _sizes(x, normalized_shape)
        dev = x.device
        x2, xs = _rows(x, rows, d)
        r2, rs = _rows(residual, rows, d) if residual is not None else (None, 0)
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        h = torch.empty_like(y) if residual is not None else None
        rstd = torch.empty(rows, device=dev) if needs_grad else None
        w = _whole(weight)
        wcode = _lib.TYPE_CODES[(w if w is not None else x).dtype]
        with torch.cuda.device(dev):
            _lib.check(_lib.load().adder_b200_rmsnorm_forward(
                x2.data_ptr(), _ptr(r2), _ptr(w), y.data_ptr(), _ptr(h), _ptr(rstd), rows, d, xs, rs, _lib.TYPE_CODES[x.dtype], wcode, eps,
                adder_cuda._stream(dev)), "adder_b200_rmsnorm_forward")
        ctx.sizes = (rows, d, wcode)
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)
        if needs_grad:
            _save(ctx, h if residual is not None else x, w, rstd)
        if residual is None:
            return y
        return y, h

    @staticmethod
    def backward(ctx, dy, dh=None):
        if dy is None and dh is None:
            return (None,) * 6
        saved = _saved(ctx)
        with torch.no_grad():
            dx, dw = _RMSNorm.gradients(ctx, saved, dy, dh)
        need_x, need_r = ctx.needs_input_grad[0], ctx.has_residual and ctx.needs_input_grad[1]
        h = saved[0] if need_x or need_r else None      # it is an output as well, and asks for gradients whatever the inputs do
        dx = _once("rms_norm", dx, dy, dh, h, saved[1])
        return dx if need_x else None, dx if need_r else None, _once("rms_norm", dw, dy, h), None, None, None

    @staticmethod
    def gradients(ctx, saved, dy, dh):
        h, (w, rstd) = saved[0], map(_whole, saved[1:])
        rows, d, wcode = ctx.sizes
        need_x = ctx.needs_input_grad[0] or (ctx.has_residual and ctx.needs_input_grad[1])
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if w is not None and ctx.needs_input_grad[2] else None
        dy = _whole(dy) if dy is not None else torch.zeros(h.shape, dtype=h.dtype, device=h.device)
        dh = _whole(dh)
        h2, hs = _rows(h, rows, d)
        dx = torch.empty(h.shape, dtype=h.dtype, device=h.device) if need_x else None
        lib = _lib.load()
        with torch.cuda.device(h.device):
            nbytes = lib.adder_b200_rmsnorm_backward_workspace_bytes(rows, d) if dw is not None else 0
            ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device) if nbytes else None
            _lib.check(lib.adder_b200_rmsnorm_backward(
                dy.data_ptr(), _ptr(dh), h2.data_ptr(), _ptr(w), rstd.data_ptr(), _ptr(dx), _ptr(dw), _ptr(ws), nbytes, rows, d, hs,
                _lib.TYPE_CODES[h.dtype], wcode, adder_cuda._stream(h.device)), "adder_b200_rmsnorm_backward")
        return dx, dw


def _check_call(x, shape, weight, eps, residual) -> None:
    _check_input(x, "x")
    if not shape or x.dim() < len(shape) or tuple(x.shape[x.dim() - len(shape):]) != shape or math.prod(shape) == 0:
        raise ValueError(f"x has shape {tuple(x.shape)}, whose last axes are not {shape}")
    if residual is not None:
        _check_input(residual, "residual", x.device)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual must have the shape and type of x: {tuple(residual.shape)} {residual.dtype}, "
                             f"expected {tuple(x.shape)} {x.dtype}")
    if weight is not None:
        _check_input(weight, "weight", x.device)
        if tuple(weight.shape) != shape:
            raise ValueError(f"weight has shape {tuple(weight.shape)}, expected {shape}")
        if weight.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"weight must be {x.dtype} or float32, got {weight.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")


def rms_norm(x: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last axes, which are `normalized_shape`.

    Without `residual` h is x, and y is returned.  With it h = x + residual, rounded to the type of both, and (y, h) is returned.
    `weight` has the shape `normalized_shape` and x's type or float32.  x and residual may be any views; those whose rows are not
    consecutive are copied.  Differentiable once, with respect to x, residual and weight: a gradient of create_graph=True raises where
    it is differentiated.  At most 2^28 - 1 rows of at most 2^30 - 2^16 elements."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    out = _native.rms_norm(x, residual, weight, shape, eps)
    if out is not None:
        return out
    _check_call(x, shape, weight, eps, residual)
    needs_grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight))
    return _RMSNorm.apply(x, residual, weight, shape, float(eps), needs_grad)


def rms_norm_8bit(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """`rms_norm` over the last axis with y in 8 bits: a `linear8.Rows8`, or with `residual` (Rows8, h).

    The codes are those of the norm before any rounding to 16 bits.  128 columns with a NaN or an infinity stand for NaN.  It has no
    gradient, and raises where one would be recorded."""
    out = _native.rms_norm_8bit(x, weight, eps, residual)
    if out is not None:
        return Rows8(*out[:2]) if residual is None else (Rows8(*out[:2]), out[2])
    _check_call(x, tuple(x.shape[-1:]) if isinstance(x, torch.Tensor) else (), weight, eps, residual)
    _refuse_gradient("rms_norm_8bit", x, residual, weight)
    out = _recorded(_norm_8bit, x, weight, float(eps), residual)
    return Rows8(*out[:2]) if residual is None else (Rows8(*out[:2]), out[2])


def _norm_8bit(x, weight, eps, residual):
    rows, d = _sizes(x, x.shape[-1:])
    dev = x.device
    x2, xs = _rows(x, rows, d)
    r2, rs = _rows(residual, rows, d) if residual is not None else (None, 0)
    out, stride = _empty_rows(x.shape, dev)
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if residual is not None else None
    w = _whole(weight)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().adder_b200_rmsnorm_forward_8bit(
            x2.data_ptr(), _ptr(r2), _ptr(w), out.values.data_ptr(), out.scales.data_ptr(), _ptr(h), rows, d, xs, rs, stride,
            _lib.TYPE_CODES[x.dtype], _lib.TYPE_CODES[(w if w is not None else x).dtype], eps, adder_cuda._stream(dev)),
            "adder_b200_rmsnorm_forward_8bit")
    return tuple(out) if residual is None else (*out, h)


class FusedRMSNorm(nn.RMSNorm):
    """nn.RMSNorm with `forward(x, residual=None, eight=False)`: with a residual it returns (norm of x + residual, x + residual), with
    `eight` the norm in 8 bits (over one axis).  Same parameters and state-dict keys; an eps of None is float32's, in which 16-bit types are
    computed, too, as there.  CPU tensors go through torch, and have no 8 bits."""

    def forward(self, x, residual=None, eight: bool = False):
        if x.is_cuda or eight:
            eps = torch.finfo(torch.float32).eps if self.eps is None else self.eps
            if not eight:
                return rms_norm(x, self.normalized_shape, self.weight, eps, residual=residual)
            if len(self.normalized_shape) != 1 or x.shape[-1:] != self.normalized_shape:
                raise ValueError(f"the norm in 8 bits is over the last axis alone, which is not {tuple(self.normalized_shape)}")
            return rms_norm_8bit(x, self.weight, eps, residual=residual)
        if residual is None:
            return super().forward(x)
        h = x + residual
        return super().forward(h), h

"""Products in 8 bits for inference: e4m3 codes with fp32 scales, on the fp8 tensor cores.

Rows (activations) have a scale for each 128 columns, a weight one for each 128 x 128; a value is code * scale.  `quantize_rows`,
`rmsnorm.rms_norm_8bit` and `quantize_weight` bring tensors to that form, `linear_8bit` multiplies them, `Linear8bit` is the layer around
it, which `inference.quantize_linear` puts in place of a network's multiply-based linear layers.

Codes: with a the largest magnitude of a block, scale = a * (1 / 448) and code = e4m3(value * (1 / a * 448)), each operation rounded to
fp32, the code to nearest even.  Blocks whose largest magnitude is below 2^-100 are zeros, blocks with a NaN or an infinity stand for NaN.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
import torch.nn as nn
from torch.autograd.forward_ad import unpack_dual

from . import _lib, _native, adder_cuda
from .layernorm import _check_input, _ptr, _recorded, _rows, _whole

BLOCK = 128


class Rows8(NamedTuple):
    """Rows in 8 bits: values float8_e4m3fn [..., columns], scales float32 [..., ceil(columns / 128)]."""
    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What the codes stand for."""
        return (self.values.float() * self.scales.repeat_interleave(BLOCK, -1)[..., :self.values.shape[-1]]).to(dtype)


class Weight8(NamedTuple):
    """A weight in 8 bits: values float8_e4m3fn [rows, columns], scales float32 [ceil(rows / 128), ceil(columns / 128)]."""
    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What the codes stand for."""
        rows, columns = self.values.shape
        scales = self.scales.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :columns]
        return (self.values.float() * scales).to(dtype)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _codes(lead, n: int, dev):
    """(codes [*lead, n] whose rows begin at multiples of 16 bytes, elements from row to row)."""
    stride = -(-n // 16) * 16
    whole = torch.empty((*lead, stride), dtype=torch.float8_e4m3fn, device=dev)
    return (whole if stride == n else whole[..., :n]), stride


def _empty_rows(shape, dev):
    values, stride = _codes(shape[:-1], shape[-1], dev)
    return Rows8(values, torch.empty((*shape[:-1], _blocks(shape[-1])), device=dev)), stride


def _refuse_gradient(name: str, *tensors) -> None:
    """Raise where a derivative of an operator that has none would be recorded, backward or forward."""
    for t in tensors:
        if t is None:
            continue
        if torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")
        if unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no gradient in forward mode either: give it the primal of a dual tensor")


def _to_8bit(name: str, x: torch.Tensor, weight: bool):
    _check_input(x, "w" if weight else "x")
    if (x.dim() != 2 if weight else x.dim() < 1) or x.shape[-1] == 0:
        raise ValueError(f"{name} takes {'a matrix' if weight else 'rows'} of at least one column, got shape {tuple(x.shape)}")
    _refuse_gradient(name, x)
    return _recorded(_convert, name, x, weight)


def _convert(name: str, x: torch.Tensor, weight: bool):
    d = x.shape[-1]
    rows = x.numel() // d
    values, stride = _codes(x.shape[:-1], d, x.device)
    lead = (_blocks(x.shape[0]),) if weight else x.shape[:-1]
    scales = torch.empty((*lead, _blocks(d)), device=x.device)
    x2, xs = _rows(x, rows, d)
    lib = _lib.load()
    with torch.cuda.device(x.device):
        entry = lib.adder_b200_quantize_weight if weight else lib.adder_b200_quantize_rows
        _lib.check(entry(x2.data_ptr(), values.data_ptr(), scales.data_ptr(), rows, d, xs, stride, _lib.TYPE_CODES[x.dtype],
                         adder_cuda._stream(x.device)), f"adder_b200_{name}")
    return values, scales


def quantize_rows(x: torch.Tensor) -> Rows8:
    """x [..., columns] (float32, bfloat16 or float16 on CUDA) in 8 bits, a scale for each 128 columns of a row.  No gradient."""
    return Rows8(*_to_8bit("quantize_rows", x, False))


def quantize_weight(w: torch.Tensor) -> Weight8:
    """w [rows, columns] in 8 bits, a scale for each 128 x 128.  No gradient."""
    return Weight8(*_to_8bit("quantize_weight", w, True))


def _check_8bit(t, name: str, kind, dev=None) -> None:
    values, scales = t
    for part, what, dtype in ((values, "values", torch.float8_e4m3fn), (scales, "scales", torch.float32)):
        if not isinstance(part, torch.Tensor):
            raise TypeError(f"{name}.{what} must be a torch.Tensor")
        if not part.is_cuda:
            raise RuntimeError(f"{name}.{what} must be a CUDA tensor")
        if part.device != (dev if dev is not None else values.device):
            raise RuntimeError(f"tensors are on different devices ({dev if dev is not None else values.device} and {part.device})")
        if part.dtype != dtype:
            raise TypeError(f"{name}.{what} must be {dtype}, got {part.dtype}")
    if (values.dim() != 2 if kind is Weight8 else values.dim() < 1) or values.shape[-1] == 0:
        raise ValueError(f"{name}.values has shape {tuple(values.shape)}")
    lead = (_blocks(values.shape[0]),) if kind is Weight8 else tuple(values.shape[:-1])
    if tuple(scales.shape) != (*lead, _blocks(values.shape[-1])):
        raise ValueError(f"{name}.scales has shape {tuple(scales.shape)}, expected {(*lead, _blocks(values.shape[-1]))}")


def _aligned(values: torch.Tensor):
    """(codes, elements from row to row), copied only where the rows do not begin at multiples of 16 bytes."""
    d = values.shape[-1]
    rows = values.numel() // d
    v, stride = _rows(values, rows, d)
    if rows <= 1:
        stride = -(-d // 16) * 16
    if v.data_ptr() % 16 == 0 and stride % 16 == 0 and stride >= d:
        return v, stride
    out, stride = _codes((rows,), d, values.device)
    out.view(torch.uint8).copy_(v.reshape(rows, d).view(torch.uint8))
    return out, stride


def _padded(values: torch.Tensor) -> torch.Tensor:
    """The same codes [rows, columns], laid out as `_codes` does."""
    if values.shape[0] <= 1 or values.stride() == (-(-values.shape[1] // 16) * 16, 1):
        return values
    out, _ = _codes(values.shape[:1], values.shape[1], values.device)
    out.view(torch.uint8).copy_(values.contiguous().view(torch.uint8))
    return out


def linear_8bit(x: Union[torch.Tensor, Rows8], weight: Weight8, bias: Optional[torch.Tensor] = None,
                dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x @ weight.T + bias with both factors in 8 bits: [..., weight rows] of `dtype`.

    x is a `Rows8`, or a float32, bfloat16 or float16 tensor [..., columns], which goes through `quantize_rows`; `dtype` (float32, bfloat16
    or float16) is x's own type where it is None, bfloat16 for a Rows8.  `bias` [weight rows] has the type `dtype`.  Sums are fp32: each
    128 columns' sum of code products is multiplied by its two scales (their product in fp32, which loses bits below 2^-126 and ends at 2^128)
    and added up, and the result is rounded once.  Codes whose
    rows do not begin at multiples of 16 bytes are copied, at every call; those of this module's functions do.  No gradient."""
    if not isinstance(weight, Weight8):
        raise TypeError(f"weight must be a Weight8, got {type(weight).__name__}")
    out = _native.linear_8bit(x, weight, bias, dtype)
    if out is not None:
        return out
    if not isinstance(x, Rows8):
        _check_input(x, "x")
        dtype = x.dtype if dtype is None else dtype
    elif dtype is None:
        dtype = torch.bfloat16
    if dtype not in _lib.TYPE_CODES:
        raise TypeError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    _check_8bit(weight, "weight", Weight8)
    dev = weight.values.device
    n, k = weight.values.shape
    if isinstance(x, Rows8):
        _check_8bit(x, "x", Rows8, dev)
    elif x.device != dev:
        raise RuntimeError(f"tensors are on different devices ({dev} and {x.device})")
    lead = x.values.shape if isinstance(x, Rows8) else x.shape
    if len(lead) < 1 or lead[-1] != k:
        raise ValueError(f"x has shape {tuple(lead)}, expected {k} columns")
    if bias is not None:
        _check_input(bias, "bias", dev)
        if bias.shape != (n,) or bias.dtype != dtype:
            raise ValueError(f"bias must have shape {(n,)} and type {dtype}, got {tuple(bias.shape)} {bias.dtype}")
    _refuse_gradient("linear_8bit", *(x if isinstance(x, Rows8) else (x,)), *weight, bias)
    if not isinstance(x, Rows8):
        x = quantize_rows(x)
    return _recorded(_product, *x, *weight, bias, dtype)


def _product(x, x_scales, weight, weight_scales, bias, dtype):
    (n, k), dev = weight.shape, weight.device
    xv, xstride = _aligned(x)
    wv, wstride = _aligned(weight)
    xs, ws, b = _whole(x_scales), _whole(weight_scales), _whole(bias)
    y = torch.empty((*x.shape[:-1], n), dtype=dtype, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().adder_b200_linear_8bit(
            xv.data_ptr(), xs.data_ptr(), wv.data_ptr(), ws.data_ptr(), _ptr(b), y.data_ptr(), y.numel() // n if n else 0, k, n, xstride, wstride,
            _lib.TYPE_CODES[dtype], adder_cuda._stream(dev)), "adder_b200_linear_8bit")
    return y


class Linear8bit(nn.Module):
    """A linear layer with its weight in 8 bits, for inference: `Linear8bit(linear)` of an nn.Linear on CUDA, or of a 1x1 nn.Conv2d (stride
    1, no padding, one group), whose input and output then are [N, C, H, W] or [C, H, W], the output in the input's memory format.  The input of
    an nn.Linear's may be a `Rows8`, as `rmsnorm.rms_norm_8bit` gives it.  The output has the type `dtype`, where it is None the input's,
    bfloat16 for a Rows8, and carries no gradient, whatever the input asks for.  There is no `weight`: the codes are `values` and `scales`."""

    def __init__(self, layer: nn.Module):
        super().__init__()
        self.check(layer)
        self.convolution = isinstance(layer, nn.Conv2d)
        weight = layer.weight.detach().flatten(1)
        self.out_features, self.in_features = weight.shape
        values, scales = quantize_weight(weight)
        self.register_buffer("values", values)
        self.register_buffer("scales", scales)
        self.register_buffer("bias", None if layer.bias is None else layer.bias.detach().to(torch.float32, copy=True))

    @staticmethod
    def check(layer: nn.Module) -> None:
        """Raise for what cannot be put in 8 bits."""
        if isinstance(layer, nn.Conv2d):
            if layer.kernel_size != (1, 1) or layer.stride != (1, 1) or layer.padding not in ((0, 0), "valid") or layer.groups != 1:
                raise ValueError("only convolutions of kernel size 1, stride 1 and one group without padding are linear layers")
        elif not isinstance(layer, nn.Linear):
            raise TypeError(f"layer must be an nn.Linear or an nn.Conv2d, got {type(layer).__name__}")
        _check_input(layer.weight, "the layer's weight")
        if layer.weight.shape[1] == 0:
            raise ValueError(f"the layer's weight has shape {tuple(layer.weight.shape)}")

    def _apply(self, fn, recurse=True):
        # a module's .half(), .float() and the like are for parameters: what is held here keeps its types, and follows to a device alone
        kept = dict(self._buffers)
        super()._apply(fn, recurse)
        for name, t in kept.items():
            if t is not None and self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        self._buffers["values"] = _padded(self._buffers["values"])
        return self

    def forward(self, x, dtype: Optional[torch.dtype] = None):
        if isinstance(x, Rows8):
            if self.convolution:
                raise TypeError("a convolution's layer takes images [N, C, H, W], not rows in 8 bits")
            dtype = torch.bfloat16 if dtype is None else dtype
        elif dtype is None:
            dtype = x.dtype
        channels_last = False
        if self.convolution:
            if x.dim() not in (3, 4):
                raise ValueError(f"a convolution's layer takes images [N, C, H, W] or [C, H, W], got shape {tuple(x.shape)}")
            channels_last = x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last)
            x = x.movedim(-3, -1)
        bias = None if self.bias is None else self.bias.to(dtype)
        with torch.no_grad():
            y = linear_8bit(x, Weight8(self.values, self.scales), bias, dtype)
        if not self.convolution:
            return y
        y = y.movedim(-1, -3)
        return y if channels_last else y.contiguous()      # in the input's order, as nn.Conv2d gives it

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"

"""AdamW over all tensors of a model in one kernel, with states in 32 bits or in 8.

`adamw_step` is one step over lists of tensors, `AdamW` the torch.optim.Optimizer around it.  Unlike the SGD of the reference's
training loop (main.py:86-101) it counts its steps on the device, so that a step can sit in a captured CUDA graph, and its launch
holds the addresses of all tensors, so that a model of any number of tensors costs one launch.

With `state_bits=8` a block of 256 values of a state is held as one byte a value and one fp32 scale (1.02 bytes a value in place of 4):
the first moment with 3 exponent bits, 4 fraction bits and a sign, the second with 4 and 4.  What lies below half a step of its code is
lost when a state is stored, so a second moment whose beta2 is near 1 follows a falling gradient late; 0.95 to 0.99 suit it better
than 0.999.  Tensors below `min_8bit_size` elements keep 32 bits.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import torch

from . import _lib, _native, adder_cuda

BLOCK = 256       # consecutive values (in memory order) that share a scale


class _Tensor(ctypes.Structure):
    """adder_b200_adamw_tensor of the C interface."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step")] + \
               [("n", ctypes.c_longlong)]


def scale_count(n: int) -> int:
    """Scales of an 8-bit state of n values."""
    return -(-n // BLOCK)


def _strides(t: torch.Tensor):
    """Strides of the extents that have more than one element: what decides where an element lies."""
    return tuple(s for s, n in zip(t.stride(), t.shape) if n > 1)


def _is_dense(t: torch.Tensor) -> bool:
    """The elements fill a stretch of memory, in whatever order of the extents."""
    want = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s != want:
            return False
        want *= n
    return True


def _check(t, name: str, dev, dtype, like=None, numel=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.layout != torch.strided:
        raise TypeError(f"{name} must be a dense tensor, got layout {t.layout}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.device != dev:
        raise RuntimeError(f"tensors are on different devices ({dev} and {t.device})")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.is_neg() and not name.startswith("grads"):
        raise ValueError(f"{name} must not be a lazily negated view")
    if like is not None and (t.shape != like.shape or _strides(t) != _strides(like)):
        raise ValueError(f"{name} must have the shape and strides of its parameter: {tuple(t.shape)} {t.stride()}, "
                         f"expected {tuple(like.shape)} {like.stride()}")
    if numel is not None and (t.numel() != numel or not t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous with {numel} elements, got {tuple(t.shape)}")


def _scalar(v, name: str, dev):
    """(host value, device pointer) of a number, or of an fp32 tensor of one element."""
    if isinstance(v, torch.Tensor):
        if not v.is_cuda:
            return float(v), None
        _check(v, name, dev, torch.float32, numel=1)
        return 0.0, v.data_ptr()
    return float(v), None


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], steps: Union[torch.Tensor, Sequence[torch.Tensor]], *,
               lr: Union[float, torch.Tensor] = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None, exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
               grad_scale: Optional[torch.Tensor] = None) -> None:
    """One AdamW step, in place, on tensors of one device:

        g = grad * grad_scale;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

    `params` are float32, bfloat16 or float16 (a mixed list takes one launch a type), dense in any order of their extents; each of
    `grads` has its parameter's type and shape (other strides are copied to the parameter's first).  `steps` is an int32 tensor
    [n, 2], or n int32 tensors of two elements: the steps that each parameter has taken, counted up by the call, and a word that is 0
    between calls.  States are float32 with the strides of their parameters, or, where scales are given, uint8 codes with
    `scale_count(numel)` float32 scales (zeros of both are a state of zeros).  `lr` and `grad_scale` may be float32 CUDA tensors of
    one element, read when the kernel runs.  `eps` is 0 or at least 2^-126.  No two of the tensors that are written may share memory: tensors that
    start at the same address are refused, other overlaps are not looked for.  The whole step runs on the current stream."""
    if _native.adamw(params, grads, exp_avgs, exp_avg_sqs, steps, lr, betas[0], betas[1], eps, weight_decay, exp_avg_scales,
                     exp_avg_sq_scales, grad_scale):
        return
    n = len(params)
    eight = exp_avg_scales is not None
    if eight != (exp_avg_sq_scales is not None):
        raise ValueError("exp_avg_scales and exp_avg_sq_scales go together")
    lists = [("grads", grads), ("exp_avgs", exp_avgs), ("exp_avg_sqs", exp_avg_sqs), ("steps", steps)]
    if eight:
        lists += [("exp_avg_scales", exp_avg_scales), ("exp_avg_sq_scales", exp_avg_sq_scales)]
    for name, values in lists:
        if len(values) != n:
            raise ValueError(f"{name} has {len(values)} tensors, params {n}")
    if n == 0:
        return
    if not isinstance(params[0], torch.Tensor) or not params[0].is_cuda:
        raise RuntimeError("params must be CUDA tensors")
    dev = params[0].device
    state_type = torch.uint8 if eight else torch.float32
    by_type: dict = {}
    written: set = set()
    kept = []             # gradients in another layout, alive until the launch
    for i in range(n):
        p, g = params[i], grads[i]
        _check(p, f"params[{i}]", dev, getattr(p, "dtype", None))
        if p.dtype not in _lib.TYPE_CODES:
            raise TypeError(f"params[{i}] must be float32, bfloat16 or float16, got {p.dtype}")
        if not _is_dense(p):
            raise ValueError(f"params[{i}] must fill its memory (strides {p.stride()} of shape {tuple(p.shape)})")
        _check(g, f"grads[{i}]", dev, p.dtype)
        if g.shape != p.shape:
            raise ValueError(f"grads[{i}] has shape {tuple(g.shape)}, expected {tuple(p.shape)}")
        if _strides(g) != _strides(p) or g.is_neg():
            g = torch.empty_like(p).copy_(g)
            kept.append(g)
        _check(exp_avgs[i], f"exp_avgs[{i}]", dev, state_type, like=p)
        _check(exp_avg_sqs[i], f"exp_avg_sqs[{i}]", dev, state_type, like=p)
        _check(steps[i], f"steps[{i}]", dev, torch.int32, numel=2)
        scales = (None, None)
        if eight:
            scales = (exp_avg_scales[i], exp_avg_sq_scales[i])
            for name, s in zip(("exp_avg_scales", "exp_avg_sq_scales"), scales):
                _check(s, f"{name}[{i}]", dev, torch.float32, numel=scale_count(p.numel()))
        if p.numel() == 0:
            continue
        out = [t.data_ptr() for t in (p, exp_avgs[i], exp_avg_sqs[i], steps[i], *scales) if t is not None]
        if len(set(out)) != len(out) or not written.isdisjoint(out):
            raise ValueError(f"params[{i}], its states or its step count are also those of another parameter")
        written.update(out)
        by_type.setdefault(p.dtype, []).append(_Tensor(
            p.data_ptr(), g.data_ptr(), exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr(),
            scales[0].data_ptr() if eight else None, scales[1].data_ptr() if eight else None, steps[i].data_ptr(), p.numel()))
    for group in by_type.values():
        for i, t in enumerate(group):
            if t.grad in written:
                raise ValueError("a gradient is also a parameter, a state or a step count")
    lr_value, lr_ptr = _scalar(lr, "lr", dev)
    if grad_scale is not None:
        if not isinstance(grad_scale, torch.Tensor):
            raise TypeError("grad_scale must be a float32 CUDA tensor of one element")
        _check(grad_scale, "grad_scale", dev, torch.float32, numel=1)
    lib = _lib.load()
    with torch.cuda.device(dev):
        for dtype, group in by_type.items():
            _lib.check(lib.adder_b200_adamw_step(
                (_Tensor * len(group))(*group), len(group), _lib.TYPE_CODES[dtype], 8 if eight else 32, lr_value, lr_ptr,
                float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
                grad_scale.data_ptr() if grad_scale is not None else None, adder_cuda._stream(dev)), "adder_b200_adamw_step")
    torch.autograd.graph.increment_version([t for ts in (params, exp_avgs, exp_avg_sqs) for t in ts if not t.is_inference()])


def adamw_state_values(codes: torch.Tensor, scales: torch.Tensor, signed: bool) -> torch.Tensor:
    """What an 8-bit state stands for, as float32 in the shape and memory order of `codes` (`signed`: a first moment, else a second)."""
    _check(codes, "codes", getattr(codes, "device", None), torch.uint8)
    if not _is_dense(codes):
        raise ValueError("codes must fill their memory")
    _check(scales, "scales", codes.device, torch.float32, numel=scale_count(codes.numel()))
    values = torch.empty_like(codes, dtype=torch.float32)
    with torch.cuda.device(codes.device):
        _lib.check(_lib.load().adder_b200_adamw_state_values(codes.data_ptr(), scales.data_ptr(), int(signed), values.data_ptr(),
                                                             codes.numel(), adder_cuda._stream(codes.device)),
                   "adder_b200_adamw_state_values")
    return values


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update on this library's kernel (CUDA parameters of float32, bfloat16 or float16; no amsgrad, no maximize).

    `state_bits=8` holds the states of tensors of `min_8bit_size` elements and more in 8 bits.  `lr` may be a float32 CUDA tensor of
    one element, so that a captured step follows a schedule.  `step(grad_scale=...)` multiplies all gradients by one device value (an
    unscaling or a clipping factor) on their way in.  A parameter's states are made at its first step, which therefore cannot be
    captured into a CUDA graph."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 min_8bit_size: int = 4096):
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"invalid learning rate: {lr}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"invalid betas: {betas}")
        if not (eps == 0.0 or eps >= 2.0 ** -126) or not weight_decay >= 0.0:
            raise ValueError(f"invalid eps or weight_decay: {eps}, {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size))

    def _init_state(self, group, fresh) -> None:
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a parameter's first step makes its states and cannot be captured: run a step before the capture")
        for p in fresh:
            if not p.is_cuda or p.dtype not in _lib.TYPE_CODES:
                raise RuntimeError(f"parameters must be float32, bfloat16 or float16 CUDA tensors, got {p.dtype} on {p.device}")
            eight = group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]
            s = self.state[p]
            s["step"] = torch.zeros(2, dtype=torch.int32, device=p.device)
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.zeros_like(p, dtype=torch.uint8 if eight else torch.float32, requires_grad=False)
                if eight:
                    s[name + "_scale"] = torch.zeros(scale_count(p.numel()), device=p.device)

    @torch.no_grad()
    def step(self, closure=None, grad_scale: Optional[torch.Tensor] = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            with_grad = [p for p in group["params"] if p.grad is not None]
            fresh = [p for p in with_grad if not self.state[p]]
            if fresh:
                self._init_state(group, fresh)
            calls: dict = {}
            for p in with_grad:
                calls.setdefault((p.device, "exp_avg_scale" in self.state[p]), []).append(p)
            for (_, eight), ps in calls.items():
                states = [self.state[p] for p in ps]
                adamw_step(ps, [p.grad for p in ps], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                           [s["step"] for s in states], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"],
                           exp_avg_scales=[s["exp_avg_scale"] for s in states] if eight else None,
                           exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states] if eight else None, grad_scale=grad_scale)
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As torch.optim.Optimizer's, but states keep their own types: torch would cast them to the parameter's."""
        super().load_state_dict(state_dict)
        given = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(given, own):
            saved = state_dict["state"].get(i)
            if not saved:
                continue
            state = {k: v.detach().to(p.device, copy=True) if isinstance(v, torch.Tensor) else v for k, v in saved.items()}
            for name in ("exp_avg", "exp_avg_sq"):
                if _strides(state[name]) != _strides(p):
                    if state[name].dtype == torch.uint8:
                        raise ValueError("8-bit states lie in the memory order of their parameter, which is another one here")
                    state[name] = torch.empty_like(p, dtype=torch.float32).copy_(state[name])
            self.state[p] = state

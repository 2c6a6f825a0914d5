"""Distillation of a network from a teacher's top logits, forward and backward.

A teacher's best classes of each row (`logprobs.token_log_probs(..., top_k=k)` gives them with their log probabilities, which serve as
logits) take some hundred bytes a row where its logits take hundreds of kilobytes, so they can be kept or sent.  `distillation` reads the
network's logits once for the divergence of its classes from the teacher's and, at temperature 1, the log probability of the label;
its backward reads them once more and writes their gradient.  `DistillationLoss` is the loss of both, beside
`logprobs.TokenCrossEntropy`; `train.TrainStep` takes it with a teacher.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import _lib, _native, adder_cuda
from .drafts import _check_whole
from .layernorm import _check_input, _once, _ptr, _rows, _save, _saved, _whole

MAX_TOP = 256


class Distillation(NamedTuple):
    """What `distillation` returns."""
    divergence: torch.Tensor                 # float32 [...]
    log_prob: Optional[torch.Tensor]         # float32 [...], with targets


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, indices, temperature, targets, ignore_index, needs_grad):
        v, k = logits.shape[-1], indices.shape[-1]
        lead = logits.shape[:-1]
        rows = logits.numel() // v
        dev = logits.device
        x, stride = _rows(logits, rows, v)
        divergence = torch.empty(lead, device=dev)
        lp = torch.empty(lead, device=dev) if targets is not None else None
        stats = torch.empty((rows, 3), device=dev) if needs_grad else None
        mass = torch.empty((rows, k), device=dev) if needs_grad else None
        with torch.cuda.device(dev):
            _lib.check(_lib.load().adder_b200_distillation_forward(
                x.data_ptr(), _lib.TYPE_CODES[logits.dtype], rows, v, stride, teacher.data_ptr(), _lib.TYPE_CODES[teacher.dtype],
                indices.data_ptr(), k, temperature, _ptr(targets), ignore_index, divergence.data_ptr(), _ptr(lp), _ptr(stats), _ptr(mass),
                adder_cuda._stream(dev)), "adder_b200_distillation_forward")
        ctx.args = (temperature, ignore_index)
        ctx.set_materialize_grads(False)
        if needs_grad:
            _save(ctx, logits, indices, targets, stats, mass)
        return divergence, lp

    @staticmethod
    def backward(ctx, g_div, g_lp):
        if g_div is None and g_lp is None:
            return (None,) * 7
        saved = _saved(ctx)
        with torch.no_grad():
            dx = _Distillation.gradient(ctx, saved, g_div, g_lp)
        return (_once("distillation", dx, saved[0], g_div, g_lp),) + (None,) * 6

    @staticmethod
    def gradient(ctx, saved, g_div, g_lp):
        logits, (indices, targets, stats, mass) = saved[0], map(_whole, saved[1:])
        temperature, ignore_index = ctx.args
        v = logits.shape[-1]
        rows = logits.numel() // v
        x, stride = _rows(logits, rows, v)
        g_div, g_lp = _whole(g_div), _whole(g_lp)
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with torch.cuda.device(logits.device):
            _lib.check(_lib.load().adder_b200_distillation_backward(
                x.data_ptr(), _lib.TYPE_CODES[logits.dtype], rows, v, stride, indices.data_ptr(), indices.shape[-1], temperature, _ptr(targets),
                ignore_index, stats.data_ptr(), mass.data_ptr(), _ptr(g_div), _ptr(g_lp), dx.data_ptr(), adder_cuda._stream(logits.device)),
                "adder_b200_distillation_backward")
        return dx


def distillation(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_indices: torch.Tensor, temperature: float = 1.0,
                 targets: Optional[torch.Tensor] = None, ignore_index: int = -100) -> Distillation:
    """How far the classes of `logits` [..., classes] (float32, bfloat16 or float16) are from a teacher's best ones.

      divergence   sum of t (log t - log p) over the classes `teacher_indices` [..., k] (int64 or int32, k at most 256), with
                   t = softmax(teacher_logits / temperature) over those k alone and p = softmax(logits / temperature) over all classes
      log_prob     log softmax(logits) at `targets` [...] (int64 or int32), at temperature 1: 0 where the target is `ignore_index`, NaN where
                   it is no class; None without targets

    Both are float32 and differentiable once with respect to the logits (a gradient of create_graph=True raises where it is
    differentiated); the teacher gets no gradient, and raises where it asks for one.  `teacher_logits` [..., k] are of any of the three types and
    need no common offset, so log probabilities will do.  An index of -1 is an empty place; a row without any has divergence 0.  A class
    named twice has both shares.  A row with an index that is no class, or with a NaN or +inf, gives NaN, and so does a NaN of the teacher's
    at an empty place: `token_log_probs` names no class in a row that has failed.  The divergence is +inf where the teacher names a class
    whose logit is -inf.  A row whose divergence has a gradient of 0 takes nothing of the teacher's.  Logits may be a view such as
    [..., :classes] of a padded buffer; views whose rows are not consecutive are copied.  The gradient of such a view takes two to three
    times as long as that of dense rows, unless row stride and classes differ by a multiple of 16 bytes."""
    out = _native.distillation(logits, teacher_logits, teacher_indices, temperature, targets, ignore_index)
    if out is not None:
        return Distillation(*out)
    _check_input(logits, "logits")
    dev = logits.device
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"logits must have a last axis of classes, got shape {tuple(logits.shape)}")
    lead = tuple(logits.shape[:-1])
    _check_input(teacher_logits, "teacher_logits", dev)
    k = teacher_logits.shape[-1] if teacher_logits.dim() else 0
    if not 1 <= k <= MAX_TOP or tuple(teacher_logits.shape[:-1]) != lead:
        raise ValueError(f"teacher_logits have shape {tuple(teacher_logits.shape)}, expected {lead} and 1 to {MAX_TOP} classes")
    indices = _check_whole(teacher_indices, "teacher_indices", (*lead, k), dev)
    if torch.is_grad_enabled() and teacher_logits.requires_grad:
        raise RuntimeError("distillation has no gradient with respect to the teacher: detach its logits")
    temperature = float(temperature)
    if not (temperature > 0.0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    if targets is not None:
        targets = _check_whole(targets, "targets", lead, dev)
    needs_grad = torch.is_grad_enabled() and logits.requires_grad
    return Distillation(*_Distillation.apply(logits, _whole(teacher_logits), indices, temperature, targets, int(ignore_index), needs_grad))


class DistillationLoss(nn.Module):
    """alpha * temperature^2 * divergence + (1 - alpha) * cross entropy, the mean over the targets that are not `ignore_index`:
    forward(logits, targets, teacher_logits, teacher_indices).  A term of weight 0 is left out.  `top_k` (at most 32) is how many classes
    `train.TrainStep` asks of its teacher.  Computed and returned in float32."""

    def __init__(self, temperature: float = 1.0, alpha: float = 0.5, ignore_index: int = -100, top_k: int = 20):
        super().__init__()
        if not 0.0 <= alpha <= 1.0:
            raise ValueError(f"alpha must be between 0 and 1, got {alpha}")
        self.temperature = temperature
        self.alpha = alpha
        self.ignore_index = ignore_index
        self.top_k = top_k

    def forward(self, logits, targets, teacher_logits, teacher_indices):
        labels = self.alpha < 1.0      # a term of weight 0 is left out: it may be infinite
        r = distillation(logits, teacher_logits, teacher_indices, self.temperature, targets if labels else None, self.ignore_index)
        if not labels:
            _check_whole(targets, "targets", logits.shape[:-1], logits.device)
        counts = targets != self.ignore_index
        loss = 0.0
        if self.alpha > 0.0:
            loss = self.alpha * self.temperature ** 2 * torch.where(counts, r.divergence, 0.0)
        if labels:
            loss = loss - (1.0 - self.alpha) * r.log_prob
        return loss.sum() / counts.sum()

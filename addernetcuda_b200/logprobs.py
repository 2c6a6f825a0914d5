"""Log probabilities of given classes, entropy and the most probable classes of rows of logits, with their gradient.

`token_log_probs` reads the logits once, in whatever type they are (float32, bfloat16, float16), and computes in fp32; its backward
reads them once more and writes their gradient.  Nothing of the size of the logits is kept between the two but the logits themselves.
`TokenCrossEntropy` is the loss that the training loop of the reference takes from nn.CrossEntropyLoss (main.py:90) on top of
it, `inference.evaluate` counts accuracy, loss and entropy with it.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import _lib, _native, adder_cuda
from .layernorm import _check_input, _once, _ptr, _rows, _save, _saved, _whole

MAX_TOP_K = 32


class TokenLogProbs(NamedTuple):
    """What `token_log_probs` returns; what was not asked for is None."""
    log_prob: Optional[torch.Tensor]           # float32 [...]
    entropy: Optional[torch.Tensor]            # float32 [...]
    top_log_probs: Optional[torch.Tensor]      # float32 [..., top_k], descending
    top_indices: Optional[torch.Tensor]        # int64 [..., top_k]


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, entropy, ignore_index, needs_grad):
        v = logits.shape[-1]
        lead = logits.shape[:-1]
        rows = logits.numel() // v
        dev = logits.device
        x, stride = _rows(logits, rows, v)

        def out(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device=dev)

        lp = out(*lead) if targets is not None else None
        ent = out(*lead) if entropy else None
        stats = out(rows, 2) if needs_grad else None
        top = out(*lead, top_k) if top_k else None
        idx = out(*lead, top_k, dtype=torch.int64) if top_k else None
        with torch.cuda.device(dev):
            _lib.check(_lib.load().adder_b200_log_probs_forward(
                x.data_ptr(), _lib.TYPE_CODES[logits.dtype], rows, v, stride, _ptr(targets), ignore_index, top_k, _ptr(lp), _ptr(ent),
                _ptr(stats), _ptr(top), _ptr(idx), adder_cuda._stream(dev)), "adder_b200_log_probs_forward")
        ctx.args = (top_k, ignore_index)
        ctx.set_materialize_grads(False)
        if needs_grad:
            _save(ctx, logits, targets, stats, ent, idx)
        if idx is not None:
            ctx.mark_non_differentiable(idx)
        return lp, ent, top, idx

    @staticmethod
    def backward(ctx, g_lp, g_ent, g_top, _):
        if g_lp is None and g_ent is None and g_top is None:
            return (None,) * 6
        saved = _saved(ctx)
        with torch.no_grad():
            dx = _LogProbs.gradient(ctx, saved, g_lp, g_ent, g_top)
        return _once("token_log_probs", dx, saved[0], g_lp, g_ent, g_top), None, None, None, None, None

    @staticmethod
    def gradient(ctx, saved, g_lp, g_ent, g_top):
        logits, (targets, stats, ent, idx) = saved[0], map(_whole, saved[1:])
        top_k, ignore_index = ctx.args
        v = logits.shape[-1]
        rows = logits.numel() // v
        x, stride = _rows(logits, rows, v)
        g_lp, g_ent, g_top = map(_whole, (g_lp, g_ent, g_top))
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        with torch.cuda.device(logits.device):
            _lib.check(_lib.load().adder_b200_log_probs_backward(
                x.data_ptr(), _lib.TYPE_CODES[logits.dtype], rows, v, stride, _ptr(targets), ignore_index, top_k, _ptr(idx), stats.data_ptr(),
                _ptr(ent), _ptr(g_lp), _ptr(g_ent), _ptr(g_top), dx.data_ptr(), adder_cuda._stream(logits.device)),
                "adder_b200_log_probs_backward")
        return dx


def token_log_probs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top_k: int = 0, entropy: bool = False,
                    ignore_index: int = -100) -> TokenLogProbs:
    """Log softmax over the last axis of `logits` [..., classes] (float32, bfloat16 or float16), as far as it is asked for:

      log_prob      at `targets` [...] (int64 or int32): 0 where the target is `ignore_index`, NaN where it is no class;
      entropy       -sum p log p of each row, with `entropy=True`;
      top_log_probs, top_indices   of the `top_k` (at most 32) most probable classes, equal logits by index from the lowest.

    All but the indices are float32 and differentiable once with respect to the logits (a gradient of create_graph=True raises where it
    is differentiated).  -inf marks classes that are out; where none is left
    the log probabilities are -inf, the entropy and the gradient 0.  A row with a NaN or +inf gives NaN, and indices of -1.  Logits may be
    a view such as [..., :classes] of a padded buffer; views whose rows are not consecutive are copied.  The gradient of such a view takes two
    to four times as long as that of dense rows, unless row stride and classes differ by a multiple of 16 bytes."""
    out = _native.log_probs(logits, targets, top_k, entropy, ignore_index)
    if out is not None:
        return TokenLogProbs(*out)
    _check_input(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"logits must have a last axis of classes, got shape {tuple(logits.shape)}")
    if targets is not None:
        if not isinstance(targets, torch.Tensor):
            raise TypeError("targets must be a torch.Tensor")
        if targets.device != logits.device:
            raise RuntimeError(f"tensors are on different devices ({logits.device} and {targets.device})")
        if targets.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"targets must be int64 or int32, got {targets.dtype}")
        if targets.shape != logits.shape[:-1]:
            raise ValueError(f"targets have shape {tuple(targets.shape)}, expected {tuple(logits.shape[:-1])}")
        targets = _whole(targets.to(torch.int64))
    top_k = int(top_k)
    if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]):
        raise ValueError(f"top_k must be between 0 and {min(MAX_TOP_K, logits.shape[-1])}, got {top_k}")
    if targets is None and not top_k and not entropy:
        raise ValueError("nothing is asked for: give targets, top_k or entropy=True")
    needs_grad = torch.is_grad_enabled() and logits.requires_grad
    return TokenLogProbs(*_LogProbs.apply(logits, targets, top_k, bool(entropy), int(ignore_index), needs_grad))


class TokenCrossEntropy(nn.Module):
    """nn.CrossEntropyLoss of class indices on `token_log_probs`: logits [..., classes], targets [...], the mean (or, by `reduction`,
    sum, or each one) of -log p over the targets that are not `ignore_index`.  Computed and returned in float32."""

    def __init__(self, ignore_index: int = -100, reduction: str = "mean"):
        super().__init__()
        if reduction not in ("mean", "sum", "none"):
            raise ValueError(f"reduction must be mean, sum or none, got {reduction}")
        self.ignore_index = ignore_index
        self.reduction = reduction

    def forward(self, logits, targets):
        loss = -token_log_probs(logits, targets, ignore_index=self.ignore_index).log_prob
        if self.reduction == "none":
            return loss
        total = loss.sum()
        return total if self.reduction == "sum" else total / (targets != self.ignore_index).sum()

"""Verification of drafted tokens: how many of a draft stand against a target's probabilities, and the token that follows them.

A small model drafts a few tokens of a sequence, each drawn from its own probabilities; the target model gives its probabilities for all of
them in one pass.  `verify_drafts` keeps the longest run of drafts so that the result is distributed as the target's own samples are,
from random numbers that the caller gives, so that a call can be repeated.  It stands beside `logprobs.token_log_probs`, which scores given tokens.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib, _native, adder_cuda
from .layernorm import _check_input, _ptr, _recorded, _whole


class VerifiedDrafts(NamedTuple):
    """What `verify_drafts` returns."""
    tokens: torch.Tensor       # int64 [sequences, drafts + 1]: the accepted drafts, one more token, then -1
    accepted: torch.Tensor     # int64 [sequences]: how many drafts were accepted


def _check_whole(t, name: str, shape, dev) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device != dev:
        raise RuntimeError(f"tensors are on different devices ({dev} and {t.device})")
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be int64 or int32, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return _whole(t.to(torch.int64))


def _planes(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t [sequences, places, classes] with consecutive classes; a copy only where they are not."""
    if t is None:
        return None
    t = t.resolve_neg()
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def verify_drafts(target_probs: torch.Tensor, draft_probs: Optional[torch.Tensor], draft_tokens: torch.Tensor, uniforms: torch.Tensor,
                  lengths: Optional[torch.Tensor] = None) -> VerifiedDrafts:
    """Accept or refuse the drafted tokens of each sequence, and draw the token behind the accepted ones.

      target_probs  [sequences, drafts + 1, classes]  float32, bfloat16 or float16: the target's, one place more than there are drafts
      draft_probs   [sequences, drafts, classes], of the same type: those that the drafts were drawn from; None where the drafter was
                    certain of its tokens (copied text, the best class)
      draft_tokens  [sequences, drafts]  int64 or int32
      uniforms      [sequences, drafts + 1]  float32 in [0, 1): one for each draft, the last for the token that is drawn
      lengths       [sequences]  int64 or int32: drafts of each sequence where they are not all of them (clipped to 0 .. drafts)

    Draft i is accepted while uniforms[i] * draft_probs[i] < target_probs[i] at its token.  At the first refusal n the next token is drawn from
    max(target_probs[n] - draft_probs[n], 0) (without draft probabilities: from target_probs[n] without the refused token), and from
    target_probs[n] where all n drafts stand, or where nothing is left of the difference: the first class c of positive weight whose sum of
    weights up to c is above uniforms[drafts] times their whole sum.  Sums are taken in 64 bits.  Probabilities need not sum to 1; what is
    below 2^-126, NaN included, weighs nothing; a token that is no class is refused; where no class has a weight, or their sum is not finite
    in float32, -1 is drawn.  Places behind a sequence's length are not looked at, but for the one at it.  Without a gradient."""
    out = _native.verify_drafts(target_probs, draft_probs, draft_tokens, uniforms, lengths)
    if out is not None:
        return VerifiedDrafts(*out)
    _check_input(target_probs, "target_probs")
    dev = target_probs.device
    if target_probs.dim() != 3 or target_probs.shape[1] == 0 or target_probs.shape[2] == 0:
        raise ValueError(f"target_probs must be [sequences, drafts + 1, classes], got shape {tuple(target_probs.shape)}")
    b, places, classes = target_probs.shape
    if draft_probs is not None:
        _check_input(draft_probs, "draft_probs", dev)
        if draft_probs.dtype != target_probs.dtype or tuple(draft_probs.shape) != (b, places - 1, classes):
            raise ValueError(f"draft_probs must have shape {(b, places - 1, classes)} and type {target_probs.dtype}, got "
                             f"{tuple(draft_probs.shape)} {draft_probs.dtype}")
    tokens = _check_whole(draft_tokens, "draft_tokens", (b, places - 1), dev)
    _check_input(uniforms, "uniforms", dev)
    if uniforms.dtype != torch.float32 or tuple(uniforms.shape) != (b, places):
        raise ValueError(f"uniforms must be float32 of shape {(b, places)}, got {tuple(uniforms.shape)} {uniforms.dtype}")
    if lengths is not None:
        lengths = _check_whole(lengths, "lengths", (b,), dev)
    with torch.no_grad():
        return VerifiedDrafts(*_recorded(_verify, target_probs, draft_probs, tokens, uniforms, lengths))


def _verify(target_probs, draft_probs, tokens, uniforms, lengths):
    (b, places, classes), dev = target_probs.shape, target_probs.device
    p, q, u = _planes(target_probs), _planes(draft_probs), _whole(uniforms)
    tokens, lengths = _whole(tokens), _whole(lengths)
    out, accepted = torch.empty((b, places), dtype=torch.int64, device=dev), torch.empty(b, dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().adder_b200_verify_drafts(
            p.data_ptr(), _ptr(q), _lib.TYPE_CODES[p.dtype], tokens.data_ptr(), u.data_ptr(), _ptr(lengths), out.data_ptr(),
            accepted.data_ptr(), b, places - 1, classes, p.stride(0), p.stride(1), q.stride(0) if q is not None else 0,
            q.stride(1) if q is not None else 0, adder_cuda._stream(dev)), "adder_b200_verify_drafts")
    return out, accepted

"""Losses on logits with their gradients: log probabilities of the targets,
the clipped policy loss with a KL term, and the preference loss of paired log
ratios.

Logits are [batch, seq, vocab] (float32, bfloat16 or float16, any strides with
a unit last one); every statistic is FP32 or wider.  A token whose mask is
False is not looked at, whatever it holds: its log probability and gradient
are 0.  A live token's target outside the vocabulary makes its log probability
and gradient NaN.  The logits alone get gradients; advantages and recorded log
probabilities are constants.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native

__all__ = ["policy_loss", "preference_loss", "token_logprobs"]

REDUCTIONS = {"token": 0, "sequence": 1}


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """log softmax(logits)[target] of every live token, [batch, seq] float32:
    what an old or reference policy is recorded as."""
    return _native.torch_ops().token_logprobs(logits, targets, mask)


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, advantages: torch.Tensor, *,
                old_logprobs: Optional[torch.Tensor] = None, ref_logprobs: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, reduction: str = "token",
                scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, logprobs): the clipped policy loss with a KL term.

    With lp the log probability of a live token's target, r = exp(lp - old)
    (old = lp, r = 1, without old_logprobs), A its advantage and g = ref - lp:

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(g) - g - 1)

    averaged over the live tokens ("token") or over the sequences of their
    means ("sequence"), times `scale`; 0 where no token is live.  advantages:
    [batch] or [batch, seq].  logprobs is lp, not differentiable.

    The gradient to float32 and bfloat16 logits is made in the pass that reads
    them.  Backward of another factor than 1 costs a pass over it and a second
    rounding: give a constant factor (one over the accumulated batches) as
    `scale`.  It can be gone through once.  The gradient to float16 logits is
    made in the backward, from a second read of them, and a loss scaler's
    factor enters it before its one rounding."""
    code = REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"policy_loss: unknown reduction {reduction!r}; expected one of {sorted(REDUCTIONS)}")
    return _native.torch_ops().policy_loss(logits, targets, advantages, old_logprobs, ref_logprobs, mask, clip_low,
                                           clip_high, kl_coef, code, scale)


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logprobs: torch.Tensor, *,
                    mask: Optional[torch.Tensor] = None, beta: float = 0.1,
                    label_smoothing: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, margins) of pairs of sequences, the chosen ones in the first half
    of the batch and their rejected counterparts in the second.

    A sequence's gain is the sum over its live tokens of lp - ref, with ref the
    reference model's ``token_logprobs``; a pair's margin m is beta times the
    chosen gain less the rejected one, and the loss the mean over pairs of
    -(1 - s) log sigmoid(m) - s log sigmoid(-m), s = label_smoothing.  margins
    is [pairs], not differentiable."""
    return _native.torch_ops().preference_loss(logits, targets, ref_logprobs, mask, beta, label_smoothing)

"""Losses on logits with their gradients: log probabilities of the targets,
the clipped policy loss with a KL term, and the preference loss of paired log
ratios.

Logits are [batch, seq, vocab] (float32, bfloat16 or float16, any strides with
a unit last one); every statistic is FP32 or wider.  A token whose mask is
False is not looked at, whatever it holds: its log probability and gradient
are 0.  A live token's target outside the vocabulary makes its log probability
and gradient NaN.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native
from ._tensors import launch, need_float, once, same_device, unit_last

__all__ = ["policy_loss", "preference_loss", "token_logprobs"]

REDUCTIONS = {"token": 0, "sequence": 1}


def _checked(what, logits, targets, mask):
    """(logits, targets, mask) as the kernels read them."""
    need_float(logits, what)
    if logits.dim() != 3 or logits.shape[2] == 0:
        raise ValueError(f"{what}: logits {tuple(logits.shape)}; expected [batch, seq, vocab]")
    if targets.shape != logits.shape[:2] or targets.is_floating_point() or targets.dtype == torch.bool:
        raise ValueError(f"{what}: targets {tuple(targets.shape)} {targets.dtype} of logits {tuple(logits.shape)}; "
                         "expected integers [batch, seq]")
    if mask is not None:
        if mask.shape != targets.shape or mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"{what}: mask {tuple(mask.shape)} {mask.dtype}; expected bool [batch, seq]")
        mask = mask.contiguous()
    same_device(what, logits, targets, mask)
    return unit_last(logits), targets.long().contiguous(), mask


def _floats(what, name, t, targets):
    """A per-token float tensor as contiguous FP32."""
    if t is None:
        return None
    if t.shape != targets.shape or not t.is_floating_point():
        raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype}; expected floats {tuple(targets.shape)}")
    same_device(what, targets, t)
    return t.detach().float().contiguous()


def _rows(logits, targets, mask):
    b, t, v = logits.shape
    return (logits.data_ptr(), _native.dtype_code(logits.dtype), b, t, v, logits.stride(0), logits.stride(1),
            targets.data_ptr(), _native.ptr(mask))


def _logprobs(logits, targets, mask, want_stats):
    lp = torch.empty(targets.shape, dtype=torch.float32, device=logits.device)
    stats = torch.empty(*targets.shape, 2, dtype=torch.float32, device=logits.device) if want_stats else None
    launch("smx_token_logprobs", logits.device, *_rows(logits, targets, mask), lp.data_ptr(), _native.ptr(stats))
    return lp, stats


def _logprobs_backward(logits, targets, mask, stats, coef, strides, scale):
    out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    launch("smx_token_logprobs_backward", logits.device, *_rows(logits, targets, mask), stats.data_ptr(),
           coef.data_ptr(), *strides, _native.ptr(scale), out.data_ptr())
    return out


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask):
        lp, stats = _logprobs(logits, targets, mask, True)
        ctx.save_for_backward(logits, targets, mask, stats)
        return lp

    @staticmethod
    @once
    def backward(ctx, grad):
        logits, targets, mask, stats = ctx.saved_tensors
        return _logprobs_backward(logits, targets, mask, stats, grad.float(), grad.stride(), None), None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """log softmax(logits)[target] of every live token, [batch, seq] float32:
    what an old or reference policy is recorded as."""
    logits, targets, mask = _checked("token_logprobs", logits, targets, mask)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogprobs.apply(logits, targets, mask)
    return _logprobs(logits, targets, mask, False)[0]


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, old, ref, adv, adv_strides, low, high, kl, reduction, scale):
        device = logits.device
        loss = torch.empty((), dtype=torch.float32, device=device)
        lp = torch.empty(targets.shape, dtype=torch.float32, device=device)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=device) if ctx.needs_input_grad[0] else None
        lib = _native.lib()
        need = lib.smx_policy_loss_workspace_bytes(*targets.shape)
        work = torch.empty(need, dtype=torch.uint8, device=device)
        launch("smx_policy_loss", logits.device, *_rows(logits, targets, mask), _native.ptr(old), _native.ptr(ref),
               adv.data_ptr(), *adv_strides, low, high, kl, reduction, scale, loss.data_ptr(), lp.data_ptr(),
               _native.ptr(grad), work.data_ptr(), need)
        ctx.grad = grad
        ctx.mark_non_differentiable(lp)
        return loss, lp

    @staticmethod
    @once
    def backward(ctx, grad_loss, _):
        grad, ctx.grad = ctx.grad, None
        if grad is None:
            raise RuntimeError("policy_loss: the gradient is made with the loss and handed out once; "
                               "call policy_loss again to go through it a second time")
        grad_loss = grad_loss.float()
        launch("smx_scale", grad.device, grad.data_ptr(), _native.dtype_code(grad.dtype), grad.numel(),
               grad_loss.data_ptr())
        return (grad,) + (None,) * 11


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

    The gradient to the logits is made in the pass that reads them.  Backward
    of another factor than 1 costs a pass over it and a second rounding: give a
    constant factor (one over the accumulated batches) as `scale`.  It can be
    gone through once."""
    what = "policy_loss"
    logits, targets, mask = _checked(what, logits, targets, mask)
    code = REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"{what}: unknown reduction {reduction!r}; expected one of {sorted(REDUCTIONS)}")
    if kl_coef and ref_logprobs is None:
        raise ValueError(f"{what}: kl_coef without ref_logprobs")
    old = _floats(what, "old_logprobs", old_logprobs, targets)
    ref = _floats(what, "ref_logprobs", ref_logprobs, targets) if kl_coef else None
    if advantages.shape not in (targets.shape[:1], targets.shape) or not advantages.is_floating_point():
        raise ValueError(f"{what}: advantages {tuple(advantages.shape)} {advantages.dtype}; expected floats [batch] or "
                         "[batch, seq]")
    same_device(what, logits, advantages)
    adv = advantages.detach().float()
    strides = adv.stride() if adv.dim() == 2 else (adv.stride(0), 0)
    return _PolicyLoss.apply(logits, targets, mask, old, ref, adv, strides, float(clip_low), float(clip_high),
                             float(kl_coef), code, float(scale))


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, ref, beta, smoothing):
        device = logits.device
        lp, stats = _logprobs(logits, targets, mask, ctx.needs_input_grad[0])
        pairs = logits.shape[0] // 2
        loss = torch.empty((), dtype=torch.float32, device=device)
        margins = torch.empty(pairs, dtype=torch.float32, device=device)
        coef = torch.empty(2 * pairs, dtype=torch.float32, device=device)
        launch("smx_preference_loss", logits.device, lp.data_ptr(), ref.data_ptr(), _native.ptr(mask), pairs,
               logits.shape[1], beta, smoothing, loss.data_ptr(), margins.data_ptr(), coef.data_ptr())
        if stats is not None:
            ctx.save_for_backward(logits, targets, mask, stats, coef)
        ctx.mark_non_differentiable(margins)
        return loss, margins

    @staticmethod
    @once
    def backward(ctx, grad_loss, _):
        logits, targets, mask, stats, coef = ctx.saved_tensors
        return (_logprobs_backward(logits, targets, mask, stats, coef, (1, 0), grad_loss.float()),) + (None,) * 5


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
    what = "preference_loss"
    logits, targets, mask = _checked(what, logits, targets, mask)
    if logits.shape[0] % 2:
        raise ValueError(f"{what}: {logits.shape[0]} sequences are no pairs")
    if ref_logprobs is None:
        raise ValueError(f"{what}: ref_logprobs is needed")
    ref = _floats(what, "ref_logprobs", ref_logprobs, targets)
    return _PreferenceLoss.apply(logits, targets, mask, ref, float(beta), float(label_smoothing))

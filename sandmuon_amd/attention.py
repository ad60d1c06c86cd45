"""RMS norms of queries and keys per head with the rotary position rotation.

Normalised queries and keys bound the attention logits whatever the
projections grow to, which updates of unit singular values let grow faster
than AdamW does.  Norm and rotation of queries and keys, forward and backward,
are one kernel launch each (two in the backward with weight gradients).
"""
from __future__ import annotations

import operator
from typing import Optional, Tuple, Union

import torch

from . import _native

__all__ = ["qk_norm_rotary", "rotary_tables"]

STYLES = {"half": 0, "interleaved": 1}


def rotary_tables(positions: int, rot: int, base: float = 10000.0,
                  device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin [positions, rot / 2] (float32) of the angles position *
    base^(-2p / rot)."""
    if positions < 0 or rot < 0 or rot % 2:
        raise ValueError(f"rotary_tables: {positions} positions of {rot} elements; expected an even number in pairs")
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                   cos: torch.Tensor, sin: torch.Tensor, positions: Union[None, int, torch.Tensor] = None, *,
                   eps: float = 1e-6, style: str = "half",
                   out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q', k'): each head of q [batch, seq, q heads, dim] and k [batch, seq, k
    heads, dim] (any strides) normalised, x * rsqrt(mean x^2 + eps) * weight,
    and its first rot elements turned by the token's position.

    cos, sin: [positions, rot / 2] float32 (``rotary_tables``), rot <= dim.
    style: "half" pairs element p with p + rot/2, "interleaved" 2p with 2p + 1.
    positions: None (0, 1, ... along seq), the first token's position, or an
    integer tensor [seq] or [batch, seq]; a position outside the tables gives
    NaN.  Weights: [dim], or None for ones.  out: (q', k') to write into, of
    any strides with a unit last one (slots of a cache, or q and k
    themselves, but no other overlap with what is read), not under autograd.  cos
    and sin are constants: no gradient.  Statistics and products are FP32, rounded
    once to q's type."""
    code = STYLES.get(style)
    if code is None:
        raise ValueError(f"qk_norm_rotary: unknown style {style!r}; expected one of {sorted(STYLES)}")
    position0 = 0
    if positions is not None and not isinstance(positions, torch.Tensor):
        positions, position0 = None, operator.index(positions)
    return _native.torch_ops().qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, position0, eps, code, out)

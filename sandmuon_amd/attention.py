"""RMS norms of queries and keys per head with the rotary position rotation.

Normalised queries and keys bound the attention logits whatever the
projections grow to, which updates of unit singular values let grow faster
than AdamW does.  Norm and rotation of queries and keys, forward and backward,
are one kernel launch each (two in the backward with weight gradients).
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple, Union

import torch

from . import _native
from ._tensors import launch, need_float, once, same_device, unit_last

__all__ = ["qk_norm_rotary", "rotary_tables"]

STYLES = {"half": 0, "interleaved": 1}

# smx_qk_desc, field by field: two sides, then the rest.
_PACK = struct.Struct("5Q10q2i" * 2 + "3Q8qd2i")
assert _PACK.size == _native.ctypes.sizeof(_native.QkDesc)
_NO_SIDE = (0,) * 17


def rotary_tables(positions: int, rot: int, base: float = 10000.0,
                  device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin [positions, rot / 2] (float32) of the angles position *
    base^(-2p / rot)."""
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _geometry(x, y):
    """heads and the strides of x and y, as a side's descriptor holds them."""
    return (x.shape[2], *x.stride()[:3], *y.stride()[:3])


def _side(x, w, geometry, y, dy=None, dw=None):
    ds = (0, 0, 0) if dy is None else dy.stride()[:3]
    return (x.data_ptr(), 0 if w is None else w.data_ptr(), 0 if dy is None else dy.data_ptr(), y.data_ptr(),
            0 if dw is None else dw.data_ptr(), *geometry, *ds, 0 if w is None else _native.dtype_code(w.dtype), 0)


def _desc(q_side, k_side, x, cos, sin, positions, rest):
    position0, eps, style = rest
    b, t, _, d = x.shape
    pos = (0, 0, 0) if positions is None else (positions.data_ptr(), *positions.stride())
    return _native.QkDesc.from_buffer(bytearray(_PACK.pack(
        *q_side, *k_side, cos.data_ptr(), sin.data_ptr(), *pos, position0, cos.shape[0], b, t, d, 2 * cos.shape[1], eps,
        _native.dtype_code(x.dtype), style)))


def _forward(q, k, qw, kw, cos, sin, positions, rest, out=None):
    """((q', k'), the sides' geometries)"""
    if out is None:
        out = (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device))
    geometries = _geometry(q, out[0]), _geometry(k, out[1])
    launch("smx_qk_norm_rotary", q.device, _desc(_side(q, qw, geometries[0], out[0]), _side(k, kw, geometries[1], out[1]),
                                                 q, cos, sin, positions, rest))
    return out, geometries


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, positions, rest):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        out, ctx.geometries = _forward(q, k, qw, kw, cos, sin, positions, rest)
        ctx.rest = rest
        return out

    @staticmethod
    @once
    def backward(ctx, dq_out, dk_out):
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        need_q, need_k, need_qw, need_kw = ctx.needs_input_grad[:4]
        # (dx is contiguous, as the result was: its strides are those of y)
        q_side, dq, dqw = _side_backward(q, qw, dq_out, ctx.geometries[0], need_q, need_qw)
        k_side, dk, dkw = _side_backward(k, kw, dk_out, ctx.geometries[1], need_k, need_kw)
        if q_side is not _NO_SIDE or k_side is not _NO_SIDE:
            work, need = None, 0
            if need_qw or need_kw:
                need = _native.lib().smx_qk_workspace_bytes(q.shape[3])
                work = torch.empty(need, dtype=torch.uint8, device=q.device)
            launch("smx_qk_norm_rotary_backward", q.device, _desc(q_side, k_side, q, cos, sin, positions, ctx.rest),
                   None if work is None else work.data_ptr(), need)
        return dq if need_q else None, dk if need_k else None, dqw, dkw, None, None, None, None


def _side_backward(x, w, dy, geometry, need_x, need_w):
    """(descriptor side, dx, dw) of one of the two, _NO_SIDE without a cotangent."""
    if dy is None or not (need_x or need_w):
        return _NO_SIDE, None, None
    dy = unit_last(dy if dy.dtype == x.dtype else dy.to(x.dtype))
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = torch.empty_like(w) if need_w else None
    return _side(x, w, geometry, dx, dy, dw), dx, dw


def _weight(w, x, name):
    if w is None:
        return None
    need_float(w, f"qk_norm_rotary: {name}")
    if w.shape != x.shape[3:]:
        raise ValueError(f"qk_norm_rotary: {name} {tuple(w.shape)} of heads of {x.shape[3]}")
    return w if w.is_contiguous() else w.contiguous()


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
    themselves), not under autograd.  Statistics and products are FP32, rounded
    once to q's type."""
    what = "qk_norm_rotary"
    need_float(q, what)
    need_float(k, what)
    code = STYLES.get(style)
    if code is None:
        raise ValueError(f"{what}: unknown style {style!r}; expected one of {sorted(STYLES)}")
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or q.dtype != k.dtype:
        raise ValueError(f"{what}: q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype}; expected "
                         "[batch, seq, heads, dim] of one type, alike but for heads")
    if (cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 or
            2 * cos.shape[1] > q.shape[3]):
        raise ValueError(f"{what}: cos {tuple(cos.shape)} {cos.dtype} and sin {tuple(sin.shape)} {sin.dtype}; expected "
                         "float32 [positions, rot / 2] with rot at most dim")
    q_weight, k_weight = _weight(q_weight, q, "q_weight"), _weight(k_weight, k, "k_weight")
    position0 = 0
    if isinstance(positions, torch.Tensor):
        if positions.is_floating_point() or positions.dtype == torch.bool or positions.dim() not in (1, 2):
            raise ValueError(f"{what}: positions {tuple(positions.shape)} {positions.dtype}; expected integers [seq] or "
                             "[batch, seq]")
        positions = positions.long().expand(q.shape[:2])
    elif positions is not None:
        positions, position0 = None, int(positions)
    same_device(what, q, k, q_weight, k_weight, cos, sin, positions)
    cos, sin = cos.contiguous(), sin.contiguous()
    rest = position0, float(eps), code
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or
                                        (q_weight is not None and q_weight.requires_grad) or
                                        (k_weight is not None and k_weight.requires_grad))
    if out is not None:
        if grad:
            raise ValueError(f"{what}: out= is not supported under autograd")
        for o, x in zip(out, (q, k)):
            if o.shape != x.shape or o.dtype != x.dtype or o.device != x.device or (o.shape[3] > 1 and o.stride(3) != 1):
                raise ValueError(f"{what}: out {tuple(o.shape)} {o.dtype} for {tuple(x.shape)} {x.dtype}; the last "
                                 "stride must be one")
    q, k = unit_last(q), unit_last(k)
    if grad:
        return _QkNormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, rest)
    return _forward(q, k, q_weight, k_weight, cos, sin, positions, rest, out)[0]

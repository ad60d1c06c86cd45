"""Activations kept in 8 bits for the backward pass.

A Linear keeps its input, and a GELU its input, from the forward to the
backward: for a GPT block that is most of the memory of a training step.
Here they are kept in one byte an element and one scale byte per 32 (33/64 of
bf16), and the backward passes read the bytes themselves:

* ``encode`` / ``decode``: any [..., d] activation to 8 bits and back;
* ``linear_backward``: a Linear's weight and bias gradients from the cotangent
  and its kept input, on BF16 MFMAs (the kept values are exact in BF16);
* ``gelu_forward`` / ``gelu_backward``: the exact GELU with its input (and, for
  the Linear behind it, its output) kept in the same pass, and its gradient;
* ``linear``, ``gelu``, ``mlp``: these as differentiable functions, under
  autocast as torch's own; ``checkpoint_linears`` puts every selected
  ``nn.Linear`` of a model on ``linear``.  The optimizer's statistics hooks see
  the unrounded inputs and cotangents, as before.

Formats.  The elements of a row in blocks of 32 neighbours share a power of
two.  ``"int8"`` (the default) holds round(x / step) with a step of 2^-6 of the
largest magnitude's power of two; ``"e4m3"`` holds a float of 3 fraction bits,
for activations whose blocks hold outliers.  A block with an infinity or a NaN
reads back as NaN.

Only what the backward reads is rounded: outputs and input gradients of a
Linear are those of torch, weight gradients those of the kept input, summed in
FP32.  Double backward is not supported.
"""
from __future__ import annotations

import functools
from typing import Callable, Optional, Tuple

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd.function import once_differentiable

from . import _native

__all__ = ["Act8", "FORMATS", "checkpoint_linears", "decode", "encode", "gelu", "gelu_backward", "gelu_forward",
           "linear", "linear_backward", "mlp"]

FORMATS = {"int8": 0, "e4m3": 1}
_BLOCK = 32


def _fmt(fmt: str, what: str) -> int:
    code = FORMATS.get(fmt)
    if code is None:
        raise ValueError(f"{what}: unknown 8-bit format {fmt!r}; expected one of {sorted(FORMATS)}")
    return code


class Act8:
    """A kept activation: codes [rows, pitch] and scale bytes [rows, pitch /
    32] in one buffer, with the activation's shape and format."""

    __slots__ = ("data", "shape", "fmt")

    def __init__(self, data: torch.Tensor, shape: torch.Size, fmt: str):
        self.data, self.shape, self.fmt = data, shape, fmt

    @property
    def rows(self) -> int:
        return self.shape[:-1].numel()

    @property
    def cols(self) -> int:
        return self.shape[-1]

    @property
    def pitch(self) -> int:
        return -(-self.shape[-1] // _BLOCK) * _BLOCK

    @property
    def codes(self) -> torch.Tensor:
        return self.data[:self.rows * self.pitch].view(self.rows, self.pitch)

    @property
    def scales(self) -> torch.Tensor:
        return self.data[self.rows * self.pitch:].view(self.rows, self.pitch // _BLOCK)

    @property
    def nbytes(self) -> int:
        return self.data.numel()


def _kept(saved: Act8, what: str) -> Act8:
    if not isinstance(saved, Act8):
        raise TypeError(f"{what}: expected an Act8, got {type(saved).__name__}")
    return saved


def encode(x: torch.Tensor, fmt: str = "int8") -> Act8:
    """x [..., d] (float32, bfloat16 or float16) in 8 bits."""
    return Act8(_native.torch_ops().act8_encode(x, _fmt(fmt, "act8.encode")), x.shape, fmt)


def decode(saved: Act8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The kept values in `dtype`: exact in bfloat16 and float32."""
    _kept(saved, "act8.decode")
    return _native.torch_ops().act8_decode(saved.data, saved.shape, FORMATS[saved.fmt], dtype)


def gelu_forward(h: torch.Tensor, fmt: str = "int8", keep_output: bool = True,
                 keep_input: bool = True) -> Tuple[torch.Tensor, Optional[Act8], Optional[Act8]]:
    """(GELU(h), h kept, the GELU's output kept) in one pass, None for what is
    not to be kept."""
    y, *kept = _native.torch_ops().act8_gelu(h, _fmt(fmt, "act8.gelu_forward"), keep_input, keep_output)
    return (y, *(None if data is None else Act8(data, h.shape, fmt) for data in kept))


def gelu_backward(dy: torch.Tensor, saved: Act8) -> torch.Tensor:
    """dy * GELU'(kept h), in dy's type."""
    _kept(saved, "act8.gelu_backward")
    return _native.torch_ops().act8_gelu_backward(dy, saved.data, saved.shape, FORMATS[saved.fmt])


def linear_backward(delta: torch.Tensor, saved: Act8, dtype: Optional[torch.dtype] = None,
                    bias: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dW [n, d], db [n] or None) of a Linear with output cotangent `delta`
    [..., n] and kept input `saved` [..., d], in `dtype` (delta's by default),
    each rounded once from FP32 sums."""
    _kept(saved, "act8.linear_backward")
    return _native.torch_ops().act8_linear_backward(delta, saved.data, saved.shape, FORMATS[saved.fmt], dtype, bias)


# ------------------------------------------------- differentiable functions ---
def _cast(t: Optional[torch.Tensor], device_type: str) -> Optional[torch.Tensor]:
    """t as autocast would hand it to a Linear (float64 and whole numbers as they
    are).  Each call casts its own; autocast keeps a weight's cast for its region."""
    if t is None or not torch.is_autocast_enabled(device_type):
        return t
    if not t.is_floating_point() or t.dtype == torch.float64:
        return t
    return t.to(torch.get_autocast_dtype(device_type))


def _input_grad(grad: torch.Tensor, weight: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    g2 = grad.reshape(grad.shape[:-1].numel(), grad.shape[-1])
    return g2.mm(weight).view(*grad.shape[:-1], weight.shape[1]).to(dtype)


# The kept bytes are saved as tensors, so that a node's backward frees them (what
# hangs on ctx lives as long as the graph, through the next step's forward where
# the loss is still referred to) and saved-tensor hooks see them.
def _data(saved: Optional[Act8]) -> Optional[torch.Tensor]:
    return None if saved is None else saved.data


def _weight_grads(grad, saved: Act8, w_dtype, b_dtype, bias: bool):
    """linear_backward with db in the bias's own type: where the two differ, both
    come in FP32 and are rounded once."""
    dw, db = linear_backward(grad, saved, w_dtype if not bias or b_dtype == w_dtype else torch.float32, bias=bias)
    return dw.to(w_dtype), None if db is None else db.to(b_dtype)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, fmt, kept):
        x_lp, w, b = (_cast(t, x.device.type) for t in (x, weight, bias))
        with torch.autocast(device_type=x.device.type, enabled=False):
            y = F.linear(x_lp, w, b)
        needs = ctx.needs_input_grad
        if not (needs[1] or needs[2]):
            kept = None
        elif kept is None:
            kept = encode(x_lp, fmt)
        ctx.save_for_backward(w if needs[0] else None, _data(kept))
        ctx.kept = None if kept is None else (kept.shape, kept.fmt)
        ctx.dtypes = x.dtype, weight.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        w, data = ctx.saved_tensors
        x_dtype, w_dtype, b_dtype = ctx.dtypes
        needs = ctx.needs_input_grad
        dx = _input_grad(grad, w, x_dtype) if needs[0] else None
        dw = db = None
        if needs[1] or needs[2]:
            dw, db = _weight_grads(grad, Act8(data, *ctx.kept), w_dtype, b_dtype, needs[2])
        return dx, dw if needs[1] else None, db, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, fmt: str = "int8",
           kept: Optional[Act8] = None) -> torch.Tensor:
    """F.linear whose input is kept in 8 bits for the weight gradient: as
    `kept`, ``encode(x)`` made once for several layers of one input, or else
    here in `fmt`."""
    if kept is None:
        _fmt(fmt, "act8.linear")
    elif _kept(kept, "act8.linear").shape != x.shape:
        raise ValueError(f"act8.linear: kept {tuple(kept.shape)} of an input {tuple(x.shape)}")
    if not torch.is_grad_enabled():
        return F.linear(x, weight, bias)
    return _Linear.apply(x, weight, bias, fmt, kept)


class _Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, fmt, grad):
        y, kept, _ = gelu_forward(h, fmt, keep_output=False, keep_input=grad and ctx.needs_input_grad[0])
        ctx.save_for_backward(_data(kept))
        ctx.kept = h.shape, fmt
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return gelu_backward(grad, Act8(*ctx.saved_tensors, *ctx.kept)), None, None


def gelu(h: torch.Tensor, fmt: str = "int8") -> torch.Tensor:
    """F.gelu (exact form) whose input is kept in 8 bits."""
    _fmt(fmt, "act8.gelu")
    return _Gelu.apply(h, fmt, torch.is_grad_enabled())


class _Mlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, fc_w, fc_b, proj_w, proj_b, fmt, grad):
        # (only what the wanted gradients read is kept)
        needs = [grad and need for need in ctx.needs_input_grad]
        x_lp, w1, b1, w2, b2 = (_cast(t, x.device.type) for t in (x, fc_w, fc_b, proj_w, proj_b))
        with torch.autocast(device_type=x.device.type, enabled=False):
            kept_x = encode(x_lp, fmt) if needs[1] or needs[2] else None
            y, kept_h, kept_y = gelu_forward(F.linear(x_lp, w1, b1), fmt, keep_output=needs[3] or needs[4],
                                             keep_input=any(needs[:3]))
            out = F.linear(y, w2, b2)
        ctx.save_for_backward(w1 if needs[0] else None, w2 if any(needs[:3]) else None, *map(_data, (kept_x, kept_h, kept_y)))
        ctx.shapes, ctx.fmt = (x.shape, y.shape), fmt
        ctx.dtypes = tuple(None if t is None else t.dtype for t in (x, fc_w, fc_b, proj_w, proj_b))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        w1, w2, x8, h8, y8 = ctx.saved_tensors
        needs, types_ = ctx.needs_input_grad, ctx.dtypes
        of_x, of_h = ctx.shapes
        out = [None] * 7
        if needs[3] or needs[4]:
            out[3], out[4] = _weight_grads(grad, Act8(y8, of_h, ctx.fmt), types_[3], types_[4], needs[4])
        if any(needs[:3]):
            dh = gelu_backward(_input_grad(grad, w2, grad.dtype), Act8(h8, of_h, ctx.fmt))
        if needs[1] or needs[2]:
            out[1], out[2] = _weight_grads(dh, Act8(x8, of_x, ctx.fmt), types_[1], types_[2], needs[2])
        if needs[0]:
            out[0] = _input_grad(dh, w1, types_[0])
        return tuple(g if k < 5 and needs[k] else None for k, g in enumerate(out))


def mlp(x: torch.Tensor, fc_weight: torch.Tensor, fc_bias: Optional[torch.Tensor], proj_weight: torch.Tensor,
        proj_bias: Optional[torch.Tensor], fmt: str = "int8") -> torch.Tensor:
    """proj(GELU(fc(x))) with x, the hidden layer and the GELU's output kept in
    8 bits: 1 byte an element where three 16-bit tensors would be kept."""
    _fmt(fmt, "act8.mlp")
    return _Mlp.apply(x, fc_weight, fc_bias, proj_weight, proj_bias, fmt, torch.is_grad_enabled())


def _checkpointed_forward(module: nn.Linear, fmt: str, x: torch.Tensor, kept: Optional[Act8] = None) -> torch.Tensor:
    if torch.is_grad_enabled() and x.is_cuda:
        return linear(x, module.weight, module.bias, fmt, kept)
    return F.linear(x, module.weight, module.bias)


class CheckpointedLinears:
    """Handle of ``checkpoint_linears``; ``close()`` restores the forwards."""

    def __init__(self, modules):
        self.modules = modules

    def close(self) -> None:
        for module in self.modules.values():
            # (not one that something else has put over it since)
            if getattr(module.__dict__.get("forward"), "func", None) is _checkpointed_forward:
                del module.forward
        self.modules = {}


def checkpoint_linears(model: nn.Module, module_filter: Optional[Callable[[str, nn.Module], bool]] = None,
                       fmt: str = "int8") -> CheckpointedLinears:
    """Puts every plain ``nn.Linear`` of `model` that `module_filter` selects
    (all of them by default) on ``linear``; their forwards take ``linear``'s
    `kept` too, for layers that share an input.  Hooks on the modules run as
    before; a module whose forward is replaced already is left as it is."""
    _fmt(fmt, "act8.checkpoint_linears")

    chosen = {}
    for name, module in model.named_modules():
        if type(module) is not nn.Linear or "forward" in module.__dict__:
            continue
        if module_filter is None or module_filter(name, module):
            # (a partial of a module's function: pickled and copied models keep it)
            module.forward = functools.partial(_checkpointed_forward, module, fmt)
            chosen[name] = module
    return CheckpointedLinears(chosen)

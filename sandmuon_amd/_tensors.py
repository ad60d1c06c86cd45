"""Argument checks and calls shared by the operators of a training step (act8,
attention, losses)."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

_CODES = _native._DTYPES
_current_device = torch._C._cuda_getDevice


def need_float(t: torch.Tensor, what: str) -> torch.Tensor:
    """t, a GPU tensor of one of the three float types."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        _native.require_gpu(t, what)
    if t.dtype not in _CODES:
        raise ValueError(f"{what}: unsupported dtype {t.dtype}; expected float32, bfloat16 or float16")
    return t


def same_device(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors on {device} and {t.device}")


def unit_last(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy where its last dimension has no unit stride."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def rows2d(t: torch.Tensor) -> torch.Tensor:
    """[..., d] -> [n, d] with unit column stride (a copy where t's strides
    allow no such view)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(t.shape[:-1].numel(), t.shape[-1])
    return unit_last(t)


def launch(name: str, device: torch.device, *args) -> None:
    """Calls entry point `name` with `args` and the current stream of `device`,
    which is made current for the call where it is not."""
    fn = getattr(_native.lib(), name)
    index = device.index
    if index == _current_device():
        rc = fn(*args, _native.stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _native.stream_of(device))
    if rc != 0:
        _native._check(rc, name)


def once(backward):
    """A Function's backward that cannot be differentiated: torch's
    once_differentiable where a graph of the backward is being made
    (create_graph), the function itself, without that wrapper's cost, else."""
    wrapped = once_differentiable(backward)

    def call(ctx, *grads):
        return wrapped(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return call

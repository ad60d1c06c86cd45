"""Argument checks shared by the operators of a training step (act8,
attention, losses)."""
from __future__ import annotations

from typing import Optional

import torch

from . import _native

FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def need_float(t: torch.Tensor, what: str) -> torch.Tensor:
    """t, a GPU tensor of one of the three float types."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(t).__name__}")
    _native.require_gpu(t, what)
    if t.dtype not in FLOATS:
        raise ValueError(f"{what}: unsupported dtype {t.dtype}; expected float32, bfloat16 or float16")
    return t


def same_device(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")


def unit_last(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy where its last dimension has no unit stride."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def rows2d(t: torch.Tensor) -> torch.Tensor:
    """[..., d] -> [n, d] with unit column stride (a copy where t's strides
    allow no such view)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(t.shape[:-1].numel(), t.shape[-1])
    return unit_last(t)


class on_device:
    """Makes t's device current for a launch, where it is not already."""

    __slots__ = ("guard",)

    def __init__(self, t: torch.Tensor):
        index = t.device.index
        self.guard = None if index is None or index == torch.cuda.current_device() else torch.cuda.device(index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)

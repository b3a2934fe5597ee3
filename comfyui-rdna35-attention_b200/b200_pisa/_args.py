"""Argument handling shared by the rotary and the differentiable attention
entry points: row views, device guard, output storage."""
from __future__ import annotations

import contextlib
import functools

import torch

from . import _lib
from ._lib import LIB, check


@functools.lru_cache(maxsize=16)
def checked_device(index: int) -> int:
    check(LIB.b2_check_device(index))
    return index


def on_device(x: torch.Tensor):
    """Context in which x's device is the current one (kernels launch on the
    current device; the caller's may be another)."""
    index = checked_device(x.device.index)
    return contextlib.nullcontext() if torch.cuda.current_device() == index else torch.cuda.device(index)


def require_one_device(name: str, *tensors: torch.Tensor | None) -> None:
    present = [t for t in tensors if t is not None]
    first = present[0].device
    if first.type != "cuda" or any(t.device != first for t in present):
        raise ValueError(f"{name} requires its tensors on one CUDA device.")


def row_strides(x: torch.Tensor) -> tuple[int, ...]:
    """Strides of x's leading dimensions, 0 where a dimension has one entry
    (its stride is never used and may be anything)."""
    return tuple(s if n > 1 else 0 for n, s in zip(x.shape[:-1], x.stride()[:-1]))


def addressable(x: torch.Tensor) -> bool:
    """Whether the 16-byte row kernels can read x in place."""
    es = x.element_size()
    return ((x.stride(-1) == 1 or x.shape[-1] == 1) and x.data_ptr() % 16 == 0
            and all(s * es % 16 == 0 and s >= 0 for s in row_strides(x)))


def row_view(x: torch.Tensor) -> _lib.View:
    """b2_view of a [B,H,T,D] tensor whose rows are addressable."""
    sb, sh, st = row_strides(x)
    batch, heads, tokens, dim = x.shape
    return _lib.View(x.data_ptr(), sb, sh, st, batch, heads, tokens, dim, _lib.dtype_code(x.dtype), _lib.ORDER_LINEAR,
                     0, 0)


def token_major(x: torch.Tensor, heads: int | None = None, tokens: int | None = None) -> torch.Tensor:
    """New [B,H,T,D] view of contiguous [B,T,H,D] storage of x's shape, type
    and device (the layout attention and the output projection read)."""
    batch, h, t, dim = x.shape
    storage = torch.empty((batch, tokens or t, heads or h, dim), device=x.device, dtype=x.dtype)
    return storage.permute(0, 2, 1, 3)

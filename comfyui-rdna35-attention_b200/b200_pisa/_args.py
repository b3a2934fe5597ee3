"""Argument handling shared by the rotary and the differentiable attention
entry points.

A call's checks depend on the shapes, strides and types of its tensors alone,
so each entry point does them once per combination, in a cached plan that also
holds the packed b2_view of every tensor but its base address.  What is left
per call is the addresses, the device and the stream: about 10 us of host time
instead of 45, which is what the smallest calls cost."""
from __future__ import annotations

import contextlib
import functools
import struct

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import LIB, check

#: calls of different shapes whose plans are kept
PLANS = 1024

_VIEW_TAIL = struct.Struct("=qqqiiiiiiii")
_POINTER = struct.Struct("=Q")
assert _POINTER.size + _VIEW_TAIL.size == _lib.ctypes.sizeof(_lib.View)


@functools.lru_cache(maxsize=16)
def checked_device(index: int) -> int:
    check(LIB.b2_check_device(index))
    return index


_HERE = contextlib.nullcontext()


def on_device(x: torch.Tensor):
    """Context in which x's device is the current one (kernels launch on the
    current device; the caller's may be another)."""
    index = checked_device(x.device.index)
    return _HERE if torch.cuda.current_device() == index else torch.cuda.device(index)


def raw_stream(x: torch.Tensor) -> int:
    """The current stream of x's device, as cudaStream_t."""
    return torch._C._cuda_getCurrentRawStream(x.device.index)


def require_one_device(name: str, *tensors: torch.Tensor | None) -> None:
    first = tensors[0].device
    one = first.type == "cuda"
    for t in tensors:
        if t is not None and t.device != first:
            one = False
    if not one:
        raise ValueError(f"{name} requires its tensors on one CUDA device.")


def refuse_tangents(name: str, *tensors: torch.Tensor | None) -> None:
    """Forward-mode derivatives do not exist here; results without them would pass for constants."""
    if forward_ad._current_level < 0:  # no dual level is open, so no tensor has a tangent
        return
    tracing = torch.compiler.is_compiling()  # a traced tensor does not show its tangent
    for t in tensors:
        if isinstance(t, torch.Tensor) and (tracing or forward_ad.unpack_dual(t).tangent is not None):
            raise ValueError(f"{name} has no forward-mode derivatives; its tensors must not carry tangents.")


def row_strides(shape, strides) -> tuple[int, ...]:
    """Strides of the leading dimensions, 0 where a dimension has one entry
    (its stride is never used and may be anything)."""
    return tuple(s if n > 1 else 0 for n, s in zip(shape[:-1], strides[:-1]))


def addressable(shape, strides, dtype: torch.dtype) -> bool:
    """Whether the 16-byte row kernels can read such a tensor in place, given
    a base address on a 16-byte boundary."""
    return ((strides[-1] == 1 or shape[-1] == 1)
            and all(s >= 0 and s * dtype.itemsize % 16 == 0 for s in row_strides(shape, strides)))


def repeats(shape, strides) -> bool:
    """Whether a dimension of several entries has stride 0 (a broadcast)."""
    return any(n > 1 and s == 0 for n, s in zip(shape, strides))


def view_tail(shape, strides, dtype: torch.dtype) -> bytes:
    """The packed b2_view of a [B,H,T,D] tensor without its base address."""
    return _VIEW_TAIL.pack(*row_strides(shape, strides), *shape, _lib.dtype_code(dtype), _lib.ORDER_LINEAR, 0, 0)


def with_base(x: torch.Tensor, tail: bytes) -> bytes:
    """The struct whose first member is x's address."""
    return _POINTER.pack(x.data_ptr()) + tail


def row_view(x: torch.Tensor) -> _lib.View:
    """b2_view of a [B,H,T,D] tensor whose rows are addressable."""
    return _lib.View.from_buffer_copy(with_base(x, view_tail(x.shape, x.stride(), x.dtype)))


def token_major_strides(shape) -> tuple[int, int, int, int]:
    """Strides of a [B,H,T,D] view of contiguous [B,T,H,D] storage, the layout
    attention and the output projection read."""
    _, h, t, d = shape
    return (t * h * d, d, h * d, 1)


def new_rows(like: torch.Tensor, shape, strides) -> torch.Tensor:
    return torch.empty_strided(shape, strides, dtype=like.dtype, device=like.device)


def signature(x: torch.Tensor):
    return x.shape, x.stride(), x.dtype


@functools.lru_cache(maxsize=PLANS)
def _tail_in_place(shape, strides, dtype: torch.dtype, broadcast: bool) -> bytes | None:
    if addressable(shape, strides, dtype) and (broadcast or not repeats(shape, strides)):
        return view_tail(shape, strides, dtype)
    return None


def as_rows(x: torch.Tensor, broadcast: bool = True) -> tuple[torch.Tensor, bytes]:
    """x where the kernels can read it in place, else a contiguous copy, and
    its packed view.  broadcast: whether stride 0 can be read in place (TMA
    cannot)."""
    tail = _tail_in_place(*signature(x), broadcast)
    if tail is None or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format) if x.data_ptr() % 16 else x.contiguous()
        tail = view_tail(*signature(x))
    return x, with_base(x, tail)


def layouts(*tensors: torch.Tensor | None):
    """What came_back() compares."""
    return tuple(None if x is None else signature(x) for x in tensors)


def came_back(name: str, tensors, were) -> bool:
    """Whether the tensors that a forward pass saved came back to its backward
    pass laid out as they ``were``, so that the forward pass's plan holds for
    them.  Saved-tensor hooks (offloading, compression) may return copies with
    other strides or off the 16-byte boundaries; copies of another shape or
    type are refused."""
    same = True
    for x, was in zip(tensors, were):
        if was is None:
            continue
        now = signature(x)
        if now != was:
            if now[0] != was[0] or now[2] != was[2]:
                raise ValueError(f"{name}: a saved tensor came back with another shape or dtype.")
            same = False
        elif x.data_ptr() % 16:
            same = False
    return same


def dense(x: torch.Tensor | None, alignment: int = 1) -> torch.Tensor | None:
    """x itself if contiguous from a multiple of ``alignment``, else a copy that is."""
    if x is None or (x.is_contiguous() and x.data_ptr() % alignment == 0):
        return x
    return x.clone(memory_format=torch.contiguous_format)

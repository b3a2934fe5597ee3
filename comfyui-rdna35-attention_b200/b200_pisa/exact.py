"""Exact softmax attention with gradients: ``attention`` (differentiable), and
its two passes ``attention_forward`` and ``attention_backward`` for callers
that keep the saved tensors themselves (e.g. inside a captured CUDA graph).

Next to ``full_attention`` (forward only, no mask) these take key/value heads
shared by groups of query heads, per-batch key counts and a causal mask.
Tensors are [B,H,T,D] (or [BH,T,D]) views, BF16 or FP16, D <= 128 a multiple
of 8; rows must start on 16-byte boundaries with a contiguous head dimension.
Results of four-dimensional calls are [B,H,T,D] views of contiguous [B,T,H,D]
storage."""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from ._args import addressable, on_device, require_one_device, row_strides, row_view, token_major
from ._lib import LIB, check, ptr, stream_of

MAX_HEAD_DIM = 128
_DTYPES = (torch.bfloat16, torch.float16)


def _four(name: str, x: torch.Tensor) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor.")
    if x.ndim not in (3, 4) or 0 in x.shape:
        raise ValueError(f"{name} must be a non-empty [B,H,T,D] or [BH,T,D] tensor.")
    return x if x.ndim == 4 else x.unsqueeze(1)


def _in_place(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy where TMA cannot read it in place: a broadcast dimension
    (stride 0), a strided head dimension, rows off the 16-byte boundaries."""
    if addressable(x) and all(s > 0 for s, n in zip(row_strides(x), x.shape) if n > 1):
        return x
    return x.contiguous()


def _check_input(name: str, x: torch.Tensor) -> torch.Tensor:
    """A checked q, k or v; expanded inputs are copied, misaligned ones refused."""
    if not addressable(x):
        raise ValueError(f"{name} needs a contiguous head dimension and rows that start on 16-byte boundaries.")
    return _in_place(x)


def _check_call(q, k, v, scale, key_lengths):
    """Checked four-dimensional (q, k, v) and the scale."""
    if len({x.ndim for x in (q, k, v) if isinstance(x, torch.Tensor)}) > 1:
        raise ValueError("q, k and v must have the same rank.")
    q, k, v = _four("q", q), _four("k", k), _four("v", v)
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[-1] != k.shape[-1]:
        raise ValueError("attention expects q [B,H,Tq,D] and matching k/v [B,Hk,Tk,D].")
    if q.shape[1] % k.shape[1]:
        raise ValueError(f"q heads ({q.shape[1]}) must be a multiple of k/v heads ({k.shape[1]}).")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("attention supports matching float16 or bfloat16 q/k/v.")
    if q.shape[-1] > MAX_HEAD_DIM or q.shape[-1] % 8:
        raise ValueError(f"attention supports D <= {MAX_HEAD_DIM}, a multiple of 8.")
    if key_lengths is not None:
        if not isinstance(key_lengths, torch.Tensor):
            raise TypeError("key_lengths must be a torch tensor or None.")
        if key_lengths.shape != (q.shape[0],) or key_lengths.dtype != torch.int32 or not key_lengths.is_contiguous():
            raise ValueError(f"key_lengths must be a contiguous int32 [B] tensor, B={q.shape[0]}.")
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if not 0.0 < ctypes.c_float(scale).value < math.inf:
        raise ValueError("scale must be representable as a positive finite float32 value.")
    return _check_input("q", q), _check_input("k", k), _check_input("v", v), scale


def _like_rank(x: torch.Tensor, rank: int) -> torch.Tensor:
    return x if rank == 4 else x.squeeze(1)


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None, *,
                      causal: bool = False, key_lengths: torch.Tensor | None = None):
    """(out, lse) of softmax(scale q k^T) v: out like q, lse FP32 [B,H,Tq]
    ([BH,Tq]) the natural log of the sum of exponentials.  key_lengths: int32
    [B] on the device, batch b attends to its first key_lengths[b] keys (what
    the K/V rows past them hold does not matter).  causal: query i sees keys
    up to i + Tk - Tq.  A query that sees no key gives out 0 and lse -inf."""
    rank = q.ndim if isinstance(q, torch.Tensor) else 0
    q, k, v, scale = _check_call(q, k, v, scale, key_lengths)
    require_one_device("attention", q, k, v, key_lengths)
    with on_device(q):
        out = token_major(q)
        lse = torch.empty(q.shape[:3], device=q.device, dtype=torch.float32)
        check(LIB.b2_attention_forward(ctypes.byref(row_view(q)), ctypes.byref(row_view(k)), ctypes.byref(row_view(v)),
                                       ctypes.byref(row_view(out)), scale, int(bool(causal)), ptr(key_lengths), ptr(lse),
                                       stream_of(q)))
    return _like_rank(out, rank), _like_rank(lse, rank)


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, scale: float | None = None, *, causal: bool = False,
                       key_lengths: torch.Tensor | None = None):
    """(dq, dk, dv) of attention_forward's call from the gradient of its out
    and what it returned.  Probabilities are recomputed from lse; dk and dv of
    a shared head are summed over its group in FP32; rows of dk and dv past a
    batch's keys are 0.  Bit-reproducible."""
    rank = q.ndim if isinstance(q, torch.Tensor) else 0
    q, k, v, scale = _check_call(q, k, v, scale, key_lengths)
    out, dout = _four("out", out), _four("dout", dout)
    for name, x in (("out", out), ("dout", dout)):
        if x.shape != q.shape or x.dtype != q.dtype:
            raise ValueError(f"{name} must have q's shape and dtype.")
    if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 or lse.numel() != math.prod(q.shape[:3]) \
            or lse.shape != (q.shape[:3] if rank == 4 else (q.shape[0], q.shape[2])):
        raise ValueError("lse must be attention_forward's float32 [B,H,Tq] tensor.")
    require_one_device("attention_backward", q, k, v, out, dout, lse, key_lengths)
    out, dout, lse = _in_place(out), _in_place(dout), lse.contiguous()
    with on_device(q):
        dq, dk, dv = token_major(q), token_major(k), token_major(v)
        ws = torch.empty(LIB.b2_attention_backward_workspace_bytes(q.shape[0], q.shape[1], k.shape[1], q.shape[2]),
                         device=q.device, dtype=torch.uint8)
        views = [ctypes.byref(row_view(x)) for x in (q, k, v, out, dout)]
        grads = [ctypes.byref(row_view(x)) for x in (dq, dk, dv)]
        check(LIB.b2_attention_backward(*views, ptr(lse), *grads, scale, int(bool(causal)), ptr(key_lengths), ptr(ws),
                                        stream_of(q)))
    return _like_rank(dq, rank), _like_rank(dk, rank), _like_rank(dv, rank)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, key_lengths):
        out, lse = attention_forward(q, k, v, scale, causal=causal, key_lengths=key_lengths)
        ctx.save_for_backward(q, k, v, out, lse, key_lengths)
        ctx.call = (scale, causal)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, key_lengths = ctx.saved_tensors
        scale, causal = ctx.call
        grads = attention_backward(dout, q, k, v, out, lse, scale, causal=causal, key_lengths=key_lengths)
        return (*grads, None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None, *, causal: bool = False,
              key_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v, differentiable in q, k and v (see
    attention_forward for the masks and layouts; scale defaults to D^-0.5)."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v)):
        return _Attention.apply(q, k, v, scale, causal, key_lengths)
    return attention_forward(q, k, v, scale, causal=causal, key_lengths=key_lengths)[0]


__all__ = ["attention", "attention_backward", "attention_forward"]

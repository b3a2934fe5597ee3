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
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from ._args import (PLANS, addressable, as_rows, came_back, dense, layouts, new_rows, on_device, raw_stream, refuse_tangents,
                    repeats, require_one_device, signature, token_major_strides, view_tail, with_base)
from ._lib import LIB, check, ptr

MAX_HEAD_DIM = 128
#: keys that a row sees up to which out's rounding error is kept for the backward pass (kLowKeys of the library)
LOW_KEYS = 64
_DTYPES = (torch.bfloat16, torch.float16)


def _four(name: str, x: torch.Tensor) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor.")
    if x.ndim == 4:
        return x
    if x.ndim != 3:
        raise ValueError(f"{name} must be a non-empty [B,H,T,D] or [BH,T,D] tensor.")
    return x.unsqueeze(1)


@functools.lru_cache(maxsize=PLANS)
def _plan(q_sig, k_sig, v_sig, lens_sig, scale):
    """Checks of a call's shapes, strides and types (four-dimensional)."""
    q_shape, k_shape, dtype = q_sig[0], k_sig[0], q_sig[2]
    for name, (shape, _, _) in (("q", q_sig), ("k", k_sig), ("v", v_sig)):
        if 0 in shape:
            raise ValueError(f"{name} must be a non-empty [B,H,T,D] or [BH,T,D] tensor.")
    if k_shape != v_sig[0] or q_shape[0] != k_shape[0] or q_shape[-1] != k_shape[-1]:
        raise ValueError("attention expects q [B,H,Tq,D] and matching k/v [B,Hk,Tk,D].")
    if q_shape[1] % k_shape[1]:
        raise ValueError(f"q heads ({q_shape[1]}) must be a multiple of k/v heads ({k_shape[1]}).")
    if dtype not in _DTYPES or k_sig[2] != dtype or v_sig[2] != dtype:
        raise ValueError("attention supports matching float16 or bfloat16 q/k/v.")
    if q_shape[-1] > MAX_HEAD_DIM or q_shape[-1] % 8:
        raise ValueError(f"attention supports D <= {MAX_HEAD_DIM}, a multiple of 8.")
    if lens_sig is not None and lens_sig != ((q_shape[0],), (1,), torch.int32):
        raise ValueError(f"key_lengths must be a contiguous int32 [B] tensor, B={q_shape[0]}.")
    scale = float(q_shape[-1] ** -0.5 if scale is None else scale)
    if not 0.0 < ctypes.c_float(scale).value < math.inf:
        raise ValueError("scale must be representable as a positive finite float32 value.")
    for name, sig in (("q", q_sig), ("k", k_sig), ("v", v_sig)):
        if not addressable(*sig):
            raise ValueError(f"{name} needs a contiguous head dimension and rows that start on 16-byte boundaries.")
    q_strides, k_strides = token_major_strides(q_shape), token_major_strides(k_shape)
    return (scale, any(repeats(*sig[:2]) for sig in (q_sig, k_sig, v_sig)),
            (view_tail(*q_sig), view_tail(*k_sig), view_tail(*v_sig)),
            (q_strides, k_strides), (view_tail(q_shape, q_strides, dtype), view_tail(k_shape, k_strides, dtype)))


def _planned(q, k, v, scale, key_lengths):
    """Checked four-dimensional (q, k, v) and their plan; expanded inputs
    (stride 0) are copied, which TMA cannot read."""
    if len({x.ndim for x in (q, k, v) if isinstance(x, torch.Tensor)}) > 1:
        raise ValueError("q, k and v must have the same rank.")
    q, k, v = _four("q", q), _four("k", k), _four("v", v)
    lens_sig = None
    if key_lengths is not None:
        if not isinstance(key_lengths, torch.Tensor):
            raise TypeError("key_lengths must be a torch tensor or None.")
        shape, strides, dtype = signature(key_lengths)
        lens_sig = (tuple(shape), strides if shape != (1,) else (1,), dtype)
    scale = None if scale is None else float(scale)
    plan = _plan(signature(q), signature(k), signature(v), lens_sig, scale)
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.data_ptr() % 16:
            raise ValueError(f"{name} needs a contiguous head dimension and rows that start on 16-byte boundaries.")
    if plan[1]:
        q, k, v = (as_rows(x, broadcast=False)[0] for x in (q, k, v))
        plan = _plan(signature(q), signature(k), signature(v), lens_sig, scale)
    return q, k, v, plan


def wants_low(dtype: torch.dtype, key_tokens: int, key_lengths, causal: bool) -> bool:
    """Whether the backward pass may need what the type cannot hold of the
    output: BF16, and rows that see at most LOW_KEYS keys."""
    return dtype == torch.bfloat16 and (key_lengths is not None or causal or key_tokens <= LOW_KEYS)


def new_low(q: torch.Tensor, strides, key_tokens: int, key_lengths, causal: bool) -> torch.Tensor | None:
    return new_rows(q, q.shape, strides) if wants_low(q.dtype, key_tokens, key_lengths, causal) else None


def with_optional(x: torch.Tensor | None, tail: bytes) -> bytes | None:
    return None if x is None else with_base(x, tail)


def _run_forward(q, k, v, plan, causal: bool, key_lengths, with_low: bool):
    """The pass on checked four-dimensional tensors."""
    scale, _, tails, strides, out_tails = plan
    with on_device(q):
        out = new_rows(q, q.shape, strides[0])
        low = new_low(q, strides[0], k.shape[2], key_lengths, causal) if with_low else None
        lse = torch.empty(q.shape[:3], device=q.device, dtype=torch.float32)
        check(LIB.b2_attention_forward(with_base(q, tails[0]), with_base(k, tails[1]), with_base(v, tails[2]),
                                       with_base(out, out_tails[0]), scale, 1 if causal else 0, ptr(key_lengths),
                                       ptr(lse), with_optional(low, out_tails[0]), raw_stream(q)))
    return out, lse, low


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None, *,
                      causal: bool = False, key_lengths: torch.Tensor | None = None, with_low: bool = False):
    """(out, lse) of softmax(scale q k^T) v: out like q, lse FP32 [B,H,Tq]
    ([BH,Tq]) the natural log of the sum of exponentials.  key_lengths: int32
    [B] on the device, batch b attends to its first key_lengths[b] keys (what
    the K/V rows past them hold does not matter).  causal: query i sees keys
    up to i + Tk - Tq.  A query that sees no key gives out 0 and lse -inf.

    with_low: (out, lse, out_low), for attention_backward: out's rounding
    error (like out, BF16) in rows that see at most 64 keys, whose gradients
    it is the largest error of (its other rows are not written); None where no
    row can see so few."""
    refuse_tangents("attention_forward", q, k, v)
    flat = isinstance(q, torch.Tensor) and q.ndim == 3
    q, k, v, plan = _planned(q, k, v, scale, key_lengths)
    require_one_device("attention", q, k, v, key_lengths)
    out, lse, low = _run_forward(q, k, v, plan, causal, key_lengths, with_low)
    if flat:
        out, lse, low = out.squeeze(1), lse.squeeze(1), None if low is None else low.squeeze(1)
    return (out, lse, low) if with_low else (out, lse)


@functools.lru_cache(maxsize=PLANS)
def _workspace_bytes(*sizes: int) -> int:
    return LIB.b2_attention_backward_workspace_bytes(*sizes)


def check_saved(q: torch.Tensor, flat: bool, lse, **rows) -> list:
    """Checked four-dimensional ``rows`` (like q) a backward pass is given."""
    got = []
    for name, x in rows.items():
        if x is not None or name != "out_low":
            x = _four(name, x)
            if x.shape != q.shape or x.dtype != q.dtype:
                raise ValueError(f"{name} must have q's shape and dtype.")
        got.append(x)
    batch, heads, tokens, _ = q.shape
    if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 \
            or lse.shape != ((batch, tokens) if flat else (batch, heads, tokens)):
        raise ValueError("lse must be the forward pass's float32 [B,H,Tq] tensor.")
    return got


def _run_backward(dout, q, k, v, out, lse, low, plan, causal: bool, key_lengths):
    scale, _, tails, strides, grad_tails = plan
    batch, heads, tokens, _ = q.shape
    with on_device(q):
        (out, out_view), (dout, dout_view) = as_rows(out, broadcast=False), as_rows(dout, broadcast=False)
        low, low_view = (None, None) if low is None else as_rows(low, broadcast=False)
        lse = dense(lse)
        dq, dk, dv = new_rows(q, q.shape, strides[0]), new_rows(k, k.shape, strides[1]), new_rows(k, k.shape, strides[1])
        ws = torch.empty(_workspace_bytes(batch, heads, k.shape[1], tokens, k.shape[2]), device=q.device,
                         dtype=torch.uint8)
        check(LIB.b2_attention_backward(
            with_base(q, tails[0]), with_base(k, tails[1]), with_base(v, tails[2]), out_view, low_view, dout_view,
            ptr(lse), with_base(dq, grad_tails[0]), with_base(dk, grad_tails[1]), with_base(dv, grad_tails[1]), scale,
            1 if causal else 0, ptr(key_lengths), ptr(ws), raw_stream(q)))
    return dq, dk, dv


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, scale: float | None = None, *, causal: bool = False,
                       key_lengths: torch.Tensor | None = None, out_low: torch.Tensor | None = None):
    """(dq, dk, dv) of attention_forward's call from the gradient of its out
    and what it returned (out_low is optional).  Probabilities are recomputed
    from lse; dk and dv of a shared head are summed over its group in FP32;
    rows of dk and dv past a batch's keys are 0.  Bit-reproducible."""
    refuse_tangents("attention_backward", dout, q, k, v, out, lse, out_low)
    flat = isinstance(q, torch.Tensor) and q.ndim == 3
    q, k, v, plan = _planned(q, k, v, scale, key_lengths)
    out, dout, out_low = check_saved(q, flat, lse, out=out, dout=dout, out_low=out_low)
    require_one_device("attention_backward", q, k, v, key_lengths, out, dout, lse, out_low)
    grads = _run_backward(dout, q, k, v, out, lse, out_low, plan, causal, key_lengths)
    return tuple(g.squeeze(1) for g in grads) if flat else grads


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, key_lengths):
        flat = isinstance(q, torch.Tensor) and q.ndim == 3
        q, k, v, plan = _planned(q, k, v, scale, key_lengths)
        require_one_device("attention", q, k, v, key_lengths)
        out, lse, low = _run_forward(q, k, v, plan, causal, key_lengths, True)
        saved = (q, k, v, out, lse, low, key_lengths)
        ctx.save_for_backward(*saved)
        ctx.call = (plan, causal, flat, layouts(*saved))
        return out.squeeze(1) if flat else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        refuse_tangents("attention", dout)
        saved = ctx.saved_tensors  # each access unpacks them anew
        q, k, v, out, lse, low, key_lengths = saved
        plan, causal, flat, were = ctx.call
        dout = dout.unsqueeze(1) if flat else dout
        require_one_device("attention", *saved, dout)
        if not came_back("attention", saved, were):
            q, k, v = (as_rows(x, broadcast=False)[0] for x in (q, k, v))
            key_lengths = dense(key_lengths)
            q, k, v, plan = _planned(q, k, v, plan[0], key_lengths)
        grads = _run_backward(dout, q, k, v, out, lse, low, plan, causal, key_lengths)
        return (*(g.squeeze(1) if flat else g for g in grads), None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None, *, causal: bool = False,
              key_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v, differentiable in q, k and v (see
    attention_forward for the masks and layouts; scale defaults to D^-0.5).
    Tensors that carry forward-mode tangents are refused."""
    refuse_tangents("attention", q, k, v)
    if torch.compiler.is_compiling():
        scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
        return torch.ops.b200_pisa.attention(q, k, v, scale, bool(causal), key_lengths)[0]
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v)):
        return _Attention.apply(q, k, v, scale, causal, key_lengths)
    return attention_forward(q, k, v, scale, causal=causal, key_lengths=key_lengths)[0]


__all__ = ["attention", "attention_backward", "attention_forward"]

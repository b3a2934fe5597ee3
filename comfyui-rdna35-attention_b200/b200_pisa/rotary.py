"""Rotary positions with several axes, alone (``axial_rope``) or in one pass
with the per-head RMS norm of queries and keys (``qk_norm_rope``): the steps
between a projection and attention.  Both are differentiable; tensors are
[B,H,T,D] views (any strides that keep rows 16-byte aligned, e.g. of an
interleaved [B,T,3,H,D] projection) and results are [B,H,T,D] views of
contiguous [B,T,H,D] storage, which the attention entry points read in place.
"""
from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._args import addressable, on_device, require_one_device, row_view, token_major
from ._lib import LIB, check, ptr, stream_of

MAX_ROTARY_DIM = 256
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_POS_CODES = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64, torch.float32: _lib.POS_F32,
              torch.float64: _lib.POS_F64}


def _check_rows(name: str, x: torch.Tensor) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor.")
    if x.ndim != 4 or 0 in x.shape:
        raise ValueError(f"{name} must be a non-empty [B,H,T,D] tensor.")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name} must be bfloat16, float16 or float32.")
    if x.shape[-1] > MAX_ROTARY_DIM or x.shape[-1] % 8:
        raise ValueError(f"rotary positions support D <= {MAX_ROTARY_DIM}, a multiple of 8.")
    if not addressable(x):
        raise ValueError(f"{name} needs a contiguous head dimension and rows that start on 16-byte boundaries.")


def _rotary(x: torch.Tensor, positions: torch.Tensor, axes_dims: Sequence[int], theta, interleaved: bool,
            inverse: bool) -> _lib.Rotary:
    """Checked b2_rotary of the call; the caller keeps ``positions`` alive."""
    if not isinstance(positions, torch.Tensor):
        raise TypeError("positions must be a torch tensor.")
    dims = [int(d) for d in axes_dims]
    if not 1 <= len(dims) <= _lib.MAX_AXES or any(d <= 0 or d % 2 for d in dims) or sum(dims) > x.shape[-1]:
        raise ValueError(f"axes_dims must be 1..{_lib.MAX_AXES} positive even sizes that sum to at most D={x.shape[-1]}.")
    thetas = [float(t) for t in theta] if isinstance(theta, Sequence) else [float(theta)] * len(dims)
    if len(thetas) != len(dims) or not all(0.0 < t < math.inf for t in thetas):
        raise ValueError("theta must be one positive number, or one for each axis.")
    batch, _, tokens, _ = x.shape
    if positions.dtype not in _POS_CODES:
        raise ValueError("positions must be int32, int64, float32 or float64.")
    if positions.requires_grad:
        raise ValueError("positions have no gradient here; detach them.")
    if tuple(positions.shape) not in ((tokens, len(dims)), (batch, tokens, len(dims))):
        raise ValueError(f"positions must be [T,{len(dims)}] or [B,T,{len(dims)}] with B={batch}, T={tokens}.")
    sb, st, sa = positions.stride() if positions.ndim == 3 else (0, *positions.stride())
    rot = _lib.Rotary(positions.data_ptr(), sb, st, sa, _POS_CODES[positions.dtype], len(dims))
    rot.axes_dims[:len(dims)] = dims
    rot.theta[:len(dims)] = thetas
    rot.interleaved, rot.inverse = int(bool(interleaved)), int(bool(inverse))
    return rot


def _rope_call(x: torch.Tensor, positions: torch.Tensor, axes_dims, theta, interleaved, inverse) -> torch.Tensor:
    rot = _rotary(x, positions, axes_dims, theta, interleaved, inverse)
    require_one_device("axial_rope", x, positions)
    with on_device(x):
        out = token_major(x)
        check(LIB.b2_axial_rope(ctypes.byref(row_view(x)), ctypes.byref(row_view(out)), ctypes.byref(rot), stream_of(x)))
    return out


class _AxialRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, *rotation):
        ctx.save_for_backward(positions)
        ctx.rotation = rotation
        return _rope_call(x, positions, *rotation)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        axes_dims, theta, interleaved, inverse = ctx.rotation
        (positions,) = ctx.saved_tensors
        dy = dy if addressable(dy) else dy.contiguous()
        return _rope_call(dy, positions, axes_dims, theta, interleaved, not inverse), None, None, None, None, None


def axial_rope(x: torch.Tensor, positions: torch.Tensor, axes_dims: Sequence[int], *, theta=10000.0,
               interleaved: bool = True, inverse: bool = False) -> torch.Tensor:
    """Rotate the first R = sum(axes_dims) columns of x [B,H,T,D] by the
    tokens' positions; the other columns pass through.

    positions: [T,A] or [B,T,A] (int32, int64, float32 or float64, any
    strides) gives a position on each of the A axes; axis a drives
    axes_dims[a] columns with rates theta^(-2j/axes_dims[a]) (``theta`` may
    be one number per axis).  interleaved: pair p is columns (2p, 2p+1), else
    (p, p + R/2).  inverse rotates back.  Angles are reduced in FP64, so far
    positions keep their accuracy; the result is rounded once to x's type.
    Differentiable in x."""
    _check_rows("x", x)
    rotation = (tuple(axes_dims), theta, interleaved, inverse)
    if torch.is_grad_enabled() and x.requires_grad:
        return _AxialRope.apply(x, positions, *rotation)
    return _rope_call(x, positions, *rotation)


def _check_weight(name: str, w: torch.Tensor | None, x: torch.Tensor) -> None:
    if w is None:
        return
    if not isinstance(w, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor or None.")
    if w.shape != (x.shape[-1],) or w.dtype not in _DTYPES:
        raise ValueError(f"{name} must be a [D] bfloat16, float16 or float32 tensor, D={x.shape[-1]}.")
    if w.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous.")


def _check_qk(q, k, q_weight, k_weight, eps) -> float:
    _check_rows("q", q)
    _check_rows("k", k)
    if q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:] or q.dtype != k.dtype:
        raise ValueError("q and k must share B, T, D and dtype (head counts may differ).")
    _check_weight("q_weight", q_weight, q)
    _check_weight("k_weight", k_weight, k)
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must share one dtype.")
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError("eps must be a finite number >= 0.")
    return eps


def _weight_code(q_weight, k_weight) -> int:
    w = q_weight if q_weight is not None else k_weight
    return _lib.B2_F32 if w is None else _lib.dtype_code(w.dtype)


def _norm_rope_call(q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved):
    rot = _rotary(q, positions, axes_dims, theta, interleaved, False)
    require_one_device("qk_norm_rope", q, k, q_weight, k_weight, positions)
    with on_device(q):
        q_out, k_out = token_major(q), token_major(k)
        check(LIB.b2_qk_norm_rope(ctypes.byref(row_view(q)), ctypes.byref(row_view(k)), ctypes.byref(row_view(q_out)),
                                  ctypes.byref(row_view(k_out)), ptr(q_weight), ptr(k_weight),
                                  _weight_code(q_weight, k_weight), eps, ctypes.byref(rot), stream_of(q)))
    return q_out, k_out


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, positions: torch.Tensor,
                          axes_dims: Sequence[int], *, eps: float = 1e-6, theta=10000.0, interleaved: bool = True,
                          weight_grads: bool = True):
    """Gradients of qk_norm_rope: (q_grad, k_grad, q_weight_grad,
    k_weight_grad) from the gradients of its two outputs; the weights' are
    None without weights or with weight_grads=False.  The statistics are
    recomputed from q and k.  Bit-reproducible."""
    eps = _check_qk(q, k, q_weight, k_weight, eps)
    for name, dy, x in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        if not isinstance(dy, torch.Tensor) or dy.shape != x.shape or dy.dtype != x.dtype:
            raise ValueError(f"{name} must be a tensor of its output's shape and dtype.")
    rot = _rotary(q, positions, axes_dims, theta, interleaved, False)
    require_one_device("qk_norm_rope_backward", q, k, dq_out, dk_out, q_weight, k_weight, positions)
    dq_out, dk_out = (x if addressable(x) else x.contiguous() for x in (dq_out, dk_out))
    with on_device(q):
        dq, dk = token_major(q), token_major(k)
        dwq, dwk = (torch.empty_like(w) if w is not None and weight_grads else None for w in (q_weight, k_weight))
        ws = None
        if dwq is not None or dwk is not None:
            ws = torch.empty(LIB.b2_qk_norm_rope_workspace_bytes(q.shape[-1]), device=q.device, dtype=torch.uint8)
        views = [ctypes.byref(row_view(x)) for x in (q, k, dq_out, dk_out, dq, dk)]
        check(LIB.b2_qk_norm_rope_backward(*views, ptr(q_weight), ptr(k_weight), _weight_code(q_weight, k_weight), eps,
                                           ctypes.byref(rot), ptr(dwq), ptr(dwk), ptr(ws), stream_of(q)))
    return dq, dk, dwq, dwk


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.rotation = dict(axes_dims=axes_dims, eps=eps, theta=theta, interleaved=interleaved)
        return _norm_rope_call(q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        wanted = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        grads = qk_norm_rope_backward(dq_out, dk_out, *ctx.saved_tensors, weight_grads=wanted, **ctx.rotation)
        return (*grads, None, None, None, None, None)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 positions: torch.Tensor, axes_dims: Sequence[int], *, eps: float = 1e-6, theta=10000.0,
                 interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS-norm every row of q [B,Hq,T,D] and k [B,Hk,T,D] over D, scale it by
    its weight [D] (None for none) and rotate it by the tokens' positions
    (``axial_rope``), in one launch with one rounding at the end.
    Differentiable in q, k and the weights."""
    eps = _check_qk(q, k, q_weight, k_weight, eps)
    args = (q, k, q_weight, k_weight, positions, tuple(axes_dims), eps, theta, interleaved)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRope.apply(*args)
    return _norm_rope_call(*args)


__all__ = ["MAX_ROTARY_DIM", "axial_rope", "qk_norm_rope", "qk_norm_rope_backward"]

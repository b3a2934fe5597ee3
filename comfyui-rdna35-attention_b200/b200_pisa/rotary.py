"""Rotary positions with several axes, alone (``axial_rope``) or in one pass
with the per-head RMS norm of queries and keys (``qk_norm_rope``): the steps
between a projection and attention.  Both are differentiable; tensors are
[B,H,T,D] views (any strides that keep rows 16-byte aligned, e.g. of an
interleaved [B,T,3,H,D] projection) and results are [B,H,T,D] views of
contiguous [B,T,H,D] storage, which the attention entry points read in place.
"""
from __future__ import annotations

import functools
import math
import operator
import struct
from collections.abc import Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._args import (PLANS, addressable, as_rows, came_back, dense, layouts, new_rows, on_device, raw_stream, refuse_tangents,
                    require_one_device, signature, token_major_strides, view_tail, with_base)
from ._lib import LIB, check, ptr

MAX_ROTARY_DIM = 256
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_POS_CODES = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64, torch.float32: _lib.POS_F32,
              torch.float64: _lib.POS_F64}
_ROTARY_TAIL = struct.Struct("=qqqii4iii4d")
assert 8 + _ROTARY_TAIL.size == _lib.ctypes.sizeof(_lib.Rotary)


def _check_rows(name: str, shape, strides, dtype) -> None:
    if len(shape) != 4 or 0 in shape:
        raise ValueError(f"{name} must be a non-empty [B,H,T,D] tensor.")
    if dtype not in _DTYPES:
        raise ValueError(f"{name} must be bfloat16, float16 or float32.")
    if shape[-1] > MAX_ROTARY_DIM or shape[-1] % 8:
        raise ValueError(f"rotary positions support D <= {MAX_ROTARY_DIM}, a multiple of 8.")
    if not addressable(shape, strides, dtype):
        raise ValueError(f"{name} needs a contiguous head dimension and rows that start on 16-byte boundaries.")


def _check_tensors(**tensors) -> None:
    """What a plan cannot know: that these are tensors, and their addresses."""
    for name, x in tensors.items():
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor.")
        if name != "positions" and x.data_ptr() % 16:
            raise ValueError(f"{name} needs a contiguous head dimension and rows that start on 16-byte boundaries.")


def _rotary_tail(shape, pos_sig, axes_dims, theta, interleaved: bool, inverse: bool) -> bytes:
    """The checked b2_rotary of a call without the positions' address."""
    dims = list(axes_dims)
    if not 1 <= len(dims) <= _lib.MAX_AXES or any(d <= 0 or d % 2 for d in dims) or sum(dims) > shape[-1]:
        raise ValueError(f"axes_dims must be 1..{_lib.MAX_AXES} positive even sizes that sum to at most D={shape[-1]}.")
    thetas = rates(dims, theta)
    if len(thetas) != len(dims) or not all(0.0 < t < math.inf for t in thetas):
        raise ValueError("theta must be one positive number, or one for each axis.")
    batch, _, tokens, _ = shape
    pos_shape, strides, dtype = pos_sig
    if dtype not in _POS_CODES:
        raise ValueError("positions must be int32, int64, float32 or float64.")
    if tuple(pos_shape) not in ((tokens, len(dims)), (batch, tokens, len(dims))):
        raise ValueError(f"positions must be [T,{len(dims)}] or [B,T,{len(dims)}] with B={batch}, T={tokens}.")
    strides = strides if len(strides) == 3 else (0, *strides)
    pad = [0] * (_lib.MAX_AXES - len(dims))
    return _ROTARY_TAIL.pack(*strides, _POS_CODES[dtype], len(dims), *dims, *pad, interleaved, inverse, *thetas, *pad)


def _hashable(axes_dims, theta):
    """The rotation's sizes and rates as plain numbers, for the plan's key."""
    theta = tuple(float(t) for t in theta) if isinstance(theta, Sequence) else float(theta)
    return tuple(operator.index(d) for d in axes_dims), theta


def rates(axes_dims, theta) -> list[float]:
    """theta of each axis, as the custom ops take it."""
    return list(theta) if isinstance(theta, tuple) else [theta] * len(axes_dims)


@functools.lru_cache(maxsize=PLANS)
def _rope_plan(sig, pos_sig, axes_dims, theta, interleaved, inverse):
    _check_rows("x", *sig)
    shape, _, dtype = sig
    out_strides = token_major_strides(shape)
    return (_rotary_tail(shape, pos_sig, axes_dims, theta, interleaved, inverse), view_tail(*sig),
            view_tail(shape, out_strides, dtype), out_strides)


def _no_position_gradient(positions) -> None:
    if isinstance(positions, torch.Tensor) and positions.requires_grad:
        raise ValueError("positions have no gradient here; detach them.")


def _rope_call(x: torch.Tensor, positions: torch.Tensor, axes_dims, theta, interleaved, inverse) -> torch.Tensor:
    _check_tensors(x=x, positions=positions)
    _no_position_gradient(positions)
    rot, tail, out_tail, out_strides = _rope_plan(signature(x), signature(positions), axes_dims, theta, interleaved, inverse)
    require_one_device("axial_rope", x, positions)
    with on_device(x):
        out = new_rows(x, x.shape, out_strides)
        check(LIB.b2_axial_rope(with_base(x, tail), with_base(out, out_tail), with_base(positions, rot), raw_stream(x)))
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
        refuse_tangents("axial_rope", dy)
        axes_dims, theta, interleaved, inverse = ctx.rotation
        (positions,) = ctx.saved_tensors
        return _rope_call(as_rows(dy)[0], positions, axes_dims, theta, interleaved, not inverse), None, None, None, None, None


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
    Differentiable in x (reverse mode; tangents are refused)."""
    refuse_tangents("axial_rope", x, positions)
    rotation = (*_hashable(axes_dims, theta), bool(interleaved), bool(inverse))
    if torch.compiler.is_compiling():
        _no_position_gradient(positions)  # the op would not see it
        return torch.ops.b200_pisa.axial_rope(x, positions, rotation[0], rates(*rotation[:2]), *rotation[2:])
    if torch.is_grad_enabled() and isinstance(x, torch.Tensor) and x.requires_grad:
        return _AxialRope.apply(x, positions, *rotation)
    return _rope_call(x, positions, *rotation)


def _check_weight(name: str, sig, dim: int) -> None:
    if sig is None:
        return
    shape, strides, dtype = sig
    if tuple(shape) != (dim,) or dtype not in _DTYPES:
        raise ValueError(f"{name} must be a [D] bfloat16, float16 or float32 tensor, D={dim}.")
    if strides[0] != 1:
        raise ValueError(f"{name} must be contiguous.")


@functools.lru_cache(maxsize=PLANS)
def _qk_plan(q_sig, k_sig, wq_sig, wk_sig, pos_sig, axes_dims, eps, theta, interleaved):
    _check_rows("q", *q_sig)
    _check_rows("k", *k_sig)
    q_shape, k_shape, dtype = q_sig[0], k_sig[0], q_sig[2]
    if q_shape[0] != k_shape[0] or q_shape[2:] != k_shape[2:] or dtype != k_sig[2]:
        raise ValueError("q and k must share B, T, D and dtype (head counts may differ).")
    _check_weight("q_weight", wq_sig, q_shape[-1])
    _check_weight("k_weight", wk_sig, q_shape[-1])
    if wq_sig is not None and wk_sig is not None and wq_sig[2] != wk_sig[2]:
        raise ValueError("q_weight and k_weight must share one dtype.")
    if not 0.0 <= eps < math.inf:
        raise ValueError("eps must be a finite number >= 0.")
    weight = wq_sig or wk_sig
    strides = tuple(token_major_strides(s) for s in (q_shape, k_shape))
    return (_rotary_tail(q_shape, pos_sig, axes_dims, theta, interleaved, False),
            (view_tail(*q_sig), view_tail(*k_sig)),
            tuple(view_tail(s, st, dtype) for s, st in zip((q_shape, k_shape), strides)), strides,
            _lib.B2_F32 if weight is None else _lib.dtype_code(weight[2]))


def _plan_of(q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved):
    _check_tensors(q=q, k=k, positions=positions)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and not isinstance(w, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor or None.")
    _no_position_gradient(positions)
    return _qk_plan(signature(q), signature(k), None if q_weight is None else signature(q_weight),
                    None if k_weight is None else signature(k_weight), signature(positions), axes_dims, eps, theta,
                    interleaved)


def _norm_rope_call(q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved):
    plan = _plan_of(q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved)
    return _run_norm_rope(q, k, q_weight, k_weight, positions, eps, plan)


def _run_norm_rope(q, k, q_weight, k_weight, positions, eps, plan):
    rot, tails, out_tails, strides, w_code = plan
    require_one_device("qk_norm_rope", q, k, q_weight, k_weight, positions)
    with on_device(q):
        q_out, k_out = new_rows(q, q.shape, strides[0]), new_rows(k, k.shape, strides[1])
        check(LIB.b2_qk_norm_rope(with_base(q, tails[0]), with_base(k, tails[1]), with_base(q_out, out_tails[0]),
                                  with_base(k_out, out_tails[1]), ptr(q_weight), ptr(k_weight), w_code, eps,
                                  with_base(positions, rot), raw_stream(q)))
    return q_out, k_out


def _run_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, positions, eps, plan, weight_grads: bool):
    """The pass on checked tensors."""
    rot, tails, out_tails, strides, w_code = plan
    with on_device(q):
        (dq_out, dq_view), (dk_out, dk_view) = as_rows(dq_out), as_rows(dk_out)
        dq, dk = new_rows(q, q.shape, strides[0]), new_rows(k, k.shape, strides[1])
        dwq, dwk = (torch.empty_like(w) if w is not None and weight_grads else None for w in (q_weight, k_weight))
        ws = None
        if dwq is not None or dwk is not None:
            ws = torch.empty(_workspace_bytes(q.shape[-1]), device=q.device, dtype=torch.uint8)
        check(LIB.b2_qk_norm_rope_backward(
            with_base(q, tails[0]), with_base(k, tails[1]), dq_view, dk_view, with_base(dq, out_tails[0]),
            with_base(dk, out_tails[1]), ptr(q_weight), ptr(k_weight), w_code, eps, with_base(positions, rot), ptr(dwq),
            ptr(dwk), ptr(ws), raw_stream(q)))
    return dq, dk, dwq, dwk


@functools.lru_cache(maxsize=PLANS)
def _workspace_bytes(dim: int) -> int:
    return LIB.b2_qk_norm_rope_workspace_bytes(dim)


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, positions: torch.Tensor,
                          axes_dims: Sequence[int], *, eps: float = 1e-6, theta=10000.0, interleaved: bool = True,
                          weight_grads: bool = True):
    """Gradients of qk_norm_rope: (q_grad, k_grad, q_weight_grad,
    k_weight_grad) from the gradients of its two outputs; the weights' are
    None without weights or with weight_grads=False.  The statistics are
    recomputed from q and k.  Bit-reproducible."""
    refuse_tangents("qk_norm_rope_backward", dq_out, dk_out, q, k, q_weight, k_weight, positions)
    axes_dims, theta = _hashable(axes_dims, theta)
    plan = _plan_of(q, k, q_weight, k_weight, positions, axes_dims, float(eps), theta, bool(interleaved))
    for name, dy, x in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        if not isinstance(dy, torch.Tensor) or dy.shape != x.shape or dy.dtype != x.dtype:
            raise ValueError(f"{name} must be a tensor of its output's shape and dtype.")
    require_one_device("qk_norm_rope_backward", q, k, q_weight, k_weight, positions, dq_out, dk_out)
    return _run_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, positions, float(eps), plan, weight_grads)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved):
        saved = (q, k, q_weight, k_weight, positions)
        ctx.save_for_backward(*saved)
        plan = _plan_of(*saved, axes_dims, eps, theta, interleaved)
        ctx.call = (axes_dims, eps, theta, interleaved)
        ctx.plan, ctx.layouts = plan, layouts(*saved)
        return _run_norm_rope(q, k, q_weight, k_weight, positions, eps, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        refuse_tangents("qk_norm_rope", dq_out, dk_out)
        wanted = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        saved, plan = ctx.saved_tensors, ctx.plan
        require_one_device("qk_norm_rope", *saved, dq_out, dk_out)
        if not came_back("qk_norm_rope", saved, ctx.layouts):
            q, k, q_weight, k_weight, positions = saved
            saved = (as_rows(q)[0], as_rows(k)[0], dense(q_weight), dense(k_weight), positions)
            plan = _plan_of(*saved, *ctx.call)
        grads = _run_norm_rope_backward(dq_out, dk_out, *saved, ctx.call[1], plan, wanted)
        return (*grads, None, None, None, None, None)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 positions: torch.Tensor, axes_dims: Sequence[int], *, eps: float = 1e-6, theta=10000.0,
                 interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS-norm every row of q [B,Hq,T,D] and k [B,Hk,T,D] over D, scale it by
    its weight [D] (None for none) and rotate it by the tokens' positions
    (``axial_rope``), in one launch with one rounding at the end.
    Differentiable in q, k and the weights (reverse mode; tangents are
    refused)."""
    refuse_tangents("qk_norm_rope", q, k, q_weight, k_weight, positions)
    axes_dims, theta = _hashable(axes_dims, theta)
    if torch.compiler.is_compiling():
        _no_position_gradient(positions)
        return torch.ops.b200_pisa.qk_norm_rope(q, k, q_weight, k_weight, positions, axes_dims, float(eps),
                                                rates(axes_dims, theta), bool(interleaved))
    args = (q, k, q_weight, k_weight, positions, axes_dims, float(eps), theta, bool(interleaved))
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args[:4]):
        return _QkNormRope.apply(*args)
    return _norm_rope_call(*args)


__all__ = ["MAX_ROTARY_DIM", "axial_rope", "qk_norm_rope", "qk_norm_rope_backward"]

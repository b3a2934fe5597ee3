"""torch.library custom ops of the rotary and the differentiable attention
entry points, with fakes and gradients, so that torch.compile keeps them in one
graph.  The public functions take these only while a graph is traced; eager
calls go to the library directly and save the dispatcher's share of a call."""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch import Tensor

from . import exact, fused, rotary
from ._args import as_rows, token_major_strides


def _like(x: Tensor) -> Tensor:
    return x.new_empty_strided(x.shape, token_major_strides(x.shape))


def _present(x: Tensor | None, like: Tensor) -> Tensor:
    """Ops return tensors: an empty one stands for None."""
    return like.new_empty(0) if x is None else x


def _optional(x: Tensor) -> Tensor | None:
    return x if x.numel() else None


# ---------------------------------------------------------------- axial_rope
@torch.library.custom_op("b200_pisa::axial_rope", mutates_args=(), device_types="cuda")
def axial_rope_op(x: Tensor, positions: Tensor, axes_dims: Sequence[int], theta: Sequence[float], interleaved: bool,
                  inverse: bool) -> Tensor:
    return rotary._rope_call(as_rows(x)[0], positions, tuple(axes_dims), tuple(theta), interleaved, inverse)


@axial_rope_op.register_fake
def _(x, positions, axes_dims, theta, interleaved, inverse):
    return _like(x)


def _rope_context(ctx, inputs, output):
    _, positions, *ctx.rotation = inputs
    ctx.save_for_backward(positions)


def _rope_backward(ctx, dy):
    axes_dims, theta, interleaved, inverse = ctx.rotation
    return axial_rope_op(dy, ctx.saved_tensors[0], axes_dims, theta, interleaved, not inverse), None, None, None, None, None


axial_rope_op.register_autograd(_rope_backward, setup_context=_rope_context)


# ---------------------------------------------------------------- qk_norm_rope
@torch.library.custom_op("b200_pisa::qk_norm_rope", mutates_args=(), device_types="cuda")
def qk_norm_rope_op(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor], positions: Tensor,
                    axes_dims: Sequence[int], eps: float, theta: Sequence[float],
                    interleaved: bool) -> tuple[Tensor, Tensor]:
    return rotary._norm_rope_call(q, k, q_weight, k_weight, positions, tuple(axes_dims), eps, tuple(theta), interleaved)


@qk_norm_rope_op.register_fake
def _(q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved):
    return _like(q), _like(k)


@torch.library.custom_op("b200_pisa::qk_norm_rope_backward", mutates_args=(), device_types="cuda")
def qk_norm_rope_backward_op(dq_out: Tensor, dk_out: Tensor, q: Tensor, k: Tensor, q_weight: Optional[Tensor],
                             k_weight: Optional[Tensor], positions: Tensor, axes_dims: Sequence[int], eps: float,
                             theta: Sequence[float], interleaved: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    dq, dk, *dw = rotary.qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, positions, axes_dims, eps=eps,
                                               theta=tuple(theta), interleaved=interleaved)
    return dq, dk, _present(dw[0], q), _present(dw[1], q)


def _weight_fake(w: Tensor | None, q: Tensor) -> Tensor:
    return q.new_empty(0) if w is None else torch.empty_like(w)


@qk_norm_rope_backward_op.register_fake
def _(dq_out, dk_out, q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved):
    return _like(q), _like(k), _weight_fake(q_weight, q), _weight_fake(k_weight, q)


def _norm_context(ctx, inputs, output):
    *tensors, axes_dims, eps, theta, interleaved = inputs
    ctx.save_for_backward(*tensors)
    ctx.rotation = (axes_dims, eps, theta, interleaved)


def _norm_backward(ctx, dq_out, dk_out):
    dq, dk, dwq, dwk = qk_norm_rope_backward_op(dq_out, dk_out, *ctx.saved_tensors, *ctx.rotation)
    return dq, dk, _optional(dwq), _optional(dwk), None, None, None, None, None


qk_norm_rope_op.register_autograd(_norm_backward, setup_context=_norm_context)


# ---------------------------------------------------------------- attention
@torch.library.custom_op("b200_pisa::attention", mutates_args=(), device_types="cuda")
def attention_op(q: Tensor, k: Tensor, v: Tensor, scale: float, causal: bool,
                 key_lengths: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor]:
    out, lse, low = exact.attention_forward(q, k, v, scale, causal=causal, key_lengths=key_lengths, with_low=True)
    return out, lse, _present(low, q)


@attention_op.register_fake
def _(q, k, v, scale, causal, key_lengths):
    four = q if q.ndim == 4 else q.unsqueeze(1)
    rows = lambda: _like(four) if q.ndim == 4 else _like(four).squeeze(1)  # noqa: E731
    low = rows() if exact.wants_low(q.dtype, k.shape[-2], key_lengths, causal) else q.new_empty(0)
    return rows(), q.new_empty(q.shape[:-1], dtype=torch.float32), low


@torch.library.custom_op("b200_pisa::attention_backward", mutates_args=(), device_types="cuda")
def attention_backward_op(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, low: Tensor, scale: float,
                          causal: bool, key_lengths: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor]:
    return exact.attention_backward(dout, q, k, v, out, lse, scale, causal=causal, key_lengths=key_lengths,
                                    out_low=_optional(low))


@attention_backward_op.register_fake
def _(dout, q, k, v, out, lse, low, scale, causal, key_lengths):
    return tuple(_like(x) if x.ndim == 4 else _like(x.unsqueeze(1)).squeeze(1) for x in (q, k, v))


def _attention_context(ctx, inputs, output):
    q, k, v, scale, causal, key_lengths = inputs
    ctx.save_for_backward(q, k, v, *output, key_lengths)
    ctx.call = (scale, causal)


def _attention_backward(ctx, dout, dlse, dlow):
    *saved, key_lengths = ctx.saved_tensors
    return (*attention_backward_op(dout, *saved, *ctx.call, key_lengths), None, None, None)


attention_op.register_autograd(_attention_backward, setup_context=_attention_context)


# ---------------------------------------------------------------- norm_rope_attention
@torch.library.custom_op("b200_pisa::norm_rope_attention", mutates_args=(), device_types="cuda")
def norm_rope_attention_op(q: Tensor, k: Tensor, v: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                           positions: Tensor, axes_dims: Sequence[int], scale: float, eps: float, theta: Sequence[float],
                           interleaved: bool, causal: bool,
                           key_lengths: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    call = (tuple(axes_dims), scale, eps, tuple(theta), interleaved, causal, key_lengths)
    out, lse, low, saved = fused._forward(q, k, v, q_weight, k_weight, positions, call, True)
    return out, lse, _present(low, q), saved


@norm_rope_attention_op.register_fake
def _(q, k, v, q_weight, k_weight, positions, axes_dims, scale, eps, theta, interleaved, causal, key_lengths):
    batch, heads, tokens, dim = q.shape
    low = _like(q) if exact.wants_low(q.dtype, tokens, key_lengths, causal) else q.new_empty(0)
    saved = fused.saved_size(batch, heads, k.shape[1], tokens, dim)
    return _like(q), q.new_empty(q.shape[:3], dtype=torch.float32), low, q.new_empty(saved, dtype=torch.uint8)


@torch.library.custom_op("b200_pisa::norm_rope_attention_backward", mutates_args=(), device_types="cuda")
def norm_rope_attention_backward_op(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, q_weight: Optional[Tensor],
                                    k_weight: Optional[Tensor], positions: Tensor, out: Tensor, lse: Tensor, low: Tensor,
                                    saved: Tensor, axes_dims: Sequence[int], scale: float, eps: float,
                                    theta: Sequence[float], interleaved: bool, causal: bool,
                                    key_lengths: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    call = (tuple(axes_dims), scale, eps, tuple(theta), interleaved, causal, key_lengths)
    dq, dk, dv, dwq, dwk = fused._backward(dout, q, k, v, q_weight, k_weight, positions, out, lse, _optional(low), saved,
                                           call, True)
    return dq, dk, dv, _present(dwq, q), _present(dwk, q)


@norm_rope_attention_backward_op.register_fake
def _(dout, q, k, v, q_weight, k_weight, positions, out, lse, low, saved, axes_dims, scale, eps, theta, interleaved, causal,
      key_lengths):
    return _like(q), _like(k), _like(v), _weight_fake(q_weight, q), _weight_fake(k_weight, q)


def _fused_context(ctx, inputs, output):
    *tensors, axes_dims, scale, eps, theta, interleaved, causal, key_lengths = inputs
    ctx.save_for_backward(*tensors, *output, key_lengths)
    ctx.call = (axes_dims, scale, eps, theta, interleaved, causal)


def _fused_backward(ctx, dout, dlse, dlow, dsaved):
    *saved, key_lengths = ctx.saved_tensors
    dq, dk, dv, dwq, dwk = norm_rope_attention_backward_op(dout, *saved, *ctx.call, key_lengths)
    return dq, dk, dv, _optional(dwq), _optional(dwk), *([None] * 8)


norm_rope_attention_op.register_autograd(_fused_backward, setup_context=_fused_context)

"""Norm, rotation and attention of a layer as one differentiable operator.

``qk_norm_rope`` followed by ``attention`` rounds the normed and rotated
queries and keys, and their gradients, to the model's type in between; in BF16
those four roundings are most of the error of the layer's gradients.
``norm_rope_attention`` keeps them in the library: FP16 held times a power of
two for the products, FP32 for the gradients.  Same kernels otherwise, and the
same results within the rounding it saves."""
from __future__ import annotations

import functools
from collections.abc import Sequence

import torch
from torch.autograd.function import once_differentiable

from . import exact, rotary
from ._args import (as_rows, came_back, dense, layouts, new_rows, on_device, raw_stream, refuse_tangents, require_one_device,
                    with_base)
from ._lib import LIB, check, ptr


@functools.lru_cache(maxsize=256)
def saved_bytes(batch: int, heads: int, kv_heads: int, tokens: int, dim: int) -> tuple[int, int]:
    sizes = (batch, heads, kv_heads, tokens, dim)
    return LIB.b2_norm_rope_attention_saved_bytes(*sizes), LIB.b2_norm_rope_attention_workspace_bytes(*sizes)


def saved_size(batch, heads, kv_heads, tokens, dim):
    """saved_bytes()[0] of sizes that need not be numbers: a traced call's are
    symbols, which neither a cache nor the library takes.  FP16 queries and keys
    and two FP32 scales, each from a multiple of 256 bytes."""
    queries, keys = (2 * batch * h * tokens * dim for h in (heads, kv_heads))
    return (queries + 255) // 256 * 256 + (keys + 255) // 256 * 256 + 256


def _checked(q, k, v, q_weight, k_weight, positions, call):
    """Both operators' checks; (q, k, v, rotation plan, attention plan)."""
    axes_dims, scale, eps, theta, interleaved, causal, key_lengths = call
    for name, x in (("q", q), ("k", k), ("v", v)):
        if isinstance(x, torch.Tensor) and x.ndim != 4:
            raise ValueError(f"{name} must be a non-empty [B,H,T,D] tensor.")
    q, k, v, attention = exact._planned(q, k, v, scale, key_lengths)
    rotation = rotary._plan_of(q, k, q_weight, k_weight, positions, axes_dims, eps, theta, interleaved)
    return q, k, v, rotation, attention


def _forward(q, k, v, q_weight, k_weight, positions, call, with_low: bool):
    q, k, v, *plans = _checked(q, k, v, q_weight, k_weight, positions, call)
    require_one_device("norm_rope_attention", q, k, v, q_weight, k_weight, positions, call[-1])
    return _run_forward(q, k, v, q_weight, k_weight, positions, call, plans, with_low)


def _run_forward(q, k, v, q_weight, k_weight, positions, call, plans, with_low: bool):
    """The pass on checked tensors."""
    _, _, eps, _, _, causal, key_lengths = call
    (rot, _, _, _, w_code), (scale, _, tails, strides, out_tails) = plans
    batch, heads, tokens, dim = q.shape
    with on_device(q):
        out = new_rows(q, q.shape, strides[0])
        low = exact.new_low(q, strides[0], tokens, key_lengths, causal) if with_low else None
        lse = torch.empty((batch, heads, tokens), device=q.device, dtype=torch.float32)
        saved = torch.empty(saved_bytes(batch, heads, k.shape[1], tokens, dim)[0], device=q.device, dtype=torch.uint8)
        check(LIB.b2_norm_rope_attention_forward(
            with_base(q, tails[0]), with_base(k, tails[1]), with_base(v, tails[2]), with_base(out, out_tails[0]),
            ptr(q_weight), ptr(k_weight), w_code, eps, with_base(positions, rot), scale, 1 if causal else 0,
            ptr(key_lengths), ptr(saved), ptr(lse), exact.with_optional(low, out_tails[0]), raw_stream(q)))
    return out, lse, low, saved


def _backward(dout, q, k, v, q_weight, k_weight, positions, out, lse, low, saved, call, weight_grads: bool):
    q, k, v, *plans = _checked(q, k, v, q_weight, k_weight, positions, call)
    return _run_backward(dout, q, k, v, q_weight, k_weight, positions, out, lse, low, saved, call, plans, weight_grads)


def _run_backward(dout, q, k, v, q_weight, k_weight, positions, out, lse, low, saved, call, plans, weight_grads: bool):
    _, _, eps, _, _, causal, key_lengths = call
    (rot, _, _, _, w_code), (scale, _, tails, strides, grad_tails) = plans
    batch, heads, tokens, dim = q.shape
    with on_device(q):
        (out, out_view), (dout, dout_view) = as_rows(out, broadcast=False), as_rows(dout, broadcast=False)
        low, low_view = (None, None) if low is None else as_rows(low, broadcast=False)
        lse, saved = dense(lse), dense(saved, 256)
        dq, dk, dv = new_rows(q, q.shape, strides[0]), new_rows(k, k.shape, strides[1]), new_rows(k, k.shape, strides[1])
        dwq, dwk = (torch.empty_like(w) if w is not None and weight_grads else None for w in (q_weight, k_weight))
        ws = torch.empty(saved_bytes(batch, heads, k.shape[1], tokens, dim)[1], device=q.device, dtype=torch.uint8)
        check(LIB.b2_norm_rope_attention_backward(
            with_base(q, tails[0]), with_base(k, tails[1]), with_base(v, tails[2]), out_view, low_view, dout_view, ptr(lse),
            ptr(q_weight), ptr(k_weight), w_code, eps, with_base(positions, rot), scale, 1 if causal else 0,
            ptr(key_lengths), ptr(saved), with_base(dq, grad_tails[0]), with_base(dk, grad_tails[1]),
            with_base(dv, grad_tails[1]), ptr(dwq), ptr(dwk), ptr(ws), raw_stream(q)))
    return dq, dk, dv, dwq, dwk


class _NormRopeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_weight, k_weight, positions, call):
        q, k, v, *plans = _checked(q, k, v, q_weight, k_weight, positions, call)
        require_one_device("norm_rope_attention", q, k, v, q_weight, k_weight, positions, call[-1])
        out, lse, low, saved = _run_forward(q, k, v, q_weight, k_weight, positions, call, plans, True)
        kept = (q, k, v, q_weight, k_weight, positions, out, lse, low, saved, call[-1])
        ctx.save_for_backward(*kept)
        ctx.call, ctx.plans, ctx.layouts = call[:-1], plans, layouts(*kept)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        refuse_tangents("norm_rope_attention", dout)
        kept = ctx.saved_tensors  # each access unpacks them anew
        q, k, v, q_weight, k_weight, positions, *results, key_lengths = kept
        wanted = ctx.needs_input_grad[3] or ctx.needs_input_grad[4]
        call, plans = (*ctx.call, key_lengths), ctx.plans
        require_one_device("norm_rope_attention", *kept, dout)
        if not came_back("norm_rope_attention", kept, ctx.layouts):
            q, k, v = (as_rows(x, broadcast=False)[0] for x in (q, k, v))
            q_weight, k_weight, call = dense(q_weight), dense(k_weight), (*ctx.call, dense(key_lengths))
            q, k, v, *plans = _checked(q, k, v, q_weight, k_weight, positions, call)
        return (*_run_backward(dout, q, k, v, q_weight, k_weight, positions, *results, call, plans, wanted), None, None)


def norm_rope_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor | None,
                        k_weight: torch.Tensor | None, positions: torch.Tensor, axes_dims: Sequence[int],
                        scale: float | None = None, *, eps: float = 1e-6, theta=10000.0, interleaved: bool = True,
                        causal: bool = False, key_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """``attention(*qk_norm_rope(q, k, ...), v)`` without rounding in between:
    q [B,H,T,D], k and v [B,Hk,T,D] (BF16 or FP16, D <= 128), weights [D] or
    None, positions and axes_dims of the rotation, scale, causal and
    key_lengths of the attention (K rows past a batch's keys are not used,
    whatever they hold).  Differentiable in q, k, v and the weights (reverse
    mode; tangents are refused)."""
    refuse_tangents("norm_rope_attention", q, k, v, q_weight, k_weight, positions)
    axes_dims, theta = rotary._hashable(axes_dims, theta)
    if torch.compiler.is_compiling():
        rotary._no_position_gradient(positions)
        scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
        return torch.ops.b200_pisa.norm_rope_attention(q, k, v, q_weight, k_weight, positions, axes_dims, scale, float(eps),
                                                       rotary.rates(axes_dims, theta), bool(interleaved), bool(causal),
                                                       key_lengths)[0]
    call = (axes_dims, None if scale is None else float(scale), float(eps), theta, bool(interleaved), bool(causal),
            key_lengths)
    leaves = (q, k, v, q_weight, k_weight)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in leaves):
        return _NormRopeAttention.apply(*leaves, positions, call)
    return _forward(*leaves, positions, call, False)[0]


__all__ = ["norm_rope_attention"]

"""Norms of queries and keys for each head, with the rotary embedding and the head-first layout in
the same pass: from a layer's projections to what its attention takes.

Per head of D values x of a query or key, with a weight w:

    y = x / sqrt(mean(x^2) + eps) * w,   then y cos + rotate_half(y) sin over its first R dimensions

Values are only moved to their place. :func:`norm_rotary_heads` takes the projections [B, N, heads * D]
and returns q, k, v [B, heads, N, D], as the attention operators take them. It serves whole sequences
and, with ``positions``, single tokens. For queries and keys of length one, as the gated delta rule asks for, give
weights of D^-1/2 (and eps / D).

Types are float32, bfloat16 or float16; sums and arithmetic are in float32, with one rounding at the
end. The backward reads the projections again and keeps nothing else. Results repeat bit by bit
from call to call.

Calls are eager: tracers, functorch's transforms and forward-mode derivatives are refused
(compiled code runs the call between its graphs).
"""

from __future__ import annotations

import math
from typing import Any, Optional

import torch

from . import _native
from .gated_delta import _FLOATS

HEAD_DIM = _native.HEAD_DIM


def _count(value, name: str) -> int:
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{name} must be an int")
    if value <= 0:
        raise ValueError(f"{name} must be positive")
    return value


def _validate(q, k, v, q_weight, k_weight, cos, sin, positions, q_heads, kv_heads, eps) -> None:
    if not all(isinstance(t, torch.Tensor) for t in (q, k, v, cos, sin)):
        raise TypeError("q, k, v, cos and sin must be torch.Tensor objects")
    q_heads, kv_heads = _count(q_heads, "q_heads"), _count(kv_heads, "kv_heads")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)):
        raise TypeError("eps must be a finite Python scalar")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError("q, k and v must be projections [B, N, heads * D]")
    if q.dtype not in _FLOATS:
        raise TypeError("q, k and v must be float16, bfloat16 or float32")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")
    b, n, width = q.shape
    if min(b, n, width) <= 0:
        raise ValueError("q, k and v dimensions must be positive")
    if width % q_heads:
        raise ValueError("q must have the same dimension for each of q_heads heads")
    d = width // q_heads
    if d > HEAD_DIM:
        raise ValueError(f"the HIP kernels support head dimensions up to {HEAD_DIM}")
    if k.shape != (b, n, kv_heads * d) or v.shape != k.shape:
        raise ValueError("k and v must be [B, N, kv_heads * D], with q's batch size, length and head dimension")
    given = [w for w in (q_weight, k_weight) if w is not None]
    for name, w, heads in (("q_weight", q_weight, q_heads), ("k_weight", k_weight, kv_heads)):
        if w is None:
            continue
        if not isinstance(w, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor or None")
        if w.dtype not in (q.dtype, torch.float32):
            raise TypeError(f"{name} must be float32 or have the dtype of q")
        if w.shape != (d,) and w.shape != (heads, d):
            raise ValueError(f"{name} must have shape [D] or [heads, D]")
    if len(given) == 2 and (given[0].dtype != given[1].dtype or given[0].ndim != given[1].ndim):
        raise ValueError("q_weight and k_weight must have the same dtype, and both one row or both one for each head")
    if cos.ndim != 2 or cos.shape != sin.shape:
        raise ValueError("cos and sin must be tables [T, R] of the same shape")
    rows, rotary = cos.shape
    if rotary < 2 or rotary > d or rotary % 2:
        raise ValueError("cos and sin must rotate an even number of dimensions, up to the head dimension")
    if cos.dtype not in (q.dtype, torch.float32) or sin.dtype != cos.dtype:
        raise TypeError("cos and sin must both be float32 or both have the dtype of q")
    if rows < (n if positions is None else 1):
        raise ValueError("cos and sin must have a row for every token")
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be an int32 or int64 tensor")
        if positions.shape != (b, n):
            raise ValueError("positions must have shape [B, N]")
    if any(t.device != q.device for t in (k, v, cos, sin, *given, *([] if positions is None else [positions]))):
        raise ValueError("all tensors must be on the same device")


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _ready(q, k, v, q_weight, k_weight, cos, sin, positions):
    """The operands as the kernels read them."""
    return (*map(_unit_rows, (q, k, v)), *(None if w is None else w.contiguous() for w in (q_weight, k_weight)),
            cos.contiguous(), sin.contiguous(), None if positions is None else positions.to(torch.int64).contiguous())


class _NormRotaryFunction(torch.autograd.Function):
    """(q, k, v, q_weight, k_weight, cos, sin, positions, options) -> head-first (q, k, v), on one ROCm device."""

    @staticmethod
    def forward(ctx: Any, q, k, v, q_weight, k_weight, cos, sin, positions, options: dict):
        ctx.set_materialize_grads(False)
        operands = _ready(q, k, v, q_weight, k_weight, cos, sin, positions)
        outs = _native.norm_rotary_forward(*operands, **options)
        ctx.save_for_backward(*operands[:2], *operands[3:])
        ctx.options = options
        return outs

    @staticmethod
    def backward(ctx: Any, dq, dk, dv):
        if torch.is_grad_enabled():
            raise RuntimeError("norm_rotary_heads does not support double backward")
        if dq is None and dk is None and dv is None:
            return (None,) * 9
        _native.require_eager("norm_rotary_heads", dq, dk, dv)
        ups = [None if t is None else _native._aligned(t.contiguous()) for t in (dq, dk, dv)]
        grads = _native.norm_rotary_backward(*ctx.saved_tensors, ups, ctx.needs_input_grad[:5], **ctx.options)
        return (*(d if need else None for d, need in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def norm_rotary_heads(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor],
    k_weight: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, *, q_heads: int, kv_heads: int,
    eps: float = 1e-6, positions: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Projections to normed, rotated, head-first q, k and to head-first v; differentiable in q, k, v and the weights.

    q [B, N, q_heads * D], k and v [B, N, kv_heads * D] of one dtype, D up to 64, at any strides (slices of one
    projection); q_weight and k_weight [D] or [heads, D], float32 or q's dtype, or None; cos and sin
    [T, R], float32 or q's dtype, R even and up to D: row p serves the token at position p.
    positions [B, N] int32 or int64 (None: 0 .. N - 1 in each sequence): a negative one means no token, whose
    results and gradients are zero; one past the tables gives NaN in its q and k. Returns
    (q [B, q_heads, N, D], k, v [B, kv_heads, N, D]), contiguous.
    """
    _validate(q, k, v, q_weight, k_weight, cos, sin, positions, q_heads, kv_heads, eps)
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise RuntimeError("norm_rotary_heads is not differentiable in cos and sin: detach them")
    _native.require_eager("norm_rotary_heads", q, k, v, q_weight, k_weight, cos, sin, positions)
    _native._require_device(q)
    options = dict(q_heads=q_heads, kv_heads=kv_heads, eps=float(eps))
    operands = (q, k, v, q_weight, k_weight, cos, sin, positions)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands[:5]):
        return _NormRotaryFunction.apply(*operands, options)
    return _native.norm_rotary_forward(*_ready(*operands), **options)  # a step's host time is most of it


__all__ = ("norm_rotary_heads",)

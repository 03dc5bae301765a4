"""Gated delta-rule attention: causal linear attention whose state is a memory that each
token corrects, over whole sequences and token by token.

Per state head, with keys k_t, values v_t, log-decays g_t <= 0 and writing strengths
beta_t in [0, 1]:

    S_t = e^(g_t) S_(t-1) + k_t u_t^T,   u_t = beta_t (v_t - e^(g_t) S_(t-1)^T k_t),
    o_t = scale S_t^T q_t

* :func:`gated_delta_attention` evaluates a whole sequence in chunks of 64 tokens, with
  its backward; it takes and returns the state, so a long text can come in pieces;
* :func:`gated_delta_step` runs the recurrence over one or a few tokens and updates the
  state in place.

Heads: k [B, Hk, ...], v, g, beta and the state [B, Hv, ...], q [B, Hq, ...]. Hk
divides Hv (state head h writes with key head h // (Hv / Hk)), and one of Hq and Hv
divides the other; the output has H = max(Hq, Hv) heads, of which head o reads with
query head o // (H / Hq) from state head o // (H / Hv).

The rule is a stable memory for keys of length one (normalise them before the call)
and beta up to 2. Sums over tokens do not depend on the type of q, k and v, which may be
float32, bfloat16 or float16: states, decays and their gradients are exact to float32.
A token with beta = 0 and g = 0 leaves the state as it is: pad batches of ragged lengths
with such tokens. Values have to be
finite: a token that is not spoils the 64 tokens of its chunk. Results repeat bit by bit from call to call;
long sequences are cut by a rule on batch and heads, so that a sequence's last bits depend on how many others
are in its batch.

Calls are eager: tracers, functorch's transforms and forward-mode derivatives are refused
(compiled code runs the call between its graphs).
"""

from __future__ import annotations

import math
from typing import Any, Optional

import torch

from . import _native

HEAD_DIM = _native.HEAD_DIM
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def _validate_scale(scale, dim: int) -> float:
    if scale is None:
        return dim ** -0.5
    if isinstance(scale, bool) or not isinstance(scale, (int, float)):
        raise TypeError("scale must be a finite Python scalar")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    return float(scale)


def _plain(q, k, v, g, beta, state) -> bool:
    """Whether the operands are as they should be, in one look: it is asked in every call."""
    try:
        (b, hq, n, d), (_, hv, _, dv), hk, dev = q.shape, v.shape, k.shape[1], q.device
        return (
            q.dtype in _FLOATS and k.dtype is v.dtype is q.dtype and g.dtype is torch.float32
            and (beta.dtype is q.dtype or beta.dtype is torch.float32)
            and k.device == dev and v.device == dev and g.device == dev and beta.device == dev
            and k.shape == (b, hk, n, d) and v.shape == (b, hv, n, dv) and g.shape == beta.shape == (b, hv, n)
            and b > 0 and hq > 0 and hk > 0 and hv > 0 and n > 0 and 0 < d <= HEAD_DIM and 0 < dv <= HEAD_DIM
            and hv % hk == 0 and (hq % hv == 0 or hv % hq == 0)
            and (state is None or (state.dtype is torch.float32 and state.shape == (b, hv, d, dv)
                                   and state.device == dev))
        )
    except (AttributeError, ValueError, IndexError):
        return False


def _validate(q, k, v, g, beta, state, name: str) -> None:
    if _plain(q, k, v, g, beta, state):
        return
    if not all(isinstance(t, torch.Tensor) for t in (q, k, v, g, beta)):
        raise TypeError("q, k, v, g and beta must be torch.Tensor objects")
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q, k and v must be rank-4 head-first tensors [B, H, N, D]")
    if q.dtype not in _FLOATS:
        raise TypeError("q, k and v must be float16, bfloat16 or float32")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")
    if g.dtype != torch.float32:
        raise TypeError("g must be float32")
    if beta.dtype not in (q.dtype, torch.float32):
        raise TypeError("beta must be float32 or have the dtype of q, k and v")
    if any(t.device != q.device for t in (k, v, g, beta)):
        raise ValueError("q, k, v, g and beta must be on the same device")
    b, hq, n, d = q.shape
    hk, hv, dv = k.shape[1], v.shape[1], v.shape[3]
    if min(b, hq, hk, hv, n, d, dv) <= 0:
        raise ValueError("q, k and v dimensions must be positive")
    if k.shape != (b, hk, n, d):
        raise ValueError("q and k must have the same batch size, sequence length and feature dimension")
    if v.shape[0] != b or v.shape[2] != n:
        raise ValueError("q, k and v must have the same batch size and sequence length")
    if g.shape != (b, hv, n) or beta.shape != (b, hv, n):
        raise ValueError("g and beta must have shape [B, Hv, N]")
    if hv % hk != 0:
        raise ValueError("value head count must be divisible by key head count")
    if hq % hv != 0 and hv % hq != 0:
        raise ValueError("one of query and value head counts must be divisible by the other")
    if max(d, dv) > HEAD_DIM:
        raise ValueError(f"the HIP kernels support head and value dimensions up to {HEAD_DIM}")
    if state is not None:
        if not isinstance(state, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if state.dtype != torch.float32:
            raise TypeError(f"{name} must be float32")
        if state.shape != (b, hv, d, dv):
            raise ValueError(f"{name} must have shape [B, Hv, D, DV]")
        if state.device != q.device:
            raise ValueError(f"{name} must be on the same device as q")


class _GatedDeltaFunction(torch.autograd.Function):
    """(q, k, v, g, beta, state or None, scale) -> (out, final state); dimensions multiples of 8, on one ROCm device."""

    @staticmethod
    def forward(ctx: Any, q, k, v, g, beta, state, scale: float):
        q, k, v = map(_native.row_tensor, (q, k, v))
        start = None if state is None else _native._aligned(state.contiguous())
        keep = any(ctx.needs_input_grad)
        out, final, saved = _native.delta_forward(q, k, v, g, beta, start, scale=scale, keep=keep)
        if keep:
            ctx.save_for_backward(q, k, v, g, beta, saved)
            ctx.scale = scale
        return out, final

    @staticmethod
    def backward(ctx: Any, dout, dfinal):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_delta_attention does not support double backward")
        _native.require_eager("gated_delta_attention", dout, dfinal)
        q, k, v, g, beta, saved = ctx.saved_tensors
        dout, dfinal = (_native._aligned(t.contiguous()) for t in (dout, dfinal))
        grads = _native.delta_backward(q, k, v, g, beta, saved, dout, dfinal, scale=ctx.scale,
                                       need_state=ctx.needs_input_grad[5])
        return (*(d if need else None for d, need in zip(grads, ctx.needs_input_grad)), None)


def _pad8(x: torch.Tensor) -> torch.Tensor:
    """x with its last dimension at the next multiple of 8, zeros behind."""
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % 8))


def gated_delta_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
    scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Gated delta rule over whole sequences; differentiable in all tensors.

    q [B, Hq, N, D], k [B, Hk, N, D], v [B, Hv, N, DV] of one dtype, D and DV up to 64;
    g [B, Hv, N] float32; beta [B, Hv, N] float32 or q's dtype; initial_state
    [B, Hv, D, DV] float32 (None: zero). scale defaults to D^-1/2. Returns out
    [B, max(Hq, Hv), N, DV] in q's dtype and the state after the last token, contiguous.
    """
    _validate(q, k, v, g, beta, initial_state, "initial_state")
    d, dv = q.shape[3], v.shape[3]
    scale = _validate_scale(scale, d)
    _native.require_eager("gated_delta_attention", q, k, v, g, beta, initial_state)
    _native._require_device(q)
    if d % 8 == 0 and dv % 8 == 0:
        return _GatedDeltaFunction.apply(q, k, v, g, beta, initial_state, scale)
    state = initial_state
    if state is not None:
        state = torch.nn.functional.pad(state, (0, -dv % 8, 0, -d % 8))
    out, final = _GatedDeltaFunction.apply(_pad8(q), _pad8(k), _pad8(v), g, beta, state, scale)
    return out[..., :dv], final[..., :d, :dv].contiguous()  # as gated_delta_step takes it


def gated_delta_step(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, state: torch.Tensor, *,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """The recurrence over one or a few tokens, for answering token by token.

    Operands as :func:`gated_delta_attention`'s; state [B, Hv, D, DV] float32,
    contiguous, is read and updated in place. Returns out [B, max(Hq, Hv), N, DV].
    Not differentiable. Calls on one state follow one another on one stream.
    """
    if state is None:
        raise TypeError("state must be a torch.Tensor")
    _validate(q, k, v, g, beta, state, "state")
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, beta, state)):
        raise RuntimeError("gated_delta_step is not differentiable: call it under torch.no_grad()")
    scale = _validate_scale(scale, q.shape[3])
    _native.require_eager("gated_delta_step", q, k, v, g, beta, state)
    _native._require_device(q)
    q, k, v = (t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous() for t in (q, k, v))
    out = _native.delta_step(q, k, v, g, beta, state, scale=scale)
    torch.autograd.graph.increment_version(state)
    return out


__all__ = ("gated_delta_attention", "gated_delta_step")

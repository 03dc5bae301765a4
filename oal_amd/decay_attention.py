"""Linear attention whose memory decays: a causal sum over all tokens before, each by what has
decayed since, over whole sequences and token by token.

Per state head, with keys k_t, values v_t and log-decays g_t <= 0:

    S_t = e^(g_t) S_(t-1) + k_t v_t^T,   o_t = scale S_t^T q_t

* :func:`decay_attention` evaluates a whole sequence in chunks of 64 tokens, with its
  backward; it takes and returns the state, so a long text can come in pieces;
* :func:`decay_step` runs the recurrence over one or a few tokens and updates the
  state in place.

Log-decays are one per state head, [Hv], or one per token, [B, Hv, N]. A token with g = -inf
forgets all before it: it begins a new text in a sequence that packs several. A token with
k = 0 and g = 0 leaves the state as it is: pad batches of ragged lengths with such tokens (with log-decays
per token: a head's one decay goes on over its padding).

Heads are those of the gated delta rule: k [B, Hk, ...], v, g and the state [B, Hv, ...], q [B, Hq, ...]. Hk
divides Hv (state head h writes with key head h // (Hv / Hk)), and one of Hq and Hv
divides the other; the output has H = max(Hq, Hv) heads, of which head o reads with
query head o // (H / Hq) from state head o // (H / Hv).

Sums over tokens do not depend on the type of q, k and v, which may be
float32, bfloat16 or float16: states, decays and their gradients are exact to float32, those of each decay by itself. 16-bit
results are rounded once, from sums whose terms are off by 2^-17 at most.
Values have to be finite: a token that is not spoils the 64 tokens of its chunk (in :func:`decay_step` itself), and with them
the state, the results behind and the gradients before. What was forgotten by g = -inf in another chunk, or in an
initial state or a step before, does not matter, whatever it is. Results repeat bit by bit from call to call;
sequences are cut into segments by a rule on batch, heads and length, so that last bits depend on those.

Calls are eager: tracers, functorch's transforms and forward-mode derivatives are refused
(compiled code runs the call between its graphs).
"""

from __future__ import annotations

from typing import Any, Optional

import torch

from . import _native
from .gated_delta import _FLOATS, _pad8, _validate_scale

HEAD_DIM = _native.HEAD_DIM


def _plain(q, k, v, g, state) -> bool:
    """Whether the operands are as they should be, in one look: it is asked in every call."""
    try:
        (b, hq, n, d), (_, hv, _, dv), hk, dev = q.shape, v.shape, k.shape[1], q.device
        return (
            q.dtype in _FLOATS and k.dtype is v.dtype is q.dtype and g.dtype is torch.float32
            and k.device == dev and v.device == dev and g.device == dev
            and k.shape == (b, hk, n, d) and v.shape == (b, hv, n, dv) and (g.shape == (b, hv, n) or g.shape == (hv,))
            and b > 0 and hq > 0 and hk > 0 and hv > 0 and n > 0 and 0 < d <= HEAD_DIM and 0 < dv <= HEAD_DIM
            and hv % hk == 0 and (hq % hv == 0 or hv % hq == 0)
            and (state is None or (state.dtype is torch.float32 and state.shape == (b, hv, d, dv)
                                   and state.device == dev))
        )
    except (AttributeError, ValueError, IndexError):
        return False


def _validate(q, k, v, g, state, name: str) -> None:
    if _plain(q, k, v, g, state):
        return
    if not all(isinstance(t, torch.Tensor) for t in (q, k, v, g)):
        raise TypeError("q, k, v and g must be torch.Tensor objects")
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q, k and v must be rank-4 head-first tensors [B, H, N, D]")
    if q.dtype not in _FLOATS:
        raise TypeError("q, k and v must be float16, bfloat16 or float32")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")
    if g.dtype != torch.float32:
        raise TypeError("g must be float32")
    if any(t.device != q.device for t in (k, v, g)):
        raise ValueError("q, k, v and g must be on the same device")
    b, hq, n, d = q.shape
    hk, hv, dv = k.shape[1], v.shape[1], v.shape[3]
    if min(b, hq, hk, hv, n, d, dv) <= 0:
        raise ValueError("q, k and v dimensions must be positive")
    if k.shape != (b, hk, n, d):
        raise ValueError("q and k must have the same batch size, sequence length and feature dimension")
    if v.shape[0] != b or v.shape[2] != n:
        raise ValueError("q, k and v must have the same batch size and sequence length")
    if g.shape != (b, hv, n) and g.shape != (hv,):
        raise ValueError("g must have shape [Hv] or [B, Hv, N]")
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


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as the kernels read it; rows that lie very far apart are copied together."""
    t = _native.row_tensor(t)
    return t if t.stride(2) < 1 << 23 or t.shape[2] == 1 else t.contiguous()


def _ready(q, k, v, g, state):
    """The operands as the kernels read them."""
    return (*map(_rows, (q, k, v)), g, None if state is None else _native._aligned(state.contiguous()))


class _DecayFunction(torch.autograd.Function):
    """(q, k, v, g, state or None, scale) -> (out, final state); dimensions multiples of 8, on one ROCm device."""

    @staticmethod
    def forward(ctx: Any, q, k, v, g, state, scale: float):
        operands = _ready(q, k, v, g, state)
        out, final, saved = _native.decay_forward(*operands, scale=scale, keep=True)
        ctx.save_for_backward(*operands[:4], saved)
        ctx.scale = scale
        return out, final

    @staticmethod
    def backward(ctx: Any, dout, dfinal):
        if torch.is_grad_enabled():
            raise RuntimeError("decay_attention does not support double backward")
        _native.require_eager("decay_attention", dout, dfinal)
        q, k, v, g, saved = ctx.saved_tensors
        dout, dfinal = (_native._aligned(t.contiguous()) for t in (dout, dfinal))
        grads = _native.decay_backward(q, k, v, g, saved, dout, dfinal, scale=ctx.scale,
                                       need_state=ctx.needs_input_grad[4])
        return (*(d if need else None for d, need in zip(grads, ctx.needs_input_grad)), None)


def decay_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, *, scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Linear attention with decays over whole sequences; differentiable in all tensors.

    q [B, Hq, N, D], k [B, Hk, N, D], v [B, Hv, N, DV] of one dtype, D and DV up to 64;
    g [Hv] or [B, Hv, N] float32; initial_state [B, Hv, D, DV] float32 (None: zero). scale
    defaults to D^-1/2. Returns out [B, max(Hq, Hv), N, DV] in q's dtype and the state after
    the last token, contiguous.
    """
    _validate(q, k, v, g, initial_state, "initial_state")
    d, dv = q.shape[3], v.shape[3]
    scale = _validate_scale(scale, d)
    _native.require_eager("decay_attention", q, k, v, g, initial_state)
    _native._require_device(q)
    operands, narrow = (q, k, v, g, initial_state), d % 8 or dv % 8
    if narrow:
        state = None if initial_state is None else torch.nn.functional.pad(initial_state, (0, -dv % 8, 0, -d % 8))
        operands = (_pad8(q), _pad8(k), _pad8(v), g, state)
    # a prompt keeps no states for a backward, also where a head's decay is a parameter
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        out, final = _DecayFunction.apply(*operands, scale)
    else:
        out, final = _native.decay_forward(*_ready(*operands), scale=scale, keep=False)[:2]
    return (out[..., :dv], final[..., :d, :dv].contiguous()) if narrow else (out, final)  # as decay_step takes it


def decay_step(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor, *,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """The recurrence over one or a few tokens, for answering token by token.

    Operands as :func:`decay_attention`'s; state [B, Hv, D, DV] float32,
    contiguous, is read and updated in place. Returns out [B, max(Hq, Hv), N, DV].
    Not differentiable. Calls on one state follow one another on one stream.
    """
    if state is None:
        raise TypeError("state must be a torch.Tensor")
    _validate(q, k, v, g, state, "state")
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, state)):
        raise RuntimeError("decay_step is not differentiable: call it under torch.no_grad()")
    scale = _validate_scale(scale, q.shape[3])
    _native.require_eager("decay_step", q, k, v, g, state)
    _native._require_device(q)
    q, k, v = (t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous() for t in (q, k, v))
    out = _native.decay_step(q, k, v, g, state, scale=scale)
    torch.autograd.graph.increment_version(state)
    return out


__all__ = ("decay_attention", "decay_step")

"""Causal softmax attention over a sliding window and a few first tokens that stay visible.

A query at position i sees the keys j <= i with i - j < window, and the first
``sinks`` keys however far they lie behind:

    out_i = sum_j softmax_j(scale q_i.k_j) v_j

* :func:`window_attention` evaluates whole sequences, with its backward;
* :func:`window_attention_step` one token per sequence over ring caches of sinks +
  window slots, which it also writes;
* :func:`window_cache` the ring caches of a prompt.

q [B, Hq, N, D], k and v [B, Hkv, N, D]; query head h reads KV head h // (Hq / Hkv), as in
the grouped quadratic operator. The token at position p is kept in slot p where p < sinks, and
else in slot sinks + (p - sinks) % window: the filled slots are just what the token sees, so
the caches never grow and nothing is masked.

bfloat16 tensors run on the matrix cores as they are, with the softmax and all sums in
float32 and its weights rounded to bfloat16 for the product with v; float32 and float16
tensors run in three and two exact bfloat16 parts per value, so that results are exact to
their type.
Padding at the end of a sequence changes nothing before it; its values have to be finite
all the same, in k, v and the gradients (a masked weight of zero times infinity is not zero).

Results repeat bit by bit from call to call. Long caches and the keys' gradients are summed in pieces
whose number follows batch and heads, so that a sequence's last bits depend on how many others are in its batch.

Calls of :func:`window_attention` and :func:`window_attention_step` are eager: tracers, functorch's
transforms and forward-mode derivatives are refused (compiled code runs the call between its graphs).
"""

from __future__ import annotations

from typing import Any, Optional

import torch

from . import _native
from .gated_delta import _FLOATS, _pad8, _validate_scale

HEAD_DIM = _native.HEAD_DIM
_MOST = 1 << 30


def _validate_window(window, sinks) -> None:
    for name, value, least in (("window", window, 1), ("sinks", sinks, 0)):
        if isinstance(value, bool) or not isinstance(value, int):
            raise TypeError(f"{name} must be an int")
        if not least <= value <= _MOST:
            raise ValueError(f"{name} must be in [{least}, {_MOST}]")


def _validate(q, k, v) -> None:
    try:  # as they should be, in one look: it is asked in every call
        (b, hq, nq, d), (_, hk, nk, dv), dev = q.shape, v.shape, q.device
        if (q.dtype in _FLOATS and k.dtype is v.dtype is q.dtype and k.device == dev and v.device == dev
                and k.shape == (b, hk, nk, d) and v.shape[0] == b and b > 0 and hq > 0 and hk > 0 and nq > 0 and nk > 0
                and 0 < d <= HEAD_DIM and 0 < dv <= HEAD_DIM and hq % hk == 0):
            return
    except (AttributeError, ValueError, IndexError):
        pass
    if not all(isinstance(t, torch.Tensor) for t in (q, k, v)):
        raise TypeError("q, k and v must be torch.Tensor objects")
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q, k and v must be rank-4 head-first tensors [B, H, N, D]")
    if q.dtype not in _FLOATS:
        raise TypeError("q, k and v must be float16, bfloat16 or float32")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on the same device")
    if min(*q.shape, *k.shape, *v.shape) <= 0:
        raise ValueError("q, k and v dimensions must be positive")
    if k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError("q and k must have the same batch size and feature dimension")
    if v.shape[:3] != k.shape[:3]:
        raise ValueError("k and v must have the same batch size, head count and length")
    if q.shape[1] % k.shape[1] != 0:
        raise ValueError("query head count must be divisible by KV head count")
    if max(q.shape[3], v.shape[3]) > HEAD_DIM:
        raise ValueError(f"the HIP kernels support head and value dimensions up to {HEAD_DIM}")


class _WindowFunction(torch.autograd.Function):
    """(q, k, v, window, sinks, scale) -> out; dimensions multiples of 8, on one ROCm device."""

    @staticmethod
    def forward(ctx: Any, q, k, v, window: int, sinks: int, scale: float):
        ctx.set_materialize_grads(False)
        q, k, v = map(_native.row_tensor, (q, k, v))
        out, lse = _native.window_forward(q, k, v, window=window, sinks=sinks, scale=scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.options = dict(window=window, sinks=sinks, scale=scale)
        return out

    @staticmethod
    def backward(ctx: Any, dout):
        if torch.is_grad_enabled():
            raise RuntimeError("window_attention does not support double backward")
        if dout is None:
            return (None,) * 6
        _native.require_eager("window_attention", dout)
        q, k, v, out, lse = ctx.saved_tensors
        dout = _native._aligned(dout.contiguous())
        grads = _native.window_backward(q, k, v, out, lse, dout, **ctx.options)
        return (*(d if need else None for d, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def window_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int, sinks: int = 0, scale: Optional[float] = None,
) -> torch.Tensor:
    """Windowed attention over whole sequences; differentiable in q, k and v.

    q [B, Hq, Nq, D], k [B, Hkv, Nk, D], v [B, Hkv, Nk, DV] of one dtype, D and DV up to
    64. Nq <= Nk: the queries are the last Nq of the Nk tokens. scale defaults to
    D^-1/2. Returns out [B, Hq, Nq, DV] in q's dtype.
    """
    _validate(q, k, v)
    _validate_window(window, sinks)
    if q.shape[2] > k.shape[2]:
        raise ValueError("there must be a key for every query")
    d, dv = q.shape[3], v.shape[3]
    scale = _validate_scale(scale, d)
    _native.require_eager("window_attention", q, k, v)
    _native._require_device(q)
    if d % 8 == 0 and dv % 8 == 0:
        return _WindowFunction.apply(q, k, v, window, sinks, scale)
    return _WindowFunction.apply(_pad8(q), _pad8(k), _pad8(v), window, sinks, scale)[..., :dv]


def window_cache(
    k: torch.Tensor, v: torch.Tensor, *, window: int, sinks: int = 0, lengths: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Ring caches [B, Hkv, sinks + window, D] of a prompt's keys and values [B, Hkv, N, D].

    lengths [B] (int32 or int64; None: N each): the tokens of each sequence of a batch padded at
    its end, from 0 to N. Empty slots are zero. The first token after the prompt has position N, or
    lengths.
    """
    _validate(k, k, v)
    _validate_window(window, sinks)
    b, _, n, _ = k.shape
    if lengths is None:
        lengths = torch.full((b,), n, dtype=torch.int64, device=k.device)
    elif not isinstance(lengths, torch.Tensor) or lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError("lengths must be an int32 or int64 tensor")
    elif lengths.shape != (b,) or lengths.device != k.device:
        raise ValueError("lengths must have shape [B], on the device of k and v")
    last = lengths.to(torch.int64).clamp(0, n)[:, None] - 1
    slot = torch.arange(sinks + window, device=k.device)[None]
    # the newest position of each slot of the ring: (position - sinks) % window == slot - sinks
    position = torch.where(slot < sinks, slot, last - torch.remainder(last - slot, window))
    filled = (position <= last) & ((slot < sinks) | (position >= sinks)) & (last >= 0)
    index = torch.where(filled, position, 0)[:, None, :, None]
    return tuple(
        torch.where(filled[:, None, :, None], torch.take_along_dim(t, index, 2), 0).to(t.dtype) for t in (k, v))


def window_attention_step(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    positions: torch.Tensor, *, window: int, sinks: int = 0, scale: Optional[float] = None,
) -> torch.Tensor:
    """One token per sequence over its ring caches, for answering token by token.

    q [B, Hq, 1, D], k [B, Hkv, 1, D], v [B, Hkv, 1, DV]; k_cache and v_cache
    [B, Hkv, sinks + window, D or DV] of the same dtype, D and DV multiples of 8 up to 64,
    rows contiguous and 16-byte aligned: the token's key and value are written into them.
    positions [B] int32 or int64, on the device: the tokens before this one; a negative position means
    that the sequence has no token now: its caches stay as they are and its output is zero.
    Returns out [B, Hq, 1, DV]. Not differentiable. Calls on one cache follow one
    another on one stream.
    """
    _validate(q, k, v)
    _validate_window(window, sinks)
    _native.require_eager("window_attention_step", q, k, v, k_cache, v_cache)  # before addresses are looked at
    (b, hk, _, d), dv = k.shape, v.shape[3]
    if q.shape[2] != 1 or k.shape[2] != 1:
        raise ValueError("a step takes one token of each sequence")
    if d % 8 or dv % 8:
        raise ValueError("head and value dimensions of a cache must be multiples of 8")
    size = sinks + window
    if size > _MOST:
        raise ValueError(f"the cache must have at most {_MOST} slots")
    for name, t, width in (("k_cache", k_cache, d), ("v_cache", v_cache, dv)):
        if (isinstance(t, torch.Tensor) and t.dtype is q.dtype and t.device == q.device
                and t.shape == (b, hk, size, width) and t.is_contiguous() and t.data_ptr() % 16 == 0):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must have the dtype of q and be on its device")
        if t.shape != (b, hk, size, width):
            raise ValueError(f"{name} must have shape [B, Hkv, sinks + window, {width}]")
        at = [s for s, n in zip(t.stride()[:3], t.shape) if n > 1]
        if t.stride(3) != 1 or any(s < width for s in at) or t.data_ptr() % 16 or any(
                s * t.element_size() % 16 for s in at):
            raise ValueError(f"the rows of {name} must be contiguous, apart from each other and 16-byte aligned")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be an int32 or int64 tensor")
    if positions.shape != (b,) or positions.device != q.device:
        raise ValueError("positions must have shape [B], on the device of q")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, k_cache, v_cache)):
        raise RuntimeError("window_attention_step is not differentiable: call it under torch.no_grad()")
    scale = _validate_scale(scale, d)
    _native._require_device(q)
    if k_cache.data_ptr() == v_cache.data_ptr():
        raise ValueError("k_cache and v_cache must be two tensors")
    q, k, v = map(_native.row_tensor, (q, k, v))
    if positions.dtype is not torch.int64 or not positions.is_contiguous():
        positions = positions.to(torch.int64).contiguous()
    out = _native.window_step(q, k, v, k_cache, v_cache, positions, window=window, sinks=sinks, scale=scale)
    for t in (k_cache, v_cache):
        torch.autograd.graph.increment_version(t)
    return out


__all__ = ("window_attention", "window_attention_step", "window_cache")

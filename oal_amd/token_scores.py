"""Log probabilities of given tokens, with the entropy of the distributions that they are from and the
most likely alternatives, in one pass over a model's logits; and the gradient in another.

    log p_v = x_v - log sum_w e^(x_w),   H = -sum_v p_v log p_v

The mean of -log p over a text is its next-token loss: :func:`token_log_probs` is differentiable in the
logits, through log_probs and entropy. It holds no float32 copy of the logits, and its backward keeps two
numbers for each row beside them.

Logits are float32, bfloat16 or float16; exponentials and results are float32, sums over a row float64, so that small
log probabilities and entropies, of a model that is sure, are as exact as others. A logit of -inf is a token
that cannot be; a row of such logits alone, and one with NaN or +inf, has NaN scores, as log_softmax has, and a gradient of NaN
if one is asked of it. Results repeat bit by bit from call to call; few rows are cut into parts by a rule on their number, so that last bits
depend on how many others are in the call.

Calls are eager: tracers, functorch's transforms and forward-mode derivatives are refused
(compiled code runs the call between its graphs).
"""

from __future__ import annotations

from typing import Any, NamedTuple, Optional

import torch

from . import _native
from .gated_delta import _FLOATS

MOST_TOP = 64


class TokenScores(NamedTuple):
    """What :func:`token_log_probs` returns; None what was not asked for."""

    log_probs: torch.Tensor
    entropy: Optional[torch.Tensor]
    top_log_probs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _validate(logits, tokens, entropy, top) -> None:
    if not isinstance(logits, torch.Tensor) or not isinstance(tokens, torch.Tensor):
        raise TypeError("logits and tokens must be torch.Tensor objects")
    if logits.dtype not in _FLOATS:
        raise TypeError("logits must be float16, bfloat16 or float32")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError("tokens must be an int32 or int64 tensor")
    if not isinstance(entropy, bool):
        raise TypeError("entropy must be a bool")
    if isinstance(top, bool) or not isinstance(top, int):
        raise TypeError("top must be an int")
    if logits.ndim < 1 or logits.shape[-1] <= 0:
        raise ValueError("logits must be [..., V], with V positive")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError("tokens must have the shape of logits without its last dimension")
    if tokens.device != logits.device:
        raise ValueError("logits and tokens must be on the same device")
    if not 0 <= top <= min(MOST_TOP, logits.shape[-1]):
        raise ValueError(f"top must be in [0, {MOST_TOP}] and not more than V")


class _TokenScoresFunction(torch.autograd.Function):
    """(logits [B, N, V], tokens [B, N] int64, entropy, top) -> the scores, on one ROCm device."""

    @staticmethod
    def forward(ctx: Any, logits, tokens, entropy: bool, top: int):
        ctx.set_materialize_grads(False)
        keep = ctx.needs_input_grad[0]
        log_probs, entropies, values, places, saved = _native.token_scores(
            logits, tokens, entropy=entropy, top=top, keep=keep)
        ctx.mark_non_differentiable(*(t for t in (values, places) if t is not None))
        if keep:
            ctx.save_for_backward(logits, tokens, saved, entropies)
        return log_probs, entropies, values, places

    @staticmethod
    def backward(ctx: Any, dlog, dentropy, _values, _places):
        if torch.is_grad_enabled():
            raise RuntimeError("token_log_probs does not support double backward")
        if dlog is None and dentropy is None:
            return (None,) * 4
        _native.require_eager("token_log_probs", dlog, dentropy)
        logits, tokens, saved, entropies = ctx.saved_tensors
        ups = (None if t is None else t.contiguous() for t in (dlog, dentropy))
        return _native.token_scores_backward(logits, tokens, saved, entropies, *ups), None, None, None


def token_log_probs(
    logits: torch.Tensor, tokens: torch.Tensor, *, entropy: bool = False, top: int = 0,
) -> TokenScores:
    """Scores of tokens [...] (int32 or int64) in logits [..., V]; differentiable in the logits.

    Returns log_probs [...] float32: zero, without a gradient, for a negative token (a place without
    one), NaN for one that is not in [0, V); with ``entropy``, entropy [...] float32; and with ``top`` (up to 64 and
    V), top_log_probs [..., top] float32 and top_tokens [..., top] int64, the most likely tokens in order, of
    equally likely ones the lowest first (not differentiable; a row with NaN may have places of -1).
    The rows of logits may lie at any strides: ``logits[:, :-1]`` is not copied.
    """
    _validate(logits, tokens, entropy, top)
    _native.require_eager("token_log_probs", logits, tokens)
    _native._require_device(logits)
    shape, vocab = tokens.shape, logits.shape[-1]
    if tokens.numel() == 0:
        # no tokens, no scores: sums of nothing carry the graph
        none = logits.float().sum(-1)
        return TokenScores(none, none.clone() if entropy else None,
                           *((none.detach().new_empty((*shape, top)), tokens.new_empty((*shape, top), dtype=torch.int64))
                             if top else (None, None)))
    rows = logits if logits.ndim == 3 else logits[None] if logits.ndim == 2 else logits.reshape(1, -1, vocab)
    if rows.stride(2) != 1 and vocab > 1:
        rows = rows.contiguous()
    tokens = tokens.reshape(rows.shape[:2]).to(torch.int64).contiguous()
    if torch.is_grad_enabled() and rows.requires_grad:
        scores = _TokenScoresFunction.apply(rows, tokens, entropy, top)
    else:  # a short call's host time is most of it
        scores = _native.token_scores(rows, tokens, entropy=entropy, top=top, keep=False)[:4]
    return TokenScores(*(None if t is None else t.reshape((*shape, *t.shape[2:])) for t in scores))


__all__ = ("TokenScores", "token_log_probs")

"""Windowed attention with first tokens that stay visible, over all pairs in float64: the definition itself."""

from __future__ import annotations

import math

import torch


def window_attention(q, k, v, *, window, sinks, scale):
    """q [B, Hq, Nq, D], k and v [B, Hkv, Nk, D]; the queries are the last Nq tokens."""
    q, k, v = (t.double() for t in (q, k, v))
    r = q.shape[1] // k.shape[1]
    k, v = (t.repeat_interleave(r, 1) for t in (k, v))
    nq, nk = q.shape[2], k.shape[2]
    i = torch.arange(nk - nq, nk, device=q.device)[:, None]
    j = torch.arange(nk, device=q.device)[None]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    score = scale * q @ k.transpose(2, 3)
    return torch.softmax(score.masked_fill(~seen, -math.inf), -1) @ v

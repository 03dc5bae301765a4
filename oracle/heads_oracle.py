"""Head norms with rotary embedding, and token scores, by their formulas in float64 on any device.

Differentiable by torch, which is how the tests take their gradients.
"""

from __future__ import annotations

import torch


def _one(x, weight, cos, sin, heads, eps):
    b, n, _ = x.shape
    y = x.double().reshape(b, n, heads, -1)
    y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.double()
    r = cos.shape[-1]
    a, rest = y[..., :r], y[..., r:]
    turned = torch.cat((-a[..., r // 2:], a[..., :r // 2]), -1)
    return torch.cat((a * cos + turned * sin, rest), -1).transpose(1, 2)


def norm_rotary(q, k, v, q_weight, k_weight, cos, sin, positions=None, *, q_heads, kv_heads, eps):
    """Projections [B, N, heads * D] -> head-first (q, k, v); a negative position's rows are zero."""
    b, n, _ = q.shape
    at = torch.arange(n, device=q.device).expand(b, n) if positions is None else positions
    cos, sin = (t.double()[at.clamp(min=0)][:, :, None] for t in (cos, sin))
    there = (at >= 0)[:, None, :, None]
    outs = (_one(q, q_weight, cos, sin, q_heads, eps), _one(k, k_weight, cos, sin, kv_heads, eps),
            v.double().reshape(b, n, kv_heads, -1).transpose(1, 2))
    return tuple(torch.where(there, t, 0) for t in outs)


def token_scores(logits, tokens):
    """(log_probs, entropy) of logits [..., V] and tokens [...]; a negative token's log probability is zero."""
    x = logits.double()
    log = torch.log_softmax(x, -1)
    p = log.exp()
    found = log.gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    # what cannot be has no share
    share = p * torch.where(torch.isinf(x), 0, log)
    return torch.where(tokens < 0, 0, found), -share.sum(-1)


def top_tokens(logits, top):
    """(values, places) of the highest logits, of equal ones the first."""
    value, place = logits.double().sort(dim=-1, descending=True, stable=True)
    return value[..., :top], place[..., :top]

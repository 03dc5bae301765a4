"""Linear attention with decays token by token, in float64 on any device: the definition itself.

    S_t = e^(g_t) S_(t-1) + k_t v_t^T,  o_t = scale S_t^T q_t

Differentiable by torch, which is how the tests take its gradients.
"""

from __future__ import annotations

import torch


def decay_attention(q, k, v, g, state=None, *, scale):
    """q [B, Hq, N, D], k [B, Hk, N, D], v [B, Hv, N, DV], g [Hv] or [B, Hv, N], state
    [B, Hv, D, DV] -> (out [B, max(Hq, Hv), N, DV], state after the last token)."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    hv, heads = v.shape[1], max(q.shape[1], v.shape[1])
    q = q.repeat_interleave(heads // q.shape[1], 1)
    k = k.repeat_interleave(hv // k.shape[1], 1)
    g = g[None, :, None].expand(v.shape[:3]) if g.ndim == 1 else g
    s = torch.zeros((*k.shape[:2], k.shape[3], v.shape[3]), dtype=torch.float64, device=q.device) if state is None else state.double()
    outs = []
    for t in range(q.shape[2]):
        s = s * g[:, :, t, None, None].exp() + k[:, :, t, :, None] * v[:, :, t, None, :]
        outs.append(scale * (s.repeat_interleave(heads // hv, 1) * q[:, :, t, :, None]).sum(2))
    return torch.stack(outs, 2), s

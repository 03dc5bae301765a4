"""Gradients of single log-decays against the recurrence in float64, token by token: a norm over all tokens does not
see the small ones among them.

Queries, keys, values and gradients are positive here, so that all terms of a sum have one sign and its error is of its
own size: chains of two products of 64 terms each, 128 roundings of 2^-24, and decays whose logarithm to base
two, up to 128, is rounded to float32, by 2^-18 ln 2 of the decay, in each of two factors at most."""

import pytest
import torch

from oal_amd.decay_attention import decay_attention
from oracle.decay_oracle import decay_attention as definition

pytestmark = pytest.mark.gpu

_TOL = 128 * 2.0 ** -24 + 2.0 ** -18 * 1.4


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _gradients(b, heads, n, dtype, strong, seed=0, with_state=True):
    """(ours, exact) of g, whose `strong` tokens have the given log-decay, the others slow ones."""
    gen = torch.Generator().manual_seed(seed)
    hq, hk, hv = heads
    q, k, v = (torch.rand(b, h, n, 64, generator=gen).to(dtype) for h in (hq, hk, hv))
    g = -0.02 * torch.rand(b, hv, n, generator=gen)
    for at, decay in strong.items():
        g[..., at] = decay
    state, dstate = (torch.rand(b, hv, 64, 64, generator=gen) * with_state for _ in range(2))
    dout = torch.rand(b, max(hq, hv), n, 64, generator=gen).to(dtype)
    dev, found = _dev(), []
    for call, cast in ((decay_attention, torch.Tensor.clone), (definition, torch.Tensor.double)):
        ins = [cast(t.to(dev)).requires_grad_() for t in (q, k, v, g, state)]
        outs = call(*ins[:4], scale=0.125, **({"initial_state": ins[4]} if call is decay_attention else {"state": ins[4]}))
        found.append(torch.autograd.grad(outs, ins[3], [cast(t.to(dev)) for t in (dout, dstate)])[0])
    return found


_PLACES = [(at, torch.float32) for at in (0, 1, 15, 16, 17, 31, 32, 40, 47, 48, 62, 63)]
_PLACES += [(at, dtype) for at in (17, 40) for dtype in (torch.bfloat16, torch.float16)]  # types differ in the operands alone


@pytest.mark.parametrize("decay", [-5.0, -12.0, -20.0, -40.0, -60.0])
@pytest.mark.parametrize("at,dtype", _PLACES)
def test_one_strong_decay_among_slow_ones(at, decay, dtype):
    """At every place of a tile and of a chunk, in a chunk with others before and behind it."""
    got, want = _gradients(1, (2, 1, 1), 192, dtype, {64 + at: decay})
    err = float(((got.double() - want) / want).abs().max())
    assert err <= _TOL, f"{err:.3g}"


@pytest.mark.parametrize("heads", [(2, 2, 2), (14, 2, 2), (2, 2, 6)])
@pytest.mark.parametrize("n", [1, 5, 16, 17, 63, 65, 130])
def test_every_token(n, heads):
    got, want = _gradients(2, heads, n, torch.float32, {n // 2: -9.0, n // 3: -25.0, n - 1: -3.0}, seed=n)
    err = float(((got.double() - want) / want).abs().max())
    assert err <= _TOL, f"{err:.3g}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_texts_apart_by_a_strong_decay_are_apart(dtype):
    """Texts of one chunk that a decay of -30 separates, without a state: the gradients of the decays that separate
    them are theirs, e^-30 of the others and less."""
    got, want = _gradients(1, (1, 1, 1), 64, dtype, {9: -30.0, 20: -30.0, 21: -30.0, 50: -30.0}, with_state=False)
    # the first text's first token has nothing before it
    assert float(got[..., 0].abs().max()) == 0.0
    err = float(((got.double() - want) / want)[..., 1:].abs().max())
    assert err <= _TOL, f"{err:.3g}"

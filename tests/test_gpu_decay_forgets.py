"""What a log-decay of -inf has forgotten does not matter any more, NaN and infinities too: not in a state that another
text left, not in another chunk of 64 tokens of a packed sequence, and not for gradients.

The results are compared with those of the same call without what is forgotten, whose terms are the same."""

import math

import pytest
import torch

from oal_amd.decay_attention import decay_attention, decay_step

pytestmark = pytest.mark.gpu

_BAD = [math.nan, math.inf, -math.inf]


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _inputs(b, heads, n, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    hq, hk, hv = heads
    q, k, v = (torch.randn(b, h, n, 64, generator=gen).to(dtype) for h in (hq, hk, hv))
    g = -0.1 * torch.rand(b, hv, n, generator=gen)
    state, dstate = (torch.randn(b, hv, 64, 64, generator=gen) for _ in range(2))
    dout = torch.randn(b, max(hq, hv), n, 64, generator=gen).to(dtype)
    dev = _dev()
    return [t.to(dev) for t in (q, k, v, g, state)], [t.to(dev) for t in (dout, dstate)]


def _run(ins, ups):
    leaves = [t.detach().clone().requires_grad_() for t in ins]
    outs = decay_attention(*leaves[:4], initial_state=leaves[4])
    return [*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, ups)]


@pytest.mark.parametrize("bad", _BAD)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 3])
def test_a_slot_that_a_step_resets(n, dtype, bad):
    (q, k, v, g, state), _ = _inputs(3, (4, 2, 2), n, dtype, seed=1)
    g[1, :, 0] = -math.inf
    clean = state.clone()
    clean[1] = 0
    want = decay_step(q, k, v, g, clean)
    state[1] = bad
    out = decay_step(q, k, v, g, state)
    assert torch.isfinite(out).all() and torch.equal(out, want) and torch.equal(state, clean)


@pytest.mark.parametrize("bad", _BAD)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at,n", [(0, 1), (0, 300), (5, 40), (70, 200)])
def test_an_initial_state_that_is_forgotten(at, n, dtype, bad):
    """Of the second sequence: what is read before is bad, what comes behind is not, and no gradient but the state's own and
    those of the tokens that read it."""
    ins, ups = _inputs(2, (4, 2, 2), n, dtype, seed=2)
    ins[3][1, :, at] = -math.inf
    want = _run(ins, ups)
    ins[4][1] = bad
    got = _run(ins, ups)
    for name, x, y in zip(("out", "state", "dq", "dk", "dv", "dg", "dstate"), got, want):
        x, y = (t if name in ("state", "dstate") else t[:, :, at:] if t.ndim > 2 else t for t in (x, y))
        if name in ("dk", "dv", "dstate"):  # of what is behind the state nothing depends on it
            assert torch.isfinite(x).all(), name
        assert torch.equal(x, y), name


@pytest.mark.parametrize("bad", _BAD)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,heads", [(1, (2, 1, 1)), (300, (2, 2, 2))])
def test_a_text_before_and_a_text_behind(b, heads, dtype, bad):
    """Texts from tokens 0, 140 and 260 on, the first and the last with a token that is not finite; in segments of one chunk
    and of several, over a whole sequence."""
    ins, ups = _inputs(b, heads, 400, dtype, seed=3)
    ins[3][..., [140, 260]] = -math.inf
    want = _run(ins, ups)
    ins[2][:, :, 50] = bad  # a value of the first text
    ups[0][:, :, 330] = bad  # a gradient of the last one's results
    got = _run(ins, ups)
    for name, x, y in zip(("out", "dq", "dk", "dv", "dg"), (got[0], *got[2:6]), (want[0], *want[2:6])):
        assert torch.isfinite(x[:, :, 140:260]).all() and torch.equal(x[:, :, 140:260], y[:, :, 140:260]), name
    assert torch.equal(got[1], want[1]) and not torch.isfinite(got[0][:, :, 50]).any()

"""Attention with decays where a block walks several chunks: the state handed on from chunk to chunk, the decays formed
four chunks at a time, the sums of gates' gradients taking turns, single segments, segments of more than eight chunks.

With U = batch times state heads and NC chunks of 64 tokens, sequences are cut into min(1024 / U, NC) segments in the forward,
min(512 / U, NC) in the backward; each case says what it gets.

Against the recurrence in float64. float32 results are sums of some hundred terms whose roundings of 2^-24 go either way,
and a state takes a rounding more with each chunk: 16 roundings in the norm. 16-bit results are compared with exact
ones rounded to their type: an error of 2^-16 before the rounding moves a result to its neighbour, up to eps
away, with a chance of 2^-16 / eps, so the norm of the differences is at most the root of 2^-16 eps."""

import math

import pytest
import torch

from oal_amd.decay_attention import decay_attention
from oracle.decay_oracle import decay_attention as definition

pytestmark = pytest.mark.gpu

_NAMES = ("out", "state", "dq", "dk", "dv", "dg", "dstate")
_SINGLE = 16 * 2.0 ** -24


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _inputs(b, heads, n, d, dv, dtype, seed, decay=0.05, per_head=False, texts=()):
    gen = torch.Generator().manual_seed(seed)
    hq, hk, hv = heads
    q, k, v = (torch.randn(b, h, n, x, generator=gen).to(dtype) for h, x in ((hq, d), (hk, d), (hv, dv)))
    g = -decay * torch.rand(b, hv, n, generator=gen)
    if per_head:
        g = g[0, :, 0].clone()
    for at in texts:
        g[..., at] = -math.inf
    state, dstate = (torch.randn(b, hv, d, dv, generator=gen) for _ in range(2))
    dout = torch.randn(b, max(hq, hv), n, dv, generator=gen).to(dtype)
    dev = _dev()
    return [t.to(dev) for t in (q, k, v, g, state)], [t.to(dev) for t in (dout, dstate)]


def _near(name, got, want, dtype):
    assert got.dtype == dtype and got.shape == want.shape and torch.isfinite(got).all(), name
    if dtype is torch.float32:
        bound = _SINGLE
    else:
        want, bound = want.to(dtype), (2.0 ** -16 * torch.finfo(dtype).eps) ** 0.5
    err = float((got.detach().double() - want.double()).norm() / want.double().norm())
    print(f"{name}: {err:.2e} of {bound:.2e}", flush=True)
    assert err <= bound, f"{name}: {err:.3g}"


def _check(ins, ups, scale=0.125):
    found = []
    for call, cast, start in ((definition, torch.Tensor.double, "state"), (decay_attention, torch.Tensor.clone, "initial_state")):
        leaves = [cast(t).requires_grad_() for t in ins]
        outs = call(*leaves[:4], scale=scale, **{start: leaves[4]})
        found.append([*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, [cast(t) for t in ups])])
    types = [ins[0].dtype, torch.float32, *(t.dtype for t in ins)]
    for name, want, got, dtype in zip(_NAMES, *found, types):
        _near(name, got, want, dtype)


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_segment_of_eleven_chunks(dtype, per_head):
    """U = 520: forward and backward walk whole sequences, with the call's own states, of narrow heads."""
    _check(*_inputs(260, (2, 2, 2), 700, 48, 40, dtype, seed=1, per_head=per_head))


@pytest.mark.parametrize("heads", [(6, 2, 2), (2, 2, 4), (4, 1, 2)])
def test_shared_heads_over_many_chunks(heads):
    """U = 520 or 1040, 9 chunks: one segment; several output heads take turns in a block, or state heads share a key."""
    _check(*_inputs(260, heads, 560, 32, 32, torch.bfloat16, seed=2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_segments_of_more_than_eight_chunks(dtype):
    """U = 500, 19 chunks: forward two segments of 10 and 9, backward one of 19; texts begin inside them, the last chunk is
    ragged."""
    _check(*_inputs(250, (2, 2, 2), 1190, 32, 32, dtype, seed=3, texts=(64, 65, 300, 710, 1189)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_segments_of_ten_chunks(dtype):
    """U = 250, 19 chunks: forward four segments of five, backward two of ten; very slow decays."""
    _check(*_inputs(125, (2, 2, 2), 1190, 32, 32, dtype, seed=4, decay=0.002))


@pytest.mark.parametrize("per_head", [False, True])
def test_the_headline_length(per_head):
    """U = 56, 64 chunks: forward 16 segments of four, backward eight of eight."""
    _check(*_inputs(4, (14, 14, 14), 4096, 32, 32, torch.bfloat16, seed=5, decay=0.01, per_head=per_head))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads", [(2, 2, 2), (6, 2, 2), (2, 1, 4)])
def test_prompts(heads, dtype):
    """U = 500 or 1000, 11 chunks, nothing kept for a backward: two segments of six and five, or one of eleven."""
    ins, _ = _inputs(250, heads, 690, 64, 64, dtype, seed=6)
    with torch.no_grad():
        want = definition(*ins, scale=0.125)
        got = decay_attention(*ins[:4], scale=0.125, initial_state=ins[4])
    _near("out", got[0], want[0], dtype)
    _near("state", got[1], want[1], torch.float32)

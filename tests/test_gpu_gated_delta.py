"""The gated delta rule's kernels against the recurrence in float64.

Tolerances, as the norm of the error over the norm of the result, are counted in
roundings. float32 results pass chains of three products of 64 terms each, 192
roundings of at most 2^-24. A bf16 result is rounded once itself and is a sum of terms
whose two factors are rounded to bf16, three roundings of at most 2^-8; a float16
one only its own, at most 2^-11, on top of the float32 chain."""

import pytest
import torch

from oal_amd.gated_delta import gated_delta_attention, gated_delta_step
from oracle.delta_oracle import gated_delta

pytestmark = pytest.mark.gpu

_TOL = {torch.float32: 192 * 2.0 ** -24, torch.bfloat16: 3 * 2.0 ** -8, torch.float16: 2.0 ** -11 + 192 * 2.0 ** -24}
_NAMES = ("out", "state", "dq", "dk", "dv", "dg", "dbeta", "dstate")


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _inputs(b, heads, n, d=64, dv=None, dtype=torch.float32, beta_dtype=None, seed=0, decay=0.3):
    hq, hk, hv = heads
    dv = dv or d
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.nn.functional.normalize(torch.randn(b, h, n, d, generator=gen), dim=-1).to(dtype) for h in (hq, hk))
    v = torch.randn(b, hv, n, dv, generator=gen).to(dtype)
    g = -decay * torch.rand(b, hv, n, generator=gen) * torch.arange(1, hv + 1)[:, None]
    beta = torch.sigmoid(torch.randn(b, hv, n, generator=gen)).to(beta_dtype or dtype)
    state = torch.randn(b, hv, d, dv, generator=gen)
    dout = torch.randn(b, max(hq, hv), n, dv, generator=gen).to(dtype)
    dstate = torch.randn(b, hv, d, dv, generator=gen)
    return [q, k, v, g, beta, state], [dout, dstate]


def _check(ins, ups, scale=0.125, with_state=True, on="cpu"):
    dev = _dev()
    want_ins = [t.to(on).double().requires_grad_() for t in ins]
    want = gated_delta(*want_ins[:5], want_ins[5] if with_state else None, scale=scale)
    leaves = want_ins if with_state else want_ins[:5]
    want = [*want, *torch.autograd.grad(want, leaves, [t.to(on).double() for t in ups])]
    got_ins = [t.to(dev).requires_grad_() for t in ins]
    got = gated_delta_attention(*got_ins[:5], scale=scale, initial_state=got_ins[5] if with_state else None)
    got = [*got, *torch.autograd.grad(got, got_ins if with_state else got_ins[:5], [t.to(dev) for t in ups])]
    types = [ups[0].dtype, torch.float32, *(t.dtype for t in (ins if with_state else ins[:5]))]
    for name, x, y, dtype in zip(_NAMES, got, want, types):
        x, y = x.detach(), y.detach()
        assert x.dtype == dtype and x.shape == y.shape, name
        err = float((x.double().to(on) - y).norm()) / max(float(y.norm()), 1e-30)
        assert err <= _TOL[dtype], f"{name}: {err:.3g}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 16, 63, 64, 65, 127, 129, 300])
def test_lengths(n, dtype):
    _check(*_inputs(2, (2, 2, 2), n, dtype=dtype, seed=n))


@pytest.mark.parametrize("heads,n", [((2, 1, 1), 6001), ((2, 2, 2), 2688)])
def test_long_sequences_walk_in_segments(heads, n):
    ins, ups = _inputs(1, heads, n, dtype=torch.bfloat16, seed=n, decay=0.02)
    _check(ins, ups, on=_dev())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(14, 2, 2), (7, 7, 14), (2, 2, 6), (4, 2, 4), (1, 1, 3), (3, 1, 1)])
def test_heads_shared_in_both_directions(heads, dtype):
    _check(*_inputs(2, heads, 100, dtype=dtype, seed=7))


@pytest.mark.parametrize("d,dv", [(64, 32), (48, 64), (1, 1), (33, 7)])
def test_narrow_heads(d, dv):
    _check(*_inputs(1, (2, 1, 2), 90, d=d, dv=dv, seed=d))


def test_no_state_and_float32_beta():
    _check(*_inputs(2, (2, 2, 2), 150, dtype=torch.bfloat16, beta_dtype=torch.float32), with_state=False)


@pytest.mark.parametrize("kind", ["keep", "forget", "mixed", "write nothing", "beta two"])
def test_gates_at_their_ends(kind):
    ins, ups = _inputs(1, (2, 2, 2), 200, seed=3)
    g, beta = ins[3], ins[4]
    if kind == "keep":
        g.zero_()
    elif kind == "forget":
        g.fill_(-30.0)
    elif kind == "mixed":  # a few tokens that forget all but nothing, slow decay elsewhere
        g.mul_(0.1)
        g[..., ::37] = -300.0
    elif kind == "write nothing":
        beta[..., ::3] = 0.0
        beta[..., 1::3] = 1.0
    else:
        beta.fill_(2.0)
    _check(ins, ups)


def test_a_decay_of_minus_infinity_starts_afresh():
    ins, ups = _inputs(1, (2, 2, 2), 150, seed=5)
    dev = _dev()
    ins[3][..., 70] = -float("inf")
    whole, _ = gated_delta_attention(*(t.to(dev) for t in ins[:5]), scale=0.125, initial_state=ins[5].to(dev))
    tail, _ = gated_delta_attention(*(t[:, :, 70:].to(dev) for t in ins[:5]), scale=0.125)
    err = float((whole[:, :, 70:] - tail).norm() / tail.norm())
    assert err <= _TOL[torch.float32]


def test_one_key_again_and_again():
    # the triangle's entries are as large as they get: every token replaces what the one before wrote
    ins, ups = _inputs(1, (2, 2, 2), 130, seed=11, decay=0.0)
    ins[1].copy_(ins[1][:, :, :1].expand_as(ins[1]).clone())
    ins[4].fill_(1.0)
    _check(ins, ups)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_rows(dtype):
    dev = _dev()
    ins, ups = _inputs(2, (4, 2, 2), 77, dtype=dtype, seed=13)
    dense = [t.to(dev) for t in ins]
    want = gated_delta_attention(*dense[:5], scale=0.125, initial_state=dense[5])
    token_major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dense[:5]]
    odd = []
    for t in dense[:3]:
        wide = torch.zeros((*t.shape[:3], 65), dtype=dtype, device=dev)
        wide[..., 1:] = t
        odd.append(wide[..., 1:])
    for views in (token_major, odd + dense[3:5]):
        got = gated_delta_attention(*views, scale=0.125, initial_state=dense[5])
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_broadcast_inputs_get_summed_gradients():
    dev = _dev()
    ins, ups = _inputs(2, (2, 2, 2), 40, seed=17)
    ins, ups = [t.to(dev) for t in ins], [t.to(dev) for t in ups]
    row = ins[4][:1, :1].clone().requires_grad_()
    full = row.detach().expand(2, 2, 40).clone().requires_grad_()
    grads = []
    for beta, leaf in ((row.expand(2, 2, 40), row), (full, full)):
        outs = gated_delta_attention(*ins[:4], beta, scale=0.125, initial_state=ins[5])
        grads.append(torch.autograd.grad(outs, leaf, ups)[0])
    assert torch.allclose(grads[0], grads[1].sum((0, 1), keepdim=True), rtol=1e-5, atol=1e-6)


def test_gradient_against_differences():
    dev = _dev()
    ins, ups = _inputs(1, (2, 1, 2), 70, d=8, seed=19)
    ups = [t.to(dev).double() for t in ups]
    ins = [t.to(dev) for t in ins]

    def loss(ts):
        outs = gated_delta_attention(*ts[:5], scale=0.3, initial_state=ts[5])
        return sum((o.double() * up).sum() for o, up in zip(outs, ups))

    leaves = [t.clone().requires_grad_() for t in ins]
    grads = torch.autograd.grad(loss(leaves), leaves)
    gen = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        way = torch.randn(ins[i].shape, generator=gen).to(dev)
        h = 1e-2 / float(way.abs().max())
        ends = [loss([t + s * h * way if j == i else t for j, t in enumerate(ins)]) for s in (1, -1)]
        slope, want = float(ends[0] - ends[1]) / (2 * h), float((grad * way).double().sum())
        # third differences of order h^2, and sums of a few hundred float32 terms over 2 h
        assert abs(slope - want) <= 2e-3 * (abs(want) + float(grad.norm() * way.norm()) * 0.1), _NAMES[i + 2]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,d,dv,n", [((2, 2, 2), 64, 64, 1), ((14, 2, 2), 64, 64, 3), ((2, 2, 6), 33, 7, 2), ((1, 1, 1), 1, 1, 5)])
def test_step(heads, d, dv, n, dtype):
    dev = _dev()
    ins, _ = _inputs(3, heads, n, d=d, dv=dv, dtype=dtype, seed=23)
    want, want_state = gated_delta(*ins, scale=0.3)
    q, k, v, g, beta, state = (t.to(dev) for t in ins)
    version = state._version
    out = gated_delta_step(q, k, v, g, beta, state, scale=0.3)
    assert out.dtype == dtype and state._version > version
    for x, y, t in ((out, want, dtype), (state, want_state, torch.float32)):
        assert float((x.double().cpu() - y).norm() / y.norm()) <= _TOL[t]


def test_pieces_and_steps_continue_a_sequence():
    """A prompt in two pieces, then token by token, is the sequence in one call."""
    dev = _dev()
    ins, _ = _inputs(2, (4, 2, 4), 200, dtype=torch.bfloat16, seed=29)
    q, k, v, g, beta, state = (t.to(dev) for t in ins)
    whole, end = gated_delta_attention(q, k, v, g, beta, initial_state=state)
    parts, cur = [], state
    for lo, hi in ((0, 90), (90, 190)):
        out, cur = gated_delta_attention(*(t[:, :, lo:hi] for t in (q, k, v, g, beta)), initial_state=cur)
        parts.append(out)
    cur = cur.clone()
    for t in range(190, 200):
        parts.append(gated_delta_step(*(x[:, :, t:t + 1] for x in (q, k, v, g, beta)), cur))
    got = torch.cat(parts, 2)
    assert float((cur - end).norm() / end.norm()) <= _TOL[torch.float32]
    assert float((got.double() - whole.double()).norm() / whole.double().norm()) <= 2 * _TOL[torch.bfloat16]


def test_padding_tokens_leave_the_state():
    dev = _dev()
    ins, _ = _inputs(2, (2, 2, 2), 100, seed=31)
    ins = [t.to(dev) for t in ins]
    ins[3][:, :, 60:] = 0
    ins[4][:, :, 60:] = 0
    _, padded = gated_delta_attention(*ins[:5], initial_state=ins[5])
    _, short = gated_delta_attention(*(t[:, :, :60] for t in ins[:5]), initial_state=ins[5])
    assert torch.equal(padded, short)


def test_repeats_streams_and_other_tensors_agree():
    dev = _dev()
    ins, ups = _inputs(2, (14, 2, 2), 333, dtype=torch.bfloat16, seed=37)
    ins, ups = [t.to(dev) for t in ins], [t.to(dev) for t in ups]

    def run():
        leaves = [t.clone().requires_grad_() for t in ins]
        outs = gated_delta_attention(*leaves[:5], initial_state=leaves[5])
        return [*outs, *torch.autograd.grad(outs, leaves, ups)]

    want = run()
    side = [torch.cuda.Stream(dev) for _ in range(2)]
    results = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream(dev))
    for s in side * 2:
        with torch.cuda.stream(s):
            results.append(run())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_captured_training_and_steps_replay():
    dev = _dev()
    ins, ups = _inputs(2, (14, 2, 2), 150, dtype=torch.bfloat16, seed=41)
    ins, ups = [t.to(dev) for t in ins], [t.to(dev) for t in ups]
    steps = [t[:, :, :1].contiguous() for t in ins[:5]]
    state = ins[5].clone()

    def train():
        leaves = [t.detach().requires_grad_() for t in ins]
        outs = gated_delta_attention(*leaves[:5], initial_state=leaves[5])
        return [*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, ups)]

    def step():
        return gated_delta_step(*steps, state)

    eager = [t.clone() for t in train()]
    graphs, results = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        train()
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    for graph, call in zip(graphs, (train, step)):
        with torch.cuda.graph(graph):
            results.append(call())
    state.copy_(ins[5])
    filler = torch.randn(1 << 20, device=dev)
    want = ins[5].clone()
    for rep in range(3):
        filler.mul_(1.0001).add_(0.5)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(results[0], eager)), rep
        out = gated_delta_step(*steps, want)
        assert torch.equal(out, results[1]) and torch.equal(want, state), rep


def test_double_backward_is_refused():
    dev = _dev()
    ins, ups = _inputs(1, (1, 1, 1), 5)
    leaves = [t.to(dev).requires_grad_() for t in ins]
    outs = gated_delta_attention(*leaves[:5], initial_state=leaves[5])
    with pytest.raises(RuntimeError, match="double backward"):
        torch.autograd.grad(outs, leaves, [t.to(dev) for t in ups], create_graph=True)

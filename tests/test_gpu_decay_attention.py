"""The kernels of attention with decays against the recurrence in float64.

Tolerances, as the norm of the error over the norm of the result, are counted in
roundings. float32 results pass chains of two products of 64 terms each, 128
roundings of at most 2^-24. A bf16 result is rounded once, by at most 2^-8, and so is the state that its
share is taken from: both in the norm by 2^-8 / sqrt(3) at most, where values are spread over a step, together
0.82 2^-8; its scores are in two parts, off by at most 2^-16 each. A float16 result is off by at most 2^-11, on top
of the float32 chain and of scores and states in two parts."""

import pytest
import torch

from oal_amd.decay_attention import decay_attention, decay_step
from oracle.decay_oracle import decay_attention as definition

pytestmark = pytest.mark.gpu

_CHAIN = 128 * 2.0 ** -24
_TOL = {torch.float32: _CHAIN, torch.bfloat16: 2.0 ** -8 + 2.0 ** -14, torch.float16: 2.0 ** -11 + 2.0 ** -14 + _CHAIN}
_NAMES = ("out", "state", "dq", "dk", "dv", "dg", "dstate")


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _inputs(b, heads, n, d=64, dv=None, dtype=torch.float32, seed=0, decay=0.3, per_head=False):
    hq, hk, hv = heads
    dv = dv or d
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(b, h, n, d, generator=gen).to(dtype) for h in (hq, hk))
    v = torch.randn(b, hv, n, dv, generator=gen).to(dtype)
    g = -decay * torch.rand(b, hv, n, generator=gen) * torch.arange(1, hv + 1)[:, None]
    if per_head:
        g = g[0, :, 0].clone()
    state = torch.randn(b, hv, d, dv, generator=gen)
    dout = torch.randn(b, max(hq, hv), n, dv, generator=gen).to(dtype)
    dstate = torch.randn(b, hv, d, dv, generator=gen)
    return [q, k, v, g, state], [dout, dstate]


def _close(name, got, want, dtype):
    got, want = got.detach().to(want.device), want.detach()
    assert got.dtype == dtype and got.shape == want.shape, name
    err = float((got.double() - want).norm()) / max(float(want.norm()), 1e-30)
    assert err <= _TOL[dtype], f"{name}: {err:.3g}"


def _check(ins, ups, scale=0.125, with_state=True, on="cpu"):
    dev = _dev()
    want_ins = [t.to(on).double().requires_grad_() for t in ins]
    want = definition(*want_ins[:4], want_ins[4] if with_state else None, scale=scale)
    count = 5 if with_state else 4
    want = [*want, *torch.autograd.grad(want, want_ins[:count], [t.to(on).double() for t in ups])]
    got_ins = [t.to(dev).requires_grad_() for t in ins]
    got = decay_attention(*got_ins[:4], scale=scale, initial_state=got_ins[4] if with_state else None)
    got = [*got, *torch.autograd.grad(got, got_ins[:count], [t.to(dev) for t in ups])]
    types = [ups[0].dtype, torch.float32, *(t.dtype for t in ins[:count])]
    for name, x, y, dtype in zip(_NAMES, got, want, types):
        _close(name, x, y, dtype)


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 16, 63, 64, 65, 127, 129, 300, 700])
def test_lengths(n, dtype, per_head):
    _check(*_inputs(2, (2, 2, 2), n, dtype=dtype, seed=n, per_head=per_head))


@pytest.mark.parametrize("heads,n", [((2, 1, 1), 6001), ((14, 14, 14), 2688)])
def test_long_sequences_of_slow_decays(heads, n):
    ins, ups = _inputs(1, heads, n, dtype=torch.bfloat16, seed=n, decay=0.002)
    _check(ins, ups, on=_dev())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(14, 2, 2), (7, 7, 14), (2, 2, 6), (4, 2, 4), (1, 1, 3), (3, 1, 1)])
def test_heads_shared_in_both_directions(heads, dtype):
    _check(*_inputs(2, heads, 200, dtype=dtype, seed=7))


@pytest.mark.parametrize("d,dv", [(64, 32), (48, 64), (1, 1), (33, 7)])
def test_narrow_heads(d, dv):
    _check(*_inputs(1, (2, 1, 2), 190, d=d, dv=dv, seed=d))


@pytest.mark.parametrize("per_head", [False, True])
def test_no_state(per_head):
    _check(*_inputs(2, (2, 2, 2), 150, dtype=torch.bfloat16, per_head=per_head), with_state=False)


@pytest.mark.parametrize("kind", ["keep", "forget", "mixed", "grow"])
def test_gates_at_their_ends(kind):
    ins, ups = _inputs(1, (2, 2, 2), 200, seed=3)
    g = ins[3]
    if kind == "keep":
        g.zero_()
    elif kind == "forget":
        g.fill_(-30.0)
    elif kind == "mixed":  # a few tokens that forget all but nothing, slow decay elsewhere
        g.mul_(0.1)
        g[..., ::37] = -300.0
    else:
        g.copy_(0.01 * torch.rand(g.shape, generator=torch.Generator().manual_seed(2)))
    _check(ins, ups)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_texts_are_texts_by_themselves(dtype):
    """Texts that begin with a decay of -inf, on a chunk's border and inside, one of a single token."""
    ins, ups = _inputs(1, (4, 2, 2), 260, dtype=dtype, seed=5)
    starts = [64, 70, 71, 128, 200]
    ins[3][..., starts] = -float("inf")
    dev = _dev()
    leaves = [t.to(dev).requires_grad_() for t in ins]
    whole, end = decay_attention(*leaves[:4], scale=0.125, initial_state=leaves[4])
    grads = torch.autograd.grad((whole, end), leaves, [t.to(dev) for t in ups])
    edges = [0, *starts, 260]
    for lo, hi in zip(edges, edges[1:]):
        part = [t[:, :, lo:hi].double().requires_grad_() for t in ins[:4]]
        part[3].data[..., 0] = ins[3][..., 0].double() if lo == 0 else 0.0
        state = ins[4].double().requires_grad_() if lo == 0 else None
        outs = definition(*part, state, scale=0.125)
        up = [ups[0][:, :, lo:hi].double(), ups[1].double() if hi == 260 else torch.zeros_like(outs[1])]
        want = torch.autograd.grad(outs, part, up)
        _close("out", whole[:, :, lo:hi], outs[0], dtype)
        for name, x, y in zip(("dq", "dk", "dv"), grads, want):
            _close(f"{name} from {lo}", x[:, :, lo:hi], y, dtype)
        dg = grads[3][:, :, lo:hi].cpu().double()
        if lo:
            assert not dg[..., 0].any()  # what was forgotten does not matter
            dg, want_dg = dg[..., 1:], want[3][..., 1:]
        else:
            want_dg = want[3]
        assert float((dg - want_dg).norm()) <= _CHAIN * float(want_dg.norm())
    _close("state", end, outs[1], torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_rows(dtype):
    dev = _dev()
    ins, _ = _inputs(2, (4, 2, 2), 77, dtype=dtype, seed=13)
    dense = [t.to(dev) for t in ins]
    want = decay_attention(*dense[:4], scale=0.125, initial_state=dense[4])
    token_major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dense[:4]]
    odd = []
    for t in dense[:3]:
        wide = torch.zeros((*t.shape[:3], 65), dtype=dtype, device=dev)
        wide[..., 1:] = t
        odd.append(wide[..., 1:])
    for views in (token_major, odd + dense[3:4]):
        got = decay_attention(*views, scale=0.125, initial_state=dense[4])
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_one_decay_per_head_is_that_decay_for_every_token():
    dev = _dev()
    ins, ups = _inputs(2, (2, 2, 2), 140, seed=17, per_head=True)
    ins, ups = [t.to(dev) for t in ins], [t.to(dev) for t in ups]
    grads, outs = [], []
    for g in (ins[3].clone(), ins[3][None, :, None].expand(2, 2, 140)):
        leaf = g.clone().requires_grad_()
        # a strided view of decays, as a head's one value expanded, serves too
        outs.append(decay_attention(*ins[:3], leaf if leaf.ndim == 1 else leaf.expand(2, 2, 140), scale=0.125, initial_state=ins[4]))
        grads.append(torch.autograd.grad(outs[-1], leaf, ups)[0])
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    # 280 float32 values of one sum, each off by half a step
    each = grads[1].double()
    assert float((grads[0].double() - each.sum((0, 2))).abs().max()) <= 2.0 ** -23 * float(each.abs().sum((0, 2)).max())
    expanded = decay_attention(*ins[:3], ins[3][None, :, None].expand(2, 2, 140), scale=0.125, initial_state=ins[4])
    assert all(torch.equal(x, y) for x, y in zip(expanded, outs[0]))


@pytest.mark.parametrize("per_head", [False, True])
def test_gradient_against_differences(per_head):
    dev = _dev()
    ins, ups = _inputs(1, (2, 1, 2), 70, d=8, seed=19, per_head=per_head)
    ups = [t.to(dev).double() for t in ups]
    ins = [t.to(dev) for t in ins]

    def loss(ts):
        outs = decay_attention(*ts[:4], scale=0.3, initial_state=ts[4])
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


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,d,dv,n", [((2, 2, 2), 64, 64, 1), ((14, 2, 2), 64, 64, 3), ((2, 2, 6), 33, 7, 2),
                                          ((1, 1, 1), 1, 1, 5), ((4, 2, 2), 40, 24, 70)])
def test_step(heads, d, dv, n, dtype, per_head):
    dev = _dev()
    ins, _ = _inputs(3, heads, n, d=d, dv=dv, dtype=dtype, seed=23, per_head=per_head)
    want, want_state = definition(*ins, scale=0.3)
    q, k, v, g, state = (t.to(dev) for t in ins)
    version = state._version
    out = decay_step(q, k, v, g, state, scale=0.3)
    assert state._version > version
    _close("out", out, want, dtype)
    _close("state", state, want_state, torch.float32)


def test_step_at_odd_addresses_and_forgetting():
    dev = _dev()
    ins, _ = _inputs(2, (4, 2, 4), 3, dtype=torch.bfloat16, seed=25)
    ins[3][0, :, 1] = -float("inf")
    want, want_state = definition(*ins, scale=0.3)
    views = []
    for t in ins[:4]:
        wide = torch.zeros((*t.shape[:-1], t.shape[-1] + 1), dtype=t.dtype, device=dev)
        wide[..., 1:] = t.to(dev)
        views.append(wide[..., 1:])
    room = torch.zeros(ins[4].numel() + 1, device=dev)
    state = room[1:].view(ins[4].shape)
    state.copy_(ins[4])
    out = decay_step(*views, state, scale=0.3)
    _close("out", out, want, torch.bfloat16)
    _close("state", state, want_state, torch.float32)
    assert float(room[0]) == 0


def test_pieces_and_steps_continue_a_sequence():
    """A prompt in two pieces, then token by token, is the sequence in one call."""
    dev = _dev()
    ins, _ = _inputs(2, (4, 2, 4), 200, dtype=torch.bfloat16, seed=29)
    q, k, v, g, state = (t.to(dev) for t in ins)
    whole, end = decay_attention(q, k, v, g, initial_state=state)
    parts, cur = [], state
    for lo, hi in ((0, 90), (90, 190)):
        out, cur = decay_attention(*(t[:, :, lo:hi] for t in (q, k, v, g)), initial_state=cur)
        parts.append(out)
    cur = cur.clone()
    for t in range(190, 200):
        parts.append(decay_step(*(x[:, :, t:t + 1] for x in (q, k, v, g)), cur))
    got = torch.cat(parts, 2)
    assert float((cur - end).norm() / end.norm()) <= _CHAIN
    assert float((got.double() - whole.double()).norm() / whole.double().norm()) <= 2 * _TOL[torch.bfloat16]


def test_padding_tokens_leave_the_state():
    dev = _dev()
    ins, _ = _inputs(2, (2, 2, 2), 300, seed=31)
    ins = [t.to(dev) for t in ins]
    ins[1][:, :, 60:] = 0
    ins[3][:, :, 60:] = 0
    _, padded = decay_attention(*ins[:4], initial_state=ins[4])
    _, short = decay_attention(*(t[:, :, :60] for t in ins[:4]), initial_state=ins[4])
    # sequences of one chunk and of five are cut into other segments: the same terms, added up in another order
    assert float((padded - short).norm()) <= _CHAIN * float(short.norm())
    # behind the chunk with the last token nothing changes any more, whatever the queries and values there
    ins[0][:, :, 64:] = 7.0
    ins[2][:, :, 64:] = -3.0
    _, other = decay_attention(*ins[:4], initial_state=ins[4])
    assert torch.equal(padded, other)


def test_a_sequence_does_not_depend_on_the_others_of_its_batch():
    dev = _dev()
    ins, _ = _inputs(3, (4, 2, 2), 333, dtype=torch.bfloat16, seed=33)
    ins = [t.to(dev) for t in ins]
    out, end = decay_attention(*ins[:4], initial_state=ins[4])
    ins[0][0] = 1e4
    ins[1][2] = -1e4
    ins[3][0] = -1.0
    other, other_end = decay_attention(*ins[:4], initial_state=ins[4])
    assert torch.equal(out[1], other[1]) and torch.equal(end[1], other_end[1])


def test_repeats_streams_and_other_tensors_agree():
    dev = _dev()
    ins, ups = _inputs(2, (14, 2, 2), 333, dtype=torch.bfloat16, seed=37)
    ins, ups = [t.to(dev) for t in ins], [t.to(dev) for t in ups]

    def run():
        leaves = [t.clone().requires_grad_() for t in ins]
        outs = decay_attention(*leaves[:4], initial_state=leaves[4])
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


@pytest.mark.parametrize("per_head", [False, True])
def test_captured_training_and_steps_replay(per_head):
    dev = _dev()
    ins, ups = _inputs(2, (14, 2, 2), 450, dtype=torch.bfloat16, seed=41, per_head=per_head)
    ins, ups = [t.to(dev) for t in ins], [t.to(dev) for t in ups]
    steps = [t[:, :, :1].contiguous() if t.ndim > 1 else t for t in ins[:4]]
    state = ins[4].clone()

    def train():
        leaves = [t.detach().requires_grad_() for t in ins]
        outs = decay_attention(*leaves[:4], initial_state=leaves[4])
        return [*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, ups)]

    def step():
        return decay_step(*steps, state)

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
    state.copy_(ins[4])
    filler = torch.randn(1 << 20, device=dev)
    want = ins[4].clone()
    for rep in range(3):
        filler.mul_(1.0001).add_(0.5)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(results[0], eager)), rep
        out = decay_step(*steps, want)
        assert torch.equal(out, results[1]) and torch.equal(want, state), rep


def test_double_backward_is_refused():
    dev = _dev()
    ins, ups = _inputs(1, (1, 1, 1), 5)
    leaves = [t.to(dev).requires_grad_() for t in ins]
    outs = decay_attention(*leaves[:4], initial_state=leaves[4])
    with pytest.raises(RuntimeError, match="double backward"):
        torch.autograd.grad(outs, leaves, [t.to(dev) for t in ups], create_graph=True)

"""The head norms with rotary embedding against their formulas in float64.

Tolerances, as the norm of the error over the norm of the result, are counted in roundings.
A float32 row passes a sum of 64 squares, its root and quotient, a mean of 64 products
and the rotation, fewer than 160 roundings of at most 2^-24; a weight's gradient adds sums over
a thread's tokens and a block's rows, fewer than 160 more. A 16-bit result is rounded once on top, by at
most half its step."""

import pytest
import torch

from oal_amd.norm_rotary import norm_rotary_heads
from oracle.heads_oracle import norm_rotary

pytestmark = pytest.mark.gpu

_ROW = 160 * 2.0 ** -24
_TOL = {torch.float32: 2 * _ROW, torch.bfloat16: 2.0 ** -8 + 2 * _ROW, torch.float16: 2.0 ** -11 + 2 * _ROW}
_NAMES = ("q", "k", "v", "dq", "dk", "dv", "dq_weight", "dk_weight")


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _tables(rows, rotary, dtype=torch.float32):
    angle = torch.outer(torch.arange(rows, dtype=torch.float64), 1e4 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary))
    return angle.repeat(1, 2).cos().to(dtype), angle.repeat(1, 2).sin().to(dtype)


def _inputs(b, heads, n, d=64, rotary=None, dtype=torch.float32, weight="shared", weight_dtype=torch.float32, seed=0,
            table_dtype=torch.float32, rows=None):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(b, n, h * d, generator=gen).to(dtype) for h in (heads[0], heads[1], heads[1]))
    ws = [None, None]
    if weight != "none":
        ws = [(1 + 0.3 * torch.randn(*((d,) if weight == "shared" else (h, d)), generator=gen)).to(weight_dtype) for h in heads]
    ups = [torch.randn(b, h, n, d, generator=gen).to(dtype) for h in (heads[0], heads[1], heads[1])]
    return [q, k, v, *ws], ups, _tables(rows or n, rotary or d, table_dtype)


def _check(ins, ups, tables, heads, positions=None, eps=1e-6, on="cpu"):
    dev = _dev()
    options = dict(q_heads=heads[0], kv_heads=heads[1], eps=eps)

    def both(leaves, call, at, tables, ups, ps):
        outs = call(*leaves, *(t.to(at) for t in tables), positions=ps, **options)
        wrt = [t for t in leaves if t is not None]
        return [*outs, *torch.autograd.grad(outs, wrt, [t.to(at) for t in ups])]

    want = both([t if t is None else t.to(on).double().requires_grad_() for t in ins], norm_rotary, on, tables,
                [t.double() for t in ups], None if positions is None else positions.to(on))
    got = both([t if t is None else t.to(dev).requires_grad_() for t in ins], norm_rotary_heads, dev, tables, ups,
               None if positions is None else positions.to(dev))
    types = [*(t.dtype for t in ups), *(t.dtype for t in ins if t is not None)]
    for name, x, y, dtype in zip(_NAMES, got, want, types):
        x, y = x.detach().to(y.device), y.detach()
        assert x.dtype == dtype and x.shape == y.shape, name
        err = float((x.double() - y).norm()) / max(float(y.norm()), 1e-30)
        assert err <= _TOL[dtype], f"{name}: {err:.3g}"
        if name in ("v", "dv"):
            assert torch.equal(x.double(), y)  # moved, not computed


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 5, 67, 1030])
def test_lengths(n, dtype):
    _check(*_inputs(2, (14, 2), n, dtype=dtype, seed=n), (14, 2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,rotary", [(64, 32), (48, 48), (32, 32), (16, 16), (64, 48), (64, 20), (40, 20), (33, 2), (7, 6), (2, 2), (63, 62)])
def test_dimensions(d, rotary, dtype):
    _check(*_inputs(2, (3, 1), 37, d=d, rotary=rotary, dtype=dtype, seed=d), (3, 1))


@pytest.mark.parametrize("weight", ["shared", "each", "none"])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (14, 14), (40, 20), (100, 50), (5, 64)])
def test_heads_and_weights(heads, weight):
    _check(*_inputs(2, heads, 41, dtype=torch.bfloat16, weight=weight, seed=heads[0]), heads)


@pytest.mark.parametrize("weight_dtype,table_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                                      (torch.bfloat16, torch.float32)])
def test_types_of_weights_and_tables(weight_dtype, table_dtype):
    _check(*_inputs(2, (4, 2), 50, dtype=torch.bfloat16, weight="each", weight_dtype=weight_dtype, table_dtype=table_dtype), (4, 2))


def test_one_weight_alone():
    ins, ups, tables = _inputs(1, (2, 2), 30)
    _check([*ins[:3], ins[3], None], ups, tables, (2, 2))
    _check([*ins[:3], None, ins[4]], ups, tables, (2, 2))


def test_many_tokens():
    # more blocks than there are sums of them: every block takes several turns
    _check(*_inputs(2, (2, 1), 9001, d=16, dtype=torch.bfloat16, seed=3), (2, 1), on=_dev())


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions(kind):
    ins, ups, tables = _inputs(3, (4, 2), 33, dtype=torch.bfloat16, rows=700)
    at = torch.randint(0, 700, (3, 33), generator=torch.Generator().manual_seed(1), dtype=kind)
    _check(ins, ups, tables, (4, 2), positions=at)


@pytest.mark.parametrize("d", [64, 40])
def test_no_token_and_positions_past_the_tables(d):
    dev = _dev()
    ins, ups, tables = _inputs(2, (4, 2), 9, d=d, rows=20)
    at = torch.arange(18).view(2, 9)
    at[0, 3], at[1, 8] = -1, -(1 << 40)
    _check(ins, ups, tables, (4, 2), positions=at)
    at[1, 0], at[1, 1] = 20, 1 << 40
    outs = norm_rotary_heads(*(t.to(dev) for t in ins), *(t.to(dev) for t in tables), q_heads=4, kv_heads=2, positions=at.to(dev))
    for t, turned in zip(outs, (True, True, False)):
        bad = torch.isnan(t).any(-1)
        assert bad[1, :, :2].all() == turned and not bad[0].any() and not bad[1, :, 2:].any()


def test_nothing_but_zeros():
    # a row of zeros is divided by the root of eps
    ins, ups, tables = _inputs(1, (2, 1), 5, dtype=torch.float32)
    ins[0][:, 2] = 0
    _check(ins, ups, tables, (2, 1), eps=1e-3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_slices_of_one_projection(dtype):
    dev = _dev()
    ins, ups, tables = _inputs(2, (4, 2), 21, dtype=dtype, seed=5)
    dense = [t.to(dev) for t in ins]
    fused = torch.cat(dense[:3], -1)
    odd = torch.zeros((2, 21, fused.shape[-1] + 1), dtype=dtype, device=dev)
    odd[..., 1:] = fused
    turned = fused.transpose(1, 2).contiguous().transpose(1, 2)
    sizes = [t.shape[-1] for t in dense[:3]]

    def run(q, k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, *dense[3:])]
        outs = norm_rotary_heads(*leaves, *(t.to(dev) for t in tables), q_heads=4, kv_heads=2)
        return [*outs, *torch.autograd.grad(outs, leaves, [t.to(dev) for t in ups])]

    want = run(*dense[:3])
    for whole in (fused, odd[..., 1:], turned):
        got = run(*whole.split(sizes, -1))
        for name, x, y in zip(_NAMES, got, want):
            # lanes that move values one by one add them up in another order
            x, y = x.detach(), y.detach()
            assert float((x.double() - y.double()).norm()) <= 2 * _TOL[x.dtype] * float(y.double().norm()), name
    # each row of the batch the same one
    one = [t[:1].expand(2, -1, -1) for t in dense[:3]]
    for x, y in zip(run(*one), run(*(t.contiguous() for t in one))):
        assert torch.equal(x, y)


def test_gradients_that_are_not_asked_for():
    dev = _dev()
    ins, ups, tables = _inputs(2, (4, 2), 21, seed=7)
    ins, ups, tables = ([t.to(dev) for t in ts] for ts in (ins, ups, tables))

    def run(wrt, used):
        leaves = [t.clone().requires_grad_(i in wrt) for i, t in enumerate(ins)]
        outs = norm_rotary_heads(*leaves, *tables, q_heads=4, kv_heads=2)
        return torch.autograd.grad([outs[i] for i in used], [leaves[i] for i in wrt], [ups[i] for i in used], allow_unused=True)

    full = run(range(5), range(3))
    for wrt in ([0], [1], [2], [3], [4], [0, 4], [3, 4], [1, 2]):
        for got, i in zip(run(wrt, range(3)), wrt):
            assert torch.equal(got, full[i]), wrt
    # a result that nothing asks about counts as zero
    dq, dk, dv, dqw, dkw = run(range(5), [0])
    assert torch.equal(dq, full[0]) and torch.equal(dqw, full[3])
    assert not dk.any() and not dv.any() and not dkw.any()


def test_gradient_against_differences():
    dev = _dev()
    ins, ups, tables = _inputs(1, (2, 1), 6, d=8, weight="each", seed=19)
    ins, tables = [t.to(dev) for t in ins], [t.to(dev) for t in tables]
    ups = [t.to(dev).double() for t in ups]

    def loss(ts):
        outs = norm_rotary_heads(*ts, *tables, q_heads=2, kv_heads=1)
        return sum((o.double() * up).sum() for o, up in zip(outs, ups))

    leaves = [t.clone().requires_grad_() for t in ins]
    grads = torch.autograd.grad(loss(leaves), leaves)
    gen = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        way = torch.randn(ins[i].shape, generator=gen).to(dev)
        h = 1e-2 / float(way.abs().max())
        ends = [loss([t + s * h * way if j == i else t for j, t in enumerate(ins)]) for s in (1, -1)]
        slope, want = float(ends[0] - ends[1]) / (2 * h), float((grad * way).double().sum())
        # third differences of order h^2, and sums of a hundred float32 terms over 2 h
        assert abs(slope - want) <= 2e-3 * (abs(want) + float(grad.norm() * way.norm()) * 0.1), _NAMES[i + 3]


def test_repeats_streams_and_captured_calls_agree():
    dev = _dev()
    ins, ups, tables = _inputs(2, (14, 2), 133, dtype=torch.bfloat16, weight="each", seed=37)
    ins, ups, tables = ([t.to(dev) for t in ts] for ts in (ins, ups, tables))
    at = torch.randint(0, 133, (2, 133), generator=torch.Generator().manual_seed(1)).to(dev)

    def run():
        leaves = [t.detach().requires_grad_() for t in ins]
        outs = norm_rotary_heads(*leaves, *tables, q_heads=14, kv_heads=2, positions=at)
        return [*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, ups)]

    want = [t.clone() for t in run()]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    filler = torch.randn(1 << 20, device=dev)
    for rep in range(3):
        filler.mul_(1.0001).add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, want)), rep


def test_agrees_with_the_rotary_embedding_alone():
    """Without a weight, rows of mean square one come out as the model's rotary embedding turns them."""
    from oal_amd.qwen_oal import rotary_heads

    dev = _dev()
    ins, _, tables = _inputs(2, (14, 2), 50, weight="none")
    q, k, v = (t.to(dev) for t in ins[:3])
    q, k = ((t.view(2, 50, -1, 64) / t.view(2, 50, -1, 64).square().mean(-1, keepdim=True).sqrt()).flatten(2) for t in (q, k))
    cos, sin = (t.to(dev) for t in tables)
    got = norm_rotary_heads(q, k, v, None, None, cos, sin, q_heads=14, kv_heads=2, eps=0.0)
    for x, y in zip(got, rotary_heads(q, k, v, cos, sin, 14, 2, 64)):
        assert float((x - y).norm()) <= _TOL[torch.float32] * float(y.norm())


def test_double_backward_is_refused():
    dev = _dev()
    ins, ups, tables = _inputs(1, (1, 1), 5)
    leaves = [t.to(dev).requires_grad_() for t in ins]
    outs = norm_rotary_heads(*leaves, *(t.to(dev) for t in tables), q_heads=1, kv_heads=1)
    with pytest.raises(RuntimeError, match="double backward"):
        torch.autograd.grad(outs, leaves, [t.to(dev) for t in ups], create_graph=True)

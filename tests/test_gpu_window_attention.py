"""The windowed attention kernels against all pairs in float64.

Tolerances, as the norm of the error over the norm of the result, are counted in
roundings. float32: two products of 64 terms and a softmax summed in tiles of 64 with
a rounding for each of its maximum's changes, 256 roundings of at most 2^-24. bfloat16: the
weights or their gradients, the output that the backward starts from, the products'
difference and the result are rounded, four roundings of at most 2^-8. float16 runs the
float32 kernels, or holds its weights to 16 bits, and rounds its result: 2^-11 on top."""

import math

import pytest
import torch

from oal_amd.gated_delta import gated_delta_attention, gated_delta_step
from oal_amd.window_attention import window_attention, window_attention_step, window_cache
from oracle.window_oracle import window_attention as dense

pytestmark = pytest.mark.gpu

_TOL = {torch.float32: 256 * 2.0 ** -24, torch.bfloat16: 4 * 2.0 ** -8, torch.float16: 2.0 ** -11 + 256 * 2.0 ** -24}


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _qkv(b, heads, nq, nk=None, d=64, dv=None, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    hq, hk = heads
    nk, dv = nk or nq, dv or d
    shapes = ((b, hq, nq, d), (b, hk, nk, d), (b, hk, nk, dv), (b, hq, nq, dv))
    return [torch.randn(s, generator=gen).to(dtype) for s in shapes]


def _near(x, y, dtype, name="out", floor=0.0):
    assert x.dtype == dtype and x.shape == y.shape, name
    err = float((x.detach().double().cpu() - y.detach().cpu()).norm())
    assert err <= _TOL[dtype] * max(float(y.detach().norm()), floor), f"{name}: {err / max(float(y.detach().norm()), 1e-30):.3g}"


def _check(qkvo, window, sinks, scale=None):
    dev = _dev()
    dtype, scale = qkvo[0].dtype, scale or qkvo[0].shape[-1] ** -0.5
    ref = [t.double().requires_grad_() for t in qkvo[:3]]
    want = dense(*ref, window=window, sinks=sinks, scale=scale)
    want_grads = torch.autograd.grad(want, ref, qkvo[3].double())
    leaves = [t.to(dev).requires_grad_() for t in qkvo[:3]]
    got = window_attention(*leaves, window=window, sinks=sinks, scale=scale)
    grads = torch.autograd.grad(got, leaves, qkvo[3].to(dev))
    _near(got, want, dtype)
    # the gradients of the scores are differences of terms of dv's size: they vanish where a row sees one key alone
    for name, x, y in zip(("dq", "dk", "dv"), grads, want_grads):
        _near(x, y, dtype, name, floor=float(want_grads[2].norm()) * 0.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (17, 4), (64, 0), (65, 70), (100, 4), (1000, 3), (5, 1000)])
@pytest.mark.parametrize("n", [1, 2, 33, 64, 65, 200, 333])
def test_lengths_and_windows(n, window, sinks, dtype):
    _check(_qkv(1, (2, 1), n, dtype=dtype, seed=n), window, sinks)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(14, 2), (1, 1), (3, 1), (8, 8), (9, 1), (17, 1)])
def test_heads(heads, dtype):
    _check(_qkv(2, heads, 150, dtype=dtype, seed=5), 40, 3)


@pytest.mark.parametrize("d,dv", [(48, 48), (64, 32), (1, 1), (33, 7)])
def test_narrow_heads(d, dv):
    _check(_qkv(1, (4, 2), 90, d=d, dv=dv, seed=d), 30, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 300), (37, 300), (64, 129), (299, 300)])
@pytest.mark.parametrize("window,sinks", [(50, 4), (400, 0), (1, 100)])
def test_queries_behind_earlier_keys(nq, nk, window, sinks, dtype):
    _check(_qkv(1, (4, 2), nq, nk, dtype=dtype, seed=nk + nq), window, sinks)


def test_long_sequence_with_sinks():
    # many tiles between the first keys and the window
    _check(_qkv(1, (2, 1), 1500, seed=3), 130, 70)


def test_large_scores():
    qkvo = _qkv(1, (2, 2), 130, seed=8)
    qkvo[0] *= 20.0
    dev = _dev()
    want = dense(*qkvo[:3], window=50, sinks=2, scale=1.0)
    got = window_attention(*(t.to(dev) for t in qkvo[:3]), window=50, sinks=2, scale=1.0)
    # scores up to about 800: a rounding of 2^-24 of one is 800 2^-24 in its weight
    assert float((got.double().cpu() - want).norm() / want.norm()) <= 64 * 800 * 2.0 ** -24


def test_scores_below_any_that_a_sum_starts_from():
    # all scores about -6e33 and equal: the weights are too
    dev = _dev()
    q, k, v, _ = (t.to(dev) for t in _qkv(1, (2, 1), 30, seed=4))
    got = window_attention(torch.full_like(q, -1e16), torch.full_like(k, 1e16), v, window=7, scale=1.0)
    want = dense(torch.zeros(1, 2, 30, 64), torch.zeros(1, 1, 30, 64), v.double().cpu(), window=7, sinks=0, scale=1.0)
    _near(got, want, torch.float32)


def test_one_query_far_from_its_heads():
    # the stride of a dimension of one row does not matter
    dev = _dev()
    q, k, v, _ = (t.to(dev) for t in _qkv(1, (2, 1), 1, 30, seed=4))
    far = q.as_strided(q.shape, (128, 64, 1 << 25, 1))
    assert torch.equal(window_attention(far, k, v, window=7, sinks=2), window_attention(q, k, v, window=7, sinks=2))


def test_widest_window_and_all_first_keys():
    dev = _dev()
    q, k, v, o = (t.to(dev) for t in _qkv(2, (4, 2), 150, dtype=torch.bfloat16, seed=6))
    results = []
    for window, sinks in ((150, 0), (150, 150), (1 << 30, 1 << 30)):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = window_attention(*leaves, window=window, sinks=sinks)
        results.append([out, *torch.autograd.grad(out, leaves, o)])
    for result in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(result, results[0]))
    _check(_qkv(2, (4, 2), 150, dtype=torch.bfloat16, seed=6), 1, 1 << 30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_rows(dtype):
    dev = _dev()
    q, k, v, _ = (t.to(dev) for t in _qkv(2, (4, 2), 77, dtype=dtype, seed=13))
    want = window_attention(q, k, v, window=20, sinks=3)
    token_major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    odd = []
    for t in (q, k, v):
        wide = torch.zeros((*t.shape[:3], 65), dtype=dtype, device=dev)
        wide[..., 1:] = t
        odd.append(wide[..., 1:])
    one_head = [t[:, :1].expand(-1, t.shape[1], -1, -1) for t in (k, v)]
    assert torch.equal(window_attention(*token_major, window=20, sinks=3), want)
    assert torch.equal(window_attention(*odd, window=20, sinks=3), want)
    assert torch.equal(window_attention(q, *one_head, window=20, sinks=3),
                       window_attention(q, *(t.contiguous() for t in one_head), window=20, sinks=3))


def test_gradient_against_differences():
    dev = _dev()
    qkvo = [t.to(dev) for t in _qkv(1, (4, 2), 70, d=8, seed=19)]

    def loss(ts):
        return (window_attention(*ts, window=20, sinks=3).double() * qkvo[3].double()).sum()

    leaves = [t.clone().requires_grad_() for t in qkvo[:3]]
    grads = torch.autograd.grad(loss(leaves), leaves)
    gen = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        way = torch.randn(qkvo[i].shape, generator=gen).to(dev)
        h = 1e-2 / float(way.abs().max())
        ends = [loss([t + s * h * way if j == i else t for j, t in enumerate(qkvo[:3])]) for s in (1, -1)]
        slope, want = float(ends[0] - ends[1]) / (2 * h), float((grad * way).double().sum())
        # third differences of order h^2, and sums of a few thousand float32 terms over 2 h
        assert abs(slope - want) <= 2e-3 * (abs(want) + float(grad.norm() * way.norm()) * 0.1)


def test_padding_at_the_end_changes_nothing_before_it():
    dev = _dev()
    q, k, v, do = (t.to(dev) for t in _qkv(2, (4, 2), 100, dtype=torch.bfloat16, seed=31))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, window=30, sinks=2)
    grads = torch.autograd.grad(out, leaves, torch.where(torch.arange(100, device=dev)[:, None] < 70, do, 0))
    short = [t[:, :, :70].clone().requires_grad_() for t in (q, k, v)]
    want = window_attention(*short, window=30, sinks=2)
    want_grads = torch.autograd.grad(want, short, do[:, :, :70].contiguous())
    assert torch.equal(out[:, :, :70], want)
    for x, y in zip(grads, want_grads):
        assert float((x[:, :, :70].double() - y.double()).norm()) <= 2.0 ** -8 * float(y.double().norm())
        assert not x[:, :, 70:].any()


# ---------------------------------------------------------------------------
# The ring cache
# ---------------------------------------------------------------------------


def _reference_step(q, k, v, history, positions, window, sinks, scale):
    """Each sequence's token over its own history of keys and values [Hkv, p, D]."""
    outs = []
    for x, p in enumerate(positions):
        hk, hv = (torch.cat((h, t[x]), 1)[None] for h, t in zip(history[x], (k, v)))
        outs.append(dense(q[x:x + 1], hk, hv, window=window, sinks=sinks, scale=scale))
    return torch.cat(outs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,d,dv", [((14, 2), 64, 64), ((1, 1), 8, 16), ((17, 1), 48, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (200, 0), (700, 70)])
def test_step_over_caches_of_any_age(window, sinks, heads, d, dv, dtype):
    dev = _dev()
    gen = torch.Generator().manual_seed(window)
    size = window + sinks
    positions = [0, 1, max(0, sinks - 1), sinks, size - 1, size, size + 1, 3 * size + 5]
    b, (hq, hk) = len(positions), heads
    q, k, v = (torch.randn(b, h, 1, w, generator=gen).to(dtype) for h, w in ((hq, d), (hk, d), (hk, dv)))
    n = max(positions)
    past = [torch.randn(b, hk, max(n, 1), w, generator=gen).to(dtype) for w in (d, dv)]
    lengths = torch.tensor(positions)
    kc, vc = window_cache(*(t.to(dev) for t in past), window=window, sinks=sinks, lengths=lengths.to(dev))
    for x, p in enumerate(positions):
        for cache, t in ((kc, past[0]), (vc, past[1])):
            want = torch.zeros(hk, size, t.shape[-1], dtype=dtype)
            for j in range(p):
                want[:, j if j < sinks else sinks + (j - sinks) % window] = t[x, :, j]
            assert torch.equal(cache[x].cpu(), want)
    # what lies in slots that no token has filled must not matter
    for cache in (kc, vc):
        for x, p in enumerate(positions):
            cache[x, :, min(p, size):] = float("nan")
    before = [kc.clone(), vc.clone()]
    out = window_attention_step(*(t.to(dev) for t in (q, k, v)), kc, vc, lengths.to(dev), window=window, sinks=sinks,
                                scale=0.2)
    history = [[t[x, :, :p] for t in past] for x, p in enumerate(positions)]
    _near(out, _reference_step(q, k, v, history, positions, window, sinks, 0.2), dtype)
    for cache, old, new in zip((kc, vc), before, (k, v)):
        for x, p in enumerate(positions):
            old[x, :, p if p < sinks else sinks + (p - sinks) % window] = new[x, :, 0].to(dev)
        assert torch.equal(cache.isnan(), old.isnan()) and torch.equal(cache.nan_to_num(), old.nan_to_num())


def test_step_without_a_token_leaves_its_caches():
    dev = _dev()
    gen = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(3, h, 1, 64, generator=gen).to(dev) for h in (4, 2, 2))
    kc, vc = (torch.randn(3, 2, 20, 64, generator=gen).to(dev) for _ in range(2))
    old = kc.clone(), vc.clone()
    version = kc._version
    out = window_attention_step(q, k, v, kc, vc, torch.tensor([5, -1, 30], dtype=torch.int32, device=dev), window=16, sinks=4)
    assert not out[1].any() and torch.equal(kc[1], old[0][1]) and torch.equal(vc[1], old[1][1])
    assert torch.equal(kc[0, :, 5], k[0, :, 0]) and torch.equal(vc[2, :, 4 + 26 % 16], v[2, :, 0])
    assert kc._version > version


@pytest.mark.parametrize("batch,window,sinks", [(1, 65536, 0), (1, 40000, 7), (130, 300, 4), (2, 128, 0)])
def test_step_in_as_many_pieces_as_the_cache_has(batch, window, sinks):
    dev = _dev()
    gen = torch.Generator().manual_seed(window)
    q, k, v = (torch.randn(batch, h, 1, 64, generator=gen) for h in (4, 2, 2))
    kc, vc = (torch.randn(batch, 2, window + sinks, 64, generator=gen) for _ in range(2))
    at = sinks + 3 * window + 5
    got = window_attention_step(*(t.to(dev) for t in (q, k, v)), kc.to(dev), vc.to(dev),
                                torch.full((batch,), at, device=dev), window=window, sinks=sinks, scale=0.2)
    kc[:, :, sinks + 5 % window], vc[:, :, sinks + 5 % window] = k[:, :, 0], v[:, :, 0]
    score = 0.2 * q.double().view(batch, 2, 2, 64) @ kc.double().transpose(2, 3)
    want = torch.softmax(score, -1) @ vc.double()
    _near(got, want.view(batch, 4, 1, 64), torch.float32)


def test_step_takes_slices_of_larger_caches():
    dev = _dev()
    gen = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(2, h, 1, 64, generator=gen).to(dev, torch.bfloat16) for h in (4, 2, 2))
    big = torch.randn(2, 30, 2, 2, 64, generator=gen).to(dev, torch.bfloat16)
    views = [big[:, :20, x].transpose(1, 2) for x in (0, 1)]
    dense_caches = [t.contiguous() for t in views]
    at = torch.tensor([11, 100], device=dev)
    outside = big[:, 20:].clone()
    got = window_attention_step(q, k, v, *views, at, window=16, sinks=4)
    want = window_attention_step(q, k, v, *dense_caches, at, window=16, sinks=4)
    assert torch.equal(got, want) and torch.equal(big[:, 20:], outside)
    assert all(torch.equal(x, y) for x, y in zip(views, dense_caches))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens_is_the_whole_sequence(dtype):
    """A stack of a windowed and a gated delta layer: a padded batch of prompts, then token
    by token, against the whole sequences in one call each."""
    dev = _dev()
    window, sinks, steps, lengths = 24, 3, 40, [50, 31]
    n = max(lengths) + steps
    q, k, v, _ = (t.to(dev) for t in _qkv(2, (4, 2), n, dtype=dtype, seed=9))
    gen = torch.Generator().manual_seed(10)
    g = (-torch.rand(2, 2, n, generator=gen)).to(dev)
    beta = torch.rand(2, 2, n, generator=gen).to(dev)
    unit = [torch.nn.functional.normalize(t.float(), dim=-1).to(dtype) for t in (q, k)]
    whole = window_attention(q, k, v, window=window, sinks=sinks)
    whole_delta, _ = gated_delta_attention(*unit, v, g, beta)
    at = torch.tensor(lengths, device=dev)
    m = max(lengths)
    pad = torch.arange(m, device=dev)[None, None] >= at[:, None, None]
    prompt = [t[:, :, :m] for t in (q, k, v)]
    caches = window_cache(*prompt[1:], window=window, sinks=sinks, lengths=at)
    _, state = gated_delta_attention(unit[0][:, :, :m], unit[1][:, :, :m], prompt[2], g[:, :, :m].masked_fill(pad, 0),
                                     beta[:, :, :m].masked_fill(pad, 0))
    state = state.contiguous()
    rows = torch.arange(2, device=dev)
    for step in range(steps):
        token = [t[rows, :, at][:, :, None] for t in (q, k, v)]
        out = window_attention_step(*token, *caches, at, window=window, sinks=sinks)
        want = whole[rows, :, at][:, :, None]
        assert float((out.double() - want.double()).norm()) <= 2 * _TOL[dtype] * float(want.double().norm()), step
        out = gated_delta_step(*(t[rows, :, at][:, :, None] for t in (*unit, v)), *(t[rows, :, at][:, :, None] for t in (g, beta)), state)
        want = whole_delta[rows, :, at][:, :, None]
        assert float((out.double() - want.double()).norm()) <= 2 * _TOL[dtype] * float(want.double().norm()), step
        at = at + 1


def test_repeats_and_streams_agree():
    dev = _dev()
    qkvo = [t.to(dev) for t in _qkv(2, (14, 2), 500, dtype=torch.bfloat16, seed=37)]
    caches = [torch.randn(2, 2, 604, 64, device=dev).to(torch.bfloat16) for _ in range(2)]
    at = torch.tensor([600, 10000], device=dev)

    def run():
        leaves = [t.detach().requires_grad_() for t in qkvo[:3]]
        out = window_attention(*leaves, window=100, sinks=4)
        own = [t.clone() for t in caches]
        with torch.no_grad():
            step = window_attention_step(*(t[:, :, :1].contiguous() for t in qkvo[:3]), *own, at, window=600, sinks=4)
        return [out.detach(), *torch.autograd.grad(out, leaves, qkvo[3]), step, *own]

    want = run()
    torch.cuda.synchronize()
    results = []
    for s in [torch.cuda.Stream(dev) for _ in range(2)] * 2:
        with torch.cuda.stream(s):
            results.append(run())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_captured_training_and_steps_replay():
    dev = _dev()
    qkvo = [t.to(dev) for t in _qkv(2, (14, 2), 300, dtype=torch.bfloat16, seed=41)]
    caches = [torch.randn(2, 2, 604, 64, device=dev).to(torch.bfloat16) for _ in range(2)]
    mine = [t.clone() for t in caches]
    token = [t[:, :, :1].contiguous() for t in qkvo[:3]]
    at = torch.tensor([601, 3], device=dev)

    def train():
        leaves = [t.detach().requires_grad_() for t in qkvo[:3]]
        out = window_attention(*leaves, window=100, sinks=4)
        return [out.detach(), *torch.autograd.grad(out, leaves, qkvo[3])]

    def step():
        return window_attention_step(*token, *caches, at, window=600, sinks=4)

    eager = [t.clone() for t in train()]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        train()
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graphs, results = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, call in zip(graphs, (train, step)):
        with torch.cuda.graph(graph):
            results.append(call())
    filler = torch.randn(1 << 20, device=dev)
    for rep in range(3):
        filler.mul_(1.0001).add_(0.5)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(results[0], eager)), rep
        out = window_attention_step(*token, *mine, at, window=600, sinks=4)
        assert torch.equal(out, results[1]) and all(torch.equal(x, y) for x, y in zip(caches, mine)), rep
        at.add_(1)


def test_double_backward_is_refused():
    dev = _dev()
    leaves = [t.to(dev).requires_grad_() for t in _qkv(1, (1, 1), 5)[:3]]
    out = window_attention(*leaves, window=3)
    with pytest.raises(RuntimeError, match="double backward"):
        torch.autograd.grad(out.sum(), leaves, create_graph=True)

"""The token scores against log_softmax in float64.

Tolerances: an exponential of a difference z to the maximum is off by the rounding of z log2 e, at most 2^-23 |z|
for |z| up to 32, and its own two; a lane's sum of some hundred terms and the tree over lanes add fewer than
100 roundings of 2^-24 on terms of one sign. Scores of a few units are differences of such logarithms: 200
roundings of 2^-24 relative to the norm, and as many for float32 gradients, whose largest terms are of
order one. A 16-bit gradient is rounded once on top, by at most half its step, and for float16 by at most
2^-25 where it is subnormal."""

import math

import pytest
import torch

from oal_amd.token_scores import token_log_probs
from oracle.heads_oracle import token_scores, top_tokens

pytestmark = pytest.mark.gpu

_SUM = 200 * 2.0 ** -24
_TOL = {torch.float32: _SUM, torch.bfloat16: 2.0 ** -8 + _SUM, torch.float16: 2.0 ** -11 + _SUM}


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _inputs(shape, vocab, dtype=torch.float32, seed=0, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    logits = (spread * torch.randn(*shape, vocab, generator=gen)).to(dtype)
    tokens = torch.randint(0, vocab, shape, generator=gen)
    return logits, tokens, [torch.randn(shape, generator=gen), torch.randn(shape, generator=gen)]


def _near(name, got, want, tol, floor=0.0):
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    assert got.shape == want.shape, name
    err = float((got - want).norm())
    assert err <= tol * float(want.norm()) + floor * math.sqrt(want.numel()), f"{name}: {err / max(float(want.norm()), 1e-30):.3g}"


def _check(logits, tokens, ups, top=0):
    dev = _dev()
    leaf = logits.double().requires_grad_()
    want = token_scores(leaf, tokens.long())
    want_grad, = torch.autograd.grad(want, leaf, [t.double() for t in ups])
    mine = logits.to(dev).requires_grad_()
    got = token_log_probs(mine, tokens.to(dev), entropy=True, top=top)
    grad, = torch.autograd.grad((got.log_probs, got.entropy), mine, [t.to(dev) for t in ups])
    assert got.log_probs.dtype == got.entropy.dtype == torch.float32 and grad.dtype == logits.dtype
    # entropies of a row that has all weight in one place are differences of numbers of order one
    _near("log_probs", got.log_probs, want[0], _SUM, _SUM)
    _near("entropy", got.entropy, want[1], _SUM, _SUM)
    _near("gradient", grad, want_grad, _TOL[logits.dtype], 2.0 ** -25 if logits.dtype is torch.float16 else 2.0 ** -24)
    if top:
        value, place = top_tokens(logits, top)
        assert got.top_tokens.dtype == torch.int64 and torch.equal(got.top_tokens.cpu(), place)
        log = torch.log_softmax(logits.double(), -1).gather(-1, place)
        fine = torch.isfinite(log)
        assert torch.equal(torch.isfinite(got.top_log_probs).cpu(), fine)
        _near("top_log_probs", got.top_log_probs.cpu()[fine], log[fine], _SUM, _SUM)
        assert not got.top_log_probs.requires_grad
    else:
        assert got.top_log_probs is None and got.top_tokens is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 64, 65, 511, 2048, 2049, 5001, 50001])
def test_vocabularies(vocab, dtype):
    _check(*_inputs((3, 5), vocab, dtype, seed=vocab), top=min(vocab, 20))


@pytest.mark.parametrize("top", [1, 2, 33, 64])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (1, 100), (3, 30011), (600, 1000)])
def test_alternatives(rows, vocab, top):
    _check(*_inputs((rows,), vocab, torch.bfloat16, seed=top), top=top)


@pytest.mark.parametrize("rows", [1, 2, 100, 1100])
def test_rows_whole_and_in_parts(rows):
    _check(*_inputs((rows,), 20003, torch.float32, seed=rows), top=3)


@pytest.mark.parametrize("order", ["rising", "falling", "equal", "two values", "zeros of both signs"])
@pytest.mark.parametrize("rows,vocab", [(2, 70000), (1030, 700)])
def test_orders_that_change_the_list_often_or_tie(order, rows, vocab):
    _, tokens, ups = _inputs((rows,), vocab, seed=1)
    line = torch.arange(vocab, dtype=torch.float32) * (8.0 / vocab)
    row = {"rising": line, "falling": -line, "equal": torch.full((vocab,), 3.0), "two values": torch.arange(vocab) % 977 // 976 * 2.0,
           "zeros of both signs": torch.where(torch.arange(vocab) % 3 == 0, -0.0, 0.0)}[order]
    _check(row.expand(rows, vocab).contiguous(), tokens, ups, top=64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_logits(dtype):
    """-inf and the type's lowest value; rows with one token left, fewer than alternatives, and first and last alone."""
    logits, tokens, ups = _inputs((6,), 9001, dtype, seed=5)
    logits[0, ::2] = -math.inf
    logits[1, 1:] = -math.inf
    logits[2, :-1] = -math.inf
    logits[3, 17:] = torch.finfo(dtype).min
    logits[4, 5:8990] = -math.inf
    for i in range(6):
        tokens[i] = int(torch.isfinite(logits[i]).nonzero()[i % 3 if i not in (1, 2) else 0])
    _check(logits, tokens, ups, top=40)


def test_a_token_that_cannot_be():
    dev = _dev()
    logits, tokens, _ = _inputs((4,), 300)
    logits[2, 7] = -math.inf
    tokens[2] = 7
    leaf = logits.to(dev).requires_grad_()
    got = token_log_probs(leaf, tokens.to(dev))
    assert float(got.log_probs[2].detach()) == -math.inf and torch.isfinite(got.log_probs[[0, 1, 3]]).all()
    grad, = torch.autograd.grad(got.log_probs[[0, 1, 3]].sum(), leaf)
    assert torch.isfinite(grad).all()


def test_rows_without_a_distribution():
    dev = _dev()
    logits, tokens, _ = _inputs((5,), 3000)
    logits[0] = -math.inf
    logits[1, 100] = math.nan
    logits[2, 2999] = math.inf
    logits[3, 0] = math.nan
    got = token_log_probs(logits.to(dev), tokens.to(dev), entropy=True, top=4)
    for t in got[:3]:
        assert torch.isnan(t[:4].flatten(1) if t.ndim > 1 else t[:4]).all() and torch.isfinite(t[4]).all()
    assert ((got.top_tokens >= -1) & (got.top_tokens < 3000)).all()


@pytest.mark.parametrize("rows", [4, 1500])
def test_places_without_a_token(rows):
    dev = _dev()
    logits, tokens, ups = _inputs((rows,), 1000, seed=9)
    tokens[1], tokens[3] = -100, -1
    _check(logits, tokens, ups)
    tokens[2] = 1000
    leaf = logits.to(dev).requires_grad_()
    got = token_log_probs(leaf, tokens.to(dev), entropy=True)
    assert float(got.log_probs[1].detach()) == 0 and torch.isnan(got.log_probs[2]) and torch.isfinite(got.entropy).all()
    grad, = torch.autograd.grad(got.log_probs, leaf, torch.ones(rows, device=dev))
    assert not grad[1].any() and torch.isnan(grad[2]).all() and torch.isfinite(grad[0]).all()
    grad, = torch.autograd.grad(token_log_probs(leaf, tokens.to(dev)).log_probs[[0, 1, 3]].sum(), leaf)
    assert not grad[1].any() and torch.isfinite(grad[0]).all()


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_tokens_of_both_types_and_any_layout(kind):
    dev = _dev()
    logits, tokens, _ = _inputs((6, 4), 99)
    want = token_log_probs(logits.to(dev), tokens.to(dev))
    turned = tokens.to(kind).t().contiguous().to(dev).t()
    assert torch.equal(token_log_probs(logits.to(dev), turned).log_probs, want.log_probs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [96, 4099])
def test_rows_at_any_place(vocab, dtype):
    """Next-token slices, rows at odd addresses, columns of a wider matrix, transposed logits, one row for all, more dimensions."""
    dev = _dev()
    logits, tokens, ups = _inputs((3, 7), vocab, dtype, seed=3)
    dense, token = logits.to(dev), tokens.to(dev)
    ups = [t.to(dev) for t in ups]

    def run(x, t=token, ups=ups):
        leaf = x.detach().requires_grad_()
        got = token_log_probs(leaf, t, entropy=True, top=5)
        return [*got, *torch.autograd.grad(got[:2], leaf, ups)]

    want = run(dense)
    longer = torch.zeros((3, 9, vocab), dtype=dtype, device=dev)
    longer[:, 1:8] = dense
    wide = torch.zeros((3, 7, vocab + 13), dtype=dtype, device=dev)
    wide[..., 5:5 + vocab] = dense
    # a row at another address is summed in another order
    for view in (longer[:, 1:8], wide[..., 5:5 + vocab], dense.transpose(1, 2).contiguous().transpose(1, 2),
                 dense.transpose(0, 1).contiguous().transpose(0, 1)):
        for x, y in zip(run(view), want):
            if x.dtype == torch.int64:
                assert torch.equal(x, y)
            else:
                _near("strided", x, y, 2 * _TOL[x.dtype], _SUM)
    flat = run(dense.flatten(0, 1), token.flatten(), [t.flatten() for t in ups])
    deep = run(dense.view(3, 1, 7, 1, vocab), token.view(3, 1, 7, 1), [t.view(3, 1, 7, 1) for t in ups])
    one = run(dense[0, 0], token[0, 0], [t[0, 0] for t in ups])
    for x, y, z, want_ in zip(flat, deep, one, want):
        assert torch.equal(x.view_as(want_), want_) and torch.equal(y.view_as(want_), want_)
        if x.dtype == torch.int64:
            assert torch.equal(z, want_[0, 0])
        else:
            _near("one row", z, want_[0, 0], 2 * _TOL[z.dtype], _SUM)
    same = dense[:1, :1].expand(3, 7, vocab)
    for x, y in zip(run(same), run(same.contiguous())):
        if vocab == 96 or x.dtype == torch.int64:
            assert torch.equal(x, y)
        else:  # rows of an odd vocabulary lie at other addresses once they are copied, and are summed in another order
            _near("one row for all", x, y, 2 * _TOL[x.dtype], _SUM)


def test_no_rows():
    dev = _dev()
    logits = torch.zeros((2, 0, 50), dtype=torch.bfloat16, device=dev, requires_grad=True)
    got = token_log_probs(logits, torch.zeros((2, 0), dtype=torch.int64, device=dev), entropy=True, top=3)
    assert got.log_probs.shape == got.entropy.shape == (2, 0) and got.top_tokens.shape == got.top_log_probs.shape == (2, 0, 3)
    grad, = torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), logits)
    assert grad.shape == logits.shape


def test_offsets_past_32_bits():
    """Rows whose elements lie past 2^31 of the first."""
    dev = _dev()
    if torch.cuda.get_device_properties(dev).total_memory < 64 << 30:
        pytest.skip("needs 16 GiB")
    rows, vocab = 15000, 151936
    logits = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=dev)
    tail, tokens, ups = _inputs((4,), vocab, torch.bfloat16, seed=21)
    logits[-4:] = tail.to(dev)
    token = torch.zeros(rows, dtype=torch.int64, device=dev)
    token[-4:] = tokens.to(dev)
    logits.requires_grad_()
    got = token_log_probs(logits, token, entropy=True, top=2)
    up = [torch.zeros(rows, device=dev) for _ in range(2)]
    for u, t in zip(up, ups):
        u[-4:] = t.to(dev)
    grad, = torch.autograd.grad(got[:2], logits, up)
    leaf = tail.double().requires_grad_()
    want = token_scores(leaf, tokens)
    _near("log_probs", got.log_probs[-4:], want[0], _SUM, _SUM)
    _near("gradient", grad[-4:], torch.autograd.grad(want, leaf, [t.double() for t in ups])[0], _TOL[torch.bfloat16])
    assert torch.equal(got.top_tokens[-4:].cpu(), top_tokens(tail, 2)[1]) and not grad[-5].any()
    assert float((got.log_probs[:-4].detach() + math.log(vocab)).abs().max()) <= _SUM * math.log(vocab)


def test_each_gradient_by_itself():
    dev = _dev()
    logits, tokens, ups = _inputs((40,), 777, seed=13)
    for i in range(2):
        leaf = logits.double().requires_grad_()
        want, = torch.autograd.grad(token_scores(leaf, tokens)[i], leaf, ups[i].double())
        mine = logits.to(dev).requires_grad_()
        got = token_log_probs(mine, tokens.to(dev), entropy=True)
        grad, = torch.autograd.grad(got[i], mine, ups[i].to(dev))
        _near(str(i), grad, want, _SUM)


def test_the_models_loss():
    """The mean of the scores is the model's loss, and so is its gradient."""
    from oal_amd.qwen_oal import causal_lm_loss

    dev = _dev()
    logits, tokens, _ = _inputs((2, 30), 4000, torch.bfloat16, seed=15)
    grads, losses = [], []
    for loss in (lambda x, t: causal_lm_loss(x, t), lambda x, t: -token_log_probs(x[:, :-1], t[:, 1:]).log_probs.mean()):
        leaf = logits.to(dev).requires_grad_()
        losses.append(loss(leaf, tokens.to(dev)))
        grads.append(torch.autograd.grad(losses[-1], leaf)[0])
    losses = [float(t.detach()) for t in losses]
    assert abs(losses[0] - losses[1]) <= _SUM * losses[0]
    _near("gradient", grads[1], grads[0], 2 * _TOL[torch.bfloat16])


def test_gradient_against_differences():
    dev = _dev()
    logits, tokens, ups = _inputs((3,), 50, seed=17)
    logits, tokens = logits.to(dev), tokens.to(dev)
    ups = [t.to(dev).double() for t in ups]

    def loss(x):
        got = token_log_probs(x, tokens, entropy=True)
        return sum((o.double() * up).sum() for o, up in zip(got, ups))

    leaf = logits.clone().requires_grad_()
    grad, = torch.autograd.grad(loss(leaf), leaf)
    way = torch.randn(logits.shape, generator=torch.Generator().manual_seed(1)).to(dev)
    h = 1e-2 / float(way.abs().max())
    slope, want = float(loss(logits + h * way) - loss(logits - h * way)) / (2 * h), float((grad * way).double().sum())
    # third differences of order h^2, and a few float32 logarithms over 2 h
    assert abs(slope - want) <= 2e-3 * (abs(want) + float(grad.norm() * way.norm()) * 0.1)


@pytest.mark.parametrize("rows,vocab", [(2, 60001), (1200, 500)])
def test_repeats_streams_and_captured_calls_agree(rows, vocab):
    dev = _dev()
    logits, tokens, ups = _inputs((rows,), vocab, torch.bfloat16, seed=19)
    logits, tokens, ups = logits.to(dev), tokens.to(dev), [t.to(dev) for t in ups]

    def run():
        leaf = logits.detach().requires_grad_()
        got = token_log_probs(leaf, tokens, entropy=True, top=7)
        return [*(t.detach() for t in got), *torch.autograd.grad(got[:2], leaf, ups)]

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


def test_double_backward_is_refused():
    dev = _dev()
    logits, tokens, ups = _inputs((3,), 50)
    leaf = logits.to(dev).requires_grad_()
    got = token_log_probs(leaf, tokens.to(dev))
    with pytest.raises(RuntimeError, match="double backward"):
        torch.autograd.grad(got.log_probs, leaf, ups[0].to(dev), create_graph=True)

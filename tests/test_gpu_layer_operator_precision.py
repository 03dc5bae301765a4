"""How exact the kernels of attention with decays, of head norms and of token scores are, at the size of the
errors that their roundings leave: a rounding more, or a term of a product lost, shows.

Errors are norms of the error over the norm of the result, against float64."""

import pytest
import torch

from oal_amd.decay_attention import decay_attention, decay_step
from oal_amd.norm_rotary import norm_rotary_heads
from oal_amd.token_scores import token_log_probs
from oracle.decay_oracle import decay_attention as definition
from oracle.heads_oracle import norm_rotary, token_scores

pytestmark = pytest.mark.gpu

_NAMES = ("out", "state", "dq", "dk", "dv", "dg", "dstate")


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _error(x, y):
    return float((x.detach().double() - y.detach().double()).norm() / y.detach().double().norm())


def _inputs(b, heads, n, dtype, seed, decay, d=64, dv=64, per_head=False):
    gen = torch.Generator().manual_seed(seed)
    hq, hk, hv = heads
    q, k, v = (torch.randn(b, h, n, x, generator=gen).to(dtype) for h, x in ((hq, d), (hk, d), (hv, dv)))
    g = -decay * torch.rand(b, hv, n, generator=gen)
    if per_head:
        g = g[0, :, 0].clone()
    state, dstate = (torch.randn(b, hv, d, dv, generator=gen) for _ in range(2))
    dout = torch.randn(b, max(hq, hv), n, dv, generator=gen).to(dtype)
    dev = _dev()
    return [t.to(dev) for t in (q, k, v, g, state)], [t.to(dev) for t in (dout, dstate)]


def _with_gradients(call, ins, ups):
    leaves = [t.detach().clone().requires_grad_() for t in ins]
    outs = call(*leaves[:4], leaves[4])
    return dict(zip(_NAMES, (*outs, *torch.autograd.grad(outs, leaves, ups))))


def _exact(ins, ups, scale=0.125):
    return _with_gradients(lambda *x: definition(*x, scale=scale), [t.double() for t in ins], [t.double() for t in ups])


def _ours(ins, ups, scale=0.125):
    return _with_gradients(lambda q, k, v, g, s: decay_attention(q, k, v, g, scale=scale, initial_state=s), ins, ups)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(2, 2, 2), (6, 2, 2), (2, 2, 6)])
def test_results_with_decays_are_rounded_once(heads, dtype):
    """16-bit results against the exact ones rounded to their type. What is rounded may be off by two parts' error,
    2^-17 of a term and 2^-16 of a sum of two such; an error e before the rounding moves a result to
    its neighbour, a step u away, with a chance of |e| / u, so that the mean square of what moves is u |e|: with
    u at most eps of the value, at most the root of 2^-16 eps in the norm. One operand of one part, 2^-9 of it, moves
    sixteen times as many."""
    ins, ups = _inputs(2, heads, 700, dtype, seed=61, decay=0.02)
    want, got = _exact(ins, ups), _ours(ins, ups)
    bound = (2.0 ** -16 * torch.finfo(dtype).eps) ** 0.5
    for name in ("out", "dq", "dk", "dv"):
        err = _error(got[name], want[name].to(dtype))
        print(f"{heads} {dtype} {name}: {err:.2e} of {bound:.2e}", flush=True)
        assert got[name].dtype == dtype and err <= bound, f"{name}: {err:.3g}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,peaks", [(24, 151936, (14, 24)), (1100, 20000, (12, 22)), (7, 1000, (10, 20))])
def test_scores_of_rows_with_nearly_all_weight_in_one_place(rows, vocab, peaks, dtype):
    """A model that is sure: the log probability of what it expects and the entropy are small sums over all the
    other tokens, whose terms have one sign. Their exponents, up to 42 in base two, are rounded by half of 2^-18 at most,
    1.4e-6 of a term, and their sums by 24 roundings of 2^-24 at most: each result is off by 4e-6 of itself at
    most. In sums of 32 bits from one on it was up to 2e-2."""
    gen = torch.Generator().manual_seed(vocab)
    logits = torch.randn(rows, vocab, generator=gen)
    tokens = torch.randint(0, vocab, (rows,), generator=gen)
    logits[torch.arange(rows), tokens] = torch.linspace(*peaks, rows)
    logits = logits.to(dtype).to(_dev())
    tokens = tokens.to(logits.device)
    log = torch.log_softmax(logits.double(), -1)
    # 1 - p as a sum, which is what float64 has left of it too
    rest = log.exp().scatter(-1, tokens[:, None], 0.0)
    sure = torch.log1p(-rest.sum(-1))
    want = {"log_probs": sure, "entropy": -(rest * log).sum(-1) - sure.exp() * sure, "top_log_probs": sure}
    got = token_log_probs(logits, tokens, entropy=True, top=1)
    assert torch.equal(got.top_tokens[:, 0], tokens)
    for name, y in want.items():
        err = float(((getattr(got, name).double().view(rows) - y) / y).abs().max())
        print(f"{rows} {vocab} {dtype} {name}: {err:.2e}", flush=True)
        assert err <= 4e-6, f"{name}: {err:.3g}"


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(2, 2, 2), (14, 2, 2), (2, 2, 6)])
def test_float32_results_with_decays(heads, dtype, per_head):
    """Sums of some hundred terms, whose roundings of 2^-24 go either way: a few of them in the norm, whatever the type
    of the tokens."""
    ins, ups = _inputs(2, heads, 400, dtype, seed=63, decay=0.1, per_head=per_head)
    want, got = _exact(ins, ups), _ours(ins, ups)
    for name in ("state", "dg", "dstate") if dtype is not torch.float32 else _NAMES:
        err = _error(got[name], want[name])
        print(f"{heads} {dtype} {name}: {err:.2e}", flush=True)
        assert got[name].dtype == torch.float32 and err <= 8 * 2.0 ** -24, f"{name}: {err:.3g}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_single_tokens_are_rounded_once(dtype):
    """Token by token through the head norms, the recurrence and the scores: norms of a token do not depend on the
    others, the recurrence's results are the exact ones rounded, and so are the scores."""
    gen = torch.Generator().manual_seed(67)
    dev = _dev()
    q, k, v = (torch.randn(2, 30, h * 64, generator=gen).to(dtype).to(dev) for h in (6, 2, 2))
    weights = [1 + 0.1 * torch.randn(64, generator=gen).to(dev) for _ in range(2)]
    angle = torch.outer(torch.arange(30, dtype=torch.float64), 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).repeat(1, 2)
    tables = [angle.cos().float().to(dev), angle.sin().float().to(dev)]
    g = -0.1 * torch.rand(2, 2, 30, generator=gen).to(dev)
    options = dict(q_heads=6, kv_heads=2)
    whole = norm_rotary_heads(q, k, v, *weights, *tables, **options)
    want, want_state = definition(*whole, g, scale=0.125)
    state = torch.zeros(2, 2, 64, 64, device=dev)
    outs = []
    for t in range(30):
        at = torch.full((2, 1), t, device=dev)
        one = norm_rotary_heads(*(x[:, t:t + 1] for x in (q, k, v)), *weights, *tables, positions=at, **options)
        assert all(torch.equal(x, y[:, :, t:t + 1]) for x, y in zip(one, whole))
        outs.append(decay_step(*one, g[:, :, t:t + 1], state, scale=0.125))
    out = torch.cat(outs, 2)
    # float32: 64 terms, and a rounding of the state a token; 16-bit: that, in a root as above
    few = 8 * 2.0 ** -24
    assert _error(state, want_state) <= few
    bound = few if dtype is torch.float32 else (few * torch.finfo(dtype).eps) ** 0.5
    assert _error(out, want.to(dtype)) <= bound
    logits = (3 * torch.randn(2, 30, 1000, generator=gen)).to(dtype).to(dev)
    tokens = torch.randint(0, 1000, (2, 30), generator=gen).to(dev)
    rows = token_log_probs(logits, tokens, entropy=True, top=5)
    for t in range(30):
        one = token_log_probs(logits[:, t:t + 1], tokens[:, t:t + 1], entropy=True, top=5)
        assert torch.equal(one.top_tokens, rows.top_tokens[:, t:t + 1])
        for x, y in zip(one[:3], rows[:3]):
            assert _error(x, y[:, t:t + 1]) <= 2 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(20, 151936), (2000, 5001), (6, 99)])
def test_scores_of_ordinary_rows(rows, vocab, dtype):
    """A score's own rounding of 2^-24, and exponentials whose errors, up to 2^-24 |z|, go either way over many terms: two
    roundings. A gradient has one exponential, of z down to -25 where it matters, and is rounded with that: 16
    roundings of 2^-24 in float32, and in 16 bits as results above."""
    gen = torch.Generator().manual_seed(vocab)
    logits = (2.5 * torch.randn(rows, vocab, generator=gen)).to(dtype).to(_dev())
    tokens = torch.randint(0, vocab, (rows,), generator=gen).to(logits.device)
    ups = [torch.randn(rows, generator=gen).to(logits.device) for _ in range(2)]
    found = []
    for call, cast in ((token_scores, torch.Tensor.double), (lambda x, t: token_log_probs(x, t, entropy=True)[:2], torch.Tensor.clone)):
        leaf = cast(logits).requires_grad_()
        outs = call(leaf, tokens)
        found.append([*outs, *torch.autograd.grad(outs, leaf, [cast(t) for t in ups])])
    for name, want, got in zip(("log_probs", "entropy", "gradient"), *found):
        eps = torch.finfo(got.dtype).eps
        bound = 2 * 2.0 ** -24 if name != "gradient" else 16 * 2.0 ** -24
        if got.dtype is not torch.float32:  # float16: what is subnormal is off by half of 2^-24 at most
            floor = 2.0 ** -25 * want.numel() ** 0.5 / float(want.detach().norm()) if got.dtype is torch.float16 else 0.0
            want, bound = want.to(got.dtype), (bound * eps) ** 0.5 + floor
        err = _error(got, want)
        print(f"{rows} {vocab} {dtype} {name}: {err:.2e} of {bound:.2e}", flush=True)
        assert err <= bound, f"{name}: {err:.3g}"


@pytest.mark.parametrize("weight", ["shared", "each"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_head_norms_are_rounded_once(dtype, weight):
    """A float32 result passes a root, a quotient and a handful of products: four roundings in the norm, back eight, and
    a weight's sum over tokens as many; a 16-bit one is that rounded, as results above."""
    gen = torch.Generator().manual_seed(71)
    dev, heads = _dev(), (6, 2)
    ins = [torch.randn(2, 700, h * 64, generator=gen).to(dtype).to(dev) for h in (6, 2, 2)]
    ins += [(1 + 0.3 * torch.randn(*((64,) if weight == "shared" else (h, 64)), generator=gen)).to(dev) for h in heads]
    ups = [torch.randn(2, h, 700, 64, generator=gen).to(dtype).to(dev) for h in (6, 2, 2)]
    angle = torch.outer(torch.arange(700, dtype=torch.float64), 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).repeat(1, 2)
    tables = [angle.cos().float().to(dev), angle.sin().float().to(dev)]
    found = []
    for call, cast in ((norm_rotary, torch.Tensor.double), (norm_rotary_heads, torch.Tensor.clone)):
        leaves = [cast(t).requires_grad_() for t in ins]
        outs = call(*leaves, *tables, q_heads=6, kv_heads=2, eps=1e-6)
        found.append([*outs, *torch.autograd.grad(outs, leaves, [cast(t) for t in ups])])
    for name, want, got in zip(("q", "k", "v", "dq", "dk", "dv", "dq_weight", "dk_weight"), *found):
        bound = (8 if name.startswith("d") else 4) * 2.0 ** -24
        if got.dtype is not torch.float32:
            want, bound = want.to(dtype), (bound * torch.finfo(dtype).eps) ** 0.5
        err = _error(got, want)
        print(f"{weight} {dtype} {name}: {err:.2e} of {bound:.2e}", flush=True)
        assert err <= bound, f"{name}: {err:.3g}"

"""How exact the kernels of attention with decays, of head norms and of token scores are, at the size of the
errors that their roundings leave: a rounding more, or a term of a product lost, shows.

Errors are norms of the error over the norm of the result, against float64."""

import pytest
import torch

from oal_amd.decay_attention import decay_attention
from oal_amd.token_scores import token_log_probs
from oracle.decay_oracle import decay_attention as definition

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

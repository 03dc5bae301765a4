"""Gradients of token scores' rows that something is wrong with: a token past the vocabulary, no
token, no distribution. What does not depend on it stays as it is.

And the alternatives of all rows of a large call.

Tolerances: 200 roundings of 2^-24 of the norm for gradients; two where exponentials' errors go either way."""

import math

import pytest
import torch

from oal_amd.token_scores import token_log_probs
from oracle.heads_oracle import token_scores, top_tokens

pytestmark = pytest.mark.gpu

_SUM = 200 * 2.0 ** -24


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _inputs(rows, vocab, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return (2 * torch.randn(rows, vocab, generator=gen), torch.randint(0, vocab, (rows,), generator=gen),
            torch.randn(rows, generator=gen))


@pytest.mark.parametrize("rows,vocab", [(4, 50), (3, 40001), (1100, 700)])
def test_the_entropys_gradient_does_not_depend_on_the_token(rows, vocab):
    dev = _dev()
    logits, tokens, up = _inputs(rows, vocab)
    leaf = logits.double().requires_grad_()
    want, = torch.autograd.grad(token_scores(leaf, tokens)[1], leaf, up.double())
    tokens[0], tokens[1 % rows] = vocab, 2 ** 40
    mine = logits.to(dev).requires_grad_()
    got = token_log_probs(mine, tokens.to(dev), entropy=True)
    assert torch.isnan(got.log_probs[0].detach()) and torch.isfinite(got.entropy).all()
    grad, = torch.autograd.grad(got.entropy, mine, up.to(dev))
    assert float((grad.cpu().double() - want).norm()) <= _SUM * float(want.norm())
    # nor does it where the other rows' log probabilities have gradients beside it
    got = token_log_probs(mine, tokens.to(dev), entropy=True)
    none = torch.zeros(rows, device=dev)
    both, = torch.autograd.grad((got.log_probs, got.entropy), mine, (none, up.to(dev)))
    assert torch.equal(both, grad)
    # one that is asked for is NaN
    none[0] = 1.0
    grad, = torch.autograd.grad(token_log_probs(mine, tokens.to(dev)).log_probs, mine, none)
    assert torch.isnan(grad[0]).all() and not grad[1:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(6, 57), (5, 40001), (1100, 700)])
def test_rows_that_nothing_is_asked_about_have_no_gradient(rows, vocab, dtype):
    """Places without a token, as a padded batch has them, whose logits are whatever is there: the others' gradients are
    those of the others alone."""
    dev = _dev()
    logits, tokens, up = _inputs(rows, vocab, seed=3)
    logits = logits.to(dtype)
    clean = logits.to(dev).requires_grad_()
    tokens[:4] = torch.tensor([-1, -100, -1, -2])
    outs = token_log_probs(clean, tokens.to(dev), entropy=True)
    up = up.to(dev)
    live = torch.zeros(rows, device=dev)
    live[4:] = 1.0
    want, = torch.autograd.grad(outs[:2], clean, (up, up * live))
    logits[0], logits[1, 5], logits[2, -1] = -math.inf, math.nan, math.inf
    logits[3, vocab // 2:] = -math.inf
    leaf = logits.to(dev).requires_grad_()
    outs = token_log_probs(leaf, tokens.to(dev), entropy=True)
    assert not outs.log_probs[:4].any() and torch.isfinite(outs.log_probs).all()
    grad, = torch.autograd.grad(outs[:2], leaf, (up, up * live))
    assert not grad[:4].any() and torch.equal(grad, want)
    grad, = torch.autograd.grad(token_log_probs(leaf, tokens.to(dev)).log_probs, leaf, up)
    assert not grad[:4].any() and torch.isfinite(grad).all() and grad[4:].any()


@pytest.mark.parametrize("scale", [1.0, 1e10, 1e30])
def test_masked_logits_under_large_gradients(scale):
    """A logit of -inf has no gradient, however large the entropy's is (a scaled loss)."""
    dev = _dev()
    logits, tokens, up = _inputs(5, 3001, seed=5)
    logits[:, ::3] = -math.inf
    tokens = tokens // 3 * 3 + 1
    leaf = logits.double().requires_grad_()
    want, = torch.autograd.grad(token_scores(leaf, tokens)[1], leaf, scale * up.double())
    mine = logits.to(dev).requires_grad_()
    grad, = torch.autograd.grad(token_log_probs(mine, tokens.to(dev), entropy=True).entropy, mine, scale * up.to(dev))
    assert not grad[:, ::3].any()
    assert float((grad.cpu().double() - want).norm()) <= _SUM * float(want.norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,top", [(1100, 20003, 20), (300, 60000, 5), (1030, 50001, 64)])
def test_alternatives_of_every_row_over_many_turns(rows, vocab, top, dtype):
    """Rows of several turns of a block's waves, whole and in parts: the lists that the waves of a row share a limit for, with
    the many equal values that 16-bit logits have."""
    gen = torch.Generator().manual_seed(top)
    logits = (2 * torch.randn(rows, vocab, generator=gen)).to(dtype).to(_dev())
    tokens = torch.randint(0, vocab, (rows,), generator=gen).to(logits.device)
    values, places = top_tokens(logits, top)
    got = token_log_probs(logits, tokens, entropy=True, top=top)
    assert torch.equal(got.top_tokens, places)
    lse = torch.logsumexp(logits.double(), -1, keepdim=True)
    for x, y in ((got.top_log_probs, values - lse), (got.log_probs, logits.double().gather(-1, tokens[:, None])[:, 0] - lse[:, 0]),
                 (got.entropy, token_scores(logits, tokens)[1])):
        assert float((x.double() - y).norm()) <= 2 * 2.0 ** -24 * float(y.norm())

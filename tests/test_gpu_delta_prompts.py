"""A prompt read in one call, then single tokens over the state that the call returned, as it is."""

import pytest
import torch

from oal_amd.gated_delta import gated_delta_attention, gated_delta_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dv", [(64, 64), (12, 20), (33, 64), (64, 7), (1, 1)])
def test_steps_go_on_from_the_returned_state(d, dv):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    dev = torch.device("cuda:0")
    gen = torch.Generator().manual_seed(d)
    n, prompt = 75, 70
    q, k = (torch.nn.functional.normalize(torch.randn(2, h, n, d, generator=gen), dim=-1).to(dev) for h in (4, 2))
    v = torch.randn(2, 2, n, dv, generator=gen).to(dev)
    g = -0.3 * torch.rand(2, 2, n, generator=gen).to(dev)
    beta = torch.rand(2, 2, n, generator=gen).to(dev)
    ops = (q, k, v, g, beta)
    with torch.no_grad():
        whole, end = gated_delta_attention(*ops)
        head, state = gated_delta_attention(*(t[:, :, :prompt] for t in ops))
        assert state.is_contiguous()
        parts = [head, *(gated_delta_step(*(t[:, :, i:i + 1] for t in ops), state) for i in range(prompt, n))]
    # both ways pass chains of three products of 64 terms, 192 roundings of at most 2^-24 each
    for x, y in ((torch.cat(parts, 2), whole), (state, end)):
        assert float((x.double() - y.double()).norm()) <= 2 * 192 * 2.0 ** -24 * float(y.double().norm())


def test_gradients_pass_through_a_narrow_state():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    dev = torch.device("cuda:0")
    gen = torch.Generator().manual_seed(2)
    ops = [torch.randn(1, 2, 30, 12, generator=gen) * 0.2 for _ in range(3)]
    ops = [t.to(dev).requires_grad_() for t in (*ops, -torch.rand(1, 2, 30, generator=gen), torch.rand(1, 2, 30, generator=gen))]
    _, state = gated_delta_attention(*(t[:, :, :20] for t in ops))
    out, end = gated_delta_attention(*(t[:, :, 20:] for t in ops), initial_state=state)
    whole_out, whole_end = gated_delta_attention(*ops)
    ups = torch.randn(out.shape, generator=gen).to(dev), torch.randn(end.shape, generator=gen).to(dev)
    got = torch.autograd.grad((out, end), ops, ups)
    want = torch.autograd.grad((whole_out[:, :, 20:], whole_end), ops, ups)
    # the decays' gradients are sums over the tokens behind that cancel: a tenth of their terms' size at least
    for x, y in zip(got, want):
        assert float((x.double() - y.double()).norm()) <= 10 * 2 * 192 * 2.0 ** -24 * float(y.double().norm())

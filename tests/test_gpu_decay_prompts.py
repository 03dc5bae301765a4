"""Prompts of attention with decays by a model whose log-decays are parameters: nothing is kept for a backward
that there is not, and a call is the same whether a tensor could have a gradient or not."""

import pytest
import torch

from oal_amd.decay_attention import decay_attention

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("d", [64, 40, 20])
def test_a_prompt_keeps_no_states(d, mode):
    dev = _dev()
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 2, 8192, d, generator=gen).to(dev, torch.bfloat16) for _ in range(3))
    g = torch.nn.Parameter(torch.full((2,), -0.05, device=dev))
    with mode():
        want = decay_attention(q, k, v, g.detach())
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated(dev)
        room = []
        for decays in (g.detach(), g):
            torch.cuda.reset_peak_memory_stats(dev)
            got = decay_attention(q, k, v, decays)
            room.append(torch.cuda.max_memory_allocated(dev) - base)
            assert all(torch.equal(x, y) for x, y in zip(got, want)) and not any(t.requires_grad for t in got)
            del got
    assert room[0] == room[1]
    # a graph that asks for one has it
    out, final = decay_attention(q, k, v, g)
    assert out.requires_grad and final.requires_grad and final.is_contiguous()
    assert torch.isfinite(torch.autograd.grad(out.float().sum() + final.sum(), g)[0]).all()

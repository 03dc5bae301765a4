"""How exact the gated delta rule's and the windowed attention's kernels are, at the size of
the errors that their roundings leave: a rounding more, or a term of a product lost, shows.

Errors are norms of the error over the norm of the result, against float64."""

import pytest
import torch

from oal_amd import _native
from oal_amd.gated_delta import gated_delta_attention
from oal_amd.window_attention import window_attention, window_attention_step
from oracle.delta_oracle import gated_delta
from oracle.window_oracle import window_attention as dense

pytestmark = pytest.mark.gpu

# A bf16 result's own rounding: up to half a step, 2^-8 of the binade's foot, evenly spread, is 2^-8 / 3^(1/2)
# of it, and over values spread over a binade 1.6e-3 to 1.7e-3 of their norm. One further independent
# rounding of what a result is a sum of makes 2.3e-3 of it.
_ONE_ROUNDING = 1.95e-3


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _error(x, y):
    return float((x.detach().double() - y.detach()).norm() / y.detach().norm())


def _delta_inputs(dtype, heads, n, seed, decay=0.3):
    gen = torch.Generator().manual_seed(seed)
    hq, hk, hv = heads
    q, k = (torch.nn.functional.normalize(torch.randn(1, h, n, 64, generator=gen), dim=-1).to(dtype) for h in (hq, hk))
    v, dout = (torch.randn(1, h, n, 64, generator=gen).to(dtype) for h in (hv, max(hq, hv)))
    g = -decay * torch.rand(1, hv, n, generator=gen)
    beta = torch.sigmoid(torch.randn(1, hv, n, generator=gen))
    state, dstate = (torch.randn(1, hv, 64, 64, generator=gen) for _ in range(2))
    dev = _dev()
    return [t.to(dev) for t in (q, k, v, g, beta, state)], [t.to(dev) for t in (dout, dstate)]


def _with_gradients(call, ins, ups):
    leaves = [t.detach().clone().requires_grad_() for t in ins]
    outs = call(leaves)
    return dict(zip(("out", "state", "dq", "dk", "dv", "dg", "dbeta", "dstate"), (*outs, *torch.autograd.grad(outs, leaves, ups))))


def _delta(ins, ups):
    return _with_gradients(lambda x: gated_delta_attention(*x[:5], scale=0.125, initial_state=x[5]), ins, ups)


def _delta_exact(ins, ups):
    return _with_gradients(lambda x: gated_delta(*x, scale=0.125), [t.double() for t in ins], [t.double() for t in ups])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["keep", "forget", "mixed", "write nothing", "beta two", "long beta two", "one key", "segments"])
def test_float32_results_do_not_depend_on_the_type_of_the_tokens(kind, dtype):
    """The same 16-bit values as 16-bit and as float32 tensors. Both ways round the same
    sums at the same places, so their errors are two samples of one distribution over
    thousands of values: no further apart than a factor of 3, or than 8 roundings where nearly nothing is
    summed. A lost product of the values' low parts, 2^-16 of a term at most, makes it 4 to 19."""
    n = {"long beta two": 2000, "segments": 6001}.get(kind, 200)
    ins, ups = _delta_inputs(dtype, (2, 1, 1) if n > 200 else (2, 2, 2), n, seed=n + len(kind), decay=0.02 if n > 200 else 0.3)
    g, beta = ins[3], ins[4]
    if kind == "keep":
        g.zero_()
    elif kind == "forget":
        g.fill_(-30.0)
    elif kind == "mixed":
        g.mul_(0.1)
        g[..., ::37] = -300.0
    elif kind == "write nothing":
        beta[..., ::3] = 0.0
        beta[..., 1::3] = 1.0
    elif kind == "one key":
        ins[1].copy_(ins[1][:, :, :1].expand_as(ins[1]).clone())
        beta.fill_(1.0)
        g.zero_()
    elif kind != "segments":
        beta.fill_(2.0)
    want, got = _delta_exact(ins, ups), _delta(ins, ups)
    wide = _delta([t.float() for t in ins], [t.float() for t in ups])
    # where all decay is strong the start's gradient is below float32's range
    for name in ("state", "dg", "dbeta", "dstate")[:3 if kind == "mixed" else 4]:
        assert got[name].dtype == torch.float32
        err, least = _error(got[name], want[name]), _error(wide[name], want[name])
        print(f"{kind} {dtype} {name}: {err:.2e} {least:.2e}", flush=True)
        assert err <= max(3 * least, 8 * 2.0 ** -24), f"{name}: {err:.3g}, as float32 {least:.3g}"


@pytest.mark.parametrize("heads", [(2, 2, 2), (6, 2, 2)])
def test_bfloat16_results_of_the_delta_rule_are_rounded_once(heads):
    ins, ups = _delta_inputs(torch.bfloat16, heads, 700, seed=51)
    want, got = _delta_exact(ins, ups), _delta(ins, ups)
    for name in ("out", "dq", "dk", "dv"):
        err = _error(got[name], want[name])
        print(f"{heads} {name}: {err:.2e}", flush=True)
        assert got[name].dtype == torch.bfloat16 and err <= _ONE_ROUNDING, f"{name}: {err:.3g}"


@pytest.mark.parametrize("n,window", [(600, 128), (1024, 256)])
def test_bfloat16_results_of_the_window(n, window):
    """The weights' rounding is in out and dv: with the result's own 2.0e-3 and 2.3e-3. dq and dk
    carry their own and, from rows that see few keys, the rounding of the out that the
    backward starts from: 1.8e-3; with score gradients in one part 2.4e-3 to 2.5e-3. These
    four are from the formula in float64 with just those roundings put in."""
    gen = torch.Generator().manual_seed(n)
    dev = _dev()
    q, k, v, do = (torch.randn(2, h, n, 64, generator=gen).to(dev, torch.bfloat16) for h in (4, 2, 2, 4))
    results = []
    for call, cast in ((dense, torch.Tensor.double), (window_attention, torch.Tensor.clone)):
        leaves = [cast(t).requires_grad_() for t in (q, k, v)]
        out = call(*leaves, window=window, sinks=4, scale=0.125)
        results.append((out, *torch.autograd.grad(out, leaves, cast(do))))
    for name, y, x, bound in zip(("out", "dq", "dk", "dv"), *results, (2.25e-3, 2.1e-3, 2.1e-3, 2.55e-3)):
        err = _error(x, y)
        print(f"{n} {name}: {err:.2e}", flush=True)
        assert err <= bound, f"{name}: {err:.3g}"


def test_float16_scores_are_exact():
    """The log-sums of rows of large scores: as 16-bit tensors as good as the same values in float32."""
    dev = _dev()
    gen = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(1, 2, 300, 64, generator=gen).to(dev, torch.float16) for _ in range(3))
    q *= 20
    i, j = torch.arange(300, device=dev)[:, None], torch.arange(300, device=dev)[None]
    score = (q.double() @ k.double().transpose(2, 3).contiguous()).masked_fill((j > i) | (i - j >= 100), -torch.inf)
    want = torch.logsumexp(score, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64))
    err, least = (_error(_native.window_forward(*(t.to(dtype) for t in (q, k, v)), window=100, sinks=0, scale=1.0)[1], want)
                  for dtype in (torch.float16, torch.float32))
    print(f"lse: {err:.2e} {least:.2e}", flush=True)
    assert err <= 3 * least, f"{err:.3g}, as float32 {least:.3g}"


@pytest.mark.parametrize("slots", [128, 2048])
def test_weights_of_a_step_average(slots):
    """The weights are summed as they meet the values: whatever their roundings, values that are all
    one have the mean one. All but every 32nd weight here are 0.5018, which is 0.5 in bf16."""
    dev = _dev()
    k = torch.zeros(1, 1, slots, 8, device=dev, dtype=torch.bfloat16)
    k[..., 0] = torch.where(torch.arange(slots, device=dev) % 32 == 0, 0.0, -1.0)
    q = torch.zeros(1, 1, 1, 8, device=dev, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    v = torch.ones_like(k)
    at = torch.full((1,), 3 * slots, device=dev)
    out = window_attention_step(q, k[:, :, :1].contiguous(), v[:, :, :1].contiguous(), k, v, at, window=slots, scale=0.68955)
    assert torch.equal(out, torch.ones_like(out))

"""Traced, transformed and forward-mode calls of attention with decays, the head norms with rotary
embedding and the token scores: the kernels work on pointers, behind the back of whatever follows the
operations, so such calls are refused, before anything reaches a device."""

import contextlib

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from oal_amd import _native
from oal_amd.decay_attention import decay_attention, decay_step
from oal_amd.norm_rotary import norm_rotary_heads
from oal_amd.token_scores import token_log_probs


def _decay():
    return [torch.zeros(2, 2, 5, 16), torch.zeros(2, 2, 5, 16), torch.zeros(2, 2, 5, 8), torch.zeros(2, 2, 5),
            torch.zeros(2, 2, 16, 8)]


def _heads():
    return [torch.zeros(2, 5, 32), torch.zeros(2, 5, 16), torch.zeros(2, 5, 16), torch.ones(8), torch.ones(8)]


def _logits():
    return [torch.zeros(2, 5, 11)]


_TABLE, _TOKENS = torch.zeros(5, 8), torch.zeros(2, 5, dtype=torch.int64)
_CALLS = {
    "decay_attention": (lambda q, k, v, g, s: decay_attention(q, k, v, g, initial_state=s), _decay),
    "decay_step": (lambda *t: decay_step(*t), _decay),
    "norm_rotary_heads": (lambda *t: norm_rotary_heads(*t, _TABLE, _TABLE, q_heads=4, kv_heads=2), _heads),
    "token_log_probs": (lambda x: tuple(token_log_probs(x, _TOKENS, entropy=True)[:2]), _logits),
}


class _Library:
    """Stands in for the built library: its calls do nothing and succeed."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 4096 if name.endswith("bytes") else 0

        return call


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(_native, "load_library", lambda: lib)
    monkeypatch.setattr(_native, "_require_device", lambda *tensors: None)
    monkeypatch.setattr(_native, "_scope", lambda *args: contextlib.nullcontext())
    monkeypatch.setattr(_native, "_stream", lambda device: 0)
    return lib


@pytest.fixture(params=list(_CALLS))
def entry(request):
    call, inputs = _CALLS[request.param]
    return request.param, call, inputs()


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_make_fx_is_refused(entry, mode, library):
    name, call, inputs = entry
    with pytest.raises(RuntimeError, match=f"{name} .*eager"):
        make_fx(call, tracing_mode=mode)(*inputs)
    assert not library.calls


def test_jit_trace_is_refused(entry, library):
    name, call, inputs = entry
    with pytest.raises(RuntimeError, match=f"{name} .*eager"):
        torch.jit.trace(call, tuple(inputs), check_trace=False)
    assert not library.calls


def test_transforms_are_refused(entry, library):
    name, call, inputs = entry
    with pytest.raises(RuntimeError, match=f"{name} .*eager"):
        torch.func.vmap(call)(*(t[None] for t in inputs))
    assert not library.calls


def test_fake_tensors_are_refused(entry, library):
    name, call, inputs = entry
    mode = torch._subclasses.FakeTensorMode()
    with pytest.raises(RuntimeError, match=f"{name} .*eager"):
        call(*(mode.from_tensor(t) for t in inputs))
    assert not library.calls


def test_forward_mode_is_refused(entry, library):
    name, call, inputs = entry
    for x in range(len(inputs)):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(inputs[x], torch.ones_like(inputs[x]))
            with pytest.raises(RuntimeError, match=f"{name} .*forward-mode"):
                call(*inputs[:x], dual, *inputs[x + 1:])
    assert not library.calls
    with forward_ad.dual_level():  # others' derivatives do not matter
        call(*inputs)
    assert library.calls


@pytest.mark.parametrize("name", ["decay_attention", "norm_rotary_heads", "token_log_probs"])
def test_traced_and_forward_mode_backwards_are_refused(name, library):
    call, inputs = _CALLS[name]
    leaves = [t.requires_grad_() for t in inputs()]
    outs = call(*leaves)
    outs = outs if isinstance(outs, tuple) else (outs,)
    ups = [torch.ones_like(t) for t in outs]

    def backward(*ups):
        return torch.autograd.grad(outs, leaves, ups, retain_graph=True)

    library.calls.clear()
    with pytest.raises(RuntimeError, match=f"{name} .*eager"):
        make_fx(backward)(*ups)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match=f"{name} .*forward-mode"):
        backward(forward_ad.make_dual(ups[0], ups[0]), *ups[1:])
    assert not library.calls
    backward(*ups)
    assert library.calls


def test_calls_of_compiled_code_and_of_subclasses_run(entry, library):
    name, call, inputs = entry

    def outer(*tensors):
        out = call(*tensors)
        return (out[0] if isinstance(out, tuple) else out) * 2

    torch._dynamo.reset()
    compiled = torch.compile(outer, backend="eager")
    for _ in range(2):
        library.calls.clear()
        with torch.no_grad():
            compiled(*inputs)
        assert library.calls
    library.calls.clear()

    class Tagged(torch.Tensor):
        pass

    with torch.no_grad():
        call(*(t.as_subclass(Tagged) for t in inputs))
    assert library.calls

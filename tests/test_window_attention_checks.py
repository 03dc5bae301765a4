"""What the windowed attention's entry points refuse, before anything reaches a device; the ring cache's slots on the CPU."""

import ctypes

import pytest
import torch

from oal_amd import _native
from oal_amd.window_attention import window_attention, window_attention_step, window_cache


def _valid(b=2, hq=4, hk=2, n=5, d=16, dv=8, dtype=torch.float32):
    return dict(q=torch.zeros(b, hq, n, d, dtype=dtype), k=torch.zeros(b, hk, n, d, dtype=dtype),
                v=torch.zeros(b, hk, n, dv, dtype=dtype), window=4, sinks=1)


_REFUSED = [
    ("not a tensor", dict(q=[1.0]), TypeError, "torch.Tensor"),
    ("rank", dict(q=torch.zeros(4, 5, 16)), ValueError, "rank-4"),
    ("float64", dict(q=torch.zeros(2, 4, 5, 16, dtype=torch.float64)), TypeError, "float16, bfloat16 or float32"),
    ("mixed types", dict(k=torch.zeros(2, 2, 5, 16, dtype=torch.bfloat16)), ValueError, "same dtype"),
    ("k features", dict(k=torch.zeros(2, 2, 5, 8)), ValueError, "feature dimension"),
    ("v length", dict(v=torch.zeros(2, 2, 6, 8)), ValueError, "k and v"),
    ("no tokens", dict(q=torch.zeros(2, 4, 0, 16)), ValueError, "positive"),
    ("heads", dict(q=torch.zeros(2, 3, 5, 16)), ValueError, "divisible"),
    ("wide heads", dict(q=torch.zeros(2, 4, 5, 72), k=torch.zeros(2, 2, 5, 72)), ValueError, "up to 64"),
    ("device", dict(v=torch.zeros(2, 2, 5, 8, device="meta")), ValueError, "same device"),
    ("window", dict(window=0), ValueError, "window"),
    ("window type", dict(window=4.0), TypeError, "window must be an int"),
    ("sinks", dict(sinks=-1), ValueError, "sinks"),
    ("more queries than keys", dict(q=torch.zeros(2, 4, 6, 16)), ValueError, "key for every query"),
    ("scale", dict(scale=float("inf")), ValueError, "finite"),
    ("CPU tensors", dict(), RuntimeError, "ROCm"),
]


@pytest.mark.parametrize("case", _REFUSED, ids=[c[0] for c in _REFUSED])
def test_refusals(case):
    _, change, error, text = case
    with pytest.raises(error, match=text):
        window_attention(**{**_valid(), **change})


def _step(**change):
    a = {**_valid(n=1), "k_cache": torch.zeros(2, 2, 5, 16), "v_cache": torch.zeros(2, 2, 5, 8),
         "positions": torch.zeros(2, dtype=torch.int64)}
    return window_attention_step(**{**a, **change})


_STEP_REFUSED = [
    ("two tokens", dict(q=torch.zeros(2, 4, 2, 16)), ValueError, "one token"),
    ("narrow", dict(k=torch.zeros(2, 2, 1, 12), q=torch.zeros(2, 4, 1, 12)), ValueError, "multiples of 8"),
    ("cache type", dict(k_cache=torch.zeros(2, 2, 5, 16, dtype=torch.bfloat16)), ValueError, "k_cache must have the dtype"),
    ("cache size", dict(v_cache=torch.zeros(2, 2, 6, 8)), ValueError, r"sinks \+ window"),
    ("cache rows", dict(k_cache=torch.zeros(2, 2, 16, 5).transpose(2, 3)), ValueError, "rows of k_cache"),
    ("one row for all", dict(k_cache=torch.zeros(2, 2, 1, 16).expand(-1, -1, 5, -1)), ValueError, "rows of k_cache"),
    ("positions type", dict(positions=torch.zeros(2)), TypeError, "positions"),
    ("positions shape", dict(positions=torch.zeros(3, dtype=torch.int64)), ValueError, "positions"),
    ("gradients", dict(q=torch.zeros(2, 4, 1, 16, requires_grad=True)), RuntimeError, "not differentiable"),
    ("CPU tensors", dict(), RuntimeError, "ROCm"),
]


@pytest.mark.parametrize("case", _STEP_REFUSED, ids=[c[0] for c in _STEP_REFUSED])
def test_step_refusals(case):
    _, change, error, text = case
    with pytest.raises(error, match=text):
        _step(**change)


@pytest.mark.parametrize("window,sinks", [(1, 0), (4, 0), (3, 2), (50, 5)])
def test_cache_slots(window, sinks):
    n = 23
    lengths = torch.tensor([0, 1, 2, 3, 5, 9, 22, 23], dtype=torch.int32)
    k = torch.arange(1, n + 1).view(1, 1, n, 1).expand(len(lengths), 2, n, 8).to(torch.float32)
    kc, vc = window_cache(k, -k, window=window, sinks=sinks, lengths=lengths)
    for x, p in enumerate(lengths.tolist()):
        want = torch.zeros(sinks + window)
        for j in range(p):
            want[j if j < sinks else sinks + (j - sinks) % window] = j + 1
        assert torch.equal(kc[x, 1, :, 3], want) and torch.equal(vc[x, 0, :, 0], -want)
    full, _ = window_cache(k, -k, window=window, sinks=sinks)
    assert torch.equal(full[0], kc[-1])
    with pytest.raises(TypeError, match="lengths"):
        window_cache(k, k, window=window, sinks=sinks, lengths=lengths.float())
    with pytest.raises(ValueError, match="lengths"):
        window_cache(k, k, window=window, sinks=sinks, lengths=lengths[:2])


def test_c_entries_check_before_they_launch():
    try:
        lib = _native.load_library()
    except RuntimeError:
        pytest.skip("liboal_amd.so not built")
    size = lib.oal_window_attention_workspace_bytes
    assert size(2, 14, 2, 100, 100, 32, 4, 1) > size(2, 14, 2, 100, 100, 32, 0, 1) > 0
    for bad, text in (((0, 14, 2, 100, 100, 32, 4, 1), b"positive"), ((2, 14, 3, 100, 100, 32, 4, 1), b"divisible"),
                      ((2, 14, 2, 101, 100, 32, 4, 1), b"key for every"), ((2, 14, 2, 100, 100, 0, 4, 1), b"window"),
                      ((1 << 20, 14, 2, 1 << 20, 1 << 20, 32, 4, 1), b"too large")):
        assert size(*bad) == 0 and text in lib.oal_last_error()
    step_size = lib.oal_window_attention_step_workspace_bytes
    assert step_size(1, 14, 2, 64, 4096, 4) > 0 and step_size(1, 14, 2, 60, 4096, 4) == 0
    p, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    rows = (ctypes.c_int64 * 15)(*[64] * 15)
    forward = lib.oal_window_attention_forward
    assert forward(p, p, None, rows, 1, 2, 2, 5, 5, 64, 64, 3, 0, 1, 0.1, p, p, None) and b"null" in lib.oal_last_error()
    assert forward(p, odd, p, rows, 1, 2, 2, 5, 5, 64, 64, 3, 0, 1, 0.1, p, p, None) and b"16-byte" in lib.oal_last_error()
    assert forward(p, p, p, rows, 1, 2, 2, 5, 5, 64, 64, 3, 0, 7, 0.1, p, p, None) and b"dtype" in lib.oal_last_error()
    backward = lib.oal_window_attention_backward
    assert backward(p, p, p, rows, 1, 2, 2, 5, 5, 64, 64, 3, 0, 1, 0.1, p, p, None, p, p, p, p, None) and b"null" in lib.oal_last_error()
    step = lib.oal_window_attention_step
    assert step(p, p, p, p, p, rows, p, 1, 2, 2, 64, 64, 3, 0, 5, 0.1, p, p, None) and b"type" in lib.oal_last_error()
    assert step(p, p, p, p, odd, rows, p, 1, 2, 2, 64, 64, 3, 0, 1, 0.1, p, p, None) and b"16-byte" in lib.oal_last_error()
    assert step(p, p, p, p, p, rows, p, 1, 2, 2, 12, 64, 3, 0, 1, 0.1, p, p, None) and b"multiples of 8" in lib.oal_last_error()


def test_workspace_follows_the_keys():
    try:
        lib = _native.load_library()
    except RuntimeError:
        pytest.skip("liboal_amd.so not built")
    size = lib.oal_window_attention_workspace_bytes
    most = (1 << 31) - 1
    assert size(1, 14, 2, 100, 100, most, most, 1) == size(1, 14, 2, 100, 100, 100, 100, 1)
    # pieces of the first keys' sums: fewer, the more first keys there are
    without, few, many = (size(1, 14, 2, 32768, 32768, 1024, sinks, 1) for sinks in (0, 4, 16384))
    assert few - without <= 64 * 2 * 2 * 64 * 64 * 4
    assert many - without <= 4 * 2 * 2 * 16384 * 64 * 4 + 4096

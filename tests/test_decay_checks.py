"""What decay_attention and decay_step refuse, before anything reaches a device."""

import ctypes

import pytest
import torch

from oal_amd import _native
from oal_amd.decay_attention import decay_attention, decay_step


def _valid(b=2, hq=4, hk=2, hv=2, n=5, d=16, dv=8, dtype=torch.float32):
    return dict(q=torch.zeros(b, hq, n, d, dtype=dtype), k=torch.zeros(b, hk, n, d, dtype=dtype),
                v=torch.zeros(b, hv, n, dv, dtype=dtype), g=torch.zeros(b, hv, n), state=torch.zeros(b, hv, d, dv))


_REFUSED = [
    ("not a tensor", dict(q=[1.0]), TypeError, "torch.Tensor"),
    ("rank", dict(q=torch.zeros(4, 5, 16)), ValueError, "rank-4"),
    ("float64", dict(q=torch.zeros(2, 4, 5, 16, dtype=torch.float64)), TypeError, "float16, bfloat16 or float32"),
    ("mixed types", dict(k=torch.zeros(2, 2, 5, 16, dtype=torch.bfloat16)), ValueError, "same dtype"),
    ("g type", dict(g=torch.zeros(2, 2, 5, dtype=torch.bfloat16)), TypeError, "g must be float32"),
    ("g shape", dict(g=torch.zeros(2, 4, 5)), ValueError, r"\[Hv\] or \[B, Hv, N\]"),
    ("g heads", dict(g=torch.zeros(4)), ValueError, r"\[Hv\] or \[B, Hv, N\]"),
    ("g scalar", dict(g=torch.zeros(())), ValueError, r"\[Hv\] or \[B, Hv, N\]"),
    ("k features", dict(k=torch.zeros(2, 2, 5, 8)), ValueError, "same batch size"),
    ("v length", dict(v=torch.zeros(2, 2, 6, 8)), ValueError, "same batch size"),
    ("no tokens", dict(q=torch.zeros(2, 4, 0, 16)), ValueError, "positive"),
    ("key heads", dict(k=torch.zeros(2, 3, 5, 16)), ValueError, "key head count"),
    ("query heads", dict(q=torch.zeros(2, 3, 5, 16)), ValueError, "query and value head counts"),
    ("wide heads", dict(q=torch.zeros(2, 4, 5, 65), k=torch.zeros(2, 2, 5, 65)), ValueError, "up to 64"),
    ("state type", dict(state=torch.zeros(2, 2, 16, 8, dtype=torch.bfloat16)), TypeError, "float32"),
    ("state shape", dict(state=torch.zeros(2, 2, 8, 16)), ValueError, r"\[B, Hv, D, DV\]"),
    ("state kind", dict(state=1.0), TypeError, "torch.Tensor"),
    ("device", dict(g=torch.zeros(2, 2, 5, device="meta")), ValueError, "same device"),
    ("scale", dict(scale=float("nan")), ValueError, "finite"),
    ("scale type", dict(scale="1"), TypeError, "scalar"),
    ("CPU tensors", dict(), RuntimeError, "ROCm"),
    ("CPU tensors, a decay per head", dict(g=torch.zeros(2)), RuntimeError, "ROCm"),
]


@pytest.mark.parametrize("case", _REFUSED, ids=[c[0] for c in _REFUSED])
def test_refusals(case):
    _, change, error, text = case
    a = {**_valid(), "scale": 0.1, **change}
    state = a.pop("state")
    with pytest.raises(error, match=text):
        decay_attention(a["q"], a["k"], a["v"], a["g"], scale=a["scale"], initial_state=state)
    with pytest.raises(error, match=text):
        decay_step(a["q"], a["k"], a["v"], a["g"], state, scale=a["scale"])


def test_step_refuses_what_it_cannot_update():
    a = _valid()
    ops = [a[x] for x in ("q", "k", "v", "g")]
    with pytest.raises(TypeError, match="state"):
        decay_step(*ops, None)
    with pytest.raises(ValueError, match="contiguous"):
        decay_step(*ops, torch.zeros(2, 2, 8, 16).transpose(2, 3))
    with pytest.raises(RuntimeError, match="not differentiable"):
        decay_step(ops[0].requires_grad_(), *ops[1:], a["state"])


def _lib():
    try:
        return _native.load_library()
    except RuntimeError:
        pytest.skip("liboal_amd.so not built")


def test_c_entries_check_before_they_launch():
    lib = _lib()
    assert lib.oal_decay_saved_bytes(2, 2, 65, 0) > 0 and lib.oal_decay_saved_bytes(2, 2, 65, 1) >= 4 * 2 * 4096 * 4
    assert lib.oal_decay_saved_bytes(0, 2, 65, 1) == 0 and b"positive" in lib.oal_last_error()
    assert lib.oal_decay_saved_bytes(1 << 20, 64, 1 << 20, 1) == 0 and b"too large" in lib.oal_last_error()
    assert lib.oal_decay_workspace_bytes(1, 3, 2, 2, 64, 64, 0) == 0 and b"divisible" in lib.oal_last_error()
    assert lib.oal_decay_workspace_bytes(1, 2, 2, 2, 64, 12, 0) == 0 and b"multiples of 8" in lib.oal_last_error()
    # shared heads need room for what is summed
    assert lib.oal_decay_workspace_bytes(1, 2, 2, 4, 64, 64, 0) > lib.oal_decay_workspace_bytes(1, 4, 4, 4, 64, 64, 0)
    p, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    rows = (ctypes.c_int64 * 12)(*[64] * 12)

    def forward(q=p, strides=rows, dtype=1, out=p, dim=64):
        return lib.oal_decay_forward(q, p, p, p, strides, 1, 2, 2, 2, 64, dim, 64, dtype, 0.1, None, out, p, p, 1, None)

    assert forward(q=None) and b"null" in lib.oal_last_error()
    assert forward(strides=None) and b"null" in lib.oal_last_error()
    assert forward(dtype=3) and b"dtype" in lib.oal_last_error()
    assert forward(dim=12) and b"multiples of 8" in lib.oal_last_error()
    assert forward(q=odd) and b"16-byte" in lib.oal_last_error()
    assert forward(strides=(ctypes.c_int64 * 12)(*[63] * 12)) and b"16-byte" in lib.oal_last_error()
    assert forward(out=odd) and b"16-byte" in lib.oal_last_error()
    assert forward(strides=(ctypes.c_int64 * 12)(*[1 << 23] * 12)) and b"too far apart" in lib.oal_last_error()
    rc = lib.oal_decay_backward(p, p, p, p, rows, 0, 1, 2, 2, 2, 64, 64, 64, 1, 0.1, p, None, None, p, p, p, p, None, p, None)
    assert rc and b"null" in lib.oal_last_error()
    rc = lib.oal_decay_backward(p, p, p, p, rows, 0, 1, 2, 2, 2, 64, 64, 64, 1, 0.1, p, odd, None, p, p, p, p, None, p, None)
    assert rc and b"16-byte" in lib.oal_last_error()
    rc = lib.oal_decay_step(p, p, p, p, rows, 1, 2, 2, 2, 1, 65, 64, 0, 0.1, p, p, None)
    assert rc and b"[1, 64]" in lib.oal_last_error()
    rc = lib.oal_decay_step(p, p, p, p, rows, 1, 2, 2, 2, 1, 64, 64, 3, 0.1, p, p, None)
    assert rc and b"type" in lib.oal_last_error()
    rc = lib.oal_decay_step(p, p, p, p, rows, 1, 2, 2, 2, 1, 64, 64, 0, 0.1, None, p, None)
    assert rc and b"null" in lib.oal_last_error()

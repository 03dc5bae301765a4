"""What norm_rotary_heads refuses, before anything reaches a device."""

import ctypes

import pytest
import torch

from oal_amd import _native
from oal_amd.norm_rotary import norm_rotary_heads


def _valid():
    z = torch.zeros
    return dict(q=z(2, 5, 32), k=z(2, 5, 16), v=z(2, 5, 16), q_weight=z(8), k_weight=z(8), cos=z(5, 8), sin=z(5, 8),
                q_heads=4, kv_heads=2, eps=1e-6, positions=None)


_z = torch.zeros
_REFUSED = [
    ("not a tensor", dict(q=[1.0]), TypeError, "torch.Tensor"),
    ("rank", dict(q=_z(5, 32)), ValueError, r"\[B, N, heads \* D\]"),
    ("float64", dict(q=_z(2, 5, 32, dtype=torch.float64)), TypeError, "float16, bfloat16 or float32"),
    ("mixed types", dict(k=_z(2, 5, 16, dtype=torch.bfloat16)), ValueError, "same dtype"),
    ("no tokens", dict(q=_z(2, 0, 32)), ValueError, "positive"),
    ("heads type", dict(q_heads=4.0), TypeError, "q_heads"),
    ("no heads", dict(kv_heads=0), ValueError, "kv_heads"),
    ("heads", dict(q_heads=3), ValueError, "q_heads heads"),
    ("wide heads", dict(q=_z(2, 5, 65 * 4)), ValueError, "up to 64"),
    ("k width", dict(k=_z(2, 5, 24)), ValueError, "k and v"),
    ("v length", dict(v=_z(2, 6, 16)), ValueError, "k and v"),
    ("weight kind", dict(q_weight=1.0), TypeError, "q_weight"),
    ("weight type", dict(k_weight=_z(8, dtype=torch.float16)), TypeError, "k_weight"),
    ("weight shape", dict(q_weight=_z(2, 8)), ValueError, "q_weight"),
    ("weights of two kinds", dict(k_weight=_z(2, 8)), ValueError, "same dtype"),
    ("tables", dict(sin=_z(5, 6)), ValueError, "same shape"),
    ("table rank", dict(cos=_z(2, 5, 8), sin=_z(2, 5, 8)), ValueError, "same shape"),
    ("table type", dict(cos=_z(5, 8, dtype=torch.float64), sin=_z(5, 8, dtype=torch.float64)), TypeError, "cos and sin"),
    ("odd rotation", dict(cos=_z(5, 7), sin=_z(5, 7)), ValueError, "even"),
    ("no rotation", dict(cos=_z(5, 0), sin=_z(5, 0)), ValueError, "even"),
    ("wide rotation", dict(cos=_z(5, 10), sin=_z(5, 10)), ValueError, "even"),
    ("short tables", dict(cos=_z(4, 8), sin=_z(4, 8)), ValueError, "every token"),
    ("empty tables", dict(cos=_z(0, 8), sin=_z(0, 8), positions=_z(2, 5, dtype=torch.int64)), ValueError, "every token"),
    ("positions type", dict(positions=_z(2, 5)), TypeError, "positions"),
    ("positions shape", dict(positions=_z(5, dtype=torch.int64)), ValueError, r"\[B, N\]"),
    ("device", dict(positions=_z(2, 5, dtype=torch.int64, device="meta")), ValueError, "same device"),
    ("eps", dict(eps=-1.0), ValueError, "eps"),
    ("eps not finite", dict(eps=float("nan")), ValueError, "eps"),
    ("eps type", dict(eps="1"), TypeError, "eps"),
    ("gradients of tables", dict(cos=_z(5, 8, requires_grad=True)), RuntimeError, "cos and sin"),
    ("CPU tensors", dict(), RuntimeError, "ROCm"),
    ("CPU tensors, weights for each head", dict(q_weight=_z(4, 8), k_weight=_z(2, 8)), RuntimeError, "ROCm"),
]


@pytest.mark.parametrize("case", _REFUSED, ids=[c[0] for c in _REFUSED])
def test_refusals(case):
    _, change, error, text = case
    with pytest.raises(error, match=text):
        norm_rotary_heads(**{**_valid(), **change})


def test_c_entries_check_before_they_launch():
    try:
        lib = _native.load_library()
    except RuntimeError:
        pytest.skip("liboal_amd.so not built")
    p, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    rows = (ctypes.c_int64 * 6)(*[64] * 6)

    def forward(q=p, strides=rows, table=5, rotary=8, position=None, n=5, d=8, dtype=1, out=p, heads=4):
        return lib.oal_norm_rotary_heads(q, p, p, strides, None, None, 0, 0, p, p, 1, table, rotary, position, 2, heads, 2, n,
                                         d, dtype, 1e-6, out, p, p, None)

    for change, text in ((dict(q=None), b"null"), (dict(strides=None), b"null"), (dict(out=None), b"null"),
                         (dict(table=4), b"every token"), (dict(table=0, position=p), b"every token"),
                         (dict(rotary=7), b"even"), (dict(rotary=10), b"even"), (dict(rotary=0), b"even"),
                         (dict(d=65), b"head_dim"), (dict(d=0), b"head_dim"), (dict(n=0), b"positive"),
                         (dict(dtype=3), b"dtype"), (dict(out=odd), b"16-byte"), (dict(heads=1 << 17), b"too large")):
        assert forward(**change) and text in lib.oal_last_error(), change

    def backward(q=p, dq=p, dw=p, work=p, up=p):
        return lib.oal_norm_rotary_heads_backward(q, p, rows, None, None, 0, 0, p, p, 1, 5, 8, None, 2, 4, 2, 5, 8, 1, 1e-6, up,
                                                  p, p, dq, p, p, dw, None, work, None)

    for change, text in ((dict(q=None), b"null"), (dict(dq=None), b"needs dq"), (dict(work=None), b"workspace"),
                         (dict(up=odd), b"16-byte")):
        assert backward(**change) and text in lib.oal_last_error(), change
    size = lib.oal_norm_rotary_heads_workspace_bytes
    # a float for each dimension of each weight row at least
    assert size(2, 4, 2, 5, 8, 0) >= 2 * 8 * 4 and size(2, 4, 2, 5, 8, 1) >= 6 * 8 * 4 and size(1, 1, 1, 1, 1, 0) > 0
    assert size(2, 0, 2, 5, 8, 0) == 0 and b"positive" in lib.oal_last_error()

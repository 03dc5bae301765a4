"""What token_log_probs refuses, before anything reaches a device."""

import ctypes

import pytest
import torch

from oal_amd import _native
from oal_amd.qwen_oal import score_tokens
from oal_amd.token_scores import token_log_probs

_z = torch.zeros
_TOKENS = _z(2, 5, dtype=torch.int64)
_REFUSED = [
    ("not a tensor", dict(logits=[1.0]), TypeError, "torch.Tensor"),
    ("tokens not a tensor", dict(tokens=[1]), TypeError, "torch.Tensor"),
    ("float64", dict(logits=_z(2, 5, 9, dtype=torch.float64)), TypeError, "float16, bfloat16 or float32"),
    ("token type", dict(tokens=_z(2, 5)), TypeError, "int32 or int64"),
    ("short type", dict(tokens=_z(2, 5, dtype=torch.int16)), TypeError, "int32 or int64"),
    ("shape", dict(tokens=_z(2, 4, dtype=torch.int64)), ValueError, "shape of logits"),
    ("broadcast", dict(tokens=_z(1, 5, dtype=torch.int64)), ValueError, "shape of logits"),
    ("scalar logits", dict(logits=_z(()), tokens=_z((), dtype=torch.int64)), ValueError, "V"),
    ("no vocabulary", dict(logits=_z(2, 5, 0)), ValueError, "V"),
    ("device", dict(tokens=_z(2, 5, dtype=torch.int64, device="meta")), ValueError, "same device"),
    ("entropy type", dict(entropy=1), TypeError, "entropy"),
    ("top type", dict(top=True), TypeError, "top"),
    ("top negative", dict(top=-1), ValueError, "top"),
    ("top past the vocabulary", dict(top=10), ValueError, "top"),
    ("top past the most", dict(logits=_z(2, 5, 100), top=65), ValueError, "top"),
    ("CPU tensors", dict(), RuntimeError, "ROCm"),
    ("CPU tensors, no rows", dict(logits=_z(0, 9), tokens=_z(0, dtype=torch.int64)), RuntimeError, "ROCm"),
]


@pytest.mark.parametrize("case", _REFUSED, ids=[c[0] for c in _REFUSED])
def test_refusals(case):
    _, change, error, text = case
    with pytest.raises(error, match=text):
        token_log_probs(**{**dict(logits=_z(2, 5, 9), tokens=_TOKENS), **change})


def test_c_entries_check_before_they_launch():
    try:
        lib = _native.load_library()
    except RuntimeError:
        pytest.skip("liboal_amd.so not built")
    p, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    rows = (ctypes.c_int64 * 2)(64, 64)

    def forward(logits=p, strides=rows, tokens=p, n=5, vocab=64, dtype=1, top=2, out=p, places=p, work=p):
        return lib.oal_token_scores(logits, strides, tokens, 2, n, vocab, dtype, top, out, None, p, places, None, work, None)

    for change, text in ((dict(logits=None), b"null"), (dict(strides=None), b"null"), (dict(tokens=None), b"null"),
                         (dict(out=None), b"null"), (dict(places=None), b"null"), (dict(work=None), b"null"),
                         (dict(n=0), b"positive"), (dict(vocab=0), b"positive"), (dict(dtype=3), b"dtype"),
                         (dict(top=65), b"top"), (dict(vocab=1), b"top"), (dict(top=-1), b"top"),
                         (dict(n=1 << 23), b"too large"), (dict(vocab=(1 << 30) + 1), b"too large"),
                         (dict(logits=ctypes.c_void_p((1 << 20) + 1)), b"aligned"), (dict(work=odd), b"16-byte")):
        assert forward(**change) and text in lib.oal_last_error(), change

    def backward(saved=p, entropy=p, dentropy=p, out=p):
        return lib.oal_token_scores_backward(p, rows, p, 2, 5, 64, 1, saved, entropy, p, dentropy, out, None)

    for change, text in ((dict(saved=None), b"null"), (dict(entropy=None), b"null"), (dict(out=None), b"null"),
                         (dict(out=odd), b"16-byte")):
        assert backward(**change) and text in lib.oal_last_error(), change
    assert lib.oal_token_scores_workspace_bytes(2, 5, 64, 2) > 0
    assert lib.oal_token_scores_workspace_bytes(2, 0, 64, 2) == 0 and b"positive" in lib.oal_last_error()


@pytest.mark.parametrize("tokens,lengths", [
    (torch.zeros(5, dtype=torch.int64), None),
    (torch.zeros(2, 5, dtype=torch.int64), torch.tensor([3])),
    (torch.zeros(2, 5, dtype=torch.int64), torch.tensor([[3, 4]])),
    (torch.zeros(2, 5, dtype=torch.int64), torch.tensor([3.0, 4.0])),
])
def test_the_model_scores_batches_of_tokens(tokens, lengths):
    with pytest.raises(ValueError, match=r"\[B"):
        score_tokens(None, tokens, lengths=lengths)

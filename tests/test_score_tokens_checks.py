"""What score_tokens refuses as lengths, before it asks the model."""

import pytest
import torch

from oal_amd.qwen_oal import score_tokens

_TOKENS = torch.zeros(2, 5, dtype=torch.int64)


@pytest.mark.parametrize("lengths", [
    [5, 3], 5, torch.tensor([True, False]), torch.tensor([5.0, 3.0]), torch.tensor([5 + 0j, 3]), torch.tensor([5]),
    torch.tensor([[5, 3]]), torch.zeros(2, dtype=torch.int64, device="meta"),
], ids=["list", "number", "bool", "float", "complex", "one", "rank", "device"])
def test_lengths_that_are_none(lengths):
    with pytest.raises(ValueError, match="lengths must be integers"):
        score_tokens(None, _TOKENS, lengths=lengths)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32, torch.int64])
def test_lengths_of_any_integer_type(dtype):
    class Asked(Exception):
        pass

    def model(tokens):
        raise Asked

    with pytest.raises(Asked):
        score_tokens(model, _TOKENS, lengths=torch.tensor([5, 3]).to(dtype))

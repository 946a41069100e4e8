"""Vocabulary masks whose last axis is not the vocabulary (CPU): refused, not regrouped into rows of another width."""
import pytest
import torch

from noetic_tensor_b200 import rl

HIDDEN, WEIGHT = torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16), torch.zeros(16, 24, dtype=torch.bfloat16)


@pytest.mark.parametrize("shape", [(2, 12), (8, 12), (16, 12), (1, 48), (24, 1), (24, 8), ()])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.bool])
def test_refused(shape, dtype):
    mask = torch.ones(shape, dtype=dtype)
    with pytest.raises(ValueError, match="vocab_mask"):
        rl.Head(HIDDEN, WEIGHT, vocab_mask=mask)
    with pytest.raises(ValueError, match="vocab_mask"):
        rl.head_sample_categorical(HIDDEN, WEIGHT, None, vocab_mask=mask)
    with pytest.raises(ValueError, match="vocab_mask"):
        rl.head_token_log_probs(HIDDEN, WEIGHT, torch.zeros(1, 2, 4, dtype=torch.int32), vocab_mask=mask)


@pytest.mark.parametrize("shape", [(24,), (1, 24), (8, 24), (1, 2, 4, 24)])
def test_taken(shape):
    assert rl.Head(HIDDEN, WEIGHT, vocab_mask=torch.ones(shape, dtype=torch.bool)).kw["allow"].shape[-1] == 24

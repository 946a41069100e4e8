"""Scoring masks that a kernel would misread (CPU): the calls that hand a mask's address to the library refuse another type, size or
order, or another device's memory, before anything is launched."""
import pytest
import torch

from noetic_tensor_b200 import capi, ops

PER = torch.zeros(2, 3, 5)
BAD = [
    PER.bool(),  # a byte per position: read as f32, four times as many bytes as there are
    PER.double(),
    PER[:1].contiguous(),
    PER[:1].expand(2, 3, 5),  # one sequence's memory
    torch.zeros(5, 3, 2).permute(2, 1, 0),  # another order
    torch.zeros(2, 3, 5, device="meta"),
]


@pytest.mark.parametrize("mask", BAD, ids=["bool", "double", "short", "expanded", "permuted", "another device"])
def test_refused(mask):
    for call in (
        lambda: ops.mask_rows(PER, mask),
        lambda: ops.reduce_tokens(PER, mask, capi.REDUCE_TOKEN_MEAN),
        lambda: ops.reduce_tokens_backward((2, 3, 5), mask, capi.REDUCE_TOKEN_MEAN, torch.ones(2)),
    ):
        with pytest.raises(ValueError, match="mask: expected"):
            call()


def test_the_masked_values_too():
    with pytest.raises(ValueError, match="x: expected"):
        ops.mask_rows(PER.double(), PER)
    with pytest.raises(ValueError, match="per: expected"):
        ops.reduce_tokens(PER.double(), PER, capi.REDUCE_SUM)

"""Upstream gradients of another size than the reduced value (CPU): refused before the library reads past their end."""
import pytest
import torch

from noetic_tensor_b200 import ops, rl

SIZES = {rl.NONE: (2, 3, 5), rl.SUM: (2,), rl.TOKEN_MEAN: (2,), rl.PER_SEQUENCE: (2, 3), rl.SEQUENCE_MEAN: (2,)}


@pytest.mark.parametrize("reduction", SIZES)
@pytest.mark.parametrize("bad", ["scalar", "half", "double", "strided"])
def test_refused(reduction, bad):
    g = torch.ones(SIZES[reduction])
    g = {"scalar": g.sum(), "half": g[:1], "double": g.double(), "strided": torch.stack((g, g), -1)[..., 0]}[bad]
    with pytest.raises(ValueError, match="upstream: expected"):
        ops.reduce_tokens_backward((2, 3, 5), None, reduction, g)

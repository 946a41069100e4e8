"""Token ids as the kernels take them (CPU): 64-bit ids outside the vocabulary do not become tokens."""
import torch

from noetic_tensor_b200 import rl


def test_ids_outside_the_vocabulary_stay_outside():
    V = 512
    ids = torch.tensor([0, 5, V - 1, V, V + 7, -1, 2**31 + 5, 2**32 + 5, -(2**32) + 5, 2**63 - 1, -(2**63)])
    got = rl._token_ids(ids, V)
    assert got.dtype == torch.int32 and got.is_contiguous()
    inside = (ids >= 0) & (ids < V)
    assert torch.equal(got[inside].long(), ids[inside]) and ((got[~inside] < 0) | (got[~inside] >= V)).all()
    same = torch.arange(6, dtype=torch.int32)
    assert rl._token_ids(same, V) is same and rl._token_ids(None, V) is None
    assert torch.equal(rl._token_ids(ids[:8].reshape(2, 4).t(), V), got[:8].reshape(2, 4).t())

"""A device named without its index is the current one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_row_forward_on_pinned_rows():
    from noetic_tensor_b200 import ops

    x = torch.randn(9, 1000, generator=torch.Generator().manual_seed(1)).pin_memory()
    a, b = ops.row_forward(x, greedy=True, device="cuda"), ops.row_forward(x, greedy=True, device="cuda:0")
    for name in ("tokens", "logp", "entropy", "rowstats"):
        assert torch.equal(getattr(a, name), getattr(b, name))
    assert torch.equal(a.tokens.cpu(), x.argmax(1).to(torch.int32))

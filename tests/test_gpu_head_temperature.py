"""Temperatures that are 0 in 32 bits: refused, since the library takes 0 for "no temperature"."""
import pytest
import torch

from noetic_tensor_b200 import rl


@pytest.mark.parametrize("tau", [1e-50, 1e-46, 0.0, -1.0, float("nan"), float("inf"), 1e39])
def test_head_refuses(tau):
    with pytest.raises(ValueError, match="temperature"):
        rl.Head(torch.zeros(1, 1, 2, 8, dtype=torch.bfloat16), torch.zeros(8, 8, dtype=torch.bfloat16), temperature=tau)


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [0.0, 1e-50])
def test_the_calls_refuse(tau):
    from noetic_tensor_b200 import ops

    x, w = torch.ones(4, 64, device="cuda").bfloat16(), torch.ones(64, 264, device="cuda").bfloat16()
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    f = ops.readout_scored_forward(x, w, tokens=tok)
    with pytest.raises(ValueError, match="temperature"):
        ops.readout_scored_forward(x, w, tokens=tok, temperature=tau)
    with pytest.raises(ValueError, match="temperature"):
        ops.readout_backward(x, w, f, tokens=tok, g_logp=torch.ones(4, device="cuda"), temperature=tau)

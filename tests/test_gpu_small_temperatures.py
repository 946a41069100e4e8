"""Temperatures that are 0 in 32 bits in the calls on head(hidden): no temperature to score with, the first maximum when drawing."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tau", [0.0, 1e-46, 1e-50])
def test_small_temperatures(tau):
    from noetic_tensor_b200 import rl

    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = torch.randn(30, 64, generator=g, device="cuda").bfloat16()
    w = (0.3 * torch.randn(64, 264, generator=g, device="cuda")).bfloat16()
    u = torch.rand(30, generator=g, device="cuda")
    tokens, logp, _ = rl.head_sample_categorical(x, w, u, temperature=tau)
    assert torch.equal(tokens.long(), (x.float() @ w.float()).argmax(1))
    best, best_logp, _ = rl.head_sample_categorical(x, w, None)
    assert torch.equal(tokens, best) and torch.equal(logp, best_logp)
    with pytest.raises(ValueError, match="temperature"):
        rl.head_token_log_probs(x, w, tokens, temperature=tau)

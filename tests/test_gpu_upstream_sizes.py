"""`.backward(upstream)` of every loss: an upstream of another size than the value is refused, and the value's size in any type is taken."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("on", ["head", "logits"])
def test_upstreams_of_every_loss(on):
    from noetic_tensor_b200 import loss, rl

    S, B, T, d, V = 2, 3, 7, 64, 264
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(6)
    x = torch.randn(S, B, T, d, generator=g, device=dev).bfloat16()
    w = (torch.randn(d, V, generator=g, device=dev) * 0.3).bfloat16()
    tok = torch.randint(0, V, (S, B, T), generator=g, device=dev, dtype=torch.int32)
    old = -torch.rand(S, B, T, generator=g, device=dev) - 3
    mask = (torch.rand(S, B, T, generator=g, device=dev) < 0.6).float()
    z = rl.Head(x, w) if on == "head" else x.float() @ w.float()
    losses = [rl.token_log_probs(z, tok, mask), rl.token_log_probs(z, tok), loss.nll(z, tok), loss.cross_entropy(z, tok), loss.masked_cross_entropy(z, tok, mask)]
    for r in (rl.NONE, rl.SUM, rl.TOKEN_MEAN, rl.PER_SEQUENCE, rl.SEQUENCE_MEAN):
        losses += [rl.policy_gradient_loss(z, tok, old, mask, r), rl.clipped_policy_loss(z, tok, old, old, mask, reduction=r), rl.categorical_entropy(z, mask, r)]
    for l in losses:
        up = torch.randn(l.value.shape, generator=g, device=dev)
        for p, q in zip(l.backward(up), l.backward(up.double())):
            assert torch.equal(p, q) and torch.isfinite(p).all()
        for bad in (torch.ones((), device=dev), torch.ones(l.value.numel() + 1, device=dev), up.reshape(-1)[:1]):
            with pytest.raises((ValueError, RuntimeError)):
                l.backward(bad)
    with pytest.raises((ValueError, RuntimeError)):
        losses[0].backward(torch.ones(losses[0].value.shape))  # on the host

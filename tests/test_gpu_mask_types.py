"""Scoring masks of other types and orders than contiguous float32: every loss of a Head and of logits takes them as the 0/1 floats they stand for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["bool", "uint8", "double", "permuted", "expanded"])
@pytest.mark.parametrize("on", ["head", "logits"])
def test_masks_of_other_types(form, on):
    from noetic_tensor_b200 import loss, rl

    S, B, T, d, V = 2, 3, 7, 64, 264
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    x = torch.randn(S, B, T, d, generator=g, device=dev).bfloat16()
    w = (torch.randn(d, V, generator=g, device=dev) * 0.3).bfloat16()
    tok = torch.randint(0, V, (S, B, T), generator=g, device=dev, dtype=torch.int32)
    old = -torch.rand(S, B, T, generator=g, device=dev) - 3
    mask = (torch.rand(S, B, T, generator=g, device=dev) < 0.6).float()
    if form == "expanded":
        mask = mask[:1].expand(S, B, T)
        other = mask
    elif form == "permuted":
        other = mask.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    else:
        other = mask.to(dict(bool=torch.bool, uint8=torch.uint8, double=torch.double)[form])
    mask = mask.contiguous()
    z = (lambda: rl.Head(x, w)) if on == "head" else (lambda: x.float() @ w.float())
    runs = [
        lambda m: rl.token_log_probs(z(), tok, m),
        lambda m: rl.policy_gradient_loss(z(), tok, old, m),
        lambda m: rl.clipped_policy_loss(z(), tok, old, old, m),
        lambda m: rl.kl_estimate(z(), tok, old, rl.K3, mask=m, reduction=rl.PER_SEQUENCE),
        lambda m: rl.categorical_entropy(z(), m, rl.SUM),
        lambda m: rl.categorical_entropy(z(), m, rl.NONE),
        lambda m: loss.masked_cross_entropy(z(), tok, m),
    ]
    for run in runs:
        a, b = run(other), run(mask)
        assert torch.equal(a.value, b.value)
        p, q = a.backward(), b.backward()
        for got, want in zip(p, q) if on == "head" else ((p, q),):
            assert torch.equal(got, want)

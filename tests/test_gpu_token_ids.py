"""Token ids of 64 bits outside the vocabulary: they have no log-prob, whatever their lower 32 bits are."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


def case():
    S, B, T, d, V = 1, 2, 10, 64, 512
    g = torch.Generator(device=dev())
    g.manual_seed(3)
    x = torch.randn(S, B, T, d, generator=g, device=dev()).bfloat16()
    w = (torch.randn(d, V, generator=g, device=dev()) * 0.3).bfloat16()
    tok = torch.randint(0, V, (S, B, T), generator=g, device=dev())
    return x, w, tok


@pytest.mark.parametrize("wrong", [2**32 + 5, -(2**32) + 5, 2**31 + 5, 2**40, 512, -1])
@pytest.mark.parametrize("form", ["head", "logits"])
def test_a_token_that_32_bits_cannot_hold(wrong, form):
    from noetic_tensor_b200 import loss, rl

    x, w, tok = case()
    z = rl.Head(x, w) if form == "head" else (x.float() @ w.float())
    fine = rl.token_log_probs(z, tok).value
    assert torch.isfinite(fine).all() and torch.equal(fine, rl.token_log_probs(z, tok.to(torch.int32)).value)
    tok[0, 1, 3] = wrong
    got = rl.token_log_probs(z, tok).value
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[0, 1, 3] = True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], fine[~nan])
    adv = torch.ones(1, 2, 10, device=dev())
    assert torch.isnan(rl.policy_gradient_loss(z, tok, adv).value).all()
    assert torch.isnan(rl.kl_estimate(z, tok, adv, rl.K1).value).all()
    if form == "head":
        assert torch.equal(torch.isnan(loss.nll(z, tok).value.reshape(1, 2, 10)), nan)
        for l in (loss.cross_entropy(z, tok), loss.masked_cross_entropy(z, tok, adv), loss.cross_entropy_with(z, tok, adv, loss.CeOptions(ignore_index=-100))):
            assert torch.isnan(l.value).all()
        assert torch.isfinite(loss.cross_entropy_with(z, tok, adv, loss.CeOptions(ignore_index=wrong)).value).all()


@pytest.mark.parametrize("wrong", [2**32 + 5, -(2**32) + 5])
def test_the_scored_rollout(wrong):
    """head_token_log_probs, untracked: as token_log_probs of its logits."""
    from noetic_tensor_b200 import rl

    x, w, tok = case()
    tok[0, 1, 3] = wrong
    lp, _ = rl.head_token_log_probs(x, w, tok)
    assert torch.isnan(lp[0, 1, 3]) and torch.isfinite(lp).sum() == lp.numel() - 1

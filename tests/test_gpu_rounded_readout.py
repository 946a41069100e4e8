"""The backward of the readout takes no forward of rounded logits: their statistics do not normalise the unrounded ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_refused():
    from noetic_tensor_b200 import ops

    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = (4 * torch.randn(20, 64, generator=g, device="cuda")).bfloat16()
    w = torch.randn(64, 264, generator=g, device="cuda").bfloat16()
    tok = torch.randint(0, 264, (20,), generator=g, device="cuda", dtype=torch.int32)
    up = torch.ones(20, device="cuda")
    rounded, plain = ops.readout_forward(x, w, tokens=tok, round_bf16=True), ops.readout_forward(x, w, tokens=tok)
    for kw in (dict(tokens=tok, g_logp=up), dict(g_ent=up)):
        with pytest.raises(ValueError, match="rounded"):
            ops.readout_backward(x, w, rounded, **kw)
        assert all(torch.isfinite(t).all() for t in ops.readout_backward(x, w, plain, **kw))

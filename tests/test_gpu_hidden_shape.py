"""`hidden_shape` of readout_backward: any sequence of sizes that the checkpoint's rows fill, ending in d."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_shapes_of_d_hidden():
    from noetic_tensor_b200 import ops

    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x = torch.randn(12, 64, generator=g, device="cuda").bfloat16()
    w = (0.3 * torch.randn(64, 264, generator=g, device="cuda")).bfloat16()
    tok = torch.randint(0, 264, (12,), generator=g, device="cuda", dtype=torch.int32)
    up = torch.ones(12, device="cuda")
    f, q = ops.readout_scored_forward(x, w, tokens=tok), ops.quantize_rows(x)
    for states in (x, q):
        flat = ops.readout_backward(states, w, f, tokens=tok, g_logp=up)[0]
        assert flat.shape == (12, 64)
        for shape in ((2, 6, 64), [3, 2, 2, 64], torch.Size((12, 64)), (12, 1, 64)):
            got = ops.readout_backward(states, w, f, tokens=tok, g_logp=up, hidden_shape=shape)[0]
            assert got.shape == tuple(shape) and torch.equal(got.reshape(12, 64), flat)
        for shape in ((64, 12), (2, 5, 64), (771,), (12, 65), (24, 32), (2, 384), ()):
            with pytest.raises(ValueError, match="hidden"):
                ops.readout_backward(states, w, f, tokens=tok, g_logp=up, hidden_shape=shape)

"""quantize_weight of [d, V] weights of every remainder of the 64 x 64 tiles it turns over, against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,V", [(1, 1), (3, 2), (17, 65), (63, 64), (64, 63), (65, 129), (130, 3), (200, 1000)])
def test_columns_as_rows(d, V):
    from noetic_tensor_b200 import ops

    g = torch.Generator(device="cuda")
    g.manual_seed(d + V)
    w = torch.randn(d, V, generator=g, device="cuda").bfloat16()
    if d > 2:
        w[1, 0] = w[:, 0].abs().max() / 2  # a tie: 63.5 goes to the even 64
    q = ops.quantize_weight(w)
    big = w.double().abs().amax(0)
    assert torch.equal(q.scales, (big / 127.0).float())
    # 127·x is exact for bf16 x and the division is correctly rounded: the integers are those of exact arithmetic
    assert torch.equal(q.values[:, :d].double(), torch.round(127.0 * w.double() / big).t()) and (q.values[:, d:] == 0).all()

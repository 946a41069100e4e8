"""An infinite logit in the fused readout: the row has no distribution (inf - inf), so its results are NaN and a draw is refused; its first
maximum is the infinite one, as in the row forward."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,V", [(5, 1000), (300, 5000)])
@pytest.mark.parametrize("column", [0, 40, 700, -1])
def test_an_infinite_logit(rows, V, column):
    from noetic_tensor_b200 import ops, rl

    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    x = torch.randn(rows, 64, generator=g, device="cuda").bfloat16()
    w = (0.3 * torch.randn(64, V, generator=g, device="cuda")).bfloat16()
    tok = torch.randint(0, V, (rows,), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(rows, generator=g, device="cuda")
    x[:, 3] = torch.where(torch.arange(rows, device="cuda") % 2 == 0, 0.5, -0.5).bfloat16()  # +inf in even rows, -inf in odd ones
    w[3] = 0
    at = column % V
    allow = torch.ones(rows, V, dtype=torch.uint8, device="cuda")
    allow[:, at] = 0
    masked = [ops.readout_forward(x, w, tokens=tok, allow=allow), ops.readout_forward(x, w, uniforms=u, allow=allow), ops.readout_forward(x, w, greedy=True, allow=allow)]
    w[3, at] = math.inf
    given, drawn, best = ops.readout_forward(x, w, tokens=tok), ops.readout_forward(x, w, uniforms=u), ops.readout_forward(x, w, greedy=True)
    for o, ref in zip((given, drawn, best), masked):
        assert torch.isnan(o.logp[::2]).all() and torch.isnan(o.entropy[::2]).all()
        odd = slice(1, None, 2)  # a logit of -inf is an excluded one
        assert (o.status[odd] == 0).all() and ((o.entropy[odd] - ref.entropy[odd]).abs() <= 1e-5).all()
    assert (drawn.status[::2] == 2).all() and (drawn.tokens[::2] == -1).all()
    assert torch.equal(drawn.tokens[1::2], masked[1].tokens[1::2]) and ((drawn.tokens[1::2] >= 0) & (drawn.tokens[1::2] < V)).all()
    assert (best.tokens[::2] == at).all() and torch.equal(best.tokens[1::2], masked[2].tokens[1::2])
    row = ops.row_forward(torch.where(torch.arange(V, device="cuda") == at, math.inf, 0.0)[None].contiguous(), greedy=True)
    assert row.tokens[0] == at and torch.isnan(row.logp).all()
    with pytest.raises(RuntimeError, match="no allowed token"):
        rl.head_sample_categorical(x, w, u)

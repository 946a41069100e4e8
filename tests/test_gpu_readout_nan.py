"""One vocabulary entry whose logit is NaN (a NaN in its column of the weight), wherever it lies in a column range of the fused
readout: every row that may draw it is refused (status bit 1, NaN results, token −1); rows whose mask excludes it are not touched."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("rows,V,one_cta", [(5, 1000, False), (300, 5000, False), (300, 5000, True)])
@pytest.mark.parametrize("column", [5, 40, 120, 250, 300, -3])
@pytest.mark.parametrize("mode", ["tokens", "rounded", "sample", "greedy"])
def test_readout_forward(rows, V, one_cta, column, mode):
    from noetic_tensor_b200 import ops

    g = torch.Generator(device=dev())
    g.manual_seed(rows + V)
    x = torch.randn(rows, 64, generator=g, device=dev()).bfloat16()
    w = (torch.randn(64, V, generator=g, device=dev()) * 0.3).bfloat16()
    tok = torch.randint(0, V, (rows,), generator=g, device=dev(), dtype=torch.int32)
    at = column % V
    tok[tok == at] = (at + 1) % V
    kw = dict(one_cta=one_cta)
    if mode in ("tokens", "rounded"):
        kw.update(tokens=tok, round_bf16=mode == "rounded")
    elif mode == "sample":
        kw.update(uniforms=torch.rand(rows, generator=g, device=dev()))
    else:
        kw.update(greedy=True)
    clean = w.clone()
    clean[:, at] = 0
    w[3, at] = math.nan
    o = ops.readout_forward(x, w, **kw)
    assert (o.status == 2).all()
    assert torch.isnan(o.logp).all() and torch.isnan(o.entropy).all() and torch.isnan(o.rowstats).all()
    if o.tokens is not None:
        assert (o.tokens == -1).all()
    allow = torch.ones(rows, V, dtype=torch.uint8, device=dev())
    allow[::2, at] = 0
    want, o = ops.readout_forward(x, clean, allow=allow, **kw), ops.readout_forward(x, w, allow=allow, **kw)
    assert (o.status[::2] == 0).all() and (o.status[1::2] == 2).all()
    for got, ref in ((o.logp, want.logp), (o.entropy, want.entropy), (o.rowstats, want.rowstats)):
        assert torch.equal(got[::2], ref[::2]) and torch.isnan(got[1::2]).all()
    if o.tokens is not None:
        assert torch.equal(o.tokens[::2], want.tokens[::2]) and (o.tokens[1::2] == -1).all()

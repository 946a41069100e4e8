"""One vocabulary entry whose logit is NaN (a NaN in its column of the weight), wherever it lies in a tile: every row that may
draw it has no distribution (status bit 1, NaN results); rows whose mask excludes it are not touched by it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


def make(rows, V, d=64):
    g = torch.Generator(device=dev())
    g.manual_seed(rows + V)
    x = torch.randn(rows, d, generator=g, device=dev()).bfloat16()
    w = (torch.randn(d, V, generator=g, device=dev()) * 0.3).bfloat16()
    tok = torch.randint(0, V, (rows,), generator=g, device=dev(), dtype=torch.int32)
    return x, w, tok


def bits_of(allow):
    rows, V = allow.shape
    a = torch.zeros(rows, (V + 31) // 32 * 32, dtype=torch.int64, device=allow.device)
    a[:, :V] = (allow != 0).long()
    words = (a.reshape(rows, -1, 32) << torch.arange(32, device=allow.device)).sum(2)
    return torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)


# halves of a tile of 64 and of 128 columns, on CTAs by themselves and on pairs
SHAPES = [(5, 1000), (5, 20008), (300, 1000), (300, 5000)]
COLUMNS = [5, 40, 70, 120, 200, -3]  # first, middle and last 32 columns of a half tile, and the vocabulary's end


@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("column", COLUMNS)
def test_scored_forward(rows, V, column):
    from noetic_tensor_b200 import ops

    x, w, tok = make(rows, V)
    at = column % V
    tok[tok == at] = (at + 1) % V
    w[3, at] = math.nan
    for entropy in (False, True):
        o = ops.readout_scored_forward(x, w, tokens=tok, want_entropy=entropy, ce_seeds=1)
        assert (o.status == 2).all()
        for t in (o.logp, o.rowstats, o.ce_loss) + ((o.entropy,) if entropy else ()):
            assert torch.isnan(t).all()
    # excluded for every other row, as bytes and as bits
    allow = torch.ones(rows, V, dtype=torch.uint8, device=dev())
    allow[::2, at] = 0
    clean = w.clone()
    clean[:, at] = 0
    want = ops.readout_scored_forward(x, clean, tokens=tok, want_entropy=True, allow=allow)
    for kw in (dict(allow=allow), dict(allow_bits=bits_of(allow))):
        o = ops.readout_scored_forward(x, w, tokens=tok, want_entropy=True, **kw)
        assert (o.status[::2] == 0).all() and (o.status[1::2] == 2).all()
        for got, ref in ((o.logp, want.logp), (o.entropy, want.entropy), (o.rowstats, want.rowstats)):
            assert torch.equal(got[::2], ref[::2]) and torch.isnan(got[1::2]).all()

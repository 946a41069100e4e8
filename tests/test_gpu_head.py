"""The readout's backward (nrl_readout_bwd), its 8-bit checkpoint and the 8-bit product, against plain
implementations in 64 bits.

Tolerances. u = 2^-8 is half a step of bf16 relative to the value. An entry of ∂/∂z is rounded to bf16
once before the products, so with D = |a|·(1[j = token] + π_j) + |b|·π_j·(|ln π_j| + H + 1) (what the
entry is a difference of) its error is at most (u + e)·D, where e covers π computed from f32 sums:
|δz| + |δ ln Z| ≤ 4·(d + 16)·2^-24·max Σ|x·w| / τ. A gradient is then off by at most (u + e)·(D·|W|) resp.
(u + e)·(|x|ᵀ·D), plus u·|gradient| where it is returned as bf16, plus the f32 sums' n·2^-24 of the same
products. With 8-bit rows the same holds for their dequantised values. The 8-bit product is exact up to the
conversion of the 32-bit sum and two products in f32 (3·2^-24) and the rounding of the result."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U16, U32 = 2.0**-8, 2.0**-24


def dev():
    return torch.device("cuda:0")


def make(rows, d, V, seed, layout="dV"):
    g = torch.Generator(device=dev())
    g.manual_seed(seed)
    w = (torch.randn(V, d, generator=g, device=dev()) * (3.0 / d**0.5)).bfloat16()
    tok = torch.randint(0, V, (rows,), generator=g, device=dev(), dtype=torch.int32)
    x = (torch.randn(rows, d, generator=g, device=dev()) + torch.rand(rows, 1, generator=g, device=dev()) * w[tok.long()].float()).bfloat16()
    return x, (w if layout == "Vd" else w.t().contiguous()), tok, g


def bits_of(allow):
    """int32 words [rows, ceil(V/32)] of a byte mask: bit v mod 32 of word v / 32."""
    rows, V = allow.shape
    a = torch.zeros(rows, (V + 31) // 32 * 32, dtype=torch.int64, device=allow.device)
    a[:, :V] = (allow != 0).long()
    words = (a.reshape(rows, -1, 32) << torch.arange(32, device=allow.device)).sum(2)
    return torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)


def truth(x, w_vd, tok, g_logp, g_ent, allow, tau, lse=None, stats=None):
    """d_hidden, d_weight [V, d] in 64 bits and their tolerances' majorants. `x` f64 [rows, d]; `stats`: (lse, H) of another forward."""
    x, w = x.double(), w_vd.double()
    rows, V = x.shape[0], w.shape[0]
    z = x @ w.t() / tau
    e = 4.0 * (x.shape[1] + 16) * U32 * (x.abs() @ w.abs().t()).max().item() / tau
    if allow is not None:
        z = torch.where(allow.expand(rows, V) != 0, z, torch.full_like(z, -math.inf))
    if stats is None:
        lse = torch.logsumexp(z, 1, keepdim=True)
        lp = z - lse
        H = -torch.where(lp > -math.inf, lp.exp() * lp, torch.zeros_like(lp)).sum(1, keepdim=True)
    else:
        lse, H = stats[0].double()[:, None], stats[1].double()[:, None]
        lp = z - lse
    pi = lp.exp()
    lp = torch.where(lp > -math.inf, lp, torch.zeros_like(lp))
    a = torch.zeros(rows, 1, dtype=torch.float64, device=x.device) if g_logp is None else g_logp.double()[:, None]
    b = torch.zeros_like(a) if g_ent is None else g_ent.double()[:, None]
    hot = torch.zeros_like(z)
    ok = (tok >= 0) & (tok < V)
    hot[torch.arange(rows, device=x.device)[ok], tok[ok].long()] = 1.0
    if allow is not None:
        hot = hot * (allow.expand(rows, V) != 0)
    dz = (a * (hot - pi) - b * pi * (lp + H)) / tau
    D = (a.abs() * (hot + pi) + b.abs() * pi * (lp.abs() + H + 1.0)) / tau
    return dz @ w, dz.t() @ x, (U16 + e) * (D @ w.abs()) + V * U32 * (D @ w.abs()), (U16 + e) * (D.t() @ x.abs()) + rows * U32 * (D.t() @ x.abs())


def held(got, want, tol, what):
    u = U16 if got.dtype == torch.bfloat16 else U32
    err, lim = (got.double() - want).abs(), tol + 2 * u * want.abs() + 1e-30
    assert torch.isfinite(got).all(), what
    assert (err <= lim).all(), f"{what}: {(err > lim).sum().item()} of {err.numel()} outside, worst {(err / lim).max().item():.2f} of its tolerance"


SHAPES = [(1, 8, 8), (16, 64, 1000), (37, 72, 776), (128, 64, 256), (129, 256, 1024), (300, 136, 4104), (257, 512, 8200), (700, 1032, 2056), (64, 2048, 32000)]


@pytest.mark.parametrize("rows,d,V", SHAPES)
@pytest.mark.parametrize("layout", ["dV", "Vd"])
def test_backward_against_64_bits(rows, d, V, layout):
    from noetic_tensor_b200 import ops

    x, w, tok, g = make(rows, d, V, rows + V, layout)
    vd = layout == "Vd"
    up = torch.randn(rows, generator=g, device=dev())
    up[torch.rand(rows, generator=g, device=dev()) < 0.3] = 0.0
    ent = 0.1 * torch.randn(rows, generator=g, device=dev())
    ent[up == 0] = 0.0
    f = ops.readout_forward(x, w, tokens=tok, weights_are_vd=vd)
    w_vd = w if vd else w.t()
    for gl, ge, dt in ((up, None, torch.bfloat16), (up, ent, torch.float32), (None, ent, torch.bfloat16)):
        dh, dw = ops.readout_backward(x, w, f, tokens=tok, g_logp=gl, g_ent=ge, weights_are_vd=vd, grad_dtype=dt)
        th, tw, eh, ew = truth(x, w_vd, tok, gl, ge, None, 1.0)
        held(dh, th, eh, "d_hidden")
        held(dw if vd else dw.t(), tw, ew, "d_weights")
        assert dh.dtype == dt and (dh[up == 0] == 0).all()
        dh2, dw2 = ops.readout_backward(x, w, f, tokens=tok, g_logp=gl, g_ent=ge, weights_are_vd=vd, grad_dtype=dt)
        assert torch.equal(dh, dh2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("rows,d,V", [(1, 16, 24), (100, 72, 776), (300, 256, 4104)])
@pytest.mark.parametrize("tau", [1.0, 0.7, 1.5])
@pytest.mark.parametrize("form", ["bytes", "row", "bits", "bits row"])
def test_masks_and_temperature(rows, d, V, tau, form):
    from noetic_tensor_b200 import ops

    x, w, tok, g = make(rows, d, V, rows + V)
    allow = (torch.rand(1 if "row" in form else rows, V, generator=g, device=dev()) < 0.4).to(torch.uint8)
    allow[:, 0] = 1
    kw = dict(allow_bits=bits_of(allow)) if "bits" in form else dict(allow=allow)
    up, ent = torch.randn(rows, generator=g, device=dev()), 0.1 * torch.randn(rows, generator=g, device=dev())
    f = ops.readout_forward(x, w, tokens=tok, temperature=tau, **kw)
    dh, dw = ops.readout_backward(x, w, f, tokens=tok, g_logp=up, g_ent=ent, temperature=tau, **kw)
    th, tw, eh, ew = truth(x, w.t(), tok, up, ent, allow, tau)
    held(dh, th, eh, "d_hidden")
    held(dw.t(), tw, ew, "d_weights")
    gone = (allow == 0).all(0)
    assert (dw[:, gone] == 0).all()  # a token that no row allows has an exactly zero gradient


@pytest.mark.parametrize("rows,d,V", [(1, 8, 8), (201, 512, 4104), (300, 136, 2056)])
@pytest.mark.parametrize("layout", ["dV", "Vd"])
def test_checkpoint_backward_against_64_bits(rows, d, V, layout):
    """From 8-bit rows: the logits and d_weights of values·scale, normalised by the unrounded forward."""
    from noetic_tensor_b200 import ops

    x, w, tok, g = make(rows, d, V, rows + V, layout)
    vd = layout == "Vd"
    x[rows // 2] = 0  # a row of zeros has scale 0
    up, ent = torch.randn(rows, generator=g, device=dev()), 0.1 * torch.randn(rows, generator=g, device=dev())
    f = ops.readout_forward(x, w, tokens=tok, weights_are_vd=vd)
    q = ops.quantize_rows(x)
    dh, dw = ops.readout_backward(q, w, f, tokens=tok, g_logp=up, g_ent=ent, weights_are_vd=vd)
    xq = q.values[:, :d].double() * q.scales.double()[:, None]
    lse = f.rowstats[:, 0].double() + f.rowstats[:, 1].double()
    th, tw, eh, ew = truth(xq, w if vd else w.t(), tok, up, ent, None, 1.0, stats=(lse, f.entropy))
    held(dh, th, eh, "d_hidden")
    held(dw if vd else dw.t(), tw, ew, "d_weights")


@pytest.mark.parametrize("rows,d", [(1, 1), (1, 8), (5, 17), (64, 1000), (33, 4096), (300, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantised_rows(rows, d, dtype):
    from noetic_tensor_b200 import ops

    g = torch.Generator(device=dev())
    g.manual_seed(rows + d)
    x = (torch.randn(rows, d, generator=g, device=dev()) * torch.exp(4 * torch.randn(rows, 1, generator=g, device=dev()))).to(dtype)
    if d > 2:
        x[0, 1] = x[0].abs().max() / 2  # a tie: 63.5 goes to the even 64
    if rows > 4:
        x[2] = 0
    q = ops.quantize_rows(x)
    big = x.double().abs().amax(1, keepdim=True)
    assert torch.equal(q.scales, (big / 127.0).float()[:, 0])
    want = torch.where(big > 0, 127.0 * x.double() / big, torch.zeros_like(big))
    got = q.values[:, :d].double()
    if dtype == torch.bfloat16:
        assert torch.equal(got, torch.round(want))
    else:  # f32: 127·x and the quotient are each rounded once, which can move a value across a tie
        assert ((got - want).abs() <= 0.5 + 127 * 4 * U32).all()
    assert (q.values[:, d:] == 0).all() and q.values.abs().max() <= 127
    back = ops.dequantize_rows(q, torch.float32)
    assert torch.equal(back, q.values[:, :d].float() * q.scales[:, None])


@pytest.mark.parametrize("d,V", [(8, 8), (72, 136), (1000, 504), (264, 4104)])
def test_quantised_weight_layouts(d, V):
    from noetic_tensor_b200 import ops

    _, w, _, _ = make(1, d, V, d + V)
    w[:, 3] = 0
    a, b = ops.quantize_weight(w), ops.quantize_weight(w.t().contiguous(), weights_are_vd=True)
    assert torch.equal(a.values, b.values) and torch.equal(a.scales, b.scales) and a.scales[3] == 0


@pytest.mark.parametrize("rows", [1, 2, 17, 33, 128, 255, 256, 257, 333, 700])
@pytest.mark.parametrize("k,n", [(16, 8), (1, 1), (1000, 257), (136, 4099), (2048, 1000)])
def test_int8_product_is_exact(rows, k, n):
    from noetic_tensor_b200 import ops

    g = torch.Generator(device=dev())
    g.manual_seed(rows + k + n)
    P = (k + 15) // 16 * 16
    xv = torch.randint(-127, 128, (rows, P), generator=g, device=dev(), dtype=torch.int8)  # what lies behind k must not matter
    wv = torch.randint(-127, 128, (n, P), generator=g, device=dev(), dtype=torch.int8)
    xs, ws = torch.rand(rows, generator=g, device=dev()), torch.rand(n, generator=g, device=dev())
    x, w = ops.Int8Rows(xv, xs, k), ops.Int8Rows(wv, ws, k)
    want = (xv[:, :k].double() @ wv[:, :k].double().t()) * xs.double()[:, None] * ws.double()
    for dt, tol in ((torch.float32, 3 * U32), (torch.bfloat16, U16 + 3 * U32)):
        got = ops.int8_matmul(x, w, dt)
        assert got.shape == (rows, n) and got.dtype == dt
        assert ((got.double() - want).abs() <= tol * want.abs() * (1 + 1e-6)).all(), (got.double() - want).abs().max()


def test_int8_extreme_integers_and_nonfinite_scales():
    from noetic_tensor_b200 import ops

    k = 131072
    x = ops.Int8Rows(torch.full((3, k), 127, dtype=torch.int8, device=dev()), torch.tensor([1.0, math.nan, math.inf], device=dev()), k)
    w = ops.Int8Rows(torch.full((40, k), -127, dtype=torch.int8, device=dev()), torch.ones(40, device=dev()), k)
    got = ops.int8_matmul(x, w)
    assert (got[0] == float(-127 * 127 * k)).all() and torch.isnan(got[1]).all() and torch.isinf(got[2]).all()

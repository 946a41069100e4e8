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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [2.0**127, 2.0**122, 2.0**-100, 2.0**-120])
def test_quantised_rows_of_extreme_magnitude(dtype, top):
    """Powers of two times small integers: exact in both types, so the integers are those of exact arithmetic, ties included."""
    from noetic_tensor_b200 import ops

    part = torch.tensor([1.0, -1.0, 0.5, -0.5, 0.25, 0.75, 2.0**-6, 2.0**-7, 2.0**-8, 0.0], device=dev(), dtype=torch.float64)
    x = (top * part).to(dtype)[None]
    assert torch.equal(x.double()[0], top * part)
    q = ops.quantize_rows(x)
    assert torch.equal(q.values[0, :10].double(), torch.round(127.0 * part))
    assert torch.equal(q.scales.double(), torch.tensor([top / 127.0], device=dev(), dtype=torch.float64).float().double())


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


def test_int8_results_past_32_bits():
    """Offsets of the result past 2^32 elements, checked where they pass it and at both ends."""
    from noetic_tensor_b200 import ops

    rows, n, k = 33600, 128256, 32
    g = torch.Generator(device=dev())
    g.manual_seed(1)
    x = torch.randint(-127, 128, (rows, k), generator=g, device=dev(), dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, device=dev(), dtype=torch.int8)
    out = ops.int8_matmul(ops.Int8Rows(x, torch.ones(rows, device=dev()), k), ops.Int8Rows(w, torch.ones(n, device=dev()), k), torch.bfloat16)
    assert out.numel() > 2**32
    for at in (0, 2**31 // n, 2**32 // n, rows - 4):
        want = x[at : at + 4].double() @ w.double().t()
        assert torch.equal(out[at : at + 4], want.float().bfloat16())  # an integer below 2^24, rounded once


def test_int8_extreme_integers_and_nonfinite_scales():
    from noetic_tensor_b200 import ops

    k = 131072
    x = ops.Int8Rows(torch.full((3, k), 127, dtype=torch.int8, device=dev()), torch.tensor([1.0, math.nan, math.inf], device=dev()), k)
    w = ops.Int8Rows(torch.full((40, k), -127, dtype=torch.int8, device=dev()), torch.ones(40, device=dev()), k)
    got = ops.int8_matmul(x, w)
    assert (got[0] == float(-127 * 127 * k)).all() and torch.isnan(got[1]).all() and torch.isinf(got[2]).all()


# ---- the forward over the scored rows ---------------------------------------------------------------


def forward_truth(x, w_vd, tok, allow, tau):
    z = x.double() @ w_vd.double().t() / tau
    if allow is not None:
        z = torch.where(allow.expand(z.shape) != 0, z, torch.full_like(z, -math.inf))
    lse = torch.logsumexp(z, 1)
    lp = z - lse[:, None]
    H = -torch.where(lp > -math.inf, lp.exp() * lp, torch.zeros_like(lp)).sum(1)
    # |δz| of an f32 sum of d products, twice (the logit and ln Z), against the largest Σ|x·w| of the row
    e = 4.0 * (x.shape[1] + 16) * U32 * (x.double().abs() @ w_vd.double().abs().t()).amax(1) / tau
    return lp[torch.arange(len(tok), device=x.device), tok.long()], H, lse, e


@pytest.mark.parametrize("rows,d,V", [(1, 8, 8), (16, 64, 1000), (129, 256, 1024), (300, 136, 4104), (700, 1032, 2056), (17000, 64, 264), (40, 2048, 32000)])
@pytest.mark.parametrize("layout", ["dV", "Vd"])
@pytest.mark.parametrize("form", [None, "bytes", "row", "bits"])
def test_scored_forward_against_64_bits(rows, d, V, layout, form):
    from noetic_tensor_b200 import ops

    x, w, tok, g = make(rows, d, V, rows + V, layout)
    w_vd, vd = (w, True) if layout == "Vd" else (w.t(), False)
    allow = None if form is None else (torch.rand(1 if form == "row" else rows, V, generator=g, device=dev()) < 0.5).to(torch.uint8)
    if allow is not None:
        allow[:, 1] = 1
    kw = {} if form is None else dict(allow_bits=bits_of(allow)) if form == "bits" else dict(allow=allow)
    scored = (torch.rand(rows, generator=g, device=dev()) < 0.7).float()
    scored[0] = 1.0
    x[scored == 0] = math.nan  # what an unscored position holds is not looked at
    tau = 1.0 if form is None else 0.7
    o = ops.readout_scored_forward(x, w, tokens=tok, scored=scored, want_entropy=True, weights_are_vd=vd, temperature=tau, ce_seeds=1, **kw)
    on = scored != 0
    lp, H, lse, e = forward_truth(x[on], w_vd, tok[on], allow if allow is None or allow.shape[0] == 1 else allow[on], tau)
    assert (o.status == 0).all()
    got = o.logp[on].double()
    assert torch.equal(got == -math.inf, lp == -math.inf)
    fin = lp > -math.inf
    assert ((got - lp).abs()[fin] <= (e + 8 * U32 * lp.abs())[fin]).all()
    assert ((o.entropy[on].double() - H).abs() <= e * (1 + lse.abs()) + 64 * U32 * (1 + H)).all()
    assert ((o.rowstats[on, 0].double() + o.rowstats[on, 1].double() - lse).abs() <= e + 8 * U32 * (1 + lse.abs())).all()
    assert (o.logp[~on] == 0).all() and (o.entropy[~on] == 0).all() and (o.rowstats[~on] == 0).all()
    # the mean cross-entropy of the same call, and the call of its own
    nll = -o.logp[on].double()
    want = nll.sum() / max(1, int(on.sum()))
    assert (torch.isinf(want) and torch.isinf(o.ce_loss[0])) or abs(o.ce_loss[0].item() - want.item()) <= 4 * U32 * abs(want.item())
    value, grad = ops.ce_mean(o.logp, 1, scored)
    assert torch.equal(value, o.ce_loss) and torch.equal(grad, o.ce_g_logp)
    assert (grad[~on] == 0).all() and ((grad[on].double() + 1.0 / int(on.sum())).abs() <= 2 * U32 / int(on.sum())).all()
    again = ops.readout_scored_forward(x, w, tokens=tok, scored=scored, want_entropy=True, weights_are_vd=vd, temperature=tau, ce_seeds=1, **kw)
    assert torch.equal(o._buf[: 4 * rows].view(torch.int32), again._buf[: 4 * rows].view(torch.int32)) and torch.equal(o.logp, again.logp) and torch.equal(o.entropy, again.entropy)


def test_scored_forward_agrees_with_the_sampling_forward():
    from noetic_tensor_b200 import ops

    x, w, tok, _ = make(300, 512, 8200, 4)
    a, b = ops.readout_scored_forward(x, w, tokens=tok, want_entropy=True), ops.readout_forward(x, w, tokens=tok)
    e = forward_truth(x, w.t(), tok, None, 1.0)[3]
    assert ((a.logp.double() - b.logp.double()).abs() <= 2 * e + 16 * U32 * b.logp.double().abs()).all()
    ga = ops.readout_backward(x, w, a, tokens=tok, g_logp=torch.ones(300, device=dev()))
    gb = ops.readout_backward(x, w, b, tokens=tok, g_logp=torch.ones(300, device=dev()))
    for p, q in zip(ga, gb):
        assert ((p.double() - q.double()).norm() <= 1e-2 * q.double().norm()).item()


def test_tokens_and_rows_that_have_no_log_prob():
    from noetic_tensor_b200 import ops

    rows, d, V = 140, 64, 1000
    x, w, tok, g = make(rows, d, V, 9)
    allow = torch.ones(rows, V, dtype=torch.uint8, device=dev())
    allow[3] = 0  # nothing allowed
    allow[4, tok[4].long()] = 0  # the token itself is excluded
    allow[5] = 0
    allow[5, 999 if tok[5] < 500 else 0] = 1  # the token's whole neighbourhood is excluded
    tok[6], tok[7], tok[8] = V, -1, V + 20
    x[9, 3] = math.nan
    o = ops.readout_scored_forward(x, w, tokens=tok, want_entropy=True, allow=allow)
    st = o.status.cpu().numpy()
    assert st[3] == 1 and st[9] == 2 and (np.delete(st, [3, 9]) == 0).all()
    lp = o.logp
    assert torch.isnan(lp[[3, 6, 7, 8, 9]]).all() and (lp[[4, 5]] == -math.inf).all() and torch.isfinite(lp[10:]).all() and torch.isfinite(o.entropy[[4, 5, 6, 7, 8]]).all()
    up = torch.zeros(rows, device=dev())
    up[10:] = 1.0
    dh, dw = ops.readout_backward(x, w, o, tokens=tok, g_logp=up, allow=allow)  # the refused rows are not scored: nothing of them arrives
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all() and (dh[:10] == 0).all()
    up[3] = 1.0  # nothing allowed: the gradient is 0 at every excluded token, here at all of them
    dh3, dw3 = ops.readout_backward(x, w, o, tokens=tok, g_logp=up, allow=allow)
    # d_weights sums the same terms, moved by one place: two f32 sums of up to 131 terms x·∂/∂z, |∂/∂z| ≤ 1, differ by at most
    # 2·131·2^-24·Σ|x| and may be rounded to neighbouring bf16 numbers
    spread = 2 * 131 * U32 * x[10:].double().abs().sum(0)[:, None]
    assert torch.equal(dh3, dh) and ((dw3.double() - dw.double()).abs() <= 2 * U16 * dw.double().abs() + spread).all()
    up[9] = 1.0  # a NaN among the hidden states
    dh, dw = ops.readout_backward(x, w, o, tokens=tok, g_logp=up, allow=allow)
    assert torch.isnan(dh[9]).all() and torch.isnan(dw).any() and torch.isfinite(dh[10:]).all()


def test_nothing_scored():
    from noetic_tensor_b200 import loss, ops, rl

    for rows in (5, 300):
        x, w, tok, _ = make(rows, 64, 264, 2)
        zero = torch.zeros(rows, device=dev())
        o = ops.readout_scored_forward(x, w, tokens=tok, scored=zero, ce_seeds=1)
        assert (o.logp == 0).all() and (o.ce_loss == 0).all()
        dh, dw = ops.readout_backward(x, w, o, tokens=tok, g_logp=zero)
        assert (dh == 0).all() and (dw == 0).all()
        l = loss.masked_cross_entropy(rl.Head(x.reshape(1, 1, rows, 64), w), tok.reshape(1, 1, rows), zero.reshape(1, 1, rows))
        dh, dw = l.backward()
        assert (l.value == 0).all() and (dh == 0).all() and (dw == 0).all()


def test_masked_positions_may_hold_anything():
    from noetic_tensor_b200 import loss, rl

    for checkpoint in (False, True):
        x, w, tok, g = make(300, 136, 1000, 11)
        mask = (torch.rand(300, generator=g, device=dev()) < 0.5).float()
        y = x.clone()
        y[mask == 0] = math.nan
        y[(mask == 0).nonzero()[0]] = math.inf
        shape = (2, 3, 50)
        a = loss.masked_cross_entropy(rl.Head(x.reshape(*shape, 136), w, checkpoint=checkpoint), tok.reshape(shape), mask.reshape(shape))
        b = loss.masked_cross_entropy(rl.Head(y.reshape(*shape, 136), w, checkpoint=checkpoint), tok.reshape(shape), mask.reshape(shape))
        assert torch.equal(a.value, b.value)
        for p, q in zip(a.backward(), b.backward()):
            assert torch.equal(p, q)


# ---- more of the backward ----------------------------------------------------------------------------


def test_several_pieces_of_the_vocabulary():
    """Enough rows that dz of the whole vocabulary would be over 512 MB: the sums of d_hidden are carried from piece to piece."""
    from noetic_tensor_b200 import ops

    rows, d, V = 16500, 64, 20008
    x, w, tok, g = make(rows, d, V, 5)
    up = torch.randn(rows, generator=g, device=dev())
    f = ops.readout_scored_forward(x, w, tokens=tok)
    dh, dw = ops.readout_backward(x, w, f, tokens=tok, g_logp=up, grad_dtype=torch.float32)
    pick = torch.arange(0, rows, 97, device=dev())
    th, _, eh, _ = truth(x[pick], w.t(), tok[pick], up[pick], None, None, 1.0)
    held(dh[pick], th, eh, "d_hidden")
    tw, ew = torch.zeros(V, d, dtype=torch.float64, device=dev()), torch.zeros(V, d, dtype=torch.float64, device=dev())
    for r in range(0, rows, 4125):
        p = slice(r, r + 4125)
        _, a, _, b = truth(x[p], w.t(), tok[p], up[p], None, None, 1.0)
        tw += a
        ew += b
    held(dw.t(), tw, ew + rows * U32 * ew / U16, "d_weights")


@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("layout", ["dV", "Vd"])
def test_pieces_whose_sums_are_split(rows, layout):
    """So many columns that few rows have two pieces too: every range of a split sum is carried from piece to piece."""
    from noetic_tensor_b200 import ops

    d, V = 64, 1060008
    x, w, tok, g = make(rows, d, V, rows, layout)
    vd = layout == "Vd"
    up = torch.randn(rows, generator=g, device=dev())
    f = ops.readout_scored_forward(x, w, tokens=tok, weights_are_vd=vd)
    w_vd = w if vd else w.t()
    th, tw, eh, ew = truth(x, w_vd, tok, up, None, None, 1.0)
    for dtype in (torch.bfloat16, torch.float32):
        dh, dw = ops.readout_backward(x, w, f, tokens=tok, g_logp=up, weights_are_vd=vd, grad_dtype=dtype)
        held(dh, th, eh, "d_hidden")
        held(dw if vd else dw.t(), tw, ew, "d_weights")


@pytest.mark.parametrize("rows,d,V", [(40, 136, 1000), (300, 264, 4104), (64, 512, 40008)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_adding_to_gradients(rows, d, V, dtype):
    from noetic_tensor_b200 import ops

    x, w, tok, g = make(rows, d, V, rows + d)
    up = torch.randn(rows, generator=g, device=dev())
    up[::5] = 0
    f = ops.readout_scored_forward(x, w, tokens=tok)
    dh, dw = ops.readout_backward(x, w, f, tokens=tok, g_logp=up, grad_dtype=torch.float32)
    h0, w0 = torch.randn(rows, d, generator=g, device=dev()).to(dtype), torch.randn(d, V, generator=g, device=dev()).to(dtype)
    ha, wa = h0.clone(), w0.clone()
    ops.readout_backward(x, w, f, tokens=tok, g_logp=up, add_hidden=ha, add_weights=wa)
    u = U16 if dtype == torch.bfloat16 else 2 * U32
    for got, old, new in ((ha, h0, dh), (wa, w0, dw)):
        want = old.double() + new.double()
        assert ((got.double() - want).abs() <= u * want.abs() + 4 * U32 * (old.double().abs() + new.double().abs())).all()
    assert torch.equal(ha[::5], h0[::5])  # rows without an upstream stay as they are
    only_h = ops.readout_backward(x, w, f, tokens=tok, g_logp=up, want_weights=False)
    only_w = ops.readout_backward(x, w, f, tokens=tok, g_logp=up, want_hidden=False)
    both = ops.readout_backward(x, w, f, tokens=tok, g_logp=up)
    assert only_h[1] is None and only_w[0] is None and torch.equal(only_h[0], both[0]) and torch.equal(only_w[1], both[1])


def test_gradients_against_differences():
    """Directional derivatives of the loss in 64 bits by central differences against the kernels' gradients."""
    from noetic_tensor_b200 import ops

    rows, d, V = 60, 72, 264
    x, w, tok, g = make(rows, d, V, 21)
    up, ent = torch.randn(rows, generator=g, device=dev()), 0.3 * torch.randn(rows, generator=g, device=dev())
    f = ops.readout_scored_forward(x, w, tokens=tok, want_entropy=True)
    dh, dw = ops.readout_backward(x, w, f, tokens=tok, g_logp=up, g_ent=ent, grad_dtype=torch.float32)
    _, _, eh, ew = truth(x, w.t(), tok, up, ent, None, 1.0)

    def value(x, w):
        lp = torch.log_softmax(x @ w, 1)
        return (up.double() * lp[torch.arange(rows), tok.long()]).sum() + (ent.double() * -(lp.exp() * lp).sum(1)).sum()

    X, W, h = x.double(), w.double(), 1e-4
    for _ in range(4):
        vx, vw = torch.randn(rows, d, generator=g, device=dev()).double(), torch.randn(d, V, generator=g, device=dev()).double()
        diff = (value(X + h * vx, W + h * vw) - value(X - h * vx, W - h * vw)) / (2 * h)
        got = (dh.double() * vx).sum() + (dw.double() * vw).sum()
        bound = (eh * vx.abs()).sum() + (ew.t() * vw.abs()).sum()
        assert (got - diff).abs() <= bound + 1e-5 * diff.abs()


# ---- rl.Head through the losses --------------------------------------------------------------------------


def head_case(S, B, T, d, V, seed, layout="dV"):
    x, w, tok, g = make(S * B * T, d, V, seed, layout)
    mask = (torch.rand(S, B, T, generator=g, device=dev()) < 0.8).float()
    return x.reshape(S, B, T, d), w, tok.reshape(S, B, T), mask, g


@pytest.mark.parametrize("S,B,T,d,V", [(1, 1, 1, 8, 8), (2, 3, 50, 136, 1000), (3, 2, 61, 512, 4104)])
@pytest.mark.parametrize("what", ["pg", "ppo", "k1", "k3", "token_log_probs", "entropy", "nll", "ce", "masked_ce", "ignore"])
def test_losses_on_a_head_against_the_losses_on_its_logits(S, B, T, d, V, what):
    """The same functions on f32 logits of the same operands: values within the f32 sums' spread of the logits, gradients
    within what the bf16 rounding of ∂/∂z allows (2-norms: at most u of the majorant, which these draws keep below 4 u of the gradient)."""
    from noetic_tensor_b200 import loss, rl

    x, w, tok, mask, g = head_case(S, B, T, d, V, S + T + V)
    logits = (x.double() @ w.double()).float()
    adv, old = torch.randn(S, B, T, generator=g, device=dev()), -2 * torch.rand(S, B, T, generator=g, device=dev()) - 3

    def run(z):
        if what == "pg":
            return rl.policy_gradient_loss(z, tok, adv, mask)
        if what == "ppo":
            return rl.clipped_policy_loss(z, tok, old, adv, mask)
        if what == "k1":
            return rl.kl_estimate(z, tok, old, rl.K1, mask=mask, reduction=rl.SEQUENCE_MEAN)
        if what == "k3":
            return rl.kl_estimate(z, tok, old, rl.K3, delta_clamp=20.0, mask=mask, reduction=rl.PER_SEQUENCE)
        if what == "token_log_probs":
            return rl.token_log_probs(z, tok, mask)
        if what == "entropy":
            return rl.categorical_entropy(z, mask, rl.SUM)
        if what == "nll":
            return loss.nll(z, tok)
        if what == "ce":
            return loss.cross_entropy(z, tok)
        if what == "masked_ce":
            return loss.masked_cross_entropy(z, tok, mask)
        return loss.cross_entropy_with(z, tok, mask, loss.CeOptions(ignore_index=int(tok[0, 0, 0])))

    a, b = run(rl.Head(x, w, grad_dtype=torch.float32)), run(logits)
    assert a.value.shape == b.value.shape
    assert ((a.value - b.value).abs() <= 1e-4 * (1 + b.value.abs())).all()
    for up in (None, torch.randn(b.value.shape, generator=g, device=dev())):
        dh, dw = a.backward(up)
        dz = b.backward(up).reshape(-1, V).double()
        th, tw = dz @ w.double().t(), x.reshape(-1, d).double().t() @ dz
        assert dh.shape == x.shape and dw.shape == w.shape
        for got, want in ((dh.reshape(-1, d), th), (dw, tw)):
            assert (got.double() - want).norm() <= 4 * U16 * want.norm() + 1e-12


@pytest.mark.parametrize("form", ["ones", "parts of one", "none kept", "no mask", "per sequence", "bool"])
def test_policy_gradient_of_a_head_and_of_its_log_probs(form):
    """The loss that the forward leaves is the reduction of its own log-probs: f64 sums of f32 terms, rounded once (and once
    more for the gradient's product); where nothing is kept both are 0, whatever the weights hold."""
    from noetic_tensor_b200 import ops, rl

    S, B, T, d, V = 3, 2, 37, 72, 1000
    x, w, tok, mask, g = head_case(S, B, T, d, V, 8)
    adv = torch.randn(S, B, T, generator=g, device=dev())
    if form == "parts of one":
        mask = mask * torch.rand(S, B, T, generator=g, device=dev())
    elif form == "none kept":
        mask[1] = 0
        adv[1] = math.nan
    elif form == "no mask":
        mask = None
    elif form == "per sequence":
        adv = adv[:, :, 0].contiguous()
    l = rl.policy_gradient_loss(rl.Head(x, w), tok, adv, mask.bool() if form == "bool" else mask)
    lp = ops.readout_scored_forward(x, w, tokens=tok, scored=mask).logp.reshape(S, B, T).double()
    k = torch.ones_like(lp) if mask is None else mask.double()
    a = (adv[:, :, None].expand(S, B, T) if adv.dim() == 2 else adv).double()
    n = k.sum((1, 2)).clamp(min=1.0)
    terms = torch.where(k != 0, -lp * a, torch.zeros_like(lp))
    want = terms.sum((1, 2)) / n
    # a term is rounded once, their sum at most once per term where it is kept in f32 (the separate reduction)
    assert ((l.value.double() - want).abs() <= (B * T + 4) * U32 * terms.abs().sum((1, 2)) / n).all()
    r = ops.readout_scored_forward(x, w, tokens=tok, scored=mask)
    g_logp = (torch.where(k != 0, -a, torch.zeros_like(a)) / n[:, None, None]).float().reshape(-1)
    for got, again in zip(l.backward(), l.backward(torch.ones_like(l.value))):
        assert torch.isfinite(got).all()
        # two roundings of the same gradient of the log-probs: at most bf16's step apart after the products
        assert (got.double() - again.double()).norm() <= 4 * U16 * got.double().norm()
    for got, ref in zip(l.backward(), ops.readout_backward(x, w, r, tokens=tok, g_logp=g_logp)):
        assert (got.double() - ref.double()).norm() <= 4 * U16 * ref.double().norm()


@pytest.mark.parametrize("S,n", [(1, 16), (2, 256), (2, 257), (1, 5000), (9, 130), (5000, 1)])
def test_means_of_many_seeds(S, n):
    from noetic_tensor_b200 import ops

    x, w, tok, g = make(S * n, 16, 64, S, "dV")
    keep = (torch.rand(S * n, generator=g, device=dev()) < 0.5).float()
    f = ops.readout_scored_forward(x, w, tokens=tok, scored=keep, ce_seeds=S)
    lp, k = f.logp.double().reshape(S, n), keep.double().reshape(S, n)
    count = k.sum(1).clamp(min=1.0)
    want = (-lp * k).sum(1) / count
    assert ((f.ce_loss.double() - want).abs() <= 2 * U32 * want.abs()).all()  # f32 products summed in f64, one rounding
    assert ((f.ce_g_logp.double().reshape(S, n) + k / count[:, None]).abs() <= 2 * U32 * k).all()
    value, g_logp = ops.ce_mean(f.logp, S, keep)
    assert torch.equal(value, f.ce_loss) and torch.equal(g_logp, f.ce_g_logp)
    for got, want in zip(ops.readout_backward(x, w, f, tokens=tok), ops.readout_backward(x, w, f, tokens=tok, g_logp=g_logp)):
        assert torch.equal(got, want)  # without an upstream: of the loss in `f`


def test_a_run_of_them_together():
    """Decode with the 8-bit head, score the drawn tokens and train on them from an 8-bit checkpoint, on another stream."""
    from noetic_tensor_b200 import ops, rl

    S, B, T, d, V = 2, 3, 17, 264, 4104
    x, w, _, mask, g = head_case(S, B, T, d, V, 3)
    adv = torch.randn(S, B, T, generator=g, device=dev())
    w8 = rl.Int8Weight.of(w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        logits = rl.head_logits(x, w8)
        tokens, lp8 = rl.sample_categorical(logits, 1.0, uniforms=torch.rand(S, B, T, generator=g, device=dev()))
        l = rl.policy_gradient_loss(rl.Head(x, w, checkpoint=True), tokens, adv, mask)
        dh, dw = l.backward()
    s.synchronize()
    exact = x.double() @ w.double()
    # the 8-bit logits: half a step of each row's and each entry's integers
    step_x, step_w = x.double().abs().amax(-1, keepdim=True) / 254, (w.double().abs().amax(0) / 254)
    tol = step_x * w.double().abs().sum(0) + step_w * x.double().abs().sum(-1, keepdim=True) + d * step_x * step_w
    assert ((logits.double() - exact).abs() <= tol * (1 + 1e-5) + 1e-4).all()
    lp = torch.log_softmax(exact, -1).gather(-1, tokens.long()[..., None])[..., 0]
    want = (-(lp * adv) * mask.double()).sum((1, 2)) / mask.double().sum((1, 2))
    assert ((l.value.double() - want).abs() <= 1e-4 * (1 + want.abs())).all()
    q = ops.quantize_rows(x.reshape(-1, d))
    xq = q.values[:, :d].double() * q.scales.double()[:, None]
    up = (-adv * mask / mask.sum((1, 2), keepdim=True)).reshape(-1)
    lse = torch.logsumexp(exact, -1).reshape(-1)
    th, tw, eh, ew = truth(xq, w.t(), tokens.reshape(-1), up, None, None, 1.0, stats=(lse, torch.zeros_like(lse)))
    held(dh.reshape(-1, d), th, eh, "d_hidden")
    held(dw.t(), tw, ew, "d_weights")


def test_the_checkpoint_does_not_keep_the_hidden_states():
    import gc
    import weakref

    from noetic_tensor_b200 import loss, rl

    x, w, tok, mask, _ = head_case(1, 2, 100, 136, 1000, 8)
    held_by = weakref.ref(x)
    l = loss.masked_cross_entropy(rl.Head(x, w, checkpoint=True), tok, mask)
    del x
    gc.collect()
    assert held_by() is None
    dh, dw = l.backward()
    assert dh.shape == (1, 2, 100, 136) and torch.isfinite(dh).all()


def test_captured_and_replayed():
    """Two graphs of whole steps with new inputs copied in, replayed in turn, give the eager results bit for bit."""
    from noetic_tensor_b200 import loss, rl

    cases = [head_case(1, 2, 100, 136, 1000, s) for s in (1, 2, 3)]
    w = cases[0][1]
    eager = []
    for x, _, tok, mask, _ in cases:
        l = loss.masked_cross_entropy(rl.Head(x, w), tok, mask)
        eager.append((l.value.clone(),) + tuple(t.clone() for t in l.backward()))
    x, tok, mask = (t.clone() for t in (cases[0][0], cases[0][2], cases[0][3]))
    w8 = rl.Int8Weight.of(w)
    graphs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            loss.masked_cross_entropy(rl.Head(x, w), tok, mask).backward()
            rl.head_logits(x, w8)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            l = loss.masked_cross_entropy(rl.Head(x, w), tok, mask)
            out = (l.value,) + tuple(l.backward())
            z = rl.head_logits(x, w8)
        graphs.append((g, out, z))
    for k in (1, 0, 2, 1):
        for dst, src in ((x, cases[k][0]), (tok, cases[k][2]), (mask, cases[k][3])):
            dst.copy_(src)
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want_z = rl.head_logits(cases[k][0], w8)
        for _, out, z in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, eager[k])) and torch.equal(z, want_z)


def test_two_streams_at_once():
    from noetic_tensor_b200 import loss, rl

    cases = [head_case(1, 2, 200, 264, 4104, s) for s in (1, 2)]
    want = []
    for x, w, tok, mask, _ in cases:
        l = loss.masked_cross_entropy(rl.Head(x, w), tok, mask)
        want.append((l.value,) + l.backward())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for k, (x, w, tok, mask, _) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                l = loss.masked_cross_entropy(rl.Head(x, w), tok, mask)
                got[k].append((l.value,) + l.backward())
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(p, q) for p, q in zip(r, want[k]))


# ---- masks and tensors at odd addresses, refusals ----------------------------------------------------------


def test_masks_at_odd_addresses():
    from noetic_tensor_b200 import ops

    rows, d, V = 140, 64, 1000
    x, w, tok, g = make(rows, d, V, 17)
    allow = (torch.rand(rows, V, generator=g, device=dev()) < 0.5).to(torch.uint8)
    allow[:, 0] = 1
    big = torch.zeros(rows * V + 8, dtype=torch.uint8, device=dev())
    up = torch.randn(rows, generator=g, device=dev())
    base = None
    for off in (0, 1, 4):
        m = big[off : off + rows * V].view(rows, V)
        m.copy_(allow * 3)  # any byte that is not 0 allows
        f = ops.readout_scored_forward(x, w, tokens=tok, allow=m)
        r = (f.logp,) + ops.readout_backward(x, w, f, tokens=tok, g_logp=up, allow=m)
        if base is None:
            base = r
        assert all(torch.equal(p, q) for p, q in zip(r, base))
    f = ops.readout_scored_forward(x, w, tokens=tok, allow=allow.bool())
    assert torch.equal(f.logp, base[0])


def test_refusals():
    from noetic_tensor_b200 import capi, loss, ops, rl

    x, w, tok, mask, _ = head_case(1, 2, 10, 64, 512, 1)
    f = ops.readout_scored_forward(x, w, tokens=tok)
    up = torch.ones(20, device=dev())
    bad = [
        (ValueError, lambda: rl.Head(x, w, temperature=0.0)),
        (ValueError, lambda: rl.Head(x, w, vocab_mask=torch.zeros(1, 512, device=dev()))),
        (ValueError, lambda: ops.readout_scored_forward(x.float(), w, tokens=tok)),
        (ValueError, lambda: ops.readout_scored_forward(x, w.t().contiguous(), tokens=tok)),
        (ValueError, lambda: ops.readout_scored_forward(x, w.t(), tokens=tok, weights_are_vd=True)),
        (ValueError, lambda: ops.readout_scored_forward(x, w, tokens=tok[:, :1])),
        (ValueError, lambda: ops.readout_scored_forward(x.cpu(), w, tokens=tok)),
        (capi.NrlError, lambda: ops.readout_scored_forward(x[..., :60].contiguous(), w[:60], tokens=tok)),
        (capi.NrlError, lambda: ops.readout_scored_forward(x, w, tokens=tok, temperature=-1.0)),
        (capi.NrlError, lambda: ops.readout_scored_forward(x, w, tokens=tok, ce_seeds=3)),
        (capi.NrlError, lambda: ops.readout_scored_forward(x, w, ce_seeds=1)),
        (capi.NrlError, lambda: ops.readout_scored_forward(x, w, tokens=tok, ce_weights=up)),
        (ValueError, lambda: ops.readout_scored_forward(x, w, tokens=tok, ce_seeds=1, ce_weights=up[:5])),
        (ValueError, lambda: rl.policy_gradient_loss(rl.Head(x, w), tok, up.reshape(1, 2, 10).double(), mask)),
        (capi.NrlError, lambda: ops.readout_scored_forward(x, w, tokens=tok, workspace=torch.empty(256, dtype=torch.uint8, device=dev()))),
        (ValueError, lambda: ops.readout_backward(x, w, f, tokens=tok)),
        (ValueError, lambda: ops.readout_scored_forward(x, w, tokens=tok, workspace=torch.empty(1 << 20, dtype=torch.uint8))),
        (ValueError, lambda: ops.readout_backward(x, w, f, tokens=tok, g_logp=up, workspace=torch.empty(1 << 22, dtype=torch.uint8))),
        (ValueError, lambda: ops.readout_backward(x, w, f, g_logp=up)),
        (ValueError, lambda: ops.readout_backward(x, w, f, g_ent=up)),
        (ValueError, lambda: ops.readout_backward(x, w, ops.readout_scored_forward(x, w, tokens=tok, ce_seeds=1))),
        (ValueError, lambda: ops.readout_backward(x, w, f, tokens=tok, g_logp=up[:5])),
        (TypeError, lambda: ops.readout_backward(x, w, f, tokens=tok, g_logp=up, grad_dtype=torch.float16)),
        (ValueError, lambda: ops.readout_backward(x, w, f, tokens=tok, g_logp=up, add_weights=w.t())),
        (ValueError, lambda: ops.readout_backward(ops.quantize_rows(x[:, :1].contiguous()), w, f, tokens=tok, g_logp=up, hidden_shape=x.shape)),
        (capi.NrlError, lambda: ops.readout_backward(x, w, f, tokens=tok, g_logp=up, workspace=torch.empty(256, dtype=torch.uint8, device=dev()))),
        (ValueError, lambda: rl.categorical_kl(rl.Head(x, w), torch.zeros(1, 2, 10, 512, device=dev()))),
        (ValueError, lambda: loss.cross_entropy_with(rl.Head(x, w), tok, mask, loss.CeOptions(smoothing=0.1))),
        (capi.NrlError, lambda: ops.readout_scored_forward(x[:, :0].contiguous(), w, tokens=tok[:, :0].contiguous())),
        (capi.NrlError, lambda: ops.readout_scored_forward(x[..., :0].contiguous(), w[:0], tokens=tok[:, :0].contiguous())),
        (capi.NrlError, lambda: ops.quantize_rows(x[..., :0].contiguous())),
        (capi.NrlError, lambda: ops.int8_linear(x[:, :0].contiguous(), ops.quantize_weight(w))),
        (ValueError, lambda: ops.Int8Rows(torch.zeros(3, 20, dtype=torch.int8, device=dev()), torch.zeros(3, device=dev()), 20)),
        (ValueError, lambda: ops.int8_matmul(ops.quantize_rows(x[0, 0]), ops.quantize_rows(x[0, 0, :, :32].contiguous()))),
        (TypeError, lambda: ops.quantize_rows(x.half())),
        (ValueError, lambda: ops.quantize_rows(x[..., ::2])),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    assert torch.isfinite(ops.readout_backward(x, w, f, tokens=tok, g_logp=up)[1]).all()  # a refused call leaves nothing behind

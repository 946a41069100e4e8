"""How far the 8-bit checkpoint's gradient is from that of the unrounded states, and the gradient of the rounded ones.

u = 2^-8 is half a step of bf16. With q·s within s / 2 of every element of x, a logit moves by at most e_j = s/2 · Σ_k |w_kj|, and a
probability normalised by the unrounded states by at most π_j·(exp(e_j) − 1). ∂/∂z is rounded to bf16 once, and the result again."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U16, U32 = 2.0**-8, 2.0**-24


def case(strong, rows=200, d=256, V=4104):
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    w = torch.randn(V, d, generator=g, device="cuda") * (3.0 / d**0.5)
    tok = torch.randint(0, V, (rows,), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randn(rows, d, generator=g, device="cuda") + torch.rand(rows, 1, generator=g, device="cuda") * w[tok.long()]
    x[:, 5] *= strong  # a channel far above the others, with a small weight on it
    w[:, 5] /= strong
    return x.bfloat16(), w.t().contiguous().bfloat16(), tok, torch.randn(rows, generator=g, device="cuda") / rows


def close(got, want, tol):
    # the result's rounding, and f32 sums of as many terms as there are
    assert ((got.double() - want).abs() <= tol * (1 + 2e-3) + 2 * U16 * want.abs() + 1e-9).all(), ((got.double() - want).abs() / (tol + 2 * U16 * want.abs() + 1e-9)).max()


@pytest.mark.parametrize("strong", [1.0, 30.0])
def test_against_the_unrounded_states(strong):
    from noetic_tensor_b200 import loss, ops, rl

    x, w, tok, _ = case(strong)
    rows, d = x.shape
    l = loss.cross_entropy(rl.Head(x.reshape(1, 1, rows, d), w, checkpoint=True), tok.reshape(1, 1, rows))
    plain = loss.cross_entropy(rl.Head(x.reshape(1, 1, rows, d), w), tok.reshape(1, 1, rows))
    assert torch.equal(l.value, plain.value)  # the value is that of the unrounded states
    dh, dw = l.backward()
    X, W = x.double(), w.double()
    pi = torch.softmax(X @ W, 1)
    hot = torch.nn.functional.one_hot(tok.long(), W.shape[1]).double()
    dz = (pi - hot) / rows
    half = ops.quantize_rows(x).scales.double()[:, None] / 2 * (1 + 2 * U32)
    e = torch.expm1(half * W.abs().sum(0)) * pi / rows  # of ∂/∂z
    D = (pi + hot) / rows + e
    t = e + U16 * 1.01 * D
    close(dh.reshape(rows, d), dz @ W.t(), t @ W.abs().t())
    close(dw, X.t() @ dz, X.abs().t() @ t + (half.expand_as(X)).t() @ D)


@pytest.mark.parametrize("strong", [1.0, 30.0, 100.0])
@pytest.mark.parametrize("what", ["ce", "policy", "entropy"])
def test_a_loss_of_the_rounded_states(strong, what):
    """Value and gradient are those of one function, the loss of q·s."""
    from noetic_tensor_b200 import loss, ops, rl

    x, w, tok, adv = case(strong)
    rows, d = x.shape
    q = ops.quantize_rows(x)
    rounded = ops.dequantize_rows(q)
    again = ops.quantize_rows(rounded)
    assert torch.equal(again.values, q.values) and torch.equal(again.scales, q.scales)
    head, tk = rl.Head(rounded.reshape(1, 1, rows, d), w, checkpoint=True), tok.reshape(1, 1, rows)
    if what == "ce":
        l, a, b = loss.cross_entropy(head, tk), torch.full((rows, 1), -1.0 / rows, device="cuda", dtype=torch.float64), 0.0
    elif what == "policy":
        l, a, b = rl.policy_gradient_loss(head, tk, adv.reshape(1, 1, rows)), -adv.double()[:, None] / rows, 0.0
    else:
        l, a, b = rl.categorical_entropy(head), 0.0, 1.0 / rows
    a = a if torch.is_tensor(a) else torch.zeros(rows, 1, device="cuda", dtype=torch.float64)
    dh, dw = l.backward()
    W = w.double()
    X = q.values[:, :d].double() * q.scales.double()[:, None]
    lp = torch.log_softmax(X @ W, 1)
    pi = lp.exp()
    H = -(pi * lp).sum(1, keepdim=True)
    hot = torch.nn.functional.one_hot(tok.long(), W.shape[1]).double()
    value = (a * (lp * hot).sum(1, keepdim=True)).sum() + (b * H).sum()
    dz = a * (hot - pi) - b * pi * (lp + H)
    # the states that the forward saw are bf16: what that moves a logit, ln Z, ln π and H by
    seen = (rounded.double() - X).abs() @ W.abs()
    e = seen + seen.amax(1, keepdim=True)
    de = torch.expm1(e) * pi * (a.abs() + b * (lp.abs() + H + e)) + b * pi * (1 + H) * 2 * e.amax(1, keepdim=True) * (1 + lp.abs().amax(1, keepdim=True))
    D = a.abs() * (hot + pi) + b * pi * (lp.abs() + H + 1.0) + de
    t = de + U16 * 1.01 * D
    close(dh.reshape(rows, d), dz @ W.t(), t @ W.abs().t())
    close(dw, X.t() @ dz, X.abs().t() @ t)
    moved = (a.abs()[:, 0] * e.amax(1)).sum() + (b * 2 * e.amax(1) * (1 + lp.abs().amax(1))).sum()
    assert abs(l.value.item() - value.item()) <= moved + 1e-4 * (1 + abs(value.item()))

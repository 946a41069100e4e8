"""Cases of the operators around the readout (`logits = hidden · W`), for timing and comparison.

Three operators, each in a plain form (elementary torch operations in 32 bits) and, where `own` is
true, through the package's public calls:

  cross_entropy / policy   a token loss on head(hidden) over a large vocabulary with its gradient to
                           the hidden states and to the weight, the logits never kept
  checkpoint               the same step when the hidden states live between forward and backward as
                           8-bit integers with a scale per token
  int8                     the head's product in 8-bit integers: hidden states quantised per token,
                           the weight laid out once as integers with a scale per vocabulary entry

Shapes follow the package: hidden [S, B, T, d], weight [d, V] (a Linear's [in, out]) or [V, d].
"""
import math

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # a single short sequence through a small head: nothing but launches and host work
        dict(name="ce_one_short_sequence", op="cross_entropy", S=1, B=1, T=16, V=1000, d=64, vd=False, scored=1.0),
        # one ordinary training micro-batch, prompt tokens unscored
        dict(name="ce_micro_batch", op="cross_entropy", S=1, B=4, T=512, V=32000, d=2048, vd=False, scored=0.75),
        # the benchmark's vocabulary and width, several seeds in one batch
        dict(name="ce_large", op="cross_entropy", S=4, B=4, T=512, V=128256, d=4096, vd=False, scored=1.0),
        # a policy-gradient step on a grammar-masked, tempered rollout; ragged everything, weight as [V, d]
        dict(name="policy_masked_ragged", op="policy", S=2, B=7, T=93, V=50264, d=1544, vd=True, scored=0.8, tau=0.7, allowed=0.3),
        # the vocabulary of the long-sequence configuration, few rows: the gradient of W is most of the traffic
        dict(name="policy_few_rows", op="policy", S=1, B=3, T=29, V=151936, d=2048, vd=True, scored=1.0, tau=1.0, allowed=1.0),
        # an 8-bit checkpoint for a small model's head
        dict(name="checkpoint_small", op="checkpoint", S=1, B=3, T=67, V=4104, d=512, vd=False, scored=0.9),
        # an 8-bit checkpoint for a full batch
        dict(name="checkpoint_batch", op="checkpoint", S=2, B=4, T=512, V=32000, d=4096, vd=False, scored=0.75),
        # a decode step for one token: the weight's bytes are the cost
        dict(name="int8_one_token", op="int8", rows=1, V=128256, d=4096, hidden="bf16", out="bf16"),
        # a decode step of a running batch, f32 logits for the sampler
        dict(name="int8_decode_batch", op="int8", rows=48, V=151936, d=2048, hidden="bf16", out="f32"),
        # scoring a short odd batch with an odd vocabulary, hidden states in f32
        dict(name="int8_ragged", op="int8", rows=333, V=50257, d=1000, hidden="f32", out="f32"),
        # scoring a whole batch
        dict(name="int8_score_batch", op="int8", rows=8192, V=32000, d=4096, hidden="bf16", out="bf16"),
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    op = rng.choice(["cross_entropy", "policy", "checkpoint", "int8"])
    if op == "int8":
        while True:
            c = dict(op=op, rows=_log_int(rng, 1, 8192), V=_log_int(rng, 500, 160000), d=_log_int(rng, 64, 4096, 8), hidden=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]))
            if c["rows"] * c["V"] <= 8192 * 32000 and c["rows"] * c["V"] * c["d"] <= 8192 * 32000 * 4096:
                return c
    while True:
        c = dict(op=op, S=rng.choice([1, 2, 3, 4]), B=_log_int(rng, 1, 16), T=_log_int(rng, 1, 700), V=_log_int(rng, 504, 160000, 8), d=_log_int(rng, 64, 4096, 8),
                 vd=rng.random() < 0.5, scored=rng.choice([1.0, round(rng.uniform(0.3, 1.0), 2)]))
        if op == "policy":
            c["tau"], c["allowed"] = rng.choice([1.0, 0.7, 1.5]), rng.choice([1.0, round(rng.uniform(0.05, 0.9), 2)])
        if c["S"] * c["B"] * c["T"] <= 8192 and c["S"] * c["B"] * c["T"] * c["V"] * c["d"] <= 8192 * 128256 * 4096:
            return c


def _rows(case):
    return case["rows"] if case["op"] == "int8" else case["S"] * case["B"] * case["T"]


def _scored(case):
    return max(1, int(case["scored"] * _rows(case)))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    N, V, d = _rows(case), case["V"], case["d"]
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    s = dict(case)
    if case["op"] == "int8":
        # normalised hidden states with a few strong channels, as a final norm's gain leaves them
        x = randn(N, d) * torch.exp(0.5 * randn(d))
        s["hidden"] = x.bfloat16() if case["hidden"] == "bf16" else x
        # the head as a server keeps it: integers [V, d rounded up to 16] with zeros behind d, one scale per vocabulary entry
        w = torch.empty(V, -(-d // 16) * 16, dtype=torch.int8, device=DEV).zero_()
        w[:, :d] = torch.randint(-127, 128, (V, d), generator=g, device=DEV, dtype=torch.int8)
        s["w_values"], s["w_scales"] = w, torch.exp(0.3 * randn(V)) * (3.0 / 73.0 / d**0.5)
        return s
    W = (randn(V, d) * (3.0 / d**0.5)).bfloat16()
    tok = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    # the token's own direction in the hidden state: log-probabilities from near 0 down to far below the mode
    h = randn(N, d) + torch.rand(N, 1, generator=g, device=DEV) * 1.5 * W[tok.long()].float()
    lead = (case["S"], case["B"], case["T"])
    s["hidden"] = h.bfloat16().reshape(*lead, d)
    if case["op"] == "policy" and case["allowed"] < 1.0:
        allow = (torch.rand(N, V, generator=g, device=DEV) < case["allowed"]).to(torch.uint8)
        allow[torch.arange(N, device=DEV), tok.long()] = 1
        s["allow"] = allow
    else:
        s["allow"] = None
    s["weight"] = W if case["vd"] else W.t().contiguous()
    s["tokens"] = tok.reshape(lead)
    mask = torch.zeros(N, device=DEV)
    mask[torch.randperm(N, generator=g, device=DEV)[: _scored(case)]] = 1.0
    s["mask"] = mask.reshape(lead)
    s["advantages"] = randn(*lead)
    return s


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "int8":
        return _plain_int8(s)
    return _plain_head(s)


# ---- the package's calls ------------------------------------------------------------------------


def _run_own(s):
    from noetic_tensor_b200 import loss, rl

    if s["op"] == "int8":
        return rl.head_logits(s["hidden"], rl.Int8Weight(s["w_values"], s["w_scales"], s["d"]), dtype=torch.bfloat16 if s["out"] == "bf16" else torch.float32)
    head = rl.Head(s["hidden"], s["weight"], temperature=s.get("tau", 1.0), vocab_mask=s["allow"], weight_is_vd=s["vd"], checkpoint=s["op"] == "checkpoint")
    if s["op"] == "policy":
        value = rl.policy_gradient_loss(head, s["tokens"], s["advantages"], s["mask"], rl.TOKEN_MEAN)
    else:
        value = loss.masked_cross_entropy(head, s["tokens"], s["mask"])
    d_hidden, d_weight = value.backward()
    return {"loss": value.value, "d_hidden": d_hidden, "d_weight": d_weight}


# ---- the plain forms ------------------------------------------------------------------------------


def _quantise(x):
    """Integers in [-127, 127] (as f32) and the f32 scale of each row: q = rint(127 x / max |x|), x ≈ q · (max |x| / 127)."""
    x = x.float()
    big = x.abs().amax(1, keepdim=True)
    q = torch.where(big > 0, torch.round(x * 127.0 / big), torch.zeros_like(x))
    return q, big / 127.0


def _plain_int8(s):
    q, scale = _quantise(s["hidden"])
    z = q @ s["w_values"][:, : s["d"]].float().t()
    z = z * scale * s["w_scales"]
    return z.bfloat16() if s["out"] == "bf16" else z


def _plain_head(s):
    S, N, V, d = s["S"], _rows(s), s["V"], s["d"]
    h = s["hidden"].reshape(N, d).float()
    W = s["weight"].float()  # [d, V], or [V, d]
    Wdv, Wvd = (W.t(), W) if s["vd"] else (W, W.t())
    tok, mask, tau = s["tokens"].reshape(N).long(), s["mask"].reshape(N), s.get("tau", 1.0)
    at = torch.arange(N, device=h.device)

    def tempered(x):
        z = x @ Wdv
        z = z / tau if tau != 1.0 else z
        return z if s["allow"] is None else z.masked_fill(s["allow"] == 0, -math.inf)

    z = tempered(h)
    top = z.amax(1, keepdim=True)
    lnZ = torch.log(torch.exp(z - top).sum(1, keepdim=True))
    logp = z[at, tok] - top[:, 0] - lnZ[:, 0]
    weight = s["advantages"].reshape(N) if s["op"] == "policy" else torch.ones_like(mask)
    count = mask.reshape(S, -1).sum(1).clamp(min=1.0)
    value = (-(logp * weight) * mask).reshape(S, -1).sum(1) / count
    if s["op"] == "checkpoint":  # the backward has the checkpoint and the forward's row statistics
        q, scale = _quantise(h)
        h = q * scale
        z = tempered(h)
    g = torch.exp(z - top - lnZ)
    del z
    g[at, tok] -= 1.0
    g *= (weight * mask / count.repeat_interleave(N // S) / tau)[:, None]
    d_hidden = (g @ Wvd).bfloat16().reshape(s["hidden"].shape)
    d_weight = (g.t() @ h if s["vd"] else h.t() @ g).bfloat16()
    return {"loss": value, "d_hidden": d_hidden, "d_weight": d_weight}


def work(case):
    N, V, d = _rows(case), case["V"], case["d"]
    if case["op"] == "int8":
        return {"bytes": N * d * (2 if case["hidden"] == "bf16" else 4) + V * d + 4 * V + N * V * (2 if case["out"] == "bf16" else 4), "flops": 2.0 * N * V * d}
    n = _scored(case)
    # hidden states and weight once in, their gradients once out; the products of the scored rows: logits, d_hidden, d_weight
    rows = 2 * n * d + 2 * N * d + 12 * N
    if case["op"] == "checkpoint":
        rows += 2 * n * d  # the checkpoint, written and read
    if case.get("allowed", 1.0) < 1.0:
        rows += n * V
    return {"bytes": rows + 4 * V * d, "flops": 6.0 * n * V * d}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int8":
        x = s["hidden"].double()
        out = torch.empty(case["rows"], case["V"], dtype=torch.float64, device=DEV)
        w = s["w_values"][:, : case["d"]].double().mul_(s["w_scales"].double()[:, None])
        for r in range(0, case["rows"], 1024):
            xr = x[r : r + 1024]
            big = xr.abs().max(dim=1, keepdim=True).values
            scale = (big / 127.0).float().double()  # scales are held in 32 bits
            out[r : r + 1024] = (torch.round(127.0 * xr / big.clamp(min=1e-300)) * scale) @ w.t()
        return out
    N, V, d, S = _rows(case), case["V"], case["d"], case["S"]
    tau = case.get("tau", 1.0)
    h = s["hidden"].reshape(N, d).double()
    W = (s["weight"].t() if case["vd"] else s["weight"]).double()  # [d, V]
    mask = s["mask"].reshape(N).double()
    per_seed = mask.reshape(S, N // S).sum(1).clamp(min=1.0)
    coef = mask / per_seed[:, None].expand(S, N // S).reshape(N)
    if case["op"] == "policy":
        coef = coef * s["advantages"].reshape(N).double()
    d_h, d_W = torch.empty_like(h), torch.zeros_like(W)
    nll = torch.empty(N, dtype=torch.float64, device=DEV)
    for r in range(0, N, 1024):
        part = slice(r, min(N, r + 1024))
        t = s["tokens"].reshape(N)[part].long()[:, None]
        c = coef[part, None]

        def logits(x):
            z = (x @ W) / tau
            return z if s["allow"] is None else torch.where(s["allow"][part].bool(), z, torch.full_like(z, -math.inf))

        x = h[part]
        z = logits(x)
        lse = torch.logsumexp(z, dim=1, keepdim=True)
        nll[part] = (lse - z.gather(1, t))[:, 0]
        if case["op"] == "checkpoint":
            big = x.abs().max(dim=1, keepdim=True).values
            x = torch.round(127.0 * x / big.clamp(min=1e-300)) * (big / 127.0).float().double()
            z = logits(x)
        p = z.sub_(lse).exp_()
        p.scatter_add_(1, t, torch.full_like(t, -1, dtype=torch.float64))
        p.mul_(c / tau)
        d_h[part] = p @ W.t()
        d_W.addmm_(x.t(), p)
    value = (nll * coef).reshape(S, N // S).sum(1)
    return {"loss": value, "d_hidden": d_h.reshape(s["hidden"].shape), "d_weight": d_W.t() if case["vd"] else d_W}

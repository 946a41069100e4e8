"""`nn::rl` over the fused kernels: the reference's function names and argument meanings
(src/nn/rl.rs), for logits that live on a CUDA device.

Each loss returns a `Loss`: `.value` is the reduced tensor the reference function returns and
`.backward(upstream)` gives d(logits) [S,B,T,V] f32 for sum(value · upstream), what the tape's
`(value * upstream).sum().backward()` yields in the reference. Where the reference builds ~40
tape nodes per PPO step, this path has one forward and one backward pass over the logits.

Masks: `mask` is the scoring mask [S,B,T] of 0/1 floats (src/nn/rl.rs:9-14; other types, bool among them,
are converted); `vocab_mask` is
either a float additive mask broadcastable as [1,V] or [rows,V] (the reference's form,
src/nn/rl.rs:471-486) or a uint8/bool allow-mask of the same shapes.
"""
import os

import torch

from . import capi, ops

NONE, SUM, TOKEN_MEAN, PER_SEQUENCE, SEQUENCE_MEAN = range(5)
K1, K2, K3 = capi.LOSS_K1, capi.LOSS_K2, capi.LOSS_K3
LOG_RATIO_CLAMP = 20.0  # src/nn/rl.rs:146
KL_DELTA_CLAMP = 20.0  # src/nn/rl.rs:150


# The reference's losses check their scored log-probabilities in debug builds only
# (`debug_check`, src/nn/rl.rs:213-221: a host read). Here the switch is this flag, set from the
# environment variable NOETIC_RL_DEBUG (any value but "" and "0") when the module is imported.
DEBUG_CHECKS = os.environ.get("NOETIC_RL_DEBUG", "0") not in ("", "0")


def check_scored_finite(what, logp, mask=None):
    """`check_scored_finite` (src/nn/rl.rs:204-211): None, or the error text naming the first scored
    position whose log-probability is not finite."""
    return ops.check_scored_finite(what, logp.contiguous(), None if mask is None else mask.contiguous())


def debug_check(what, logp, mask=None):
    """`debug_check` (src/nn/rl.rs:213-221): raises the check's message when DEBUG_CHECKS is on."""
    if DEBUG_CHECKS:
        e = check_scored_finite(what, logp, mask)
        if e is not None:
            raise RuntimeError(e)


class Clip:
    """`Clip` (src/nn/rl.rs:160-198)."""

    def __init__(self, low, high, dual=None, log_ratio_clamp=LOG_RATIO_CLAMP):
        self.low, self.high, self.dual, self.log_ratio_clamp = low, high, dual, log_ratio_clamp

    @staticmethod
    def symmetric(eps):
        return Clip(eps, eps)

    def with_dual(self, c):
        return Clip(self.low, self.high, c, self.log_ratio_clamp)

    def with_log_ratio_clamp(self, b):
        return Clip(self.low, self.high, self.dual, b)


class Tempered:
    """`tempered_logits(logits, temperature, mask)` (src/nn/rl.rs:475-486) without materialising
    it: the kernels apply the temperature and the mask as they stream the row."""

    def __init__(self, logits, temperature=1.0, vocab_mask=None):
        if not (temperature > 0.0):
            raise ValueError(f"tempered_logits: temperature {temperature} (must be positive)")
        self.logits = logits
        self.shape = tuple(logits.shape)
        self.V = logits.shape[-1]
        self.flat = logits.reshape(-1, self.V)
        self.temperature = float(temperature)
        self.allow = self.add = None
        if vocab_mask is not None:
            if vocab_mask.shape[-1] != self.V:
                raise ValueError("tempered_logits: mask does not broadcast to the logits")
            m = vocab_mask.reshape(-1, self.V)
            if m.dtype in (torch.uint8, torch.bool):
                self.allow = m.contiguous()
            else:
                self.add = m.to(torch.float32).contiguous()

    def kw(self):
        return dict(allow=self.allow, add_mask=self.add, temperature=self.temperature)


class Head:
    """`Decoder::head(hidden)` (src/nn/decoder.rs:270-279) in place of logits, without computing them:
    every function here and in `loss` that takes logits [S, B, T, V] and returns a `Loss` takes a Head,
    runs the fused readout instead (the logits are never kept, forward or backward), and its
    `.backward(upstream)` returns the pair (d_hidden [S, B, T, d], d_weight in the weight's layout).

    `hidden` bf16 [S, B, T, d]; `weight` bf16 [d, V] (the Linear's [in, out] layout) or, with
    `weight_is_vd`, [V, d]; d and V multiples of 8. `temperature` and `vocab_mask` make the logits the
    tempered ones (src/nn/rl.rs:475-486); the mask is a uint8/bool allow-mask [..., V] or [1, V], or int32
    words of one bit per token. With `checkpoint` a loss keeps the hidden states for its backward as 8-bit
    integers with a scale per position (half the memory) instead of keeping `hidden`. `grad_dtype`:
    bfloat16 or float32 (d(logits) is rounded to bf16 on the way to either).

    The checkpoint's gradient takes the logits of the rounded states and the normaliser of the unrounded ones, those of
    the loss's value, so its probabilities add up to 1 only as far as the rounding leaves the logits alone. Hidden
    states of about one size: 1 % of the gradient's norm. With a channel far above the others the integers hold
    the others badly, and the gradient is off by several times what the rounding itself costs (d 2048, a channel 100
    times the others with a weight as much smaller: 67 % against 14 %). Give the loss the rounded states then, and value and gradient are those of one function:

        rounded = ops.dequantize_rows(ops.quantize_rows(hidden)).reshape(hidden.shape)
        Head(rounded, weight, checkpoint=True)  # its integers are the first ones; d_hidden is taken as that of `hidden`

    Positions that a loss's `mask` leaves out are not read and cost nothing: their d_hidden is 0 whatever
    they hold. Nothing is read back to the host: a token outside the vocabulary makes its log-prob, and with
    it the loss, NaN, as does a position with no allowed token."""

    def __init__(self, hidden, weight, temperature=1.0, vocab_mask=None, weight_is_vd=False, checkpoint=False, grad_dtype=torch.bfloat16):
        if not (0.0 < ops.nearest_f32(temperature) < float("inf")):
            raise ValueError(f"tempered_logits: temperature {temperature} (must be positive, in 32 bits too)")
        if vocab_mask is not None and vocab_mask.dtype not in (torch.uint8, torch.bool, torch.int32):
            raise ValueError("Head: vocab_mask is a uint8/bool allow-mask or int32 words of bits")
        self.V = weight.shape[0 if weight_is_vd else 1]
        self.shape = hidden.shape[:-1] + (self.V,)
        self.hidden, self.weight = hidden.contiguous(), weight
        allow, bits = _vocab_mask_args(vocab_mask, self.V)
        self.kw = dict(weights_are_vd=weight_is_vd, allow=allow, allow_bits=bits, temperature=float(temperature))
        self.checkpoint, self.grad_dtype = checkpoint, grad_dtype

    def run(self, tokens=None, scored=None, want_entropy=False, ce_seeds=0, ce_weights=None):
        return _HeadRun(self, tokens, scored, want_entropy, ce_seeds, ce_weights)


def _as(t, dtype):
    """`t` as a contiguous tensor of `dtype`: itself where it is one."""
    return t if t is None or (t.dtype is dtype and t.is_contiguous()) else t.to(dtype).contiguous()


def _token_ids(tokens, V):
    """Tokens as contiguous int32. An id of 64 bits outside the vocabulary stays outside: its lower 32 bits may be a token."""
    if tokens is not None and tokens.dtype is torch.int64:
        tokens = tokens.clamp(-1, V)
    return _as(tokens, torch.int32)


class _HeadRun:
    """A forward of a Head and what its backward needs (not the hidden states when they are checkpointed)."""

    def __init__(self, head, tokens, scored, want_entropy, ce_seeds, ce_weights):
        self.tokens, self.weight, self.kw, self.grad_dtype, self.shape = _token_ids(tokens, head.V), head.weight, head.kw, head.grad_dtype, head.hidden.shape
        self.fwd = ops.readout_scored_forward(head.hidden, head.weight, tokens=self.tokens, scored=_as(scored, torch.float32), want_entropy=want_entropy, ce_seeds=ce_seeds, ce_weights=ce_weights,
                                              **head.kw)
        self.saved = ops.quantize_rows(head.hidden) if head.checkpoint else head.hidden

    def backward_of_loss(self):
        return ops.readout_backward_of_loss(self.fwd, self.saved, self.weight, self.tokens, grad_dtype=self.grad_dtype, hidden_shape=self.shape, **self.kw)

    def backward(self, g_logp=None, g_ent=None):
        return ops.readout_backward(self.saved, self.weight, self.fwd, tokens=self.tokens, g_logp=_as(g_logp, torch.float32), g_ent=_as(g_ent, torch.float32), grad_dtype=self.grad_dtype,
                                    hidden_shape=self.shape, **self.kw)


class Int8Weight(ops.Int8Rows):
    """A readout weight laid out once as 8-bit integers [V, pitch] with a scale per vocabulary entry
    (pitch: d rounded up to a multiple of 16). `Int8Weight.of(weight)` makes it from bf16 [d, V], or
    [V, d] with `weight_is_vd`."""

    __slots__ = ()

    @staticmethod
    def of(weight, weight_is_vd=False):
        q = ops.quantize_weight(weight, weight_is_vd)
        return Int8Weight(q.values, q.scales, q.d)


def head_logits(hidden, weight, dtype=torch.float32):
    """`head(x)` (src/nn/decoder.rs:270-279) in 8-bit integers: `hidden` [..., d] (bf16 or f32) is
    quantised with a scale per position, `weight` is an Int8Weight; logits [..., V] of `dtype` (float32 or
    bfloat16), ready for `sample_categorical` and the other functions here that take logits."""
    return ops.int8_linear(hidden.contiguous(), weight, dtype)


def _tempered(x):
    return x if isinstance(x, (Tempered, Head)) else Tempered(x)


class Loss:
    def __init__(self, value, backward, unit=None):
        self.value = value
        self._backward = backward
        self._unit = unit  # the backward for an upstream of ones, where the forward has left its gradient already

    def backward(self, upstream=None):
        if upstream is None and self._unit is not None:
            return self._unit()
        if upstream is None:
            upstream = torch.ones_like(self.value)
        return self._backward(upstream.to(torch.float32).contiguous())


def sample_categorical(logits, temperature=1.0, vocab_mask=None, uniforms=None):
    """Tokens [...] (int32) from softmax(logits/τ + mask): inverse CDF against `uniforms` (one per
    position); τ = 0 is the first maximum. Refuses a position with no allowed token or a NaN with
    the reference's message (src/nn/rl.rs:516-519). Returns (tokens, log-probs of the tokens)."""
    if temperature < 0:
        raise ValueError(f"sample_categorical: temperature {temperature} (must be ≥ 0)")
    z = Tempered(logits, 1.0 if temperature == 0.0 else temperature, vocab_mask)
    lead = z.shape[:-1]
    if temperature == 0.0:
        f = ops.row_forward(z.flat, greedy=True, want_entropy=False, **z.kw())
    else:
        f = ops.row_forward(z.flat, uniforms=uniforms.reshape(-1).contiguous(), want_entropy=False, **z.kw())
    ops.check_status(f.status)
    return f.tokens.reshape(lead), f.logp.reshape(lead)


class ChaChaStream:
    """The position of a `ChaCha20Rng` (src/rng.rs:10-17 derives its 32-byte seed): the seed and
    the number of 32-bit words drawn so far. `sample_categorical_reference` advances it as the
    reference's sampler advances its generator."""

    def __init__(self, seed, words=0):
        if len(seed) != 32:
            raise ValueError("seed: 32 bytes")
        self.seed, self.words = bytes(seed), int(words)


def sample_categorical_reference(logits, temperature, vocab_mask, rng):
    """`sample_categorical(logits, temperature, mask, rng)` with the reference's own noise
    (src/nn/rl.rs:510-529): Gumbel-max, one `next_u64` of `rng` per logit in row-major order, so the
    tokens are the reference's for the same generator state. Temperature 0 is the first maximum
    and draws nothing. Refuses a position with no allowed token before drawing, as the reference
    does. Returns tokens [...] (int32)."""
    if temperature < 0:
        raise ValueError(f"sample_categorical: temperature {temperature} (must be ≥ 0)")
    z = Tempered(logits, 1.0 if temperature == 0.0 else temperature, vocab_mask)
    lead = z.shape[:-1]
    if temperature == 0.0:
        f = ops.row_forward(z.flat, greedy=True, want_entropy=False, want_logp=False, **z.kw())
        ops.check_status(f.status)
        return f.tokens.reshape(lead)
    tokens, status = ops.sample_gumbel(z.flat, rng.seed, word_offset=rng.words, **z.kw())
    ops.check_status(status)
    rng.words += 2 * z.flat.shape[0] * z.V
    return tokens.reshape(lead)


class _TokenLogProbs:
    """token_log_probs (src/nn/rl.rs:134-141) and its backward to the logits."""

    def __init__(self, logits, tokens, mask=None):
        self.z = _tempered(logits)
        self.lead = self.z.shape[:-1]
        if isinstance(self.z, Head):
            self.run, self.z = self.z.run(tokens, mask), None
            self.logp = self.run.fwd.logp.reshape(self.lead)
            return
        self.fwd = ops.row_forward(self.z.flat, tokens=_token_ids(tokens.reshape(-1), self.z.V), want_entropy=False, **self.z.kw())
        self.logp = self.fwd.logp.reshape(self.lead)

    def grad_logits(self, g_logp):
        """d(logits), or (d_hidden, d_weight) of a Head."""
        if self.z is None:
            return self.run.backward(g_logp=g_logp)
        d = ops.row_backward(self.z.flat, self.fwd, g_logp=g_logp.reshape(-1).contiguous(), **self.z.kw())
        return d.reshape(self.z.shape)


def token_log_probs(logits, tokens, mask=None):
    mask = _as(mask, torch.float32)
    t = _TokenLogProbs(logits, tokens, mask)
    value = t.logp if mask is None else ops.mask_rows(t.logp, mask)

    def backward(up):
        g = up if mask is None else ops.mask_rows(up, mask)
        return t.grad_logits(g)

    return Loss(value, backward)


_CHECK_NAMES = {
    capi.LOSS_PG: ("policy_gradient_loss", None),
    capi.LOSS_PPO: ("clipped_policy_loss", "clipped_policy_loss (old log-probabilities)"),
    capi.LOSS_K1: ("kl_estimate", "kl_estimate (reference log-probabilities)"),
    capi.LOSS_K2: ("kl_estimate", "kl_estimate (reference log-probabilities)"),
    capi.LOSS_K3: ("kl_estimate", "kl_estimate (reference log-probabilities)"),
}


def _token_level(kind, logits, tokens, mask, reduction, **kw):
    lead, mask = logits.shape[:-1], _as(mask, torch.float32)
    if len(lead) != 3:
        raise ValueError("logp must be [S, B, T]")
    if isinstance(logits, Head) and kind == capi.LOSS_PG and reduction == TOKEN_MEAN and kw["weights"].shape == lead and (mask is None or mask.shape == lead):
        return _head_policy_gradient(logits, tokens, mask, kw["weights"])
    t = _TokenLogProbs(logits, tokens, mask)
    lp = t.logp
    # the checks of src/nn/rl.rs:230, 268-269, 386-387
    what, what_other = _CHECK_NAMES[kind]
    debug_check(what, lp, mask)
    if what_other is not None:
        debug_check(what_other, kw["other"], mask)
    if t.z is None and reduction in (SUM, TOKEN_MEAN, SEQUENCE_MEAN):
        o = ops.token_objective(kind, lp, reduction, mask=mask, **kw)  # the value and its gradient in one launch
        return Loss(o.policy, lambda up: t.grad_logits(ops.token_objective(kind, lp, reduction, mask=mask, up_policy=up, **kw).g_logp), lambda: t.grad_logits(o.g_logp))
    per, _ = ops.token_loss(kind, lp, mask=mask, want_grad=False, **kw)
    value = ops.reduce_tokens(per, mask, reduction)

    def backward(up):
        d_per = ops.reduce_tokens_backward(tuple(lp.shape), mask, reduction, up)
        _, g_logp = ops.token_loss(kind, lp, mask=mask, upstream=d_per, **kw)
        return t.grad_logits(g_logp)

    return Loss(value, backward)


def _head_policy_gradient(head, tokens, mask, weights):
    """A Head's token-mean policy gradient comes out of the forward call itself, value and gradient."""
    lead = head.shape[:-1]
    run = head.run(tokens, mask, ce_seeds=lead[0], ce_weights=weights)
    if DEBUG_CHECKS:
        debug_check("policy_gradient_loss", run.fwd.logp.reshape(lead), mask)

    def backward(up):
        o = ops.token_objective(capi.LOSS_PG, run.fwd.logp.reshape(lead), TOKEN_MEAN, mask=mask, up_policy=up, weights=weights)
        return run.backward(g_logp=o.g_logp)

    return Loss(run.fwd.ce_loss, backward, run.backward_of_loss)


def policy_gradient_loss(logits, tokens, weights, mask=None, reduction=TOKEN_MEAN):
    """policy_gradient_loss(token_log_probs(logits, tokens), weights, mask, reduction), src/nn/rl.rs:228-235."""
    return _token_level(capi.LOSS_PG, logits, tokens, mask, reduction, weights=weights)


def clipped_policy_loss(logits, tokens, old_logp, advantages, mask=None, clip=None, reduction=TOKEN_MEAN):
    """clipped_policy_loss (src/nn/rl.rs:265-287) of the tokens' log-probabilities."""
    clip = clip or Clip.symmetric(0.2)
    return _token_level(capi.LOSS_PPO, logits, tokens, mask, reduction, other=old_logp, weights=advantages, clip_low=clip.low, clip_high=clip.high,
                        dual=clip.dual, clamp=clip.log_ratio_clamp)


def kl_estimate(logits, tokens, ref_logp, estimator, delta_clamp=None, mask=None, reduction=TOKEN_MEAN):
    """kl_estimate (src/nn/rl.rs:380-400) of the tokens' log-probabilities."""
    return _token_level(estimator, logits, tokens, mask, reduction, other=ref_logp, clamp=delta_clamp)


def clip_fraction(logp, old_logp, advantages, mask=None, clip=None):
    """clip_fraction (src/nn/rl.rs:293-317), untracked."""
    clip = clip or Clip.symmetric(0.2)
    return ops.clip_fraction(logp, old_logp, advantages, mask=mask, clip_low=clip.low, clip_high=clip.high, dual=clip.dual, clamp=clip.log_ratio_clamp)


def _row_level(which, logits, ref_logits, mask, reduction):
    z = _tempered(logits)
    if len(z.shape) != 4:
        raise ValueError("logits [S, B, T, V]")
    lead, mask = z.shape[:-1], _as(mask, torch.float32)
    if isinstance(z, Head):
        if which != "entropy":
            raise ValueError("the exact KL to a reference needs both sides' logits: a Head has none (kl_estimate takes one)")
        run = z.run(scored=mask, want_entropy=True)
        per = run.fwd.entropy.reshape(lead) if mask is None else ops.mask_rows(run.fwd.entropy.reshape(lead), mask)
        return Loss(ops.reduce_tokens(per, mask, reduction), lambda up: run.backward(g_ent=ops.reduce_tokens_backward(lead, mask, reduction, up)))
    ref = None if ref_logits is None else ref_logits.reshape(-1, z.V)
    f = ops.row_forward(z.flat, ref_logits=ref, want_entropy=(which == "entropy"), want_kl=(which == "kl"), want_ref_logp=False, **z.kw())
    raw = (f.kl if which == "kl" else f.entropy).reshape(lead)
    per = raw if mask is None else ops.mask_rows(raw, mask)
    value = ops.reduce_tokens(per, mask, reduction)

    def backward(up):
        d_per = ops.reduce_tokens_backward(lead, mask, reduction, up).reshape(-1)
        kw = dict(g_kl=d_per) if which == "kl" else dict(g_ent=d_per)
        return ops.row_backward(z.flat, f, ref_logits=ref, **kw, **z.kw()).reshape(z.shape)

    return Loss(value, backward)


def categorical_kl(logits, ref_logits, mask=None, reduction=TOKEN_MEAN):
    """categorical_kl (src/nn/rl.rs:327-338). Pass `Tempered(...)` logits for reference_kl."""
    return _row_level("kl", logits, ref_logits, mask, reduction)


def reference_kl(logits, ref_logits, temperature, vocab_mask=None, mask=None, reduction=TOKEN_MEAN):
    """reference_kl (src/nn/rl.rs:347-351): both sides at the sampling temperature, same vocabulary mask."""
    return _row_level("kl", Tempered(logits, temperature, vocab_mask), ref_logits, mask, reduction)


def categorical_entropy(logits, mask=None, reduction=TOKEN_MEAN):
    """categorical_entropy (src/nn/rl.rs:405-414)."""
    return _row_level("entropy", logits, None, mask, reduction)


def _vocab_mask_args(vocab_mask, V):
    """(allow bytes, allow bits) for ops.readout_forward from a bool/uint8 mask [..., V] / [1, V] or
    int32 words of one bit per token [..., ceil(V/32)] / [1, ceil(V/32)]."""
    if vocab_mask is None:
        return None, None
    if vocab_mask.dtype == torch.int32:
        return None, vocab_mask.reshape(-1, vocab_mask.shape[-1]).contiguous()
    if vocab_mask.shape[-1:] != (V,):
        raise ValueError(f"vocab_mask: [..., {V}] or [1, {V}], got {tuple(vocab_mask.shape)}")
    allow = vocab_mask.reshape(-1, V)
    return (allow.view(torch.uint8) if allow.dtype == torch.bool else allow).contiguous(), None


def head_token_log_probs(hidden, weight, tokens, round_bf16=False, vocab_mask=None, temperature=1.0):
    """`token_log_probs(head(x), tokens)` and `categorical_entropy(head(x))` per position without the
    logits in between (src/nn/decoder.rs:270-279, then src/nn/rl.rs:134-141, 405-414): `hidden`
    bf16 [..., d], `weight` bf16 [d, V] (the Linear's [in, out] layout), tokens [...]. With
    `vocab_mask` / `temperature` the logits are the tempered ones (src/nn/rl.rs:475-486): what a
    rollout drawn by `head_sample_categorical` under the same mask and temperature is scored with.
    Returns (log-probs [...], entropies [...]). Untracked; needs a compute-capability-10 device."""
    lead = hidden.shape[:-1]
    if not (0.0 < ops.nearest_f32(temperature) < float("inf")):
        raise ValueError(f"tempered_logits: temperature {temperature} (must be positive, in 32 bits too)")
    allow, bits = _vocab_mask_args(vocab_mask, weight.shape[1])
    o = ops.readout_forward(hidden.reshape(-1, hidden.shape[-1]).contiguous(), weight, tokens=_token_ids(tokens.reshape(-1), weight.shape[1]), round_bf16=round_bf16, allow=allow, allow_bits=bits,
                            temperature=temperature)
    ops.check_status(o.status)
    return o.logp.reshape(lead), o.entropy.reshape(lead)


def head_sample_categorical(hidden, weight, uniforms, vocab_mask=None, temperature=1.0):
    """`sample_categorical(head(x), temperature, mask, ·)` by inverse CDF against `uniforms` (one per
    position; None or temperature 0: the first maximum) without the logits in between: tokens [...]
    (int32), their log-probs and the per-position entropies (of the tempered distribution).
    `vocab_mask`: a uint8/bool allow-mask [..., V] or [1, V], or int32 words of one bit per token
    [..., ceil(V/32)] or [1, ceil(V/32)]. Refuses a position with no allowed token
    with the reference's message (src/nn/rl.rs:516-519)."""
    lead = hidden.shape[:-1]
    V = weight.shape[1]
    allow, bits = _vocab_mask_args(vocab_mask, V)
    x = hidden.reshape(-1, hidden.shape[-1]).contiguous()
    if not (temperature >= 0.0 and temperature == temperature and temperature != float("inf")):
        raise ValueError("sample_categorical: temperature (must be >= 0)")
    if uniforms is None or ops.nearest_f32(temperature) == 0.0:  # the library takes 0 for no temperature
        o = ops.readout_forward(x, weight, greedy=True, allow=allow, allow_bits=bits)
    else:
        o = ops.readout_forward(x, weight, uniforms=uniforms.reshape(-1).contiguous(), allow=allow, allow_bits=bits, temperature=temperature)
    ops.check_status(o.status)
    return o.tokens.reshape(lead), o.logp.reshape(lead), o.entropy.reshape(lead)

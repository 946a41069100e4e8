"""Calls into the C ABI with torch tensors as the device buffers.

torch is used for device memory and the current stream only; every computation happens in
libnrl.so. The functions here are thin: they check devices/dtypes, allocate the outputs the C ABI
wants the caller to own, fill the argument struct and launch on torch's current stream.
"""
import ctypes as C
import functools

import torch

from . import capi


def _dt(t):
    if t.dtype == torch.float32:
        return capi.F32
    if t.dtype == torch.bfloat16:
        return capi.BF16
    raise TypeError(f"logits must be float32 or bfloat16, got {t.dtype}")


def nearest_f32(x):
    """The 32-bit float nearest to `x`, as the library takes it."""
    return C.c_float(x).value


def _p(t):
    return 0 if t is None else t.data_ptr()


def _stream(dev):
    index = torch.cuda.current_device() if dev.index is None else dev.index  # torch.device("cuda") is the current one
    return torch._C._cuda_getCurrentRawStream(index)  # the handle of torch.cuda.current_stream(dev)


def _launch(dev, name, *args):
    """The library's function `name` on `dev` and torch's current stream there."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _launch(dev, name, *args)
    rc = getattr(capi.lib(), name)(*args, _stream(dev))
    if rc != 0:
        capi.check(rc, name)


def _need(t, dtype, shape, what, dev):
    if t.dtype is not dtype or t.shape != tuple(shape) or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{what}: expected contiguous {dtype} {tuple(shape)} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _need_flat(t, dtype, n, what, dev):
    """The address of a contiguous tensor of `n` elements, whatever its shape; None is 0."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.numel() != n or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{what}: expected {n} contiguous {dtype} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _masks(V, rows, allow, add, dev):
    a_stride = d_stride = 0
    if allow is not None:
        allow = allow.view(torch.uint8) if allow.dtype == torch.bool else allow
        if allow.dtype != torch.uint8 or not allow.is_contiguous() or allow.device != dev or allow.numel() not in (V, rows * V):
            raise ValueError("allow mask: contiguous uint8/bool of [rows, V] or [1, V]")
        a_stride = 0 if allow.numel() == V and rows != 1 else V
    if add is not None:
        if add.dtype != torch.float32 or not add.is_contiguous() or add.device != dev or add.numel() not in (V, rows * V):
            raise ValueError("additive mask: contiguous float32 of [rows, V] or [1, V]")
        d_stride = 0 if add.numel() == V and rows != 1 else V
    return allow, a_stride, add, d_stride


def _bit_mask(V, rows, allow_bits, dev):
    """(tensor, stride in words) of a bit-packed allow-mask: int32 [rows, words >= ceil(V/32)] or
    [1, words] (broadcast), bit v of a row = bit (v mod 32) of its word v / 32."""
    if allow_bits.dtype != torch.int32 or allow_bits.dim() != 2 or not allow_bits.is_contiguous() or allow_bits.device != dev:
        raise ValueError(f"allow_bits: contiguous int32 [rows, words] on {dev}")
    if allow_bits.shape[1] < (V + 31) // 32 or allow_bits.shape[0] not in (1, rows):
        raise ValueError("allow_bits: [rows, >= ceil(V/32)] or [1, >= ceil(V/32)]")
    return allow_bits, (0 if allow_bits.shape[0] == 1 and rows != 1 else allow_bits.shape[1])


class RowForward:
    """Outputs of nrl_row_fwd over [rows, V] logits (fields are None when not requested)."""

    __slots__ = ("tokens", "logp", "ref_logp", "kl", "entropy", "rowstats", "status")


def row_forward(logits, *, ref_logits=None, allow=None, add_mask=None, temperature=1.0, uniforms=None, tokens=None, greedy=False,
                want_logp=True, want_entropy=True, want_kl=None, want_ref_logp=None, workspace=None, device=None, allow_bits=None, row_per_block=False):
    """Fused sample / log-prob / KL / entropy over logits [rows, V] (f32 or bf16, CUDA).

    Exactly one of: `uniforms` (sample by inverse CDF), `greedy=True`, `tokens` (given, int32), or
    none (row statistics, entropy and KL only).

    With `device` given, `logits`, `ref_logits` and the masks may be PINNED host tensors: pinned
    memory is mapped into the device's address space, so the kernel reads them in place over the
    host link (with a byte mask, only the mask and the vectors it allows cross it). Everything else
    (uniforms, tokens, the outputs) lives on `device`.

    `allow_bits` instead of `allow`: the mask bit-packed, int32 [rows, ceil(V/32)] (or [1, …]) on
    the device, bit v of a row = bit (v mod 32) of word v / 32; the kernels read V/8 mask bytes
    per row instead of V.

    `row_per_block=True` (NRL_FWD_ROW_PER_BLOCK): the kernel with one thread block per row also
    where the call has enough rows for the grouped kernel."""
    in_dev = logits.device
    dev = torch.device(device) if device is not None else in_dev
    if dev.type != "cuda":
        raise ValueError("row_forward needs CUDA tensors: this library has no CPU path")
    if in_dev.type != "cuda":
        for t in (logits, ref_logits, allow, add_mask):
            if t is not None and t.device != dev and not (t.device.type == "cpu" and t.is_pinned()):
                raise ValueError("row_forward: host inputs must all be pinned (page-locked) tensors")
    if logits.dim() != 2 or not logits.is_contiguous():
        raise ValueError("logits: contiguous [rows, V]")
    rows, V = logits.shape
    a = capi.RowFwdArgs()
    a.struct_size = C.sizeof(a)
    a.dtype, a.V, a.rows, a.temperature = _dt(logits), V, rows, float(temperature)
    a.logits = _p(logits)
    if ref_logits is not None:
        _need(ref_logits, logits.dtype, logits.shape, "ref_logits", in_dev)
        a.ref_logits = _p(ref_logits)
    # with host logits a mask may already be on the device (it is read whole; copying it ahead is cheaper than reading it in place)
    allow, a.allow_row_stride, _, _ = _masks(V, rows, allow, None, dev if (allow is not None and allow.device == dev) else in_dev)
    _, _, add_mask, a.add_row_stride = _masks(V, rows, None, add_mask, dev if (add_mask is not None and add_mask.device == dev) else in_dev)
    a.allow_mask, a.add_mask = _p(allow), _p(add_mask)
    bits_flag = 0
    if allow_bits is not None:
        if allow is not None:
            raise ValueError("give `allow` or `allow_bits`, not both")
        allow_bits, a.allow_row_stride = _bit_mask(V, rows, allow_bits, dev)
        a.allow_mask, bits_flag = _p(allow_bits), capi.FWD_MASK_BITS
    out = RowForward()
    f32 = dict(dtype=torch.float32, device=dev)
    mode = 0
    if uniforms is not None:
        _need(uniforms, torch.float32, (rows,), "uniforms", dev)
        mode, a.uniforms = capi.FWD_SAMPLE, _p(uniforms)
        out.tokens = torch.empty(rows, dtype=torch.int32, device=dev)
    elif greedy:
        mode = capi.FWD_GREEDY
        out.tokens = torch.empty(rows, dtype=torch.int32, device=dev)
    elif tokens is not None:
        _need(tokens, torch.int32, (rows,), "tokens", dev)
        mode = capi.FWD_TOKENS_IN
        out.tokens = tokens
    else:
        out.tokens = None
    a.flags, a.tokens = mode | bits_flag | (capi.FWD_ROW_PER_BLOCK if row_per_block else 0), _p(out.tokens)
    has_ref = ref_logits is not None
    want_kl = has_ref if want_kl is None else want_kl
    want_ref_logp = (has_ref and mode != 0) if want_ref_logp is None else want_ref_logp
    out.logp = torch.empty(rows, **f32) if (want_logp and mode) else None
    out.ref_logp = torch.empty(rows, **f32) if want_ref_logp else None
    out.kl = torch.empty(rows, **f32) if want_kl else None
    out.entropy = torch.empty(rows, **f32) if want_entropy else None
    out.rowstats = torch.empty(rows, 4, **f32)
    out.status = torch.empty(rows, dtype=torch.uint8, device=dev)
    a.logp, a.ref_logp, a.kl, a.entropy, a.rowstats, a.status = _p(out.logp), _p(out.ref_logp), _p(out.kl), _p(out.entropy), _p(out.rowstats), _p(out.status)
    need = capi.lib().nrl_row_fwd_workspace_bytes(rows, V)
    if need:
        if workspace is None or workspace.numel() * workspace.element_size() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = _p(workspace), workspace.numel() * workspace.element_size()
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_row_fwd(C.byref(a), _stream(dev)), "nrl_row_fwd")
    return out


def row_backward(logits, fwd, *, ref_logits=None, allow=None, add_mask=None, temperature=1.0, g_logp=None, g_kl=None, g_ent=None, out=None, accumulate=False,
                 g_uniform=None, d_ref=None, want_d_logits=True, allow_bits=None):
    """d(logits) [rows, V] f32 from the forward's saved statistics and per-row upstream gradients.
    `g_uniform`: upstream of −mean_v log π_v (label smoothing). `d_ref=True` (or a tensor) also
    returns the KL term's gradient w.r.t. ref_logits, g_kl·(ρ − π): the result is then the pair
    (d_logits or None when `want_d_logits` is False, d_ref_logits)."""
    dev = logits.device
    rows, V = logits.shape
    a = capi.RowBwdArgs()
    a.struct_size = C.sizeof(a)
    a.dtype, a.V, a.rows, a.temperature = _dt(logits), V, rows, float(temperature)
    a.logits, a.ref_logits = _p(logits), _p(ref_logits)
    allow, a.allow_row_stride, add_mask, a.add_row_stride = _masks(V, rows, allow, add_mask, dev)
    a.allow_mask, a.add_mask = _p(allow), _p(add_mask)
    if allow_bits is not None:
        if allow is not None:
            raise ValueError("give `allow` or `allow_bits`, not both")
        allow_bits, a.allow_row_stride = _bit_mask(V, rows, allow_bits, dev)
        a.allow_mask, a.mask_bits = _p(allow_bits), 1
    for name, g in (("g_logp", g_logp), ("g_kl", g_kl), ("g_ent", g_ent), ("g_uniform", g_uniform)):
        if g is not None:
            _need(g, torch.float32, (rows,), name, dev)
    a.tokens, a.rowstats, a.kl, a.entropy = _p(fwd.tokens), _p(fwd.rowstats), _p(fwd.kl), _p(fwd.entropy)
    a.g_logp, a.g_kl, a.g_ent = _p(g_logp), _p(g_kl), _p(g_ent)
    a.g_uniform = _p(g_uniform)
    if not want_d_logits:
        out = None
    elif out is None:
        out = torch.empty(rows, V, dtype=torch.float32, device=dev)
    else:
        _need(out, torch.float32, (rows, V), "d_logits", dev)
    a.d_logits = _p(out)
    if d_ref is True:
        d_ref = torch.empty(rows, V, dtype=torch.float32, device=dev)
    elif d_ref is not None and d_ref is not False:
        _need(d_ref, torch.float32, (rows, V), "d_ref_logits", dev)
    else:
        d_ref = None
    a.d_ref_logits = _p(d_ref)
    a.accumulate = 1 if accumulate else 0
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_row_bwd(C.byref(a), _stream(dev)), "nrl_row_bwd")
    return out if d_ref is None else (out, d_ref)


def _tok_args(kind, logp, other, weights, mask, clip_low=0.0, clip_high=0.0, dual=None, clamp=None):
    shape, dev = logp.shape, logp.device
    S, B, T = shape
    _need(logp, torch.float32, shape, "logp", dev)
    w_per_seq = 0
    if other is not None:
        _need(other, torch.float32, shape, "old/ref log-probs", dev)
    if weights is not None:
        w_per_seq = 1 if weights.dim() == 2 else 0
        _need(weights, torch.float32, (S, B) if w_per_seq else shape, "weights", dev)
    if mask is not None:
        _need(mask, torch.float32, shape, "mask", dev)
    return capi.TokenLossArgs(C.sizeof(capi.TokenLossArgs), kind, S, B, T, logp.data_ptr(), _p(other), _p(weights), w_per_seq, dual is not None, _p(mask), clip_low, clip_high,
                              0.0 if dual is None else dual, 0.0 if clamp is None else clamp, clamp is not None)


def token_loss(kind, logp, *, other=None, weights=None, mask=None, clip_low=0.0, clip_high=0.0, dual=None, clamp=None, want_grad=True, upstream=None, accumulate_into=None):
    """Per-token loss [S,B,T] (0 at unscored positions) and upstream · its derivative w.r.t. logp
    (added into `accumulate_into` when that is given: a logp tensor that feeds two losses)."""
    dev = logp.device
    a = _tok_args(kind, logp, other, weights, mask, clip_low, clip_high, dual, clamp)
    if upstream is not None:
        _need(upstream, torch.float32, logp.shape, "upstream", dev)
        a.upstream = _p(upstream)
    loss = torch.empty_like(logp)
    dl = torch.empty_like(logp) if want_grad else None
    if accumulate_into is not None:
        _need(accumulate_into, torch.float32, logp.shape, "accumulate_into", dev)
        dl, a.accumulate = accumulate_into, 1
    a.loss, a.dloss_dlogp = _p(loss), _p(dl)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_token_loss(C.byref(a), _stream(dev)), "nrl_token_loss")
    return loss, dl


class TokenObjective:
    """Outputs of nrl_token_objective: reduced values [S] and per-token gradients [S,B,T] (None when not requested)."""

    __slots__ = ("policy", "kl", "entropy", "g_logp", "g_kl", "g_ent")


def token_objective(kind, logp, reduction, *, other=None, weights=None, mask=None, clip_low=0.0, clip_high=0.0, dual=None, clamp=None, kl=None, entropy=None,
                    up_policy=None, up_kl=None, up_entropy=None, want_grads=True):
    """A token loss of `logp` plus the per-token KL and entropy, all reduced per seed with one
    TokenReduction, and the per-token upstream gradients of the row backward, in one launch
    (nrl_token_objective). `up_*` are the upstream gradients [S] of the three reduced values (None = ones)."""
    shape, dev = logp.shape, logp.device
    S = shape[0]
    policy = _tok_args(kind, logp, other, weights, mask, clip_low, clip_high, dual, clamp)
    for name, t in (("kl", kl), ("entropy", entropy)):
        if t is not None:
            _need(t, torch.float32, shape, name, dev)
    for name, t in (("up_policy", up_policy), ("up_kl", up_kl), ("up_entropy", up_entropy)):
        if t is not None:
            _need(t, torch.float32, (S,), name, dev)
    out = TokenObjective()

    def new(size, want):
        return torch.empty(size, dtype=torch.float32, device=dev) if want else None

    out.policy, out.kl, out.entropy = new(S, True), new(S, kl is not None), new(S, entropy is not None)
    out.g_logp, out.g_kl, out.g_ent = new(shape, want_grads), new(shape, want_grads and kl is not None), new(shape, want_grads and entropy is not None)
    a = capi.TokenObjectiveArgs(C.sizeof(capi.TokenObjectiveArgs), reduction, policy, _p(kl), _p(entropy), _p(up_policy), _p(up_kl), _p(up_entropy), out.policy.data_ptr(), _p(out.kl), _p(out.entropy),
                                _p(out.g_logp), _p(out.g_kl), _p(out.g_ent))
    _launch(dev, "nrl_token_objective", C.byref(a))
    return out


def clip_fraction(logp, old_logp, advantages, *, mask=None, clip_low, clip_high, dual=None, clamp=None):
    dev = logp.device
    a = _tok_args(capi.LOSS_PPO, logp, old_logp, advantages, mask, clip_low, clip_high, dual, clamp)
    out = torch.empty(logp.shape[0], dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_clip_fraction(C.byref(a), _p(out), _stream(dev)), "nrl_clip_fraction")
    return out


def reduce_tokens(per, mask, reduction):
    S, B, T = per.shape
    dev = per.device
    _need(per, torch.float32, per.shape, "per", dev)
    mask_at = _need_flat(mask, torch.float32, S * B * T, "mask", dev)
    shape = {capi.REDUCE_NONE: (S, B, T), capi.REDUCE_PER_SEQUENCE: (S, B)}.get(reduction, (S,))
    out = torch.empty(shape, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_reduce_tokens(reduction, S, B, T, _p(per), mask_at, _p(out), _stream(dev)), "nrl_reduce_tokens")
    return out


def reduce_tokens_backward(shape, mask, reduction, g_out):
    S, B, T = shape
    dev = g_out.device
    mask_at = _need_flat(mask, torch.float32, S * B * T, "mask", dev)
    g_at = _need_flat(g_out, torch.float32, {capi.REDUCE_NONE: S * B * T, capi.REDUCE_PER_SEQUENCE: S * B}.get(reduction, S), "upstream", dev)
    d = torch.empty(shape, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_reduce_tokens_bwd(reduction, S, B, T, mask_at, g_at, _p(d), _stream(dev)), "nrl_reduce_tokens_bwd")
    return d


def mask_rows(x, mask):
    _need(x, torch.float32, x.shape, "x", x.device)
    mask_at = _need_flat(mask, torch.float32, x.numel(), "mask", x.device)
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        capi.check(capi.lib().nrl_mask_rows(x.numel(), _p(x), mask_at, _p(out), _stream(x.device)), "nrl_mask_rows")
    return out


def group_advantages(rewards, *, norm_std=False, eps=0.0, unbiased=True):
    """group_advantages_tensor (src/nn/rl.rs:465-469) over the last axis of f32 rewards [..., N], on the device."""
    if rewards.dtype != torch.float32 or not rewards.is_contiguous() or rewards.device.type != "cuda":
        raise ValueError("rewards: a contiguous float32 CUDA tensor [..., N]")
    n = rewards.shape[-1]
    out = torch.empty_like(rewards)
    with torch.cuda.device(rewards.device):
        capi.check(capi.lib().nrl_group_advantages(rewards.numel() // n, n, int(norm_std), float(eps), int(unbiased), _p(rewards), _p(out), _stream(rewards.device)),
                   "nrl_group_advantages")
    return out


def expand_bitmask(bits, V, rows=None, out=None):
    """U8 allow-mask [rows, V] from bit-packed masks: `bits` int32 [rows, ceil(V/32)] (or [1, …]
    with `rows` given, broadcast), bit v of a row = bit (v mod 32) of word v / 32."""
    dev = bits.device
    if bits.dtype != torch.int32 or bits.dim() != 2 or not bits.is_contiguous() or dev.type != "cuda" or bits.shape[1] < (V + 31) // 32:
        raise ValueError("bits: contiguous int32 CUDA tensor [rows, >= ceil(V/32)]")
    stride = bits.shape[1]
    if rows is None:
        rows = bits.shape[0]
    elif bits.shape[0] == 1 and rows != 1:
        stride = 0
    elif bits.shape[0] != rows:
        raise ValueError("bits: [rows, words] or [1, words]")
    if out is None:
        out = torch.empty(rows, V, dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_expand_bitmask(rows, V, _p(bits), stride, _p(out), _stream(dev)), "nrl_expand_bitmask")
    return out


def check_status(status):
    """Raises the reference's error (src/nn/rl.rs:517-519) if any row was refused."""
    bad, bits = C.c_uint64(0), C.c_uint32(0)
    with torch.cuda.device(status.device):
        rc = capi.lib().nrl_check_status(_p(status), status.numel(), _stream(status.device), C.byref(bad), C.byref(bits))
    if rc == capi.E_ROW_STATUS:
        raise RuntimeError(f"sample_categorical: position {bad.value} has no allowed token (every logit −∞ or a NaN)")
    capi.check(rc, "nrl_check_status")


def _rust_float(v):
    """How Rust's `{}` prints a non-finite f64 (the reference's message carries the value)."""
    if v != v:
        return "NaN"
    return "inf" if v > 0 else "-inf"


def check_scored_finite(what, logp, mask=None):
    """`check_scored_finite(what, logp, mask)` (src/nn/rl.rs:204-211): None when every scored
    log-probability (mask != 0; no mask: all) is finite, else the reference's error text, which
    names the first flat position. A host read: it synchronises the stream."""
    dev = logp.device
    if dev.type != "cuda" or logp.dtype != torch.float32 or not logp.is_contiguous():
        raise ValueError("check_scored_finite: a contiguous float32 CUDA tensor")
    if mask is not None:
        _need(mask, torch.float32, logp.shape, "mask", dev)
    result = torch.empty(2, dtype=torch.int64, device=dev)
    pos, val = C.c_uint64(0), C.c_float(0.0)
    with torch.cuda.device(dev):
        rc = capi.lib().nrl_check_scored_finite(_p(logp), _p(mask), logp.numel(), _p(result), _stream(dev), C.byref(pos), C.byref(val))
    if rc == capi.E_NOT_FINITE:
        return f"{what}: the scored log-probability at flat position {pos.value} is {_rust_float(val.value)} (not finite)"
    capi.check(rc, "nrl_check_scored_finite")
    return None


def reduce_tokens_partial(per, mask):
    """Step 1 of a TokenReduction on the sequences this caller holds: `per`, `mask` [n_seq, T] ->
    pairs [n_seq, 2] = (sum of per, sum of mask) per sequence (nrl_reduce_tokens_partial)."""
    n_seq, T = per.shape
    dev = per.device
    _need(per, torch.float32, (n_seq, T), "per", dev)
    if mask is not None:
        _need(mask, torch.float32, (n_seq, T), "mask", dev)
    pairs = torch.empty(n_seq, 2, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_reduce_tokens_partial(n_seq, T, _p(per), _p(mask), _p(pairs), _stream(dev)), "nrl_reduce_tokens_partial")
    return pairs


def reduce_tokens_fold(pairs, S, B, reduction):
    """Step 2: the pairs of all S·B sequences, in sequence order, folded per seed (nrl_reduce_tokens_fold)."""
    dev = pairs.device
    _need(pairs, torch.float32, (S * B, 2), "pairs", dev)
    out = torch.empty((S, B) if reduction == capi.REDUCE_PER_SEQUENCE else (S,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_reduce_tokens_fold(reduction, S, B, _p(pairs), _p(out), _stream(dev)), "nrl_reduce_tokens_fold")
    return out


def reduce_tokens_backward_pairs(reduction, S, B, T, seq_begin, n_seq, pairs, mask, g_out):
    """d_per [n_seq, T] of the local sequences from the whole reduced value's gradient and the
    gathered pairs (nrl_reduce_tokens_bwd_pairs)."""
    dev = g_out.device
    d = torch.empty(n_seq, T, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_reduce_tokens_bwd_pairs(reduction, S, B, T, seq_begin, n_seq, _p(pairs), _p(mask), _p(g_out), _p(d), _stream(dev)), "nrl_reduce_tokens_bwd_pairs")
    return d


class Readout:
    """Outputs of nrl_readout_fwd (fields are None when not requested); `rounded`: of logits rounded to bf16."""

    __slots__ = ("logp", "entropy", "rowstats", "status", "logits", "tokens", "rounded")


def _readout_masks(a, V, rows, allow, allow_bits, dev):
    """The allow-mask fields of a readout call; returns the byte mask as the call reads it (keep it alive until the launch)."""
    if allow is not None and allow_bits is not None:
        raise ValueError("give `allow` or `allow_bits`, not both")
    if allow is not None:
        allow, a.allow_row_stride, _, _ = _masks(V, rows, allow, None, dev)
        a.allow_mask = _p(allow)
    if allow_bits is not None:
        words = (V + 31) // 32
        if allow_bits.dtype != torch.int32 or allow_bits.dim() != 2 or allow_bits.shape[0] not in (1, rows) or allow_bits.shape[1] < words or allow_bits.device != dev or not allow_bits.is_contiguous():
            raise ValueError("allow_bits: contiguous int32 [rows, >= ceil(V/32)] or [1, ...] on the logits' device")
        a.allow_mask, a.allow_row_stride = _p(allow_bits), (0 if allow_bits.shape[0] == 1 else allow_bits.shape[1])
        a.flags |= capi.READOUT_MASK_BITS
    return allow


def readout_forward(hidden, weights, *, tokens=None, weights_are_vd=False, round_bf16=False, want_logits=False, workspace=None, one_cta=False, uniforms=None, allow=None, greedy=False, temperature=1.0, allow_bits=None):
    """Row statistics of logits = hidden [rows, d] · W without writing the logits (nrl_readout_fwd):
    `hidden` bf16 [rows, d]; `weights` bf16 [d, V] (the reference's Linear layout) or, with
    `weights_are_vd`, [V, d]; `tokens` int32 [rows] (given tokens) for `logp`. `round_bf16` folds
    the logits rounded to bf16; `want_logits` also returns those bf16 logits [rows, V]. With
    `uniforms` (float32 [rows]) the tokens are drawn by inverse CDF instead of given (`tokens` of the
    result), with `greedy` they are each row's first maximum; `allow` is a uint8 allow-mask [rows, V]
    or [1, V], `allow_bits` the same as int32 words [rows, ceil(V/32)] or [1, ceil(V/32)] (bit v of a row =
    bit v mod 32 of word v / 32); `temperature` divides the logits before they are folded (the returned `logits` are the
    undivided ones)."""
    dev = hidden.device
    if dev.type != "cuda":
        raise ValueError("readout_forward needs CUDA tensors: this library has no CPU path")
    rows, d = hidden.shape
    V = weights.shape[0] if weights_are_vd else weights.shape[1]
    _need(hidden, torch.bfloat16, (rows, d), "hidden", dev)
    _need(weights, torch.bfloat16, (V, d) if weights_are_vd else (d, V), "weights", dev)
    a = capi.ReadoutArgs()
    a.struct_size = C.sizeof(a)
    a.flags = (capi.READOUT_W_VD if weights_are_vd else 0) | (capi.READOUT_ROUND_BF16 if round_bf16 else 0) | (capi.READOUT_ONE_CTA if one_cta else 0) | (capi.READOUT_SAMPLE if uniforms is not None else 0) | (capi.READOUT_GREEDY if greedy else 0)
    a.V, a.d, a.rows, a.temperature = V, d, rows, float(temperature)
    a.hidden, a.weights = _p(hidden), _p(weights)
    out = Readout()
    out.rounded = round_bf16
    out.logp = out.tokens = None
    if uniforms is not None:
        if tokens is not None or greedy:
            raise ValueError("give one of `tokens`, `uniforms`, `greedy`")
        _need(uniforms, torch.float32, (rows,), "uniforms", dev)
        a.uniforms = _p(uniforms)
        tokens = out.tokens = torch.empty(rows, dtype=torch.int32, device=dev)
    elif greedy:
        if tokens is not None:
            raise ValueError("give `tokens` or `greedy`, not both")
        tokens = out.tokens = torch.empty(rows, dtype=torch.int32, device=dev)
    elif tokens is not None:
        _need(tokens, torch.int32, (rows,), "tokens", dev)
    if tokens is not None:
        a.tokens = _p(tokens)
        out.logp = torch.empty(rows, dtype=torch.float32, device=dev)
    allow = _readout_masks(a, V, rows, allow, allow_bits, dev)
    out.entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    out.rowstats = torch.empty(rows, 4, dtype=torch.float32, device=dev)
    out.status = torch.empty(rows, dtype=torch.uint8, device=dev)
    out.logits = torch.empty(rows, V, dtype=torch.bfloat16, device=dev) if want_logits else None
    a.logp, a.entropy, a.rowstats, a.status, a.logits_out = _p(out.logp), _p(out.entropy), _p(out.rowstats), _p(out.status), _p(out.logits)
    if workspace is None:
        workspace = torch.empty(capi.lib().nrl_readout_workspace_bytes(rows, V, d, a.flags), dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = _p(workspace), workspace.numel() * workspace.element_size()
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_readout_fwd(C.byref(a), _stream(dev)), "nrl_readout_fwd")
    return out


def _readout_weight(weights, d, weights_are_vd, dev):
    """The vocabulary size of a readout weight for `d`-wide hidden states, checked."""
    shape = weights.shape
    if len(shape) != 2 or shape[1 if weights_are_vd else 0] != d:
        raise ValueError(f"weights: expected {'[V, d]' if weights_are_vd else '[d, V]'} with d = {d}, got {tuple(shape)}")
    V = shape[0 if weights_are_vd else 1]
    _need_flat(weights, torch.bfloat16, d * V, "weights", dev)
    return V


@functools.lru_cache(maxsize=1024)
def _scored_workspace_bytes(rows, V, d, has_scored):
    return capi.lib().nrl_readout_scored_workspace_bytes(rows, V, d, has_scored)


@functools.lru_cache(maxsize=1024)
def _bwd_workspace_bytes(rows, V, d):
    return capi.lib().nrl_readout_bwd_workspace_bytes(rows, V, d)


def _no_zero_temperature(temperature):
    if nearest_f32(temperature) == 0.0:  # the library's word for "no temperature"
        raise ValueError(f"temperature {temperature}: 0 in 32 bits (must be positive)")


class ScoredReadout:
    """Outputs of nrl_readout_scored_fwd, in one buffer: `rowstats` [rows, 4], `status` uint8 [rows] and,
    when requested (else None), `logp`, `entropy`, `ce_g_logp` [rows] and `ce_loss` [seeds]."""

    __slots__ = ("rows", "seeds", "_buf", "_logp", "_entropy", "_g", "_loss", "_status")

    def __init__(self, rows, want_logp, want_entropy, seeds, dev):
        # offsets in floats; 0 is the row statistics, so 0 elsewhere means "not requested"
        self.rows, self.seeds = rows, seeds
        self._status = at = 4 * rows
        at += (rows + 3) // 4
        self._logp = self._entropy = self._g = self._loss = 0
        if want_logp:
            self._logp, at = at, at + rows
        if want_entropy:
            self._entropy, at = at, at + rows
        if seeds:
            self._g, self._loss, at = at, at + rows, at + rows + seeds
        self._buf = torch.empty(at, dtype=torch.float32, device=dev)

    def _vector(self, at, n):
        return self._buf[at : at + n] if at else None

    rowstats = property(lambda self: self._buf[: 4 * self.rows].reshape(self.rows, 4))
    status = property(lambda self: self._buf[self._status :].view(torch.uint8)[: self.rows])
    logp = property(lambda self: self._vector(self._logp, self.rows))
    entropy = property(lambda self: self._vector(self._entropy, self.rows))
    ce_g_logp = property(lambda self: self._vector(self._g, self.rows))
    ce_loss = property(lambda self: self._vector(self._loss, self.seeds))


def readout_scored_forward(hidden, weights, *, tokens=None, scored=None, want_entropy=False, weights_are_vd=False, allow=None, allow_bits=None, temperature=1.0, workspace=None, ce_seeds=0, ce_weights=None):
    """`readout_forward` of given tokens over the positions of a training batch that `scored` (float32
    [rows], 0: not scored; None: all) lets into the loss (nrl_readout_scored_fwd): a ScoredReadout with `logp`
    (with `tokens`), `entropy` (with `want_entropy`), `rowstats` and `status`, all 0 at the other positions,
    which are not read. A token outside the vocabulary has log-prob NaN. `hidden` may have any leading shape,
    `tokens` and `scored` the same. With `ce_seeds` = S the result also has what `ce_mean` of S seeds with
    keep = scored gives, `ce_loss` [S] and `ce_g_logp` [rows]; with `ce_weights` (float32 [rows]) besides, the
    token-mean policy-gradient loss of these signed weights in its place. `readout_backward` is its backward."""
    dev = hidden.device
    if dev.type != "cuda":
        raise ValueError("readout_scored_forward needs CUDA tensors: this library has no CPU path")
    d, n = hidden.shape[-1], hidden.numel()
    rows = n // d if d else 0
    V = _readout_weight(weights, d, weights_are_vd, dev)
    _no_zero_temperature(temperature)
    xp, tp, sp = _need_flat(hidden, torch.bfloat16, n, "hidden", dev), _need_flat(tokens, torch.int32, rows, "tokens", dev), _need_flat(scored, torch.float32, rows, "scored", dev)
    out = ScoredReadout(rows, tokens is not None, want_entropy, ce_seeds, dev)
    buf = out._buf.data_ptr()
    at = lambda offset: buf + 4 * offset if offset else 0  # noqa: E731
    if workspace is None:
        workspace = torch.empty(_scored_workspace_bytes(rows, V, d, scored is not None), dtype=torch.uint8, device=dev)
    elif workspace.device != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace: contiguous, on {dev}")
    a = capi.ReadoutScoredArgs(C.sizeof(capi.ReadoutScoredArgs), 1 if weights_are_vd else 0, V, d, rows, xp, weights.data_ptr(), tp, sp, at(out._logp), at(out._entropy), buf, at(out._status), 0, 0,
                               workspace.data_ptr(), workspace.numel() * workspace.element_size(), temperature, 0, ce_seeds, at(out._loss), at(out._g), _need_flat(ce_weights, torch.float32, rows, "weights", dev))
    if allow is not None or allow_bits is not None:
        allow = _readout_masks(a, V, rows, allow, allow_bits, dev)
    _launch(dev, "nrl_readout_scored_fwd", C.byref(a))
    return out


def ce_mean(logp, S, keep=None, upstream=None, want_loss=True):
    """masked_cross_entropy of given log-probs, S seeds of logp.numel() / S positions: (value [S] or None,
    d(Σ value · upstream) / d(logp) in logp's shape) in one launch (nrl_ce_mean); `upstream` None: ones."""
    dev = logp.device
    if dev.type != "cuda":
        raise ValueError("ce_mean needs CUDA tensors: this library has no CPU path")
    n = logp.numel()
    if S < 1 or n % S:
        raise ValueError(f"ce_mean: {n} positions of {S} seeds")
    lp, kp, up = _need_flat(logp, torch.float32, n, "logp", dev), _need_flat(keep, torch.float32, n, "keep", dev), _need_flat(upstream, torch.float32, S, "upstream", dev)
    value = torch.empty(S, dtype=torch.float32, device=dev) if want_loss else None
    g = torch.empty_like(logp)
    _launch(dev, "nrl_ce_mean", S, n // S, lp, kp, up, _p(value), g.data_ptr())
    return value, g


class Int8Rows:
    """Rows as 8-bit integers with an f32 scale each: `values` int8 [rows, pitch] (pitch: `d` rounded up
    to a multiple of 16), `scales` f32 [rows], x ≈ values[:, :d] · scales[:, None]."""

    __slots__ = ("values", "scales", "d")

    def __init__(self, values, scales, d):
        if values.dim() != 2 or not 0 < d <= values.shape[1] or values.shape[1] % 16:
            raise ValueError("values: int8 [rows, pitch], pitch >= d and a multiple of 16")
        _need_flat(values, torch.int8, values.numel(), "values", values.device)
        _need(scales, torch.float32, values.shape[:1], "scales", values.device)
        self.values, self.scales, self.d = values, scales, d


def _int8_rows(rows, d, dev):
    q = Int8Rows.__new__(Int8Rows)
    q.values, q.scales, q.d = torch.empty(rows, (d + 15) // 16 * 16, dtype=torch.int8, device=dev), torch.empty(rows, dtype=torch.float32, device=dev), d
    return q


def quantize_rows(x):
    """`x` [..., d] (float32 or bfloat16) as Int8Rows, a row per leading position: q = rint(127 x / max|x|),
    scale max|x| / 127 (nrl_i8_quantize_rows). A row with an infinity or a NaN gets a non-finite scale."""
    dev = x.device
    if dev.type != "cuda":
        raise ValueError("quantize_rows needs CUDA tensors: this library has no CPU path")
    d = x.shape[-1]
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    q = _int8_rows(x.numel() // d if d else 0, d, dev)
    _launch(dev, "nrl_i8_quantize_rows", _dt(x), q.values.shape[0], d, x.data_ptr(), q.values.data_ptr(), q.values.shape[1], q.scales.data_ptr())
    return q


def quantize_weight(weights, weights_are_vd=False):
    """A readout weight, bf16 [d, V] (or [V, d] with `weights_are_vd`), as Int8Rows [V, d]: a scale per
    vocabulary entry (nrl_i8_quantize_columns / nrl_i8_quantize_rows)."""
    if weights_are_vd:
        return quantize_rows(weights)
    dev = weights.device
    if dev.type != "cuda":
        raise ValueError("quantize_weight needs CUDA tensors: this library has no CPU path")
    d, V = weights.shape
    _need(weights, torch.bfloat16, (d, V), "weights", dev)
    q = _int8_rows(V, d, dev)
    _launch(dev, "nrl_i8_quantize_columns", d, V, weights.data_ptr(), q.values.data_ptr(), q.values.shape[1], q.scales.data_ptr())
    return q


def dequantize_rows(q, dtype=torch.bfloat16):
    """values · scale as [rows, d] of `dtype` (nrl_i8_dequantize_rows)."""
    dev = q.values.device
    if dev.type != "cuda":
        raise ValueError("dequantize_rows needs CUDA tensors: this library has no CPU path")
    out = torch.empty(q.values.shape[0], q.d, dtype=dtype, device=dev)
    _launch(dev, "nrl_i8_dequantize_rows", _dt(out), out.shape[0], q.d, q.values.data_ptr(), q.values.shape[1], q.scales.data_ptr(), out.data_ptr())
    return out


def int8_matmul(x, w, dtype=torch.float32):
    """out[r, v] = Σ_k x[r, k] w[v, k] (exact) · x.scales[r] · w.scales[v], [rows, V] of `dtype`
    (nrl_i8_matmul); `x`, `w`: Int8Rows of the same d."""
    dev = x.values.device
    if dev.type != "cuda":
        raise ValueError("int8_matmul needs CUDA tensors: this library has no CPU path")
    if x.d != w.d or w.values.device != dev:
        raise ValueError(f"int8_matmul: rows of {x.d} and of {w.d} integers on {dev} and {w.values.device}")
    (rows, x_pitch), (n, w_pitch) = x.values.shape, w.values.shape
    out = torch.empty(rows, n, dtype=dtype, device=dev)
    a = capi.I8MatmulArgs(C.sizeof(capi.I8MatmulArgs), _dt(out), rows, n, x.d, x.values.data_ptr(), x_pitch, x.scales.data_ptr(), w.values.data_ptr(), w_pitch, w.scales.data_ptr(), out.data_ptr())
    _launch(dev, "nrl_i8_matmul", C.byref(a))
    return out


def int8_linear(x, w, dtype=torch.float32):
    """`int8_matmul(quantize_rows(x), w, dtype)` in one call (nrl_i8_linear): `x` [..., d] float32 or bfloat16,
    `w` Int8Rows [V, d], result [..., V]."""
    dev = x.device
    if dev.type != "cuda":
        raise ValueError("int8_linear needs CUDA tensors: this library has no CPU path")
    d = x.shape[-1]
    (n, w_pitch), rows = w.values.shape, x.numel() // d if d else 0
    if d != w.d or w.values.device != dev or not x.is_contiguous():
        raise ValueError(f"int8_linear: contiguous rows of {w.d} values on {w.values.device}, got {tuple(x.shape)} on {dev}")
    out = torch.empty(x.shape[:-1] + (n,), dtype=dtype, device=dev)
    a = capi.I8MatmulArgs(C.sizeof(capi.I8MatmulArgs), _dt(out), rows, n, d, x.data_ptr(), 0, 0, w.values.data_ptr(), w_pitch, w.scales.data_ptr(), out.data_ptr())
    workspace = torch.empty(capi.lib().nrl_i8_linear_workspace_bytes(rows, d), dtype=torch.uint8, device=dev)
    _launch(dev, "nrl_i8_linear", _dt(x), C.byref(a), workspace.data_ptr(), workspace.numel())
    return out


def readout_backward(hidden, weights, fwd, *, tokens=None, g_logp=None, g_ent=None, weights_are_vd=False, allow=None, allow_bits=None, temperature=1.0, want_hidden=True,
                     want_weights=True, grad_dtype=torch.bfloat16, add_hidden=None, add_weights=None, workspace=None, hidden_shape=None):
    """(d_hidden, d_weights) of Σ g_logp·logp + Σ g_ent·entropy of the results `fwd` of
    `readout_scored_forward` or `readout_forward` (their `rowstats` and, with `g_ent`, `entropy`; not of rounded logits), the
    logits computed again in pieces (nrl_readout_bwd). `hidden`: the bf16 [..., d] of the forward call, or
    an Int8Rows checkpoint of it (d_hidden then has `hidden_shape`, default [rows, d]). Gradients are
    `grad_dtype` (bfloat16 or float32); `add_hidden` / `add_weights` are tensors they are added to in place
    (their own dtype counts). Rows whose upstreams are 0 are not read. With neither upstream given, it is the
    gradient of the loss that `fwd` holds (`ce_g_logp`)."""
    quant = hidden if isinstance(hidden, Int8Rows) else None
    x = quant.values if quant else hidden
    dev = x.device
    if dev.type != "cuda":
        raise ValueError("readout_backward needs CUDA tensors: this library has no CPU path")
    d = quant.d if quant else x.shape[-1]
    if hidden_shape is None:
        hidden_shape = (x.shape[0], d) if quant else x.shape
    hidden_shape = torch.Size(hidden_shape)
    rows = hidden_shape.numel() // d if d else 0
    if hidden_shape[-1:] != (d,):
        raise ValueError(f"hidden_shape: [..., {d}], got {tuple(hidden_shape)}")
    V = _readout_weight(weights, d, weights_are_vd, dev)
    if grad_dtype is not torch.bfloat16 and grad_dtype is not torch.float32:
        raise TypeError(f"gradients must be bfloat16 or float32, got {grad_dtype}")
    _no_zero_temperature(temperature)
    if type(fwd) is Readout and fwd.rounded:
        raise ValueError("fwd: of logits rounded to bf16, which have no gradient here")
    own = type(fwd) is ScoredReadout and fwd.rows == rows and fwd._buf.device == dev
    from_loss = 4 * fwd._g if own and g_logp is None and g_ent is None else 0  # where fwd's gradient of the log-probs lies, 0: not used
    if g_logp is None and g_ent is None and not from_loss:
        raise ValueError("give `g_logp`, `g_ent` or both, or a forward with a loss")
    flags = capi.READOUT_W_VD if weights_are_vd else 0
    if quant:
        if x.shape[0] != rows:
            raise ValueError(f"hidden: {x.shape[0]} rows of integers for {rows} positions")
        flags |= capi.READOUT_BWD_HIDDEN_I8
        xp, sp, pitch = x.data_ptr(), quant.scales.data_ptr(), x.shape[1]
    else:
        xp, sp, pitch = _need_flat(x, torch.bfloat16, rows * d, "hidden", dev), 0, 0
    if (g_logp is not None or from_loss) and tokens is None:
        raise ValueError("`g_logp` needs the tokens")

    def out(add, want, shape, f32_flag, add_flag, what):
        nonlocal flags
        if add is not None:
            if add.dtype not in (torch.bfloat16, torch.float32):
                raise TypeError(f"{what}: bfloat16 or float32, got {add.dtype}")
            _need(add, add.dtype, shape, what, dev)
            flags |= add_flag
        elif want:
            add = torch.empty(shape, dtype=grad_dtype, device=dev)
        if add is not None and add.dtype is torch.float32:
            flags |= f32_flag
        return add

    d_hidden = out(add_hidden, want_hidden, hidden_shape, capi.READOUT_BWD_D_HIDDEN_F32, capi.READOUT_BWD_ADD_D_HIDDEN, "add_hidden")
    d_weights = out(add_weights, want_weights, weights.shape, capi.READOUT_BWD_D_WEIGHTS_F32, capi.READOUT_BWD_ADD_D_WEIGHTS, "add_weights")
    if workspace is not None and (workspace.device != dev or not workspace.is_contiguous()):
        raise ValueError(f"workspace: contiguous, on {dev}")
    if own:
        stats = fwd._buf.data_ptr()
        ent = stats + 4 * fwd._entropy if fwd._entropy else 0
    else:
        stats, ent = _need_flat(fwd.rowstats, torch.float32, rows * 4, "rowstats", dev), _need_flat(fwd.entropy, torch.float32, rows, "entropy", dev)
    if g_ent is not None and not ent:
        raise ValueError("`g_ent` needs a forward with entropies")
    tp = 0 if g_logp is None and not from_loss else _need_flat(tokens, torch.int32, rows, "tokens", dev)
    gp, ep = stats + from_loss if from_loss else _need_flat(g_logp, torch.float32, rows, "g_logp", dev), _need_flat(g_ent, torch.float32, rows, "g_ent", dev)
    _launch_backward(dev, flags, V, d, rows, xp, sp, pitch, weights.data_ptr(), tp, stats, ent if ep else 0, gp, ep, _p(d_hidden), _p(d_weights), workspace, temperature, allow, allow_bits)
    return d_hidden, d_weights


def _launch_backward(dev, flags, V, d, rows, x, scales, pitch, weights, tokens, stats, ent, g_logp, g_ent, d_hidden, d_weights, workspace, temperature, allow, allow_bits):
    """nrl_readout_bwd of checked addresses."""
    if workspace is None:
        workspace = torch.empty(_bwd_workspace_bytes(rows, V, d), dtype=torch.uint8, device=dev)
    a = capi.ReadoutBwdArgs(C.sizeof(capi.ReadoutBwdArgs), flags, V, d, rows, x, scales, pitch, weights, tokens, stats, ent, g_logp, g_ent, d_hidden, d_weights, 0, 0,
                            workspace.data_ptr(), workspace.numel() * workspace.element_size(), temperature)
    if allow is not None or allow_bits is not None:
        allow = _readout_masks(a, V, rows, allow, allow_bits, dev)
    _launch(dev, "nrl_readout_bwd", C.byref(a))


def readout_backward_of_loss(fwd, hidden, weights, tokens, *, weights_are_vd=False, allow=None, allow_bits=None, temperature=1.0, grad_dtype=torch.bfloat16, hidden_shape=None):
    """`readout_backward` of the loss that `fwd` holds, for the arguments that the forward call has checked
    already: `hidden` as it was there or its Int8Rows, the other arguments as they were."""
    flags, x, scales, pitch = (capi.READOUT_W_VD if weights_are_vd else 0), hidden, 0, 0
    if type(hidden) is Int8Rows:
        flags, x, scales, pitch = flags | capi.READOUT_BWD_HIDDEN_I8, hidden.values, hidden.scales.data_ptr(), hidden.values.shape[1]
    else:
        hidden_shape = hidden.shape
    if grad_dtype is torch.float32:
        flags |= capi.READOUT_BWD_D_HIDDEN_F32 | capi.READOUT_BWD_D_WEIGHTS_F32
    elif grad_dtype is not torch.bfloat16:
        raise TypeError(f"gradients must be bfloat16 or float32, got {grad_dtype}")
    dev, stats = x.device, fwd._buf.data_ptr()
    d_hidden, d_weights = torch.empty(hidden_shape, dtype=grad_dtype, device=dev), torch.empty_like(weights, dtype=grad_dtype)
    _launch_backward(dev, flags, weights.shape[0 if weights_are_vd else 1], hidden_shape[-1], fwd.rows, x.data_ptr(), scales, pitch, weights.data_ptr(), tokens.data_ptr(), stats, 0, stats + 4 * fwd._g, 0,
                     d_hidden.data_ptr(), d_weights.data_ptr(), None, temperature, allow, allow_bits)
    return d_hidden, d_weights


def row_sum(logits):
    """Σ_v logits[r, v] per row in f32 (nrl_row_sum)."""
    dev = logits.device
    rows, V = logits.shape
    if not logits.is_contiguous():
        raise ValueError("logits must be contiguous")
    out = torch.empty(rows, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_row_sum(_dt(logits), rows, V, _p(logits), _p(out), _stream(dev)), "nrl_row_sum")
    return out


def ce_tokens(V, logp, *, smoothing=0.0, rowstats=None, logit_sum=None, keep=None, upstream=None, want_loss=True):
    """The O(rows) part of the cross-entropy family (nrl_ce_tokens): returns (loss, g_logp,
    g_uniform), each [n] f32 or None."""
    dev = logp.device
    n = logp.numel()
    a = capi.CeArgs()
    a.struct_size = C.sizeof(a)
    a.V, a.n, a.smoothing = V, n, float(smoothing)
    _need(logp, torch.float32, logp.shape, "logp", dev)
    a.logp, a.rowstats, a.logit_sum, a.keep = _p(logp), _p(rowstats), _p(logit_sum), _p(keep)
    if keep is not None:
        _need(keep, torch.float32, logp.shape, "keep", dev)
    loss = torch.empty_like(logp) if want_loss else None
    g_logp = g_uni = None
    if upstream is not None:
        _need(upstream, torch.float32, logp.shape, "upstream", dev)
        g_logp = torch.empty_like(logp)
        g_uni = torch.empty_like(logp) if smoothing > 0.0 else None
    a.loss, a.upstream, a.g_logp, a.g_uniform = _p(loss), _p(upstream), _p(g_logp), _p(g_uni)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_ce_tokens(C.byref(a), _stream(dev)), "nrl_ce_tokens")
    return loss, g_logp, g_uni


def sample_gumbel(logits, seed, *, word_offset=0, temperature=1.0, allow=None, add_mask=None):
    """The reference's Gumbel-max sampler on the device (nrl_sample_gumbel): `seed` is the 32-byte
    ChaCha20 key, `word_offset` the 32-bit words already drawn. Returns (tokens int32 [rows],
    status uint8 [rows]); the call consumes 2·rows·V words of the stream."""
    dev = logits.device
    rows, V = logits.shape
    if not logits.is_contiguous():
        raise ValueError("logits must be contiguous")
    if len(seed) != 32:
        raise ValueError("seed: 32 bytes")
    a = capi.GumbelArgs()
    a.struct_size = C.sizeof(a)
    a.dtype, a.V, a.rows, a.temperature = _dt(logits), V, rows, float(temperature)
    a.logits = _p(logits)
    allow, a.allow_row_stride, add_mask, a.add_row_stride = _masks(V, rows, allow, add_mask, dev)
    a.allow_mask, a.add_mask = _p(allow), _p(add_mask)
    a.seed[:] = list(seed)
    a.word_offset = int(word_offset)
    tokens = torch.empty(rows, dtype=torch.int32, device=dev)
    status = torch.empty(rows, dtype=torch.uint8, device=dev)
    a.tokens, a.status = _p(tokens), _p(status)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_sample_gumbel(C.byref(a), _stream(dev)), "nrl_sample_gumbel")
    return tokens, status


def _lane(op, x, *, g=None, lse=None, full_out=True, index=False):
    dev = x.device
    if dev.type != "cuda":
        raise ValueError("lane ops run on CUDA tensors only")
    if x.dim() != 2 or not x.is_contiguous():
        raise ValueError("x must be a contiguous [rows, V] tensor")
    rows, V = x.shape
    a = capi.LaneArgs()
    a.struct_size = C.sizeof(a)
    a.op, a.dtype, a.V, a.rows = op, _dt(x), V, rows
    a.x = _p(x)
    if g is not None:
        _need(g, torch.float32, (rows, V) if op != capi.LANE_LOGSUMEXP_BWD else (rows,), "g", dev)
        a.g = _p(g)
    if lse is not None:
        _need(lse, torch.float32, (rows,), "lse", dev)
        a.lse = _p(lse)
    out = torch.empty((rows, V) if full_out else (rows,), dtype=torch.float32, device=dev)
    a.out = _p(out)
    idx = None
    if index:
        idx = torch.empty(rows, dtype=torch.int32, device=dev)
        a.out_index = _p(idx)
    with torch.cuda.device(dev):
        capi.check(capi.lib().nrl_lane_op(C.byref(a), _stream(dev)), "nrl_lane_op")
    return (idx, out) if index else out


def softmax(x):
    """softmax along the last axis of [rows, V] (src/tensor/activation.rs:15-26), f32 out."""
    return _lane(capi.LANE_SOFTMAX, x)


def log_softmax(x):
    """log_softmax along the last axis (src/tensor/activation.rs:30-42), f32 out."""
    return _lane(capi.LANE_LOG_SOFTMAX, x)


def logsumexp(x):
    """log Σ exp along the last axis with the ±inf rule (src/tensor/activation.rs:71-77), [rows]."""
    return _lane(capi.LANE_LOGSUMEXP, x, full_out=False)


def argmax(x):
    """(index i32 [rows], value f32 [rows]): the first maximum, the first NaN of a row that holds one
    (src/tensor/kernels.rs:184-209)."""
    return _lane(capi.LANE_ARGMAX, x, full_out=False, index=True)


def sum_last(x):
    """Σ along the last axis in the reference's operand order (src/tensor/kernels.rs:122-148)."""
    return _lane(capi.LANE_SUM, x, full_out=False)


def softmax_backward(y, g):
    """y · (g − Σ g·y) from the saved output."""
    return _lane(capi.LANE_SOFTMAX_BWD, y, g=g)


def log_softmax_backward(y, g):
    """g − exp(y) · Σ g from the saved output."""
    return _lane(capi.LANE_LOG_SOFTMAX_BWD, y, g=g)


def logsumexp_backward(x, lse, g):
    """g[row] · exp(x − lse[row])."""
    return _lane(capi.LANE_LOGSUMEXP_BWD, x, g=g, lse=lse)

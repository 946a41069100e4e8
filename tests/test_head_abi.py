"""CPU checks of the C entries of the readout's backward and its 8-bit forms: struct sizes, argument refusals that need no
device, and the scratch sizes' shape."""
import ctypes as C

from noetic_tensor_b200 import capi


def test_struct_layouts():
    assert C.sizeof(capi.ReadoutScoredArgs) == 4 * 4 + 8 + 8 * 8 + 2 * 8 + 2 * 8 + 4 + 4 + 4 * 8
    assert C.sizeof(capi.ReadoutBwdArgs) == 4 * 4 + 8 + 15 * 8 + 4 + 4
    assert C.sizeof(capi.I8MatmulArgs) == 2 * 4 + 8 + 2 * 4 + 7 * 8


def scored():
    a = capi.ReadoutScoredArgs()
    a.struct_size, a.V, a.d, a.rows = C.sizeof(a), 512, 64, 10
    a.hidden = a.weights = a.rowstats = a.workspace = 4096
    return a


def backward():
    a = capi.ReadoutBwdArgs()
    a.struct_size, a.V, a.d, a.rows = C.sizeof(a), 512, 64, 10
    a.hidden = a.weights = a.rowstats = a.workspace = a.g_logp = a.tokens = a.d_hidden = 4096
    return a


def product():
    a = capi.I8MatmulArgs()
    a.struct_size, a.dtype, a.rows, a.n, a.k = C.sizeof(a), capi.F32, 4, 100, 50
    a.x = a.w = a.x_scales = a.w_scales = a.out = 4096
    a.x_pitch = a.w_pitch = 64
    return a


def refused(make, call, changes):
    for want, change in changes:
        a = make()
        for k, v in change.items():
            setattr(a, k, v)
        assert call(a) == want, (change, want)


def test_scored_forward_refuses():
    l = capi.lib()
    B, U = capi.E_BAD_ARG, capi.E_UNSUPPORTED
    refused(scored, lambda a: l.nrl_readout_scored_fwd(C.byref(a), None), [
        (B, dict(struct_size=0)), (B, dict(rows=0)), (B, dict(hidden=0)), (B, dict(weights=0)), (B, dict(rowstats=0)), (B, dict(flags=2)), (B, dict(flags=1 << 30)),
        (U, dict(V=510)), (U, dict(d=60)), (U, dict(hidden=4104)), (U, dict(rows=1 << 31)), (B, dict(rowstats=4100)), (B, dict(workspace=4112)), (B, dict(logp=4096)), (B, dict(tokens=2)),
        (B, dict(temperature=-1.0)), (B, dict(temperature=float("nan"))), (B, dict(reserved=1)), (B, dict(allow_mask=4096, allow_row_stride=100)),
        (B, dict(flags=capi.READOUT_MASK_BITS)), (B, dict(flags=capi.READOUT_MASK_BITS, allow_mask=4096, allow_row_stride=3)),
        (B, dict(seeds=1)), (B, dict(seeds=3, tokens=4096, logp=4096, ce_loss=4096)), (B, dict(seeds=2, tokens=4096, logp=4096)), (B, dict(ce_loss=4096)), (B, dict(ce_weights=4096)),
    ])
    assert l.nrl_readout_scored_fwd(None, None) == B


def test_backward_refuses():
    l = capi.lib()
    B, U = capi.E_BAD_ARG, capi.E_UNSUPPORTED
    I8 = capi.READOUT_BWD_HIDDEN_I8
    refused(backward, lambda a: l.nrl_readout_bwd(C.byref(a), None), [
        (B, dict(struct_size=8)), (B, dict(rows=0)), (B, dict(d_hidden=0)), (B, dict(rowstats=0)), (B, dict(g_logp=0)), (B, dict(tokens=0)), (B, dict(g_ent=4096)), (B, dict(flags=1 << 20)),
        (U, dict(V=4)), (U, dict(d_hidden=4104)), (B, dict(hidden_scales=4096)), (B, dict(hidden_pitch=80)), (B, dict(flags=I8)), (B, dict(flags=I8, hidden_scales=4096, hidden_pitch=60)),
        (B, dict(flags=I8, hidden_scales=4096, hidden_pitch=72)), (B, dict(temperature=float("inf"))), (B, dict(allow_mask=4096, allow_row_stride=8)), (B, dict(workspace=4097)),
    ])


def test_int8_entries_refuse():
    l = capi.lib()
    B, U = capi.E_BAD_ARG, capi.E_UNSUPPORTED
    refused(product, lambda a: l.nrl_i8_matmul(C.byref(a), None), [
        (B, dict(struct_size=0)), (B, dict(rows=0)), (B, dict(n=0)), (B, dict(k=0)), (B, dict(w=0)), (B, dict(out=0)), (U, dict(dtype=5)), (B, dict(x_pitch=40)), (B, dict(w_pitch=56)), (B, dict(x=4100)),
        (B, dict(out=4097)), (U, dict(k=131088, x_pitch=131088, w_pitch=131088)), (U, dict(rows=1 << 31)),
    ])
    a = product()
    assert l.nrl_i8_linear(capi.BF16, C.byref(a), 4096, 1 << 20, None) == B  # x_pitch and x_scales belong to the call
    a.x_pitch = a.x_scales = 0
    assert l.nrl_i8_linear(capi.BF16, C.byref(a), 4096, 16, None) == capi.E_WORKSPACE
    assert l.nrl_i8_linear(capi.BF16, C.byref(a), 4100, 1 << 20, None) == B
    assert l.nrl_i8_quantize_rows(capi.F32, 0, 8, 4096, 4096, 16, 4096, None) == B
    assert l.nrl_i8_quantize_rows(capi.F32, 4, 20, 4096, 4096, 16, 4096, None) == B
    assert l.nrl_i8_quantize_rows(7, 4, 8, 4096, 4096, 16, 4096, None) == U
    assert l.nrl_i8_quantize_columns(8, 0, 4096, 4096, 16, 4096, None) == B
    assert l.nrl_i8_dequantize_rows(capi.BF16, 4, 8, 4096, 4, 4096, 4096, None) == B
    assert l.nrl_ce_mean(0, 4, 4096, 0, 0, 4096, 0, None) == B and l.nrl_ce_mean(1, 4, 0, 0, 0, 4096, 0, None) == B and l.nrl_ce_mean(1, 4, 4096, 0, 0, 0, 0, None) == B


def test_scratch_sizes():
    l = capi.lib()
    # dz of a piece of the vocabulary, never more than 512 MB of it unless 4096 columns are more
    assert l.nrl_readout_bwd_workspace_bytes(8192, 128256, 4096) < 512 * 2**20 + 8192 * 4096 * 6 + 2**20
    assert l.nrl_readout_bwd_workspace_bytes(0, 512, 64) == 0
    assert l.nrl_readout_scored_workspace_bytes(262144, 128256, 4096, 0) < 16384 * 128256 // 128 * 2 * 16 + 2**20
    assert l.nrl_readout_scored_workspace_bytes(262144, 128256, 4096, 1) > 262144 * 4096 * 2
    assert l.nrl_i8_linear_workspace_bytes(3, 100) == 256 + 3 * 128

// The C ABI of the readout's backward pass and of its 8-bit forms: argument checks, the
// decomposition of a call into pieces of the vocabulary, and launches. No allocation, no synchronisation.
#include <atomic>
#include <cstring>

#include "head_ops.cuh"

using namespace nrl;

extern std::atomic<uint64_t> nrl_g_launches;

// One launch in stream order, counted. The products start early (launch_next), and small grids; a larger grid of small blocks that
// waits beside a product's last tiles delayed the pass by 7 us (the statistics of 2048 rows at V = 32 000, d = 1024: 121 against 114 us).
template <typename... Params, typename... Args>
static int launch_as(unsigned cluster, void (*kernel)(Params...), dim3 grid, unsigned block, size_t smem, cudaStream_t stream, const Args&... args) {
    nrl_g_launches.fetch_add(1, std::memory_order_relaxed);
    const cudaError_t e = launch_next(smem != 0 || grid.x <= 2 * kPairs, cluster, kernel, grid, dim3(block), smem, stream, args...);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? NRL_OK : (int)e;
}
template <typename... Params, typename... Args>
static int launch(void (*kernel)(Params...), dim3 grid, unsigned block, size_t smem, cudaStream_t stream, const Args&... args) {
    return launch_as(1, kernel, grid, block, smem, stream, args...);
}

static int need_cc10() {
    int dev = 0, cc_major = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&cc_major, cudaDevAttrComputeCapabilityMajor, dev);
    if (e != cudaSuccess) return (int)e;
    return cc_major == 10 ? NRL_OK : NRL_E_UNSUPPORTED;  // tcgen05 / tensor memory
}

template <int EPI, int MASK, bool PAIR>
static int launch_tiles(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, HeadGemm p, uint64_t tiles, cudaStream_t st) {
    constexpr unsigned ctas = PAIR ? 2 : 1;
    p.stages = kHgSmemTiles / (kHgABytes + (p.bn / ctas) * 128);
    if (p.stages > kHgMaxStages) p.stages = kHgMaxStages;
    if (tiles > 0x7fffffffull) return NRL_E_UNSUPPORTED;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    static std::atomic<uint64_t> ready{0};  // devices on which this kernel may have its shared memory
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1u)) {
        e = cudaFuncSetAttribute(head_gemm_kernel<EPI, MASK, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kHgSmemBytes);
        if (e != cudaSuccess) return (int)e;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const uint64_t most = 2 * kPairs / ctas;
    return launch_as(ctas, head_gemm_kernel<EPI, MASK, PAIR>, dim3(ctas * (unsigned)(tiles < most ? (tiles ? tiles : 1) : most)), kHgThreads, kHgSmemBytes, st, ma, mb, mo, p);
}
// on pairs of CTAs or, `single`, on CTAs by themselves
template <int EPI, int MASK = kMaskNone>
static int launch_gemm(bool single, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, const HeadGemm& p, uint64_t tiles, cudaStream_t st) {
    return single ? launch_tiles<EPI, MASK, false>(ma, mb, mo, p, tiles, st) : launch_tiles<EPI, MASK, true>(ma, mb, mo, p, tiles, st);
}
template <int EPI>
static int launch_masked(bool single, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, const HeadGemm& p, uint32_t allow_bits, uint64_t tiles, cudaStream_t st) {
    if (!p.allow) return launch_gemm<EPI, kMaskNone>(single, ma, mb, mo, p, tiles, st);
    return allow_bits ? launch_gemm<EPI, kMaskBits>(single, ma, mb, mo, p, tiles, st) : launch_gemm<EPI, kMaskBytes>(single, ma, mb, mo, p, tiles, st);
}

static inline uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }
static inline uint32_t tiles256(uint64_t x) { return (uint32_t)((x + 255) / 256); }

// Columns per tile of a bf16 product over `rows` × `cols`: half the width where that puts twice the pairs to work (140 rows at
// V = 1120, d = 1808: five pairs took 20 us).
// With `single` CTAs there are twice as many workers.
static uint32_t tile_width(uint64_t rows, uint64_t cols, bool single) { return (uint64_t)tiles256(rows) * tiles256(cols) <= (single ? kPairs : kPairs / 2) ? 128u : 256u; }
// At most one CTA's rows: single CTAs instead of pairs.
static bool runs_single(uint64_t rows) { return rows <= kHgBM; }
static uint64_t tiles_of(uint64_t rows, uint64_t cols, uint32_t bn) { return (uint64_t)tiles256(rows) * ((cols + bn - 1) / bn); }

static int launch_rows(HeadRows& hr, cudaStream_t st) {
    // a block owns 8 rows, one per warp; more when there would be over 1024 blocks, since each looks at every row's upstream
    hr.per_block = (uint32_t)((hr.rows + 1023) / 1024);
    if (hr.per_block < 8) hr.per_block = 8;
    return launch(head_rows_kernel, dim3((unsigned)((hr.rows + hr.per_block - 1) / hr.per_block)), kRowsThreads, 0, st, hr);
}

// the mask fields that the forward and the backward share: what a call may give
static bool bad_mask(uint32_t flags, nrl_devptr mask, uint64_t stride, uint32_t V) {
    if (flags & NRL_READOUT_MASK_BITS) return !mask || (mask & 3u) || (stride != 0 && stride < (V + 31u) / 32u);
    return mask && stride != 0 && stride != V;
}
static void set_mask(HeadGemm& g, nrl_devptr mask, uint64_t stride) {
    g.allow = (const uint8_t*)mask;
    g.allow_stride = stride;
    g.allow_wide = (mask | stride) % 4 == 0 ? 1u : 0u;
}

// How a backward call is cut: pieces of `vc` vocabulary columns; their dz is what exists of [rows, V] at any time. A function of
// (rows, V, d) only.
struct BwdPlan {
    uint64_t rows_pad;
    uint32_t vc, pieces, chunks, grad_bn, hidden_bn, side_by_side;
    bool may_split, single;
    uint64_t off_coef, off_more, off_rows, off_x, off_dz, off_acc, bytes;
};
static BwdPlan bwd_plan(uint64_t rows, uint32_t V, uint32_t d) {
    BwdPlan b;
    b.rows_pad = up(rows, 256);
    b.single = runs_single(rows);
    // dz of a piece is at most 512 MB, but not narrower than 4096 columns: dx's f32 sums are read and written once per piece
    uint64_t vc = (512ull << 20) / (b.rows_pad * 2) / 256 * 256;
    if (vc < 4096) vc = 4096;
    if (vc > up(V, 256)) vc = up(V, 256);
    b.pieces = (uint32_t)((V + vc - 1) / vc);
    b.vc = (uint32_t)up((V + b.pieces - 1) / b.pieces, 256);  // pieces of about the same width
    b.pieces = (V + b.vc - 1) / b.vc;
    b.chunks = b.vc / 64;
    b.grad_bn = tile_width(rows, b.vc, b.single);
    // any number of scored rows up to `rows` may turn up: whether one of them would have dx's K split
    b.side_by_side = b.single ? 2 * kPairs : kPairs;
    // half-width tiles of dx where even its ranges leave pairs idle
    b.hidden_bn = (uint64_t)tiles256(rows) * tiles256(d) * (b.chunks >= 24 ? b.chunks / 12 : 1) < b.side_by_side ? 128u : 256u;
    uint64_t split_units = 0;
    const uint32_t tn = (d + b.hidden_bn - 1) / b.hidden_bn, tm = tiles256(rows);
    for (uint32_t m = 1; m <= tm && m * tn <= b.side_by_side; m++) {
        const uint32_t s = hidden_split(m * tn, b.chunks, b.side_by_side);
        if (s > 1 && (uint64_t)m * s > split_units) split_units = (uint64_t)m * s;
    }
    b.may_split = split_units > 0;
    uint64_t at = 256;
    b.off_coef = at; at += up(rows * 16, 256);
    b.off_more = at; at += up(rows * 16, 256);
    b.off_rows = at; at += up(rows * 4, 256);
    b.off_x = at; at += b.rows_pad * up(d, 64) * 2;
    b.off_dz = at; at += b.rows_pad * b.vc * 2;
    b.off_acc = at;
    uint64_t acc = split_units * 256 * d * 4;
    if (b.pieces > 1 && acc < b.rows_pad * d * 4) acc = b.rows_pad * d * 4;
    b.bytes = at + acc;
    return b;
}

extern "C" uint64_t nrl_readout_bwd_workspace_bytes(uint64_t rows, uint32_t V, uint32_t d) {
    if (rows == 0 || V == 0 || d == 0) return 0;
    return bwd_plan(rows, V, d).bytes;
}

extern "C" int nrl_readout_bwd(const nrl_readout_bwd_args* a, nrl_stream stream) {
    if (!a || a->struct_size != sizeof(nrl_readout_bwd_args)) return NRL_E_BAD_ARG;
    if (a->rows == 0 || a->V == 0 || a->d == 0 || !a->hidden || !a->weights || !a->rowstats || (!a->d_hidden && !a->d_weights)) return NRL_E_BAD_ARG;
    const uint32_t known = NRL_READOUT_W_VD | NRL_READOUT_MASK_BITS | NRL_READOUT_BWD_HIDDEN_I8 | NRL_READOUT_BWD_D_HIDDEN_F32 | NRL_READOUT_BWD_D_WEIGHTS_F32 |
                           NRL_READOUT_BWD_ADD_D_HIDDEN | NRL_READOUT_BWD_ADD_D_WEIGHTS;
    if (a->flags & ~known) return NRL_E_BAD_ARG;
    if (a->V % 8 != 0 || a->d % 8 != 0 || ((a->hidden | a->weights | a->d_hidden | a->d_weights) & 15u)) return NRL_E_UNSUPPORTED;
    if (a->V > 0x40000000u || a->d > 0x40000000u || a->rows > 0x40000000ull) return NRL_E_UNSUPPORTED;  // TMA coordinates are 32-bit
    if (!a->g_logp && !a->g_ent) return NRL_E_BAD_ARG;
    if ((a->g_logp && !a->tokens) || (a->g_ent && !a->entropy)) return NRL_E_BAD_ARG;
    if ((a->rowstats & 15u) || ((a->tokens | a->entropy | a->g_logp | a->g_ent | a->hidden_scales) & 3u) || (a->workspace & 255u)) return NRL_E_BAD_ARG;
    if (a->reserved != 0 || !(a->temperature >= 0.f) || !isfinite(a->temperature)) return NRL_E_BAD_ARG;
    const bool i8 = (a->flags & NRL_READOUT_BWD_HIDDEN_I8) != 0;
    if (i8 ? (!a->hidden_scales || a->hidden_pitch < a->d || a->hidden_pitch % 16 != 0) : (a->hidden_scales || (a->hidden_pitch != 0 && a->hidden_pitch != a->d))) return NRL_E_BAD_ARG;
    if (bad_mask(a->flags, a->allow_mask, a->allow_row_stride, a->V)) return NRL_E_BAD_ARG;
    int rc = need_cc10();
    if (rc) return rc;
    const BwdPlan b = bwd_plan(a->rows, a->V, a->d);
    if (!a->workspace || a->workspace_bytes < b.bytes) return NRL_E_WORKSPACE;
    const cudaStream_t st = (cudaStream_t)stream;
    const uint64_t ws = a->workspace;
    const bool vd = (a->flags & NRL_READOUT_W_VD) != 0;
    const float tau = a->temperature == 0.f ? 1.f : a->temperature;

    HeadRows hr;
    memset(&hr, 0, sizeof hr);
    hr.rows = a->rows;
    hr.d = a->d;
    hr.g_logp = (const float*)a->g_logp;
    hr.g_ent = (const float*)a->g_ent;
    hr.rowstats = (const float*)a->rowstats;
    hr.entropy = (const float*)a->entropy;
    hr.tokens = (const int32_t*)a->tokens;
    hr.tau = tau;
    hr.hidden = (const void*)a->hidden;
    hr.pitch = a->hidden_pitch;
    hr.scales = i8 ? (const float*)a->hidden_scales : nullptr;
    hr.count = (uint32_t*)ws;
    hr.alpha = (float*)(ws + 4);
    hr.coef = (float4*)(ws + b.off_coef);
    hr.more = (float4*)(ws + b.off_more);
    hr.rows_at = (uint32_t*)(ws + b.off_rows);
    hr.x = (uint16_t*)(ws + b.off_x);
    hr.x_pitch = (uint32_t)up(a->d, 64);
    hr.d_hidden = (a->flags & NRL_READOUT_BWD_ADD_D_HIDDEN) ? nullptr : (void*)a->d_hidden;
    hr.d_hidden_f32 = (a->flags & NRL_READOUT_BWD_D_HIDDEN_F32) ? 1u : 0u;
    rc = launch_rows(hr, st);
    if (rc) return rc;

    HeadGemm g;
    memset(&g, 0, sizeof g);
    g.bn = 256;
    g.group_m = 16;
    g.coef = hr.coef;
    g.more = hr.more;
    g.rows_at = hr.rows_at;
    g.zscale = logit_scale(a->d, tau);
    g.entropy_term = a->g_ent ? 1u : 0u;
    set_mask(g, a->allow_mask, a->allow_row_stride);
    const uint32_t allow_bits = a->flags & NRL_READOUT_MASK_BITS;
    g.vocab = a->V;
    g.alpha = hr.alpha;

    const uint64_t x = ws + b.off_x, dz = ws + b.off_dz;
    // boxes of 64 elements of K × 128 rows, or of 64 columns × 64 elements of K; the weight is read along K by one product and across
    // it by the other
    const uint64_t w_in = vd ? a->d : a->V, w_rows = vd ? a->V : a->d;
    CUtensorMap x_k, x_mn, w_rows_k, w_k, w_mn, dz_k, dz_mn, dz_out, dw_out;
    const bool dw32 = (a->flags & NRL_READOUT_BWD_D_WEIGHTS_F32) != 0;
    memset(&dw_out, 0, sizeof dw_out);
    if ((rc = encode_2d(&x_k, false, x, a->d, b.rows_pad, hr.x_pitch, 64, 128)) || (rc = encode_2d(&x_mn, false, x, a->d, b.rows_pad, hr.x_pitch, 64, 64)) ||
        (rc = encode_2d(&dz_k, false, dz, b.vc, b.rows_pad, b.vc, 64, 128)) || (rc = encode_2d(&dz_mn, false, dz, b.vc, b.rows_pad, b.vc, 64, 64)) ||
        (rc = encode_2d(&dz_out, false, dz, b.vc, b.rows_pad, b.vc, 64, 32)) || (rc = vd ? encode_2d(&w_rows_k, false, a->weights, w_in, w_rows, w_in, 64, b.single ? b.grad_bn : b.grad_bn / 2) : encode_2d(&w_k, false, a->weights, w_in, w_rows, w_in, 64, b.single ? b.hidden_bn : b.hidden_bn / 2)) ||
        (rc = encode_2d(&w_mn, false, a->weights, w_in, w_rows, w_in, 64, 64)))
        return rc;
    if (a->d_weights) {
        rc = dw32 ? encode_2d_f32(&dw_out, a->d_weights, vd ? a->d : a->V, vd ? a->V : a->d, 32, 32) : encode_2d(&dw_out, false, a->d_weights, vd ? a->d : a->V, vd ? a->V : a->d, vd ? a->d : a->V, 64, 32);
        if (rc) return rc;
    }

    for (uint32_t piece = 0; piece < b.pieces; piece++) {
        const uint32_t v0 = piece * b.vc, cols = a->V - v0 < b.vc ? a->V - v0 : b.vc;
        {  // dz of this piece: x [count, d] · W[:, v0 …]
            HeadGemm p = g;
            p.m = (uint32_t)a->rows;
            p.m_count = hr.count;
            p.n = cols;
            p.k = a->d;
            p.b_mn = vd ? 0u : 1u;
            p.b_n0 = v0;
            p.v0 = v0;
            p.bn = b.grad_bn;
            rc = launch_masked<kEpiGrad>(b.single, x_k, vd ? w_rows_k : w_mn, dz_out, p, allow_bits, tiles_of(a->rows, cols, p.bn), st);
            if (rc) return rc;
        }
        if (a->d_hidden) {  // dx += dz · Wᵀ
            HeadGemm p = g;
            p.m = (uint32_t)a->rows;
            p.m_count = hr.count;
            p.n = a->d;
            p.k = cols;
            p.b_mn = vd ? 1u : 0u;
            p.b_k0 = v0;
            p.bn = b.hidden_bn;
            p.split = b.may_split ? b.chunks : 0u;
            p.acc = (float*)(ws + b.off_acc);
            p.acc_in = piece > 0 ? 1u : 0u;
            p.acc_out = piece + 1 < b.pieces ? 1u : 0u;
            p.out = (void*)a->d_hidden;
            p.out_pitch = a->d;
            p.out_f32 = hr.d_hidden_f32;
            p.out_add = (a->flags & NRL_READOUT_BWD_ADD_D_HIDDEN) ? 1u : 0u;
            p.wide = (a->d_hidden % 32 == 0 && (p.out_f32 || a->d % 16 == 0)) ? 1u : 0u;
            rc = launch_gemm<kEpiHidden>(b.single, dz_k, vd ? w_mn : w_k, dz_out, p, b.may_split ? 2 * kPairs : tiles_of(a->rows, a->d, p.bn), st);
            if (rc) return rc;
            if (b.may_split && piece + 1 == b.pieces) {
                const uint64_t most = (a->rows < (uint64_t)kPairs * 256 ? a->rows : (uint64_t)kPairs * 256) * ((a->d + 127) / 128);  // more rows are never split
                rc = launch(head_fold_kernel, dim3((unsigned)(most < 8 * 148 ? most : 8 * 148)), 256, 0, st, hr.count, hr.alpha, hr.more, hr.rows_at, p.acc, b.chunks, b.side_by_side, b.hidden_bn, a->d, (void*)a->d_hidden, p.out_f32, p.out_add);
                if (rc) return rc;
            }
        }
        if (a->d_weights) {  // dW[:, v0 …] = xᵀ · dz, or its transpose
            HeadGemm p = g;
            p.m = vd ? cols : a->d;
            p.n = vd ? a->d : cols;
            p.k = (uint32_t)a->rows;
            p.k_count = hr.count;
            p.b_mn = 1u;
            p.out = (void*)a->d_weights;
            p.out_pitch = vd ? a->d : a->V;
            p.out_row0 = vd ? v0 : 0u;
            p.out_col0 = vd ? 0u : v0;
            p.out_f32 = dw32 ? 1u : 0u;
            p.out_add = (a->flags & NRL_READOUT_BWD_ADD_D_WEIGHTS) ? 1u : 0u;
            p.wide = (a->d_weights % 32 == 0 && (p.out_f32 || p.out_pitch % 16 == 0)) ? 1u : 0u;
            p.staged = p.out_add ? 0u : 1u;  // sums into what is there go through registers
            p.bn = tile_width(p.m, p.n, false);
            rc = launch_tiles<kEpiWeight, kMaskNone, true>(vd ? dz_mn : x_mn, vd ? x_mn : dz_mn, dw_out, p, tiles_of(p.m, p.n, p.bn), st);
            if (rc) return rc;
        }
    }
    return NRL_OK;
}

// ---- forward over the scored rows -----------------------------------------------------------------------

// 512 threads for up to four positions each (1.8 us against 2.8 with 1024), else 1024 (8192 positions of a seed: 6.3 us against 9.7)
static int mean_of_log_probs(const CeMean& ce, cudaStream_t st) { return launch(ce_mean_kernel, dim3((unsigned)ce.seeds), ce.n <= 2048 ? 512u : (unsigned)kMeanThreads, 0, st, ce); }
// The loss of a small call is taken by the merge's last block: 0.6 us more on the device for 64 positions (a launch of its own takes the
// host 3 us, and such a call waits for the host). Else a launch with a block per seed: that last block took 10 us longer for 8192
// positions, and 4 us longer for four seeds of 64.
static bool mean_at_the_end(uint64_t seeds, uint64_t rows) { return seeds <= 2 && rows <= 512; }
constexpr uint64_t kScoredChunk = 16384;  // rows per launch: what bounds the partial statistics' scratch (16 bytes per row and 128 columns)

struct ScoredPlan {
    bool gather;  // the scored rows are brought together first
    bool single;
    uint32_t bn, parts_pitch;
    uint64_t rows_pad, off_rows, off_x, off_parts, bytes;
};
static ScoredPlan scored_plan(uint64_t rows, uint32_t V, uint32_t d, bool scored) {
    ScoredPlan s;
    s.gather = scored && rows > 256;  // up to one row block nothing is saved by leaving rows out
    s.rows_pad = up(rows, 256);
    s.single = runs_single(rows);
    s.bn = tile_width(rows, V, s.single);
    s.parts_pitch = 2 * ((V + s.bn - 1) / s.bn);
    uint64_t at = 256;
    s.off_rows = at; at += s.gather ? up(rows * 4, 256) : 0;
    s.off_x = at; at += s.gather ? s.rows_pad * up(d, 64) * 2 : 0;
    s.off_parts = at; at += (s.rows_pad < kScoredChunk ? s.rows_pad : kScoredChunk) * s.parts_pitch * 16;
    s.bytes = at;
    return s;
}

extern "C" uint64_t nrl_readout_scored_workspace_bytes(uint64_t rows, uint32_t V, uint32_t d, uint32_t has_scored) {
    if (rows == 0 || V == 0 || d == 0) return 0;
    return scored_plan(rows, V, d, has_scored != 0).bytes;
}

extern "C" int nrl_readout_scored_fwd(const nrl_readout_scored_args* a, nrl_stream stream) {
    if (!a || a->struct_size != sizeof(nrl_readout_scored_args)) return NRL_E_BAD_ARG;
    if (a->rows == 0 || a->V == 0 || a->d == 0 || !a->hidden || !a->weights || !a->rowstats) return NRL_E_BAD_ARG;
    if (a->flags & ~(uint32_t)(NRL_READOUT_W_VD | NRL_READOUT_MASK_BITS)) return NRL_E_BAD_ARG;
    if (a->V % 8 != 0 || a->d % 8 != 0 || ((a->hidden | a->weights) & 15u)) return NRL_E_UNSUPPORTED;
    if (a->V > 0x40000000u || a->d > 0x40000000u || a->rows > 0x40000000ull) return NRL_E_UNSUPPORTED;  // TMA coordinates are 32-bit
    if (((a->tokens | a->scored | a->logp | a->entropy) & 3u) || (a->rowstats & 15u) || (a->workspace & 255u)) return NRL_E_BAD_ARG;
    if (a->logp && !a->tokens) return NRL_E_BAD_ARG;
    if (a->seeds ? (!a->logp || a->rows % a->seeds != 0 || (!a->ce_loss && !a->ce_g_logp) || ((a->ce_loss | a->ce_g_logp | a->ce_weights) & 3u)) : (a->ce_loss || a->ce_g_logp || a->ce_weights)) return NRL_E_BAD_ARG;
    if (a->reserved != 0 || !(a->temperature >= 0.f) || !isfinite(a->temperature)) return NRL_E_BAD_ARG;
    if (bad_mask(a->flags, a->allow_mask, a->allow_row_stride, a->V)) return NRL_E_BAD_ARG;
    int rc = need_cc10();
    if (rc) return rc;
    const ScoredPlan s = scored_plan(a->rows, a->V, a->d, a->scored != 0);
    if (!a->workspace || a->workspace_bytes < s.bytes) return NRL_E_WORKSPACE;
    const cudaStream_t st = (cudaStream_t)stream;
    const uint64_t ws = a->workspace;
    const bool vd = (a->flags & NRL_READOUT_W_VD) != 0;
    if (s.gather) {
        HeadRows hr;
        memset(&hr, 0, sizeof hr);
        hr.rows = a->rows;
        hr.d = a->d;
        hr.scored = (const float*)a->scored;
        hr.tau = 1.f;
        hr.hidden = (const void*)a->hidden;
        hr.count = (uint32_t*)ws;
        hr.rows_at = (uint32_t*)(ws + s.off_rows);
        hr.x = (uint16_t*)(ws + s.off_x);
        hr.x_pitch = (uint32_t)up(a->d, 64);
        hr.logp = (float*)a->logp;
        hr.out_entropy = (float*)a->entropy;
        hr.out_rowstats = (float4*)a->rowstats;
        hr.status = (uint8_t*)a->status;
        rc = launch_rows(hr, st);
        if (rc) return rc;
    }
    CUtensorMap mx, mw;
    rc = encode_2d(&mx, false, s.gather ? ws + s.off_x : a->hidden, a->d, s.gather ? s.rows_pad : a->rows, s.gather ? up(a->d, 64) : a->d, 64, 128);
    if (rc) return rc;
    rc = vd ? encode_2d(&mw, false, a->weights, a->d, a->V, a->d, 64, s.single ? s.bn : s.bn / 2) : encode_2d(&mw, false, a->weights, a->V, a->d, a->V, 64, 64);
    if (rc) return rc;
    const CeMean ce = {a->seeds, a->seeds ? a->rows / a->seeds : 0, (const float*)a->logp, (const float*)a->scored, (const float*)a->ce_weights, nullptr, (float*)a->ce_loss, (float*)a->ce_g_logp};
    for (uint64_t r0 = 0; r0 < a->rows; r0 += kScoredChunk) {
        const uint64_t n = a->rows - r0 < kScoredChunk ? a->rows - r0 : kScoredChunk;
        HeadGemm p;
        memset(&p, 0, sizeof p);
        p.bn = s.bn;
        p.group_m = 16;
        p.m = (uint32_t)n;
        p.m_count = s.gather ? (const uint32_t*)ws : nullptr;
        p.m_first = (uint32_t)r0;
        p.a_m0 = (uint32_t)r0;
        p.n = a->V;
        p.k = a->d;
        p.b_mn = vd ? 0u : 1u;
        p.rows_at = s.gather ? (const uint32_t*)(ws + s.off_rows) + r0 : nullptr;
        p.tokens = a->tokens ? (const int32_t*)a->tokens + (s.gather ? 0 : r0) : nullptr;
        p.zscale = logit_scale(a->d, a->temperature == 0.f ? 1.f : a->temperature);
        p.entropy_term = a->entropy ? 1u : 0u;
        set_mask(p, a->allow_mask, a->allow_row_stride);
        if (!s.gather && a->allow_mask) p.allow += r0 * a->allow_row_stride * ((a->flags & NRL_READOUT_MASK_BITS) ? 4u : 1u);
        p.vocab = a->V;
        p.zero = (uint32_t*)(ws + 8);
        p.parts = (float4*)(ws + s.off_parts);
        p.parts_pitch = s.parts_pitch;
        rc = launch_masked<kEpiStats>(s.single, mx, mw, mx, p, a->flags & NRL_READOUT_MASK_BITS, tiles_of(n, a->V, s.bn), st);
        if (rc) return rc;
        HeadFinish f;
        memset(&f, 0, sizeof f);
        f.rows = (uint32_t)n;
        f.count = p.m_count;
        f.first = (uint32_t)r0;
        f.rows_at = p.rows_at;
        const uint64_t at = s.gather ? 0 : r0;
        f.scored = a->scored ? (const float*)a->scored + at : nullptr;
        f.parts = p.parts;
        f.nparts = p.parts_pitch;
        f.logp = a->logp ? (float*)a->logp + at : nullptr;
        f.entropy = a->entropy ? (float*)a->entropy + at : nullptr;
        f.rowstats = (float4*)a->rowstats + at;
        f.status = a->status ? (uint8_t*)a->status + at : nullptr;
        if (a->seeds && mean_at_the_end(a->seeds, a->rows)) {  // one launch of rows then
            f.ce = ce;
            f.done = (uint32_t*)(ws + 8);
        }
        rc = n <= 8 * 148 ? launch(head_finish_kernel<8>, dim3((unsigned)n), 256, 0, st, f) : launch(head_finish_kernel<1>, dim3((unsigned)((n + 7) / 8)), 256, 0, st, f);
        if (rc) return rc;
    }
    if (a->seeds && !mean_at_the_end(a->seeds, a->rows)) return mean_of_log_probs(ce, st);
    return NRL_OK;
}

extern "C" int nrl_ce_mean(uint64_t s, uint64_t n, nrl_devptr logp, nrl_devptr keep, nrl_devptr upstream, nrl_devptr out, nrl_devptr g_logp, nrl_stream stream) {
    if (s == 0 || n == 0 || (!out && !g_logp) || (out && !logp)) return NRL_E_BAD_ARG;
    if ((logp | keep | upstream | out | g_logp) & 3u) return NRL_E_BAD_ARG;
    if (s > 0x7fffffffull) return NRL_E_UNSUPPORTED;
    return mean_of_log_probs(CeMean{s, n, (const float*)logp, (const float*)keep, nullptr, (const float*)upstream, (float*)out, (float*)g_logp}, (cudaStream_t)stream);
}

// ---- 8-bit integers -----------------------------------------------------------------------------------

extern "C" int nrl_i8_quantize_rows(uint32_t dtype, uint64_t rows, uint32_t d, nrl_devptr x, nrl_devptr values, uint64_t pitch, nrl_devptr scales, nrl_stream stream) {
    if (rows == 0 || d == 0 || !x || !values || !scales || (scales & 3u)) return NRL_E_BAD_ARG;
    if (dtype != NRL_F32 && dtype != NRL_BF16) return NRL_E_UNSUPPORTED;
    if (pitch < d || pitch % 16 != 0 || (values & 15u) || (x & (dtype == NRL_F32 ? 3u : 1u))) return NRL_E_BAD_ARG;
    if (rows > 0x7fffffffull) return NRL_E_UNSUPPORTED;
    const bool vec = d % 8 == 0 && (x & 15u) == 0;
    const cudaStream_t st = (cudaStream_t)stream;
    const void* xp = (const void*)x;
    int8_t* q = (int8_t*)values;
    float* sp = (float*)scales;
    // a warp per row where that fills the device and the rows in flight stay in L2 for their second look (8192 rows: 30 against 35 us
    // for 8 KB of bf16, 53 against 35 for 16 KB of f32)
    const bool many = rows >= 8 * 148 && (uint64_t)d * (dtype == NRL_F32 ? 4 : 2) <= 8192;
    const unsigned grid = (unsigned)(many ? (rows + 7) / 8 : rows);
    const dim3 g(grid);
    if (dtype == NRL_BF16) return many ? launch(quantise_rows_kernel<NRL_BF16, 1>, g, 256, 0, st, xp, rows, d, pitch, q, sp, vec) : launch(quantise_rows_kernel<NRL_BF16, 8>, g, 256, 0, st, xp, rows, d, pitch, q, sp, vec);
    return many ? launch(quantise_rows_kernel<NRL_F32, 1>, g, 256, 0, st, xp, rows, d, pitch, q, sp, vec) : launch(quantise_rows_kernel<NRL_F32, 8>, g, 256, 0, st, xp, rows, d, pitch, q, sp, vec);
}

extern "C" int nrl_i8_quantize_columns(uint32_t d, uint32_t V, nrl_devptr weights, nrl_devptr values, uint64_t pitch, nrl_devptr scales, nrl_stream stream) {
    if (d == 0 || V == 0 || !weights || !values || !scales || (scales & 3u) || (weights & 1u)) return NRL_E_BAD_ARG;
    if (pitch < d || pitch % 16 != 0 || (values & 15u)) return NRL_E_BAD_ARG;
    return launch(quantise_columns_kernel, dim3((V + 63) / 64), 256, 0, (cudaStream_t)stream, (const uint16_t*)weights, d, V, pitch, (int8_t*)values, (float*)scales);
}

extern "C" int nrl_i8_dequantize_rows(uint32_t dtype, uint64_t rows, uint32_t d, nrl_devptr values, uint64_t pitch, nrl_devptr scales, nrl_devptr out, nrl_stream stream) {
    if (rows == 0 || d == 0 || !values || !scales || !out || (scales & 3u)) return NRL_E_BAD_ARG;
    if (dtype != NRL_F32 && dtype != NRL_BF16) return NRL_E_UNSUPPORTED;
    if (pitch < d || (out & (dtype == NRL_F32 ? 3u : 1u))) return NRL_E_BAD_ARG;
    if (rows > 0x7fffffffull) return NRL_E_UNSUPPORTED;
    return launch(dequantise_rows_kernel, dim3((unsigned)rows), 256, 0, (cudaStream_t)stream, (const int8_t*)values, (const float*)scales, d, pitch, (void*)out, dtype == NRL_F32 ? 1u : 0u);
}

static int i8_check(const nrl_i8_matmul_args* a) {
    if (!a || a->struct_size != sizeof(nrl_i8_matmul_args)) return NRL_E_BAD_ARG;
    if (a->rows == 0 || a->n == 0 || a->k == 0 || !a->x || !a->x_scales || !a->w || !a->w_scales || !a->out) return NRL_E_BAD_ARG;
    if (a->dtype != NRL_F32 && a->dtype != NRL_BF16) return NRL_E_UNSUPPORTED;
    if (a->x_pitch < a->k || a->w_pitch < a->k || a->x_pitch % 16 != 0 || a->w_pitch % 16 != 0 || ((a->x | a->w) & 15u) || ((a->x_scales | a->w_scales) & 3u) ||
        (a->out & (a->dtype == NRL_F32 ? 3u : 1u)))
        return NRL_E_BAD_ARG;
    if (a->rows > 0x40000000ull || a->n > 0x40000000u) return NRL_E_UNSUPPORTED;  // TMA coordinates are 32-bit
    if (a->k > 131072u) return NRL_E_UNSUPPORTED;                                  // 127·127·k must fit 31 bits
    return need_cc10();
}

extern "C" uint64_t nrl_i8_linear_workspace_bytes(uint64_t rows, uint32_t k) { return up(rows * 4, 256) + rows * up(k, 128); }

extern "C" int nrl_i8_linear(uint32_t x_dtype, const nrl_i8_matmul_args* a, nrl_devptr workspace, uint64_t workspace_bytes, nrl_stream stream) {
    if (!a || a->struct_size != sizeof(nrl_i8_matmul_args) || a->x_scales || a->x_pitch) return NRL_E_BAD_ARG;
    if (a->rows == 0 || a->k == 0 || (workspace & 255u)) return NRL_E_BAD_ARG;
    if (!workspace || workspace_bytes < nrl_i8_linear_workspace_bytes(a->rows, a->k)) return NRL_E_WORKSPACE;
    nrl_i8_matmul_args q = *a;
    q.x_scales = workspace;
    q.x = workspace + up(a->rows * 4, 256);
    q.x_pitch = up(a->k, 128);  // TMA reads then cover whole lines
    int rc = i8_check(&q);  // nothing is launched for a product that is refused
    if (rc) return rc;
    rc = nrl_i8_quantize_rows(x_dtype, a->rows, a->k, a->x, q.x, q.x_pitch, q.x_scales, stream);
    return rc ? rc : nrl_i8_matmul(&q, stream);
}

extern "C" int nrl_i8_matmul(const nrl_i8_matmul_args* a, nrl_stream stream) {
    int rc = i8_check(a);
    if (rc) return rc;
    // M = the weight's rows, N = the tokens: few tokens make a narrow tile, and the weight streams through it
    HeadGemm p;
    memset(&p, 0, sizeof p);
    const uint64_t tiles_n = (a->rows + 255) / 256;
    p.bn = (uint32_t)up((a->rows + tiles_n - 1) / tiles_n, 32);
    p.m = a->n;
    p.n = (uint32_t)a->rows;
    p.k = a->k;
    p.group_m = 16;
    p.m_scale = (const float*)a->w_scales;
    p.n_scale = (const float*)a->x_scales;
    p.out = (void*)a->out;
    p.out_pitch = a->n;
    p.out_f32 = a->dtype == NRL_F32 ? 1u : 0u;
    CUtensorMap mw, mx;
    // the extent along K is k, not the pitch: what lies behind a row's k integers is read as zeros
    rc = encode_2d(&mw, true, a->w, a->k, a->n, a->w_pitch, 128, 128);
    if (rc) return rc;
    rc = encode_2d(&mx, true, a->x, a->k, a->rows, a->x_pitch, 128, p.bn / 2);
    if (rc) return rc;
    return launch_tiles<kEpiInt8, kMaskNone, true>(mw, mx, mw, p, (uint64_t)tiles256(a->n) * ((a->rows + p.bn - 1) / p.bn), (cudaStream_t)stream);
}

// The matrix products of the readout's backward pass and of its 8-bit form: one kernel on CTA pairs
// (tcgen05.mma.cta_group::2, f32 or 32-bit integer accumulators in tensor memory), five epilogues.
//
//   kEpiStats   z = x · W for the scored rows x; the epilogue keeps, per row and half tile, the maximum,
//               Σ exp(z − max), Σ exp(z − max)·(z − max) and the given token's logit
//   kEpiGrad    z = x · W for the scored rows x and a piece of the vocabulary; the epilogue turns the
//               accumulators into dz = ∂/∂z of the per-row terms and writes them as bf16:
//               π_j = exp((z_j − m) − ln Z), dz_j = a·1[j = token] − π_j·(a + b·(ln π_j + H)).
//               The logits themselves are never written.
//   kEpiHidden  dx = dz · Wᵀ over a piece of the vocabulary (f32 sums carried from piece to piece)
//   kEpiWeight  dW = xᵀ · dz for a piece of the vocabulary
//   kEpiInt8    z[r, v] = s_r·w_v·Σ_k q[r, k]·p[v, k] in 8-bit integers (sums exact in 32 bits)
//
// A pair of CTAs (tcgen05 cta_group::2) owns 256 rows × `bn` columns of the output; each CTA loads its 128 rows of A and half
// of B per stage (TMA, 128-byte swizzle, no multicast), one thread of the first CTA issues the products
// for both, and the 256-column accumulators are double-buffered so that a tile's epilogue runs under the
// next tile's products. The grid is persistent: 74 pairs walk the tiles in a fixed order, so every sum
// has a fixed order and results are bitwise reproducible. A and B may each be contiguous along K or along
// their other axis (the descriptors' major bits), so dz, x and W are read as they lie in memory. With at most 128 rows every CTA
// works by itself (cta_group::1, PAIR = false): a pair would multiply 128 rows of zeros, and the pass is then bound by the weight's
// bytes instead of the tensor pipe.
//
// Bound: the tensor pipe for the large products (1536 rows, V = 32 000, d = 2048: 130 to 138 us each, the pipe busy 76 to 84 % of the
// time at the clock that power leaves, 1.53 GHz), HBM for the few-row forms (87 rows, V = 151 936, d = 2048: 98 to 115 us for the
// weight's 622 MB, which each reads once; d_weights writes as much in 158 us, what a fill takes; 8 bits, one token, V = 128 256,
// d = 4096: 86 us, 6.1 TB/s). Waits are bounded as in the readout forward; a role that gives up raises its
// CTA's abort flag, on which that CTA's other roles stop (the partner's stop at their own limit), and the tiles not reached are
// written as NaN.
#pragma once
#include "tcgen05.cuh"

namespace nrl {

constexpr int kHgBM = 128;           // rows per CTA (256 per pair)
constexpr int kHgEpiWarps = 8;       // two per quarter of tensor memory: each takes half of the columns
constexpr int kHgThreads = 64 + 32 * kHgEpiWarps;
constexpr uint32_t kHgABytes = kHgBM * 128;      // one stage of A: 128 rows × 128 bytes of K
constexpr uint32_t kHgMaxStages = 10;
constexpr uint32_t kHgStageOut = 4096;           // 32 rows × 128 bytes of an epilogue warp's results on their way out
// bytes of input stages: six of 32 KB at bn = 256, more when B is narrower. A second staging tile per warp in the place of the sixth
// stage cost dW 1 to 6 %.
constexpr uint32_t kHgSmemTiles = 6 * 2 * kHgABytes;
constexpr uint32_t kHgSmemBytes = kHgSmemTiles + kHgEpiWarps * kHgStageOut + 1024 + 256;

template <bool V>
struct Const {
    static constexpr bool value = V;
};
enum { kEpiGrad = 0, kEpiHidden = 1, kEpiWeight = 2, kEpiInt8 = 3, kEpiStats = 4 };
enum { kMaskNone = 0, kMaskBytes = 1, kMaskBits = 2 };

// An accumulator drops what lies below its last bit at each of the d / 16 steps that add into it, toward zero: a sum comes out
// smaller by 1.6e-8 of itself per step on average (measured: 2.4e-7, 1.0e-6, 2.1e-6, 4.1e-6 of the row maximum at
// d = 256, 1024, 2048, 4096, the expectation for partial sums that grow in proportion to the step). The logits are scaled back.
constexpr float kAccumulatorLoss = 1.6e-8f;
inline float logit_scale(uint32_t d, float tau) { return (1.f + kAccumulatorLoss * (float)((d + 15) / 16)) / tau; }

// Ranges of K in dx = dz·Wᵀ for `tiles` tiles of dx and `chunks` steps of K: with few tiles the steps of a tile go to several
// pairs (or single CTAs), whose sums are added afterwards. As many ranges as fill one wave of those, or two where that takes 5 % fewer steps, each of
// at least 12 steps (201 rows at V = 4104, d = 512: dz, dx and the adding-up 33 us with at least 24, 27 with 12; with 8, 140 rows at
// V = 1120 took 10 % longer). Decided where the number of scored rows is known, on
// the device, and the same there and in the kernel that adds up.
constexpr uint32_t kPairs = 74;  // CTA pairs that run side by side (148 SMs)
__host__ __device__ inline uint32_t hidden_split(uint32_t tiles, uint32_t chunks, uint32_t side_by_side) {
    if (tiles == 0 || tiles > side_by_side) return 1u;
    const uint32_t most = chunks / 12u, a = side_by_side / tiles, b = 2 * side_by_side / tiles;
    const uint32_t one = most < a ? (most ? most : 1u) : a, two = most < b ? (most ? most : 1u) : b;  // steps of a tile: 1 / one, or 2 / two
    return 200u * one < 95u * two ? two : one;
}

// n / d for n < 2^32 without a division: m = floor((2^32 − 1) / d) gives the quotient or one less.
struct FastDiv {
    uint32_t d, m;
    __device__ __forceinline__ explicit FastDiv(uint32_t by) : d(by), m(by > 1u ? 0xffffffffu / by : 0u) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        if (d <= 1u) return n;
        const uint32_t q = __umulhi(n, m);
        return n - q * d >= d ? q + 1u : q;
    }
};

struct HeadGemm {
    uint32_t m, n, k;          // extents of the product
    const uint32_t* m_count;   // device: the rows in use along M, of which this launch takes m from m_first on; or null: all m
    uint32_t m_first;
    const uint32_t* k_count;   // device: the extent along K (≤ k), or null
    uint32_t bn;               // columns per tile: 256 or 128, kEpiInt8 a multiple of 32 up to 256
    uint32_t stages;
    uint32_t b_mn;             // B contiguous along N instead of K (kEpiWeight: both operands always lie across K; A of the others never)
    uint32_t b_n0, b_k0;       // where this piece of the vocabulary begins in B, along N / along K
    uint32_t a_m0;             // … in A, along M
    uint32_t split;            // kEpiHidden: ranges of K, each with its own output buffer, where that fills the device better (hidden_split); the steps of K that rule is given, 0: never
    uint32_t group_m;          // 256-row blocks that are walked side by side (L2 reuse of B)
    // kEpiGrad, kEpiStats
    const float4* coef;        // kEpiGrad [rows] of the scored rows: (a·xs, b·xs, (m + ln Z)·log2 e, a·xs + b·xs·H)
    const float4* more;        // [rows] (xs, 1 / xs, token bits, ·): xs is the scale of an 8-bit row, else 1
    const uint32_t* rows_at;   // [rows] the row in the caller's order, or null: the same
    const int32_t* tokens;     // kEpiStats [rows in the caller's order] or null
    float zscale;              // logit = accumulator · zscale (· xs)
    uint32_t entropy_term;     // kEpiGrad: some b ≠ 0 is possible; kEpiStats: the entropy sum is wanted
    uint32_t* zero;            // kEpiStats: a counter that the kernel behind this one starts from
    const uint8_t* allow;
    uint64_t allow_stride;
    uint32_t allow_wide;       // every row of the byte mask is 4-byte aligned
    uint32_t vocab;            // V
    uint32_t v0;               // first column of this piece
    float4* parts;             // kEpiStats [rows, parts_pitch]: (max, sum, entropy sum, token's logit) per half tile
    uint32_t parts_pitch;
    // kEpiHidden, kEpiWeight
    const float* alpha;        // device scalar
    float* acc;                // f32 sums between pieces / ranges of K: [ranges, rows in use rounded up to 256, n]
    uint32_t acc_in, acc_out;  // start from acc; end in acc (otherwise in out, unless K is split)
    void* out;
    uint64_t out_pitch;
    uint32_t out_f32, out_add; // type of `out`; add to what it holds
    uint32_t out_col0;         // kEpiWeight: first column (or first row, with out_row0) of this piece
    uint32_t out_row0;
    uint32_t wide;             // rows of out are 32-byte aligned
    uint32_t staged;           // results leave through shared memory and TMA stores (map_out)
    __host__ __device__ static uint32_t acc_rows(uint32_t rows_in_use) { return (rows_in_use + 255u) & ~255u; }
    // kEpiInt8
    const float* m_scale;      // [m]
    const float* n_scale;      // [n]
};

__device__ __forceinline__ void tc_mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void stg32(void* p, const uint32_t r[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// four bytes read once, past L1; not as read-only data: the kernel that wrote them may still run when this one starts
__device__ __forceinline__ uint32_t ldg4(const void* p) {
    uint32_t v;
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ void ldg32(const void* p, uint32_t r[8]) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p) : "memory");
}
// 128 bytes of this thread's row (lane) into the warp's staging tile, 128-byte swizzle: 16-byte piece j of row r lies at j ^ (r mod 8)
__device__ __forceinline__ void sts_piece(uint32_t stage, int lane, int j, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 128 + ((j ^ (lane & 7)) << 4)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// the warp's staging tile may be written again (its last store has read it)
__device__ __forceinline__ void stage_free(int lane) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}
// the warp's staging tile is complete: send it off
__device__ __forceinline__ void stage_send(const CUtensorMap* map, uint32_t stage, int lane, int32_t x, int32_t y) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) tma_store_2d(map, stage, x, y);
}
__device__ __forceinline__ void scale32(float* z, float by) {
    const f32x2 b2 = pack2(by, by);
#pragma unroll
    for (int i = 0; i < 32; i += 2) unpack2(mul2(pack2(z[i], z[i + 1]), b2), z[i], z[i + 1]);
}
// An arrival on a barrier of either CTA of the pair that hands tensor memory back (mbar_try_wait_pair waits for it). A release at
// this scope waits for what the thread has stored: the statistics of 2048 x 50264 x 512 took 125 us with one, 100 without.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar_cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}
// keeps what reads z behind this point
__device__ __forceinline__ void pin32(float* z) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile("" : "+f"(z[i]), "+f"(z[i + 1]), "+f"(z[i + 2]), "+f"(z[i + 3]), "+f"(z[i + 4]), "+f"(z[i + 5]), "+f"(z[i + 6]), "+f"(z[i + 7]));
}
__device__ __forceinline__ void pin16(uint32_t* z) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
        asm volatile("" : "+r"(z[i]), "+r"(z[i + 1]), "+r"(z[i + 2]), "+r"(z[i + 3]), "+r"(z[i + 4]), "+r"(z[i + 5]), "+r"(z[i + 6]), "+r"(z[i + 7]));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {  // nearest, ties to even; NaN stays NaN
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The allow-mask of the warp's 32 rows × 128 columns: loads that go out before the accumulators are waited for, and what they become
// in each lane, a bit per column of its row (columns past the vocabulary: 0). Of a byte mask the warp reads one row at a time, four
// bytes a lane, one 128-byte line per load (eight bytes a lane of 32 rows at a time touched 32 lines per load, and L1 with them: the
// product with such a mask ran at 0.66 of its rate without), and four ballots hand row r's bits to lane r: column c is bit c / 4 of
// word c mod 4. Of a bit mask each lane reads its row's four words: column c is bit c mod 32 of word c / 32.
template <int MASK>
struct MaskAhead {
    uint32_t raw[MASK == kMaskBytes ? 32 : 4];
    uint32_t keep[4];
    __device__ __forceinline__ void load(const HeadGemm& p, uint32_t caller_row, uint32_t v, bool live, int lane) {
        if constexpr (MASK == kMaskBits) {
            const uint32_t* mp = reinterpret_cast<const uint32_t*>(p.allow) + (uint64_t)caller_row * p.allow_stride + (v >> 5);
#pragma unroll
            for (int c = 0; c < 4; c++) raw[c] = live && v + 32 * c < p.vocab ? ldg4(mp + c) : 0u;
        } else if constexpr (MASK == kMaskBytes) {
            const uint32_t here = v + 4 * lane;
            const uint32_t lives = __ballot_sync(0xffffffffu, live);
            const uint8_t* mp = p.allow + here;
#pragma unroll
            for (int r = 0; r < 32; r++) {
                const uint32_t row = __shfl_sync(0xffffffffu, caller_row, r);
                const uint8_t* q = mp + (uint64_t)row * p.allow_stride;
                uint32_t x = 0u;
                if ((lives >> r & 1u) && here < p.vocab) {  // V is a multiple of 8: a lane's four columns exist or do not
                    if (p.allow_wide) x = ldg4(q);
                    else x = (uint32_t)q[0] | (uint32_t)q[1] << 8 | (uint32_t)q[2] << 16 | (uint32_t)q[3] << 24;
                }
                raw[r] = x;
            }
        }
    }
    __device__ __forceinline__ void settle(const HeadGemm& p, uint32_t v, int lane) {
        if constexpr (MASK == kMaskBytes) {
#pragma unroll
            for (int r = 0; r < 32; r++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t b = __ballot_sync(0xffffffffu, (raw[r] & (0xffu << (8 * j))) != 0u);
                    if (lane == r) keep[j] = b;
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t left = v + 32 * c < p.vocab ? p.vocab - v - 32 * c : 0u;
                const uint32_t k = left >= 32u ? 0xffffffffu : (1u << left) - 1u;
                keep[c] = MASK == kMaskBits ? k & raw[c] : k;
            }
        }
    }
    // the 32 columns from 32·c on: one word, or (bytes) eight columns in each of four
    struct Chunk {
        uint32_t w[MASK == kMaskBytes ? 4 : 1];
        __device__ __forceinline__ bool any() const {
            if constexpr (MASK == kMaskBytes) return (w[0] | w[1] | w[2] | w[3]) & 0xffu;
            return w[0] != 0u;
        }
        __device__ __forceinline__ bool all() const { return MASK != kMaskBytes && w[0] == 0xffffffffu; }
        __device__ __forceinline__ bool column(int i) const {
            if constexpr (MASK == kMaskBytes) return w[i & 3] & (1u << (i >> 2));
            return w[0] & (1u << i);
        }
    };
    __device__ __forceinline__ Chunk chunk(int c) const {
        Chunk k;
        if constexpr (MASK == kMaskBytes) {
#pragma unroll
            for (int j = 0; j < 4; j++) k.w[j] = keep[j] >> (8 * c);
        } else {
            k.w[0] = c < 2 ? (c == 0 ? keep[0] : keep[1]) : (c == 2 ? keep[2] : keep[3]);
        }
        return k;
    }
};

// What an epilogue thread needs to know of its row, fetched while the tile before is worked on.
struct RowInfo {
    uint32_t caller_row;
    int32_t token;
    float4 cf;
    float2 xs;  // scale of an 8-bit row and its inverse
    bool live;
};

// ∂/∂z of 32 columns of one row from the accumulators y, as 16 packed bf16 pairs. With the row's coefficients pre-multiplied
// (a′ = a·xs, …): ln π in units of log2 is one fused multiply-add of y, dz = −π·(a′ + b′·(ln π + H)), and the token's entry gets a′.
template <int MASK>
__device__ __forceinline__ void epi_grad(const HeadGemm& p, bool live, uint32_t v, const float y[32], const float4& cf, float ys, int32_t token, const typename MaskAhead<MASK>::Chunk& mask, uint32_t out[16]) {
    if (!live || !mask.any()) {
#pragma unroll
        for (int i = 0; i < 16; i++) out[i] = 0u;
        return;
    }
    const f32x2 ys2 = pack2(ys, ys), lse2 = pack2(-cf.z, -cf.z);
    float g[32];
    if (p.entropy_term) {
        const float nb2 = -cf.y * 0.69314718055994531f;
        const f32x2 b2 = pack2(nb2, nb2), ab2 = pack2(-cf.w, -cf.w);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float l0, l1;
            unpack2(fma2(pack2(y[i], y[i + 1]), ys2, lse2), l0, l1);
            // a −inf logit: π = 0, and 0·inf cannot appear
            unpack2(mul2(pack2(ex2_approx(l0), ex2_approx(l1)), fma2(pack2(fmaxf(l0, -1e30f), fmaxf(l1, -1e30f)), b2, ab2)), g[i], g[i + 1]);
        }
    } else {
        const f32x2 na2 = pack2(-cf.x, -cf.x);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float l0, l1;
            unpack2(fma2(pack2(y[i], y[i + 1]), ys2, lse2), l0, l1);
            unpack2(mul2(pack2(ex2_approx(l0), ex2_approx(l1)), na2), g[i], g[i + 1]);
        }
    }
    const uint32_t tk = (uint32_t)(token - (int32_t)v);
    if (tk < 32u) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if ((uint32_t)i == tk) g[i] += cf.x;
    }
    if (!mask.all()) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if (!mask.column(i)) g[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) out[i] = pack_bf16(g[2 * i], g[2 * i + 1]);
}

// 32 columns of one row folded into (m, S, W): m in accumulator units, W in units of log2.
template <int MASK>
__device__ __forceinline__ void epi_stats(const HeadGemm& p, uint32_t v, float y[32], float c2, int32_t token, const typename MaskAhead<MASK>::Chunk& mask, float& m, float& S, float& W, float& ytok) {
    const uint32_t tk = (uint32_t)(token - (int32_t)v);
    if (!mask.any()) {
        if (tk < 32u) ytok = -FLT_MAX;  // the token itself is excluded
        return;
    }
    if (!mask.all()) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if (!mask.column(i)) y[i] = -FLT_MAX;
    }
    if (tk < 32u) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if ((uint32_t)i == tk) ytok = y[i];
    }
    float c4[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        c4[k] = fmax3_nan(y[8 * k], y[8 * k + 1], y[8 * k + 2]);
        c4[k] = fmax3_nan(c4[k], y[8 * k + 3], y[8 * k + 4]);
        c4[k] = fmax3_nan(c4[k], y[8 * k + 5], fmax_nan(y[8 * k + 6], y[8 * k + 7]));
    }
    const float cm = fmax_nan(fmax3_nan(c4[0], c4[1], c4[2]), c4[3]);
    if (cm <= -FLT_MAX) return;  // every column here is excluded or −inf (a NaN goes on)
    if (!(cm <= m)) {
        if (m > -FLT_MAX) {
            const float dm = (m - cm) * c2, sc = ex2_approx(dm);
            W = (W + S * dm) * sc;
            S *= sc;
        }
        m = fmax_nan(m, cm);  // a NaN stays: the sums it went into must not be taken for the other columns'
    }
    const float m2 = -m * c2;
    const f32x2 c22 = pack2(c2, c2), m22 = pack2(m2, m2);
    f32x2 s0 = pack2(0.f, 0.f), s1 = s0, w0 = s0, w1 = s0;
    if (p.entropy_term) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float t0, t1;
            unpack2(fma2(pack2(y[i], y[i + 1]), c22, m22), t0, t1);
            t0 = fmaxf(t0, -1e30f);
            t1 = fmaxf(t1, -1e30f);
            const f32x2 e = pack2(ex2_approx(t0), ex2_approx(t1)), t = pack2(t0, t1);
            if (i & 2) { s1 = add2(s1, e); w1 = fma2(e, t, w1); }
            else { s0 = add2(s0, e); w0 = fma2(e, t, w0); }
        }
        float a0, a1;
        unpack2(add2(w0, w1), a0, a1);
        W += a0 + a1;
    } else {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float t0, t1;
            unpack2(fma2(pack2(y[i], y[i + 1]), c22, m22), t0, t1);
            const f32x2 e = pack2(ex2_approx(t0), ex2_approx(t1));
            if (i & 2) s1 = add2(s1, e);
            else s0 = add2(s0, e);
        }
    }
    float a0, a1;
    unpack2(add2(s0, s1), a0, a1);
    S += a0 + a1;
}

// 32 consecutive results of one output row to `out` (bf16 or f32), added to what it holds if asked.
// `left` columns exist; `wide`: the row start is 32-byte aligned.
__device__ __forceinline__ void store_row32(void* out, uint64_t at, bool f32, bool add, bool wide, uint32_t left, const float y[32]) {
    if (left >= 32 && wide) {
        if (f32) {
            float* o = reinterpret_cast<float*>(out) + at;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t r[8];
                if (add) ldg32(o + 8 * c, r);
#pragma unroll
                for (int i = 0; i < 8; i++) r[i] = __float_as_uint(add ? __uint_as_float(r[i]) + y[8 * c + i] : y[8 * c + i]);
                stg32(o + 8 * c, r);
            }
        } else {
            uint16_t* o = reinterpret_cast<uint16_t*>(out) + at;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t r[8];
                if (add) ldg32(o + 16 * c, r);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float lo = y[16 * c + 2 * i], hi = y[16 * c + 2 * i + 1];
                    r[i] = add ? pack_bf16(bf16_lo(r[i]) + lo, bf16_hi(r[i]) + hi) : pack_bf16(lo, hi);
                }
                stg32(o + 16 * c, r);
            }
        }
        return;
    }
    // rows are a multiple of 8 elements long and 16-byte aligned: pieces of 8 columns
#pragma unroll
    for (int c = 0; c < 4; c++) {
        if (8u * c + 8u <= left) {
            if (f32) {
                float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at + 8 * c);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float4 q = add ? o[h] : make_float4(0.f, 0.f, 0.f, 0.f);
                    q.x += y[8 * c + 4 * h]; q.y += y[8 * c + 4 * h + 1]; q.z += y[8 * c + 4 * h + 2]; q.w += y[8 * c + 4 * h + 3];
                    o[h] = q;
                }
            } else {
                uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + at + 8 * c);
                uint4 q = add ? *o : make_uint4(0u, 0u, 0u, 0u);
                uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float lo = y[8 * c + 2 * i], hi = y[8 * c + 2 * i + 1];
                    r[i] = add ? pack_bf16(bf16_lo(r[i]) + lo, bf16_hi(r[i]) + hi) : pack_bf16(lo, hi);
                }
                *o = make_uint4(r[0], r[1], r[2], r[3]);
            }
        }
    }
}

// launched in clusters of two with PAIR, of one without
template <int EPI, int MASK, bool PAIR>
__global__ void __launch_bounds__(kHgThreads, 1)
    head_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out, const __grid_constant__ HeadGemm p) {
    extern __shared__ uint8_t smem_raw[];
    constexpr bool kI8 = EPI == kEpiInt8;
    constexpr uint32_t kKStep = kI8 ? 128 : 64;  // elements of K per stage (128 bytes)
    const uint32_t smem_base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    constexpr uint32_t kCtas = PAIR ? 2 : 1, kRows = kCtas * kHgBM;  // CTAs that share a tile, and its rows
    const uint32_t b_bytes = (p.bn / kCtas) * 128, stage_bytes = kHgABytes + b_bytes;
    const uint32_t bars = smem_base + kHgSmemTiles + kHgEpiWarps * kHgStageOut;
    const uint32_t bar_full = bars, bar_empty = bars + 8 * kHgMaxStages, bar_acc_full = bars + 16 * kHgMaxStages, bar_acc_empty = bar_acc_full + 16, bar_done = bar_acc_empty + 16;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_cta_rank() : 0u;
    const uint32_t pair = blockIdx.x / kCtas, pairs = gridDim.x / kCtas;
    if (threadIdx.x == 0) {
        abort_flag = 0u;
        for (uint32_t s = 0; s < kHgMaxStages; s++) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(bar_acc_full + 8 * a, 1);
            mbar_init(bar_acc_empty + 8 * a, kCtas * kHgEpiWarps);
        }
        mbar_init(bar_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_slot)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_slot)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
    }
    if (threadIdx.x == 64) {
        prefetch_map(&map_a);
        prefetch_map(&map_b);
        if (EPI == kEpiGrad || EPI == kEpiWeight) prefetch_map(&map_out);
    }
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();  // both CTAs' barriers exist before anything crosses between them
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    after_previous_kernel();  // what came before is done; nothing above reads or writes global memory
    if (EPI == kEpiStats && blockIdx.x == 0 && threadIdx.x == 0 && p.zero) *p.zero = 0u;
    const uint32_t in_use = p.m_count ? *p.m_count : 0u;
    const uint32_t mm = p.m_count ? min(in_use - min(in_use, p.m_first), p.m) : p.m, kk = p.k_count ? min(*p.k_count, p.k) : p.k;
    const uint32_t tiles_m = (mm + kRows - 1) / kRows, tiles_n = (p.n + p.bn - 1) / p.bn;
    const uint32_t kchunks = (kk + kKStep - 1) / kKStep, nsplit = p.split ? hidden_split(tiles_m * tiles_n, p.split, PAIR ? kPairs : 2 * kPairs) : 1u, kper = (kchunks + nsplit - 1) / nsplit;
    const bool to_acc = p.acc_out || nsplit > 1;
    const uint32_t tiles = tiles_m * tiles_n * nsplit;  // the host keeps this below 2^31
    struct Item {
        uint32_t split, tm, tn, k0, k1;
    };
    const FastDiv by_tiles(tiles_m * tiles_n), by_group(p.group_m * tiles_n), by_full(p.group_m), by_last(tiles_m > 0 ? tiles_m - (tiles_m - 1) / p.group_m * p.group_m : 1u);
    auto item = [&](uint32_t t) {
        Item it;
        it.split = by_tiles(t);
        t -= it.split * by_tiles.d;
        const uint32_t g = by_group(t), first = g * p.group_m;
        t -= g * by_group.d;
        const bool full = first + p.group_m <= tiles_m;
        it.tn = full ? by_full(t) : by_last(t);
        it.tm = first + t - it.tn * (full ? by_full.d : by_last.d);
        it.k0 = min(it.split * kper, kchunks);
        it.k1 = min(it.k0 + kper, kchunks);
        return it;
    };

    if (warp < 2) next_kernel_may_start();
    if (warp == 0) {
        // ---- loader (both CTAs) -------------------------------------------------------------------
        auto load = [&](auto b_across) {
            constexpr bool b_mn = decltype(b_across)::value;
            const uint32_t full_first = PAIR ? in_first_cta(bar_full) : bar_full;
            uint32_t s = 0, phase = 1u, issued = 0, a_at = smem_base;
            bool ok = true;
            for (uint32_t t = pair; t < tiles && ok; t += pairs) {
                const Item w = item(t);
                const int32_t m0 = (int32_t)(p.a_m0 + w.tm * kRows + rank * kHgBM), n0 = (int32_t)(p.b_n0 + w.tn * p.bn + rank * (p.bn / kCtas));
                for (uint32_t kc = w.k0; kc < w.k1; kc++) {
                    if (!mbar_wait(bar_empty + 8 * s, phase, &abort_flag)) { ok = false; break; }
                    if (rank == 0) mbar_expect_tx(bar_full + 8 * s, kCtas * stage_bytes);  // both CTAs' copies land on the first CTA's barrier
                    const uint32_t bar = full_first + 8 * s, b_at = a_at + kHgABytes;
                    const int32_t k0 = (int32_t)(kc * kKStep), kb = (int32_t)p.b_k0 + k0;
                    if constexpr (PAIR) {
                        if constexpr (EPI == kEpiWeight) {  // two boxes of 64 m × 64 k
                            tma_load_2d_pair(a_at, &map_a, m0, k0, bar);
                            tma_load_2d_pair(a_at + 8192, &map_a, m0 + 64, k0, bar);
                        } else {
                            tma_load_2d_pair(a_at, &map_a, k0, m0, bar);
                        }
                        if constexpr (b_mn) {
                            tma_load_2d_pair(b_at, &map_b, n0, kb, bar);
                            if (p.bn == 256) tma_load_2d_pair(b_at + 8192, &map_b, n0 + 64, kb, bar);
                        } else {
                            tma_load_2d_pair(b_at, &map_b, kb, n0, bar);
                        }
                    } else {  // A is contiguous along K in the products that run on single CTAs
                        tma_load_2d(a_at, &map_a, k0, m0, bar);
                        if constexpr (b_mn) {
                            for (uint32_t j = 0; j < p.bn / 64; j++) tma_load_2d(b_at + 8192 * j, &map_b, n0 + (int32_t)(64 * j), kb, bar);
                        } else {
                            tma_load_2d(b_at, &map_b, kb, n0, bar);
                        }
                    }
                    issued++;
                    a_at += stage_bytes;
                    if (++s == p.stages) { s = 0; phase ^= 1u; a_at = smem_base; }
                }
            }
            if ((!ok || abort_flag) && issued) {  // copies in flight get time to land before the pair may end
                const unsigned long long t_start = global_ns();
                while (global_ns() - t_start < 2000000ull) {}
            }
        };
        if (lane == 0) {
            if (EPI == kEpiWeight || (!kI8 && p.b_mn)) load(Const<true>());
            else load(Const<false>());
        }
    } else if (warp == 1) {
        // ---- tensor-core issue (first CTA only) -------------------------------------------------------
        auto issue = [&](auto b_across) {
            constexpr bool a_mn = EPI == kEpiWeight, b_mn = decltype(b_across)::value;
            const uint32_t shape = ((p.bn >> 3) << 17) | ((kRows >> 4) << 24);
            // f32 accumulators of bf16 products, or s32 accumulators of s8 products
            const uint32_t idesc = kI8 ? ((2u << 4) | (1u << 7) | (1u << 10) | shape) : ((1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | shape);
            // contiguous along K: rows of 128 bytes, groups of 8 rows 1024 bytes apart, 32 bytes of K per product; contiguous along M / N:
            // 64-wide blocks 8 KB apart, groups of 8 k-rows 1024 bytes apart, 16 k-rows per product. One descriptor per operand, the
            // rest are additions to its address field. This thread's instructions between two products are what the tensor pipe waits for:
            // a vote or a test of a barrier more per stage cost 2 to 8 %, the descriptors' upper halves kept out of the additions gave 10,
            // two stages to an iteration 2 (8 bits: 3)
            const uint64_t da0 = a_mn ? smem_desc_sw128(smem_base, 8192, 1024) : smem_desc_sw128(smem_base, 16, 1024);
            const uint64_t db0 = b_mn ? smem_desc_sw128(smem_base + kHgABytes, 8192, 1024) : smem_desc_sw128(smem_base + kHgABytes, 16, 1024);
            constexpr uint32_t a_step = (a_mn ? 2048u : 32u) >> 4, b_step = (b_mn ? 2048u : 32u) >> 4;
            const uint32_t s_step = stage_bytes >> 4;
            auto commit = [](uint32_t bar) {
                if constexpr (PAIR) tc_commit_pair(bar);
                else tc_commit(bar);
            };
            uint32_t s = 0, phase = 0u, n = 0;
            // no address carries into the upper half
            const uint32_t a_hi = (uint32_t)(da0 >> 32), b_hi = (uint32_t)(db0 >> 32);
            uint32_t a_lo = (uint32_t)da0, b_lo = (uint32_t)db0;
            auto desc = [](uint32_t hi, uint32_t lo) { return (uint64_t)hi << 32 | lo; };
            bool ok = true;
            for (uint32_t t = pair; t < tiles && ok; t += pairs) {
                const Item w = item(t);
                if (w.k0 == w.k1) continue;  // an empty sum: the epilogue writes zeros by itself
                const uint32_t acc = n & 1u;
                if (!mbar_wait<PAIR>(bar_acc_empty + 8 * acc, ((n >> 1) & 1u) ^ 1u, &abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem + acc * 256;
#pragma unroll 2
                for (uint32_t kc = w.k0; kc < w.k1; kc++) {
                    if (!mbar_wait(bar_full + 8 * s, phase, &abort_flag)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t add = k ? 1u : kc != w.k0;
                        const uint64_t da = desc(a_hi, a_lo + k * a_step), db = desc(b_hi, b_lo + k * b_step);
                        if constexpr (kI8) tc_mma_i8_pair(d_tmem, da, db, idesc, add);
                        else if constexpr (PAIR) tc_mma_bf16_pair(d_tmem, da, db, idesc, add);
                        else tc_mma_bf16(d_tmem, da, db, idesc, add);
                    }
                    commit(bar_empty + 8 * s);
                    a_lo += s_step;
                    b_lo += s_step;
                    if (++s == p.stages) { s = 0; phase ^= 1u; a_lo = (uint32_t)da0; b_lo = (uint32_t)db0; }
                }
                if (ok) commit(bar_acc_full + 8 * acc);
                n++;
            }
            commit(bar_done);
        };
        if (rank == 0 && lane == 0) {
            if (EPI == kEpiWeight || (!kI8 && p.b_mn)) issue(Const<true>());
            else issue(Const<false>());
        }
    } else {
        // ---- epilogue (both CTAs): thread = row of the output (of the transposed one for kEpiInt8) ---------
        const uint32_t quarter = (uint32_t)warp & 3u, half = ((uint32_t)warp - 2u) >> 2;
        const uint32_t half_cols = p.bn / 2;  // this warp's columns: [half · bn/2, + bn/2), a multiple of 16
        const int chunks = (int)half_cols / 32;  // four or two of 32 columns in the bf16 products
        const uint32_t stage_out = smem_base + kHgSmemTiles + ((uint32_t)warp - 2u) * kHgStageOut;
        float alpha = 1.f;
        if constexpr (EPI == kEpiHidden || EPI == kEpiWeight) alpha = p.alpha ? *p.alpha : 1.f;
        // plain loads: the kernel before this one may have written these while this one was starting, so they are not read-only data
        auto row_info = [&](const Item& w) {
            RowInfo r;
            const uint32_t row = w.tm * kRows + rank * kHgBM + quarter * 32u + (uint32_t)lane;
            r.live = row < mm;
            r.caller_row = row;
            r.token = -1;
            r.cf = make_float4(0.f, 0.f, 0.f, 0.f);
            r.xs = make_float2(1.f, 1.f);
            if (r.live) {
                if constexpr (EPI == kEpiGrad || EPI == kEpiStats || EPI == kEpiHidden)
                    if (p.rows_at) r.caller_row = p.rows_at[row];
                if constexpr (EPI == kEpiGrad) r.cf = p.coef[row];
                if constexpr (EPI == kEpiGrad || EPI == kEpiHidden) {
                    const float4 mo = p.more[row];
                    r.xs = make_float2(mo.x, mo.y);
                    r.token = __float_as_int(mo.z);
                }
                if constexpr (EPI == kEpiInt8) r.xs.x = p.m_scale[row];
            }
            return r;
        };
        uint32_t n = 0, scales_of = 0xffffffffu;  // kEpiInt8: the column of tiles whose scales are staged
        bool ok = true;
        RowInfo ahead;
        MaskAhead<MASK> mask;
        if (pair < tiles) {
            const Item w = item(pair);
            ahead = row_info(w);
            mask.load(p, ahead.caller_row, p.v0 + w.tn * p.bn + half * half_cols, ahead.live, lane);
        }
        for (uint32_t t = pair; t < tiles; t += pairs) {
            const Item w = item(t);
            const bool some = w.k0 != w.k1, more_tiles = t + pairs < tiles;
            const RowInfo r = ahead;
            Item next = w;
            if (more_tiles) {
                next = item(t + pairs);
                ahead = row_info(next);
            }
            const uint32_t acc = n & 1u;
            auto wait = [&] {
                if (some && ok) {
                    ok = __all_sync(0xffffffffu, mbar_wait(bar_acc_full + 8 * acc, (n >> 1) & 1u, &abort_flag));
                    tc_fence_after();
                }
                if (!more_tiles) next_kernel_may_start();
            };
            // the accumulator may be overwritten: this warp has it in registers. Before the results are stored: the arrival waits for
            // whatever the warp has stored.
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0) {
                    if constexpr (PAIR) mbar_arrive_remote(in_first_cta(bar_acc_empty + 8 * acc));
                    else mbar_arrive(bar_acc_empty + 8 * acc);
                }
            };
            const uint32_t row0 = w.tm * kRows + rank * kHgBM + quarter * 32u, row = row0 + (uint32_t)lane;
            const bool live = r.live;
            const uint32_t taddr = tmem + ((quarter * 32u) << 16) + acc * 256 + half * half_cols;
            const uint32_t col0 = w.tn * p.bn + half * half_cols;
            if constexpr (EPI == kEpiGrad || EPI == kEpiStats) {
                const float ys = p.zscale * kLog2e * r.xs.x;
                int32_t token = r.token;
                if (EPI == kEpiStats && live && p.tokens) {
                    token = p.tokens[r.caller_row];
                    if ((uint32_t)token >= p.vocab) token = -1;  // no such column, not even past the vocabulary's end in its last tile
                }
                float m = -FLT_MAX, S = 0.f, W = 0.f, ytok = __int_as_float(0x7fc00000);
                wait();
                mask.settle(p, p.v0 + col0, lane);
#pragma unroll 1
                for (int c = 0; c < chunks; c++) {
                    float y[32];
                    __syncwarp();
                    tc_ld32(taddr + 32 * c, reinterpret_cast<uint32_t*>(y));
                    tc_wait_ld();
                    pin32(y);
                    if (c == chunks - 1) release();
                    if (c == 0 && more_tiles) mask.load(p, ahead.caller_row, p.v0 + next.tn * p.bn + half * half_cols, ahead.live, lane);
                    if (!ok) {
#pragma unroll
                        for (int i = 0; i < 32; i++) y[i] = __int_as_float(0x7fc00000);
                    }
                    const uint32_t v = p.v0 + col0 + 32 * c;
                    if constexpr (EPI == kEpiGrad) {
                        uint32_t g[16];
                        epi_grad<MASK>(p, live, v, y, r.cf, ys, token, mask.chunk(c), g);
                        if ((c & 1) == 0) stage_free(lane);
#pragma unroll
                        for (int j = 0; j < 4; j++) sts_piece(stage_out, lane, 4 * (c & 1) + j, g[4 * j], g[4 * j + 1], g[4 * j + 2], g[4 * j + 3]);
                        if (c & 1) stage_send(&map_out, stage_out, lane, (int32_t)(col0 + 32 * (c - 1)), (int32_t)row0);
                    } else {
                        epi_stats<MASK>(p, v, y, ys, token, mask.chunk(c), m, S, W, ytok);
                    }
                }
                if constexpr (EPI == kEpiStats) {
                    // the maximum and the token's logit in logit units, the entropy sum in natural units; S = −1: this pair gave up
                    if (live) p.parts[(uint64_t)row * p.parts_pitch + w.tn * 2 + half] = make_float4(m > -FLT_MAX || m != m ? m * p.zscale : -FLT_MAX, ok ? S : -1.f, W * 0.69314718055994531f, ytok <= -FLT_MAX ? -FLT_MAX : ytok * p.zscale);
                }
            } else if constexpr (EPI != kEpiInt8) {
                uint64_t orow = (uint64_t)p.out_row0 + row;
                float scale = alpha;
                if (EPI == kEpiHidden && !to_acc) {
                    orow = r.caller_row;
                    scale = alpha * r.xs.y;
                }
                wait();
                const bool there = some && ok;
                if (EPI == kEpiWeight && p.staged && !p.out_f32) {
                    // 64 columns at a time: one wait for tensor memory and one store of whole lines per 64
#pragma unroll 1
                    for (int c = 0; c < chunks; c += 2) {
                        float z[64];
                        if (there) {
                            __syncwarp();
                            tc_ld32(taddr + 32 * c, reinterpret_cast<uint32_t*>(z));
                            tc_ld32(taddr + 32 * c + 32, reinterpret_cast<uint32_t*>(z + 32));
                            tc_wait_ld();
                            pin32(z);
                            pin32(z + 32);
                            if (c + 2 >= chunks) release();
                        } else {
#pragma unroll
                            for (int i = 0; i < 64; i++) z[i] = ok ? 0.f : __int_as_float(0x7fc00000);
                        }
                        scale32(z, scale);
                        scale32(z + 32, scale);
                        const uint32_t col = col0 + 32 * c;
                        stage_free(lane);
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            sts_piece(stage_out, lane, j, pack_bf16(z[8 * j], z[8 * j + 1]), pack_bf16(z[8 * j + 2], z[8 * j + 3]), pack_bf16(z[8 * j + 4], z[8 * j + 5]), pack_bf16(z[8 * j + 6], z[8 * j + 7]));
                        if (row0 < mm && col < p.n) stage_send(&map_out, stage_out, lane, (int32_t)(p.out_col0 + col), (int32_t)(p.out_row0 + row0));
                    }
                } else {
#pragma unroll 1
                for (int c = 0; c < chunks; c++) {
                    float z[32];
                    if (there) {
                        __syncwarp();
                        tc_ld32(taddr + 32 * c, reinterpret_cast<uint32_t*>(z));
                        tc_wait_ld();
                        pin32(z);
                        if (c == chunks - 1) release();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i++) z[i] = ok ? 0.f : __int_as_float(0x7fc00000);
                    }
                    const uint32_t col = col0 + 32 * c;
                    if (EPI == kEpiWeight && p.staged) {
                        scale32(z, scale);
                        stage_free(lane);
#pragma unroll
                        for (int j = 0; j < 8; j++) sts_piece(stage_out, lane, j, __float_as_uint(z[4 * j]), __float_as_uint(z[4 * j + 1]), __float_as_uint(z[4 * j + 2]), __float_as_uint(z[4 * j + 3]));
                        if (row0 < mm && col < p.n) stage_send(&map_out, stage_out, lane, (int32_t)(p.out_col0 + col), (int32_t)(p.out_row0 + row0));
                    } else if (live && col < p.n) {
                        float* part = p.acc + ((uint64_t)w.split * p.acc_rows(mm) + row) * p.n + col;
                        if (p.acc_in) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                if (col + i < p.n) {
                                    const float4 q = *reinterpret_cast<const float4*>(part + i);
                                    z[i] += q.x; z[i + 1] += q.y; z[i + 2] += q.z; z[i + 3] += q.w;
                                }
                        }
                        if (to_acc) {
                            store_row32(part, 0, true, false, true, p.n - col, z);
                        } else {
                            scale32(z, scale);
                            store_row32(p.out, orow * p.out_pitch + p.out_col0 + col, p.out_f32, p.out_add, p.wide, p.n - col, z);
                        }
                    }
                }
                }
            } else {
                // thread = vocabulary entry, registers = tokens: a warp's store covers 32 consecutive entries of a row. The tokens' scales
                // pass through the warp's staging tile, four to a read. Instructions are what such a tile costs where K is short (bf16 results
                // of 256 tokens at K = 512: 74 -> 52 us for 202 752 entries without a comparison per result, with packed products and the scales staged)
                if (w.tn != scales_of) {
                    scales_of = w.tn;
                    __syncwarp();
                    float s4[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) s4[j] = 4u * lane + j < half_cols && col0 + 4 * lane + j < p.n ? p.n_scale[col0 + 4 * lane + j] : 0.f;
                    asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(stage_out + 16 * lane), "f"(s4[0]), "f"(s4[1]), "f"(s4[2]), "f"(s4[3]) : "memory");
                    __syncwarp();
                }
                wait();
                const float scale = ok ? r.xs.x : __int_as_float(0x7fc00000);
                const f32x2 scale2 = pack2(scale, scale);
                const uint32_t pitch = (uint32_t)p.out_pitch, size = p.out_f32 ? 4u : 2u;
                uint8_t* o = reinterpret_cast<uint8_t*>(p.out) + ((uint64_t)col0 * pitch + row) * size;
#pragma unroll 1
                for (uint32_t c = 0; c < half_cols; c += 16, o += (uint64_t)(16u * size) * pitch) {
                    const uint32_t col = col0 + c, left = col < p.n ? min(16u, p.n - col) : 0u;  // tokens here
                    float y[16];
                    if (some && ok) {
                        uint32_t z[16];
                        __syncwarp();
                        tc_ld16(taddr + c, z);
                        tc_wait_ld();
                        pin16(z);
                        if (c + 16 >= half_cols) release();
#pragma unroll
                        for (int i = 0; i < 16; i++) y[i] = (float)(int32_t)z[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++) y[i] = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float t0, t1, t2, t3;
                        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(t0), "=f"(t1), "=f"(t2), "=f"(t3) : "r"(stage_out + 4 * (c + i)) : "memory");
                        unpack2(mul2(mul2(pack2(y[i], y[i + 1]), pack2(t0, t1)), scale2), y[i], y[i + 1]);
                        unpack2(mul2(mul2(pack2(y[i + 2], y[i + 3]), pack2(t2, t3)), scale2), y[i + 2], y[i + 3]);
                    }
                    if (!live) continue;
                    if (p.out_f32) {
                        if (left == 16u) {
#pragma unroll
                            for (int i = 0; i < 16; i++) *reinterpret_cast<float*>(o + (uint64_t)(4u * i) * pitch) = y[i];
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if ((uint32_t)i < left) *reinterpret_cast<float*>(o + (uint64_t)(4u * i) * pitch) = y[i];
                        }
                    } else if (left == 16u) {
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const uint32_t two = pack_bf16(y[i], y[i + 1]);
                            *reinterpret_cast<uint16_t*>(o + (uint64_t)(2u * i) * pitch) = (uint16_t)two;
                            *reinterpret_cast<uint16_t*>(o + (uint64_t)(2u * i + 2u) * pitch) = (uint16_t)(two >> 16);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const uint32_t two = pack_bf16(y[i], y[i + 1]);
                            if ((uint32_t)i < left) *reinterpret_cast<uint16_t*>(o + (uint64_t)(2u * i) * pitch) = (uint16_t)two;
                            if ((uint32_t)i + 1 < left) *reinterpret_cast<uint16_t*>(o + (uint64_t)(2u * i + 2u) * pitch) = (uint16_t)(two >> 16);
                        }
                    }
                }
            }
            if (some) n++;
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // this warp's last stores are written
    }

    // ---- teardown ------------------------------------------------------------------------------------
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (lane == 0) {
            volatile uint32_t never = 0u;
            mbar_wait(bar_done, 0u, &never, 20000000ull);  // every product has finished (multicast to both CTAs)
        }
        __syncwarp();
    }
    if constexpr (PAIR) cluster_sync_all();  // neither CTA leaves while the other may still reach into its shared or tensor memory
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace nrl

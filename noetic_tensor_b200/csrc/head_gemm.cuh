// The matrix products of the readout's backward pass and of its 8-bit form: one kernel on CTA pairs
// (tcgen05.mma.cta_group::2, f32 or 32-bit integer accumulators in tensor memory), five epilogues.
//
//   kEpiStats   z = x · W for the scored rows x; the epilogue keeps, per row and 128 columns, the maximum,
//               Σ exp(z − max), Σ exp(z − max)·(z − max) and the given token's logit
//   kEpiGrad    z = x · W for the scored rows x and a piece of the vocabulary; the epilogue turns the
//               accumulators into dz = ∂/∂z of the per-row terms and writes them as bf16:
//               π_j = exp((z_j − m) − ln Z), dz_j = a·1[j = token] − π_j·(a + b·(ln π_j + H)).
//               The logits themselves are never written.
//   kEpiHidden  dx = dz · Wᵀ over a piece of the vocabulary (f32 sums carried from piece to piece)
//   kEpiWeight  dW = xᵀ · dz for a piece of the vocabulary
//   kEpiInt8    z[r, v] = s_r·w_v·Σ_k q[r, k]·p[v, k] in 8-bit integers (sums exact in 32 bits)
//
// A pair of CTAs owns 256 rows × `bn` columns of the output; each CTA loads its 128 rows of A and half
// of B per stage (TMA, 128-byte swizzle, no multicast), one thread of the first CTA issues the products
// for both, and the 256-column accumulators are double-buffered so that a tile's epilogue runs under the
// next tile's products. The grid is persistent: 74 pairs walk the tiles in a fixed order, so every sum
// has a fixed order and results are bitwise reproducible. A and B may each be contiguous along K or along
// their other axis (the descriptors' major bits), so dz, x and W are read as they lie in memory.
//
// Bound: the tensor pipe for the large products, HBM for the few-row forms (the weight is read once per
// call). Waits are bounded as in the readout forward; a role that gives up raises the pair's abort flag
// and the tiles not reached are written as NaN.
#pragma once
#include "tcgen05.cuh"

namespace nrl {

constexpr int kHgBM = 128;           // rows per CTA (256 per pair)
constexpr int kHgEpiWarps = 8;       // two per quarter of tensor memory: each takes half of the columns
constexpr int kHgThreads = 64 + 32 * kHgEpiWarps;
constexpr uint32_t kHgABytes = kHgBM * 128;      // one stage of A: 128 rows × 128 bytes of K
constexpr uint32_t kHgSmemTiles = 6 * 2 * kHgABytes;  // 192 KB of stages: six of 32 KB at bn = 256, more when B is narrower
constexpr uint32_t kHgMaxStages = 10;
constexpr uint32_t kHgStageOut = 4096;  // per epilogue warp: 32 rows × 128 bytes on their way out
constexpr uint32_t kHgSmemBytes = kHgSmemTiles + kHgEpiWarps * kHgStageOut + 1024 + 256;

enum { kEpiGrad = 0, kEpiHidden = 1, kEpiWeight = 2, kEpiInt8 = 3, kEpiStats = 4 };
enum { kMaskNone = 0, kMaskBytes = 1, kMaskBits = 2 };

// An accumulator drops what lies below its last bit at each of the d / 16 steps that add into it, toward zero: a sum comes out
// smaller by 1.6e-8 of itself per step on average (measured: 2.4e-7, 1.0e-6, 2.1e-6, 4.1e-6 of the row maximum at
// d = 256, 1024, 2048, 4096, the expectation for partial sums that grow in proportion to the step). The logits are scaled back.
constexpr float kAccumulatorLoss = 1.6e-8f;
inline float logit_scale(uint32_t d, float tau) { return (1.f + kAccumulatorLoss * (float)((d + 15) / 16)) / tau; }

struct HeadGemm {
    uint32_t m, n, k;          // extents of the product
    const uint32_t* m_count;   // device: the rows in use along M, of which this launch takes m from m_first on; or null: all m
    uint32_t m_first;
    const uint32_t* k_count;   // device: the extent along K (≤ k), or null
    uint32_t bn;               // columns per tile (a multiple of 32, ≤ 256)
    uint32_t stages;
    uint32_t a_mn, b_mn;       // A / B contiguous along M / N instead of K
    uint32_t b_n0, b_k0;       // where this piece of the vocabulary begins in B, along N / along K
    uint32_t a_m0;             // … in A, along M
    uint32_t nsplit;           // ranges of K, each with its own output buffer
    uint32_t group_m;          // 256-row blocks that are walked side by side (L2 reuse of B)
    // kEpiGrad, kEpiStats
    const float4* coef;        // kEpiGrad [rows] of the scored rows: (a·xs, b·xs, (m + ln Z)·log2 e, a·xs + b·xs·H)
    const float4* more;        // [rows] (xs, 1 / xs, token bits, ·): xs is the scale of an 8-bit row, else 1
    const uint32_t* rows_at;   // [rows] the row in the caller's order, or null: the same
    const int32_t* tokens;     // kEpiStats [rows in the caller's order] or null
    float zscale;              // logit = accumulator · zscale (· xs)
    uint32_t entropy_term;     // kEpiGrad: some b ≠ 0 is possible; kEpiStats: the entropy sum is wanted
    const uint8_t* allow;
    uint64_t allow_stride;
    uint32_t allow_wide;       // every row of the byte mask is 8-byte aligned
    uint32_t vocab;            // V
    uint32_t v0;               // first column of this piece
    float4* parts;             // kEpiStats [rows, parts_pitch]: (max, sum, entropy sum, token's logit) per 128 columns
    uint32_t parts_pitch;
    // kEpiHidden, kEpiWeight
    const float* alpha;        // device scalar
    float* acc;                // f32 sums between pieces / ranges of K: [nsplit, acc_rows, n]
    uint64_t acc_rows;
    uint32_t acc_in, acc_out;  // start from acc; end in acc (otherwise in out)
    void* out;
    uint64_t out_pitch;
    uint32_t out_f32, out_add; // type of `out`; add to what it holds
    uint32_t out_col0;         // kEpiWeight: first column (or first row, with out_row0) of this piece
    uint32_t out_row0;
    uint32_t wide;             // rows of out are 32-byte aligned
    uint32_t staged;           // results leave through shared memory and TMA stores (map_out)
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
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {  // nearest, ties to even; NaN stays NaN
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The allow-mask of 32 columns of one row, fetched ahead of its use. Bytes: eight words, four columns each; bits: one word.
template <int MASK>
struct MaskWords {
    uint32_t w[MASK == kMaskBytes ? 8 : 1];
    __device__ __forceinline__ void load(const HeadGemm& p, uint64_t caller_row, uint32_t v, bool live) {
        if constexpr (MASK == kMaskBits) {
            w[0] = live && v < p.vocab ? __ldg(reinterpret_cast<const uint32_t*>(p.allow) + caller_row * p.allow_stride + (v >> 5)) : 0u;
        } else if constexpr (MASK == kMaskBytes) {
            const uint8_t* mp = p.allow + caller_row * p.allow_stride + v;
            if (live && p.allow_wide && v + 32 <= p.vocab) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint2 q = ldg_stream8(mp + 8 * i);
                    w[2 * i] = q.x;
                    w[2 * i + 1] = q.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    uint32_t x = 0u;
#pragma unroll 1
                    for (int j = 0; j < 4; j++)
                        if (live && v + 4 * i + j < p.vocab) x |= (uint32_t)mp[4 * i + j] << (8 * j);
                    w[i] = x;
                }
            }
            // bit 7 of a byte: the byte is not 0
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] |= (w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu;
        }
    }
    __device__ __forceinline__ bool allows(int i) const {
        if constexpr (MASK == kMaskBits) return (w[0] >> i) & 1u;
        if constexpr (MASK == kMaskBytes) return w[i >> 2] & (0x80u << (8 * (i & 3)));
        return true;
    }
};

// ∂/∂z of 32 columns of one row from the accumulators y, as 16 packed bf16 pairs. With the row's coefficients pre-multiplied
// (a′ = a·xs, …): ln π in units of log2 is one fused multiply-add of y, dz = −π·(a′ + b′·(ln π + H)), and the token's entry gets a′.
template <int MASK>
__device__ __forceinline__ void epi_grad(const HeadGemm& p, bool live, uint32_t v, const float y[32], const float4& cf, float ys, int32_t token, const MaskWords<MASK>& mask, uint32_t out[16]) {
    if (!live || v >= p.vocab) {
#pragma unroll
        for (int i = 0; i < 16; i++) out[i] = 0u;
        return;
    }
    const float na = -cf.x, lse2 = -cf.z, nb2 = -cf.y * 0.69314718055994531f, nab = -cf.w;
    float g[32];
    if (p.entropy_term) {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const float l2 = fmaf(y[i], ys, lse2);
            g[i] = ex2_approx(l2) * fmaf(fmaxf(l2, -1e30f), nb2, nab);  // a −inf logit: π = 0, and 0·inf cannot appear
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) g[i] = ex2_approx(fmaf(y[i], ys, lse2)) * na;
    }
    const uint32_t tk = (uint32_t)(token - (int32_t)v);
    if (tk < 32u) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if ((uint32_t)i == tk) g[i] += cf.x;
    }
    if constexpr (MASK != kMaskNone) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if (!mask.allows(i)) g[i] = 0.f;
    }
    if (v + 32 > p.vocab) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if (v + i >= p.vocab) g[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) out[i] = pack_bf16(g[2 * i], g[2 * i + 1]);
}

// 32 columns of one row folded into (m, S, W): m in accumulator units, W in units of log2.
template <int MASK>
__device__ __forceinline__ void epi_stats(const HeadGemm& p, uint32_t v, float y[32], float c2, int32_t token, const MaskWords<MASK>& mask, float& m, float& S, float& W, float& ytok) {
    if constexpr (MASK != kMaskNone) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if (!mask.allows(i)) y[i] = -FLT_MAX;
    }
    if (v + 32 > p.vocab) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if (v + i >= p.vocab) y[i] = -FLT_MAX;
    }
    const uint32_t tk = (uint32_t)(token - (int32_t)v);
    if (tk < 32u) {
#pragma unroll
        for (int i = 0; i < 32; i++)
            if ((uint32_t)i == tk) ytok = y[i];
    }
    float cm = fmax3_nan(y[0], y[1], y[2]);
#pragma unroll
    for (int i = 3; i < 31; i += 2) cm = fmax3_nan(cm, y[i], y[i + 1]);
    cm = fmax_nan(cm, y[31]);
    if (cm <= -FLT_MAX) return;  // every column here is excluded or −inf (a NaN goes on)
    if (!(cm <= m)) {
        if (m > -FLT_MAX) {
            const float dm = (m - cm) * c2, sc = ex2_approx(dm);
            W = (W + S * dm) * sc;
            S *= sc;
        }
        m = cm;
    }
    const float m2 = -m * c2;
    float s0 = 0.f, s1 = 0.f, w0 = 0.f, w1 = 0.f;
    if (p.entropy_term) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float t0 = fmaxf(fmaf(y[i], c2, m2), -1e30f), t1 = fmaxf(fmaf(y[i + 1], c2, m2), -1e30f);
            const float e0 = ex2_approx(t0), e1 = ex2_approx(t1);
            s0 += e0; s1 += e1;
            w0 = fmaf(e0, t0, w0); w1 = fmaf(e1, t1, w1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            s0 += ex2_approx(fmaf(y[i], c2, m2));
            s1 += ex2_approx(fmaf(y[i + 1], c2, m2));
        }
    }
    S += s0 + s1;
    W += w0 + w1;
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

template <int EPI, int MASK>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kHgThreads, 1)
    head_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out, const __grid_constant__ HeadGemm p) {
    extern __shared__ uint8_t smem_raw[];
    constexpr bool kI8 = EPI == kEpiInt8;
    constexpr uint32_t kKStep = kI8 ? 128 : 64;  // elements of K per stage (128 bytes)
    const uint32_t smem_base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t b_bytes = (p.bn / 2) * 128, stage_bytes = kHgABytes + b_bytes;
    const uint32_t bars = smem_base + kHgSmemTiles + kHgEpiWarps * kHgStageOut;
    const uint32_t bar_full = bars, bar_empty = bars + 8 * kHgMaxStages, bar_acc_full = bars + 16 * kHgMaxStages, bar_acc_empty = bar_acc_full + 16, bar_done = bar_acc_empty + 16;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t in_use = p.m_count ? *p.m_count : 0u;
    const uint32_t mm = p.m_count ? min(in_use - min(in_use, p.m_first), p.m) : p.m, kk = p.k_count ? min(*p.k_count, p.k) : p.k;
    const uint32_t tiles_m = (mm + 2 * kHgBM - 1) / (2 * kHgBM), tiles_n = (p.n + p.bn - 1) / p.bn;
    const uint32_t kchunks = (kk + kKStep - 1) / kKStep, kper = (kchunks + p.nsplit - 1) / p.nsplit;
    const uint32_t tiles = tiles_m * tiles_n * p.nsplit;  // the host keeps this below 2^31
    struct Item {
        uint32_t split, tm, tn, k0, k1;
    };
    auto item = [&](uint32_t t) {
        Item it;
        it.split = t / (tiles_m * tiles_n);
        t -= it.split * (tiles_m * tiles_n);
        const uint32_t per = p.group_m * tiles_n, g = t / per, first = g * p.group_m, here = min(p.group_m, tiles_m - first);
        t -= g * per;
        it.tm = first + t % here;
        it.tn = t / here;
        it.k0 = min(it.split * kper, kchunks);
        it.k1 = min(it.k0 + kper, kchunks);
        return it;
    };

    if (threadIdx.x == 0) {
        abort_flag = 0u;
        for (uint32_t s = 0; s < kHgMaxStages; s++) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(bar_acc_full + 8 * a, 1);
            mbar_init(bar_acc_empty + 8 * a, 2 * kHgEpiWarps);
        }
        mbar_init(bar_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before anything crosses between them
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        // ---- loader (both CTAs) -------------------------------------------------------------------
        if (lane == 0) {
            uint32_t s = 0, phase = 1u, issued = 0;
            bool ok = true;
            for (uint32_t t = pair; t < tiles && ok; t += pairs) {
                const Item w = item(t);
                const int32_t m0 = (int32_t)(p.a_m0 + w.tm * 2 * kHgBM + rank * kHgBM), n0 = (int32_t)(p.b_n0 + w.tn * p.bn + rank * (p.bn / 2));
                for (uint32_t kc = w.k0; kc < w.k1; kc++) {
                    if (!mbar_wait(bar_empty + 8 * s, phase, &abort_flag)) { ok = false; break; }
                    const uint32_t full_first = in_first_cta(bar_full + 8 * s);
                    if (rank == 0) mbar_expect_tx(bar_full + 8 * s, 2 * stage_bytes);  // both CTAs' copies land on this barrier
                    const uint32_t a_at = smem_base + s * stage_bytes, b_at = a_at + kHgABytes;
                    const int32_t k0 = (int32_t)(kc * kKStep);
                    if (p.a_mn) {  // two boxes of 64 m × 64 k
                        tma_load_2d_pair(a_at, &map_a, m0, k0, full_first);
                        tma_load_2d_pair(a_at + 8192, &map_a, m0 + 64, k0, full_first);
                    } else {
                        tma_load_2d_pair(a_at, &map_a, k0, m0, full_first);
                    }
                    const int32_t kb = (int32_t)p.b_k0 + k0;
                    if (p.b_mn) {
                        for (uint32_t j = 0; j < p.bn / 128; j++) tma_load_2d_pair(b_at + j * 8192, &map_b, n0 + (int32_t)(64 * j), kb, full_first);
                    } else {
                        tma_load_2d_pair(b_at, &map_b, kb, n0, full_first);
                    }
                    issued++;
                    if (++s == p.stages) { s = 0; phase ^= 1u; }
                }
            }
            if ((!ok || abort_flag) && issued) {  // copies in flight get time to land before the pair may end
                const unsigned long long t_start = global_ns();
                while (global_ns() - t_start < 2000000ull) {}
            }
        }
    } else if (warp == 1) {
        // ---- tensor-core issue (first CTA only) -------------------------------------------------------
        if (rank == 0 && lane == 0) {
            const uint32_t shape = ((p.bn >> 3) << 17) | ((uint32_t)((2 * kHgBM) >> 4) << 24);
            // f32 accumulators of bf16 products, or s32 accumulators of s8 products
            const uint32_t idesc = kI8 ? ((2u << 4) | (1u << 7) | (1u << 10) | shape) : ((1u << 4) | (1u << 7) | (1u << 10) | (p.a_mn << 15) | (p.b_mn << 16) | shape);
            uint32_t s = 0, phase = 0u, n = 0;
            bool ok = true;
            for (uint32_t t = pair; t < tiles && ok; t += pairs) {
                const Item w = item(t);
                if (w.k0 == w.k1) continue;  // an empty sum: the epilogue writes zeros by itself
                const uint32_t acc = n & 1u;
                if (!mbar_wait(bar_acc_empty + 8 * acc, ((n >> 1) & 1u) ^ 1u, &abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem + acc * 256;
                for (uint32_t kc = w.k0; kc < w.k1; kc++) {
                    if (!mbar_wait(bar_full + 8 * s, phase, &abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t a_addr = smem_base + s * stage_bytes, b_addr = a_addr + kHgABytes;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        // contiguous along K: rows of 128 bytes, groups of 8 rows 1024 bytes apart, 32 bytes of K per product;
                        // contiguous along M / N: 64-wide blocks 8 KB apart, groups of 8 k-rows 1024 bytes apart, 16 k-rows per product
                        const uint64_t da = p.a_mn ? smem_desc_sw128(a_addr + k * 2048, 8192, 1024) : smem_desc_sw128(a_addr + k * 32, 16, 1024);
                        const uint64_t db = p.b_mn ? smem_desc_sw128(b_addr + k * 2048, 8192, 1024) : smem_desc_sw128(b_addr + k * 32, 16, 1024);
                        if constexpr (kI8) tc_mma_i8_pair(d_tmem, da, db, idesc, (kc != w.k0) | (uint32_t)(k != 0));
                        else tc_mma_bf16_pair(d_tmem, da, db, idesc, (kc != w.k0) | (uint32_t)(k != 0));
                    }
                    tc_commit_pair(bar_empty + 8 * s);
                    if (++s == p.stages) { s = 0; phase ^= 1u; }
                }
                if (ok) tc_commit_pair(bar_acc_full + 8 * acc);
                n++;
            }
            tc_commit_pair(bar_done);
        }
    } else {
        // ---- epilogue (both CTAs): thread = row of the output (of the transposed one for kEpiInt8) ---------
        const uint32_t quarter = (uint32_t)warp & 3u, half = ((uint32_t)warp - 2u) >> 2;
        const uint32_t half_cols = p.bn / 2;  // this warp's columns: [half · bn/2, + bn/2), a multiple of 16
        const uint32_t stage_out = smem_base + kHgSmemTiles + ((uint32_t)warp - 2u) * kHgStageOut;
        float alpha = 1.f;
        if constexpr (EPI == kEpiHidden || EPI == kEpiWeight) alpha = p.alpha ? *p.alpha : 1.f;
        uint32_t n = 0;
        bool ok = true;
        for (uint32_t t = pair; t < tiles; t += pairs) {
            const Item w = item(t);
            const bool some = w.k0 != w.k1;
            const uint32_t acc = n & 1u;
            if (some && ok) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar_acc_full + 8 * acc, (n >> 1) & 1u, &abort_flag));
                tc_fence_after();
            }
            const uint32_t row0 = w.tm * 2 * kHgBM + rank * kHgBM + quarter * 32u, row = row0 + (uint32_t)lane;
            const bool live = row < mm;
            const uint32_t taddr = tmem + ((quarter * 32u) << 16) + acc * 256 + half * half_cols;
            const uint32_t col0 = w.tn * p.bn + half * half_cols;
            if constexpr (EPI == kEpiGrad || EPI == kEpiStats) {
                float4 cf = make_float4(0.f, 0.f, 0.f, 0.f);
                uint64_t caller_row = row;
                int32_t token = -1;
                float ys = p.zscale * kLog2e;
                if (live) {
                    if (p.rows_at) caller_row = __ldg(p.rows_at + row);
                    if constexpr (EPI == kEpiGrad) {
                        cf = __ldg(p.coef + row);
                        const float4 mo = __ldg(p.more + row);
                        ys *= mo.x;
                        token = __float_as_int(mo.z);
                    } else if (p.tokens) {
                        token = __ldg(p.tokens + caller_row);
                    }
                }
                float m = -FLT_MAX, S = 0.f, W = 0.f, ytok = __int_as_float(0x7fc00000);
                MaskWords<MASK> mask;
                mask.load(p, caller_row, p.v0 + col0, live);
#pragma unroll 1
                for (uint32_t c = 0; c < half_cols; c += 32) {
                    float y[32];
                    tc_ld32(taddr + c, reinterpret_cast<uint32_t*>(y));
                    MaskWords<MASK> next;
                    if (c + 32 < half_cols) next.load(p, caller_row, p.v0 + col0 + c + 32, live);
                    tc_wait_ld();
                    if (!ok) {
#pragma unroll
                        for (int i = 0; i < 32; i++) y[i] = __int_as_float(0x7fc00000);
                    }
                    const uint32_t v = p.v0 + col0 + c;
                    if constexpr (EPI == kEpiGrad) {
                        uint32_t g[16];
                        epi_grad<MASK>(p, live, v, y, cf, ys, token, mask, g);
                        if ((c & 32) == 0) stage_free(lane);
#pragma unroll
                        for (int j = 0; j < 4; j++) sts_piece(stage_out, lane, (int)(c & 32) / 8 + j, g[4 * j], g[4 * j + 1], g[4 * j + 2], g[4 * j + 3]);
                        if (c & 32) stage_send(&map_out, stage_out, lane, (int32_t)(col0 + c - 32), (int32_t)row0);
                    } else {
                        if (v < p.vocab) epi_stats<MASK>(p, v, y, ys, token, mask, m, S, W, ytok);
                    }
                    mask = next;
                }
                if constexpr (EPI == kEpiStats) {
                    // the maximum and the token's logit in logit units, the entropy sum in natural units; S = −1: this pair gave up
                    if (live) p.parts[(uint64_t)row * p.parts_pitch + w.tn * 2 + half] = make_float4(m > -FLT_MAX || m != m ? m * p.zscale : -FLT_MAX, ok ? S : -1.f, W * 0.69314718055994531f, ytok <= -FLT_MAX ? -FLT_MAX : ytok * p.zscale);
                }
            } else if constexpr (EPI != kEpiInt8) {
                uint64_t orow = (uint64_t)p.out_row0 + row;
                float scale = alpha;
                if constexpr (EPI == kEpiHidden) {
                    if (live && !p.acc_out) {
                        orow = __ldg(p.rows_at + row);
                        scale = alpha * __ldg(p.more + row).y;
                    }
                }
#pragma unroll 1
                for (uint32_t c = 0; c < half_cols; c += 32) {
                    float y[32];
                    if (some && ok) {
                        tc_ld32(taddr + c, reinterpret_cast<uint32_t*>(y));
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i++) y[i] = ok ? 0.f : __int_as_float(0x7fc00000);
                    }
                    const uint32_t col = col0 + c;
                    if (EPI == kEpiWeight && p.staged) {
#pragma unroll
                        for (int i = 0; i < 32; i++) y[i] *= scale;
                        if (p.out_f32) {
                            stage_free(lane);
#pragma unroll
                            for (int j = 0; j < 8; j++)
                                sts_piece(stage_out, lane, j, __float_as_uint(y[4 * j]), __float_as_uint(y[4 * j + 1]), __float_as_uint(y[4 * j + 2]), __float_as_uint(y[4 * j + 3]));
                            if (col < p.n && row0 < mm) stage_send(&map_out, stage_out, lane, (int32_t)(p.out_col0 + col), (int32_t)(p.out_row0 + row0));
                        } else {
                            if ((c & 32) == 0) stage_free(lane);
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                sts_piece(stage_out, lane, (int)(c & 32) / 8 + j, pack_bf16(y[8 * j], y[8 * j + 1]), pack_bf16(y[8 * j + 2], y[8 * j + 3]), pack_bf16(y[8 * j + 4], y[8 * j + 5]),
                                          pack_bf16(y[8 * j + 6], y[8 * j + 7]));
                            if ((c & 32) && col - 32 < p.n && row0 < mm) stage_send(&map_out, stage_out, lane, (int32_t)(p.out_col0 + col - 32), (int32_t)(p.out_row0 + row0));
                        }
                    } else if (live && col < p.n) {
                        float* part = p.acc ? p.acc + ((uint64_t)w.split * p.acc_rows + row) * p.n + col : nullptr;
                        if (p.acc_in) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                if (col + i < p.n) {
                                    const float4 q = *reinterpret_cast<const float4*>(part + i);
                                    y[i] += q.x; y[i + 1] += q.y; y[i + 2] += q.z; y[i + 3] += q.w;
                                }
                        }
                        if (p.acc_out) {
                            store_row32(part, 0, true, false, true, p.n - col, y);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++) y[i] *= scale;
                            store_row32(p.out, orow * p.out_pitch + p.out_col0 + col, p.out_f32, p.out_add, p.wide, p.n - col, y);
                        }
                    }
                }
            } else {
                // thread = vocabulary entry, registers = tokens: a warp's store covers 32 consecutive entries of a row
                const float scale = live ? __ldg(p.m_scale + row) : 0.f;
#pragma unroll 1
                for (uint32_t c = 0; c < half_cols; c += 16) {
                    uint32_t r[16];
                    if (some && ok) {
                        tc_ld16(taddr + c, r);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++) r[i] = 0u;
                    }
                    const uint32_t col = col0 + c;
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            if (col + i < p.n) {
                                float y = ((float)(int32_t)r[i] * __ldg(p.n_scale + col + i)) * scale;
                                if (!ok) y = __int_as_float(0x7fc00000);
                                const uint64_t at = (uint64_t)(col + i) * p.out_pitch + row;
                                if (p.out_f32) reinterpret_cast<float*>(p.out)[at] = y;
                                else reinterpret_cast<uint16_t*>(p.out)[at] = (uint16_t)pack_bf16(y, 0.f);
                            }
                        }
                    }
                }
            }
            if (some) {
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive_cluster(in_first_cta(bar_acc_empty + 8 * acc));
                n++;
            }
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
    cluster_sync_all();  // neither CTA leaves while the other may still reach into its shared or tensor memory
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace nrl

// The matrix products of the readout's backward pass and of its 8-bit form: one kernel on CTA pairs
// (tcgen05.mma.cta_group::2, f32 or 32-bit integer accumulators in tensor memory), four epilogues.
//
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
constexpr uint32_t kHgSmemBytes = kHgSmemTiles + 1024 + 256;

enum { kEpiGrad = 0, kEpiHidden = 1, kEpiWeight = 2, kEpiInt8 = 3 };

struct HeadGemm {
    uint32_t m, n, k;          // extents of the product
    const uint32_t* m_count;   // device: the extent along M (≤ m) when only some rows are in use, or null
    const uint32_t* k_count;   // device: the extent along K (≤ k), or null
    uint32_t bn;               // columns per tile (a multiple of 32, ≤ 256)
    uint32_t stages;
    uint32_t a_mn, b_mn;       // A / B contiguous along M / N instead of K
    uint32_t b_n0, b_k0;       // where this piece of the vocabulary begins in B, along N / along K
    uint32_t a_m0;             // … in A, along M
    uint32_t nsplit;           // ranges of K, each with its own output buffer
    uint32_t group_m;          // 256-row blocks that are walked side by side (L2 reuse of B)
    // kEpiGrad
    const float4* coef;        // [rows] (a, b, m, ln Z) of the scored rows
    const float4* more;        // [rows] (H, scale of x, 1 / scale, token bits)
    const uint32_t* rows_at;   // [rows] the row in the caller's order
    float tau;
    uint32_t round_bf16;
    uint32_t entropy_term;     // some b ≠ 0 is possible
    const uint8_t* allow;
    uint64_t allow_stride;
    uint32_t allow_bits;
    uint32_t vocab;            // V
    uint32_t v0;               // first column of this piece
    uint16_t* dz;              // [rows, dz_pitch]
    uint64_t dz_pitch;
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
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {  // nearest, ties to even; NaN stays NaN
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 32 columns of one row of dz (thread = row).
__device__ __forceinline__ void epi_grad(const HeadGemm& p, uint32_t row, bool live, uint32_t col, float z[32], const float4& cf, const float4& mo, uint64_t caller_row) {
    const uint32_t v = p.v0 + col;
    uint32_t packed[16];
    if (!live || v >= p.vocab) {
#pragma unroll
        for (int i = 0; i < 16; i++) packed[i] = 0u;
    } else {
        uint32_t keep = 0xffffffffu;  // columns that exist and are allowed
        if (v + 32 > p.vocab) keep = 0xffffffffu >> (v + 32 - p.vocab);
        if (p.allow) {
            if (p.allow_bits) {
                keep &= __ldg(reinterpret_cast<const uint32_t*>(p.allow) + caller_row * p.allow_stride + (v >> 5));
            } else {
                const uint8_t* mp = p.allow + caller_row * p.allow_stride + v;
                uint32_t bits = 0u;
                if (v + 32 <= p.vocab && (reinterpret_cast<uintptr_t>(mp) & 15u) == 0) {
                    const uint4 q0 = ldg_stream16(mp), q1 = ldg_stream16(mp + 16);
                    const uint32_t w[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if ((w[i >> 2] >> (8 * (i & 3))) & 0xffu) bits |= 1u << i;
                } else {
                    for (int i = 0; i < 32; i++)
                        if (v + i < p.vocab && mp[i]) bits |= 1u << i;
                }
                keep &= bits;
            }
        }
        const float a = cf.x, b = cf.y, m = cf.z, lnZ = cf.w, H = mo.x, xs = mo.y;
        const int32_t tok = __float_as_int(mo.w) - (int32_t)v;
        float g[32];
#pragma unroll
        for (int i = 0; i < 32; i++) {
            float zi = z[i] * xs;  // xs = 1 for bf16 hidden states
            if (p.round_bf16) zi = round_through_bf16(zi);
            if (p.tau != 1.f) zi = __fdiv_rn(zi, p.tau);
            const float lp = fmaxf((zi - m) - lnZ, -1e30f);  // a −inf logit: π = 0, and 0·inf cannot appear
            const float pi = ex2_approx(lp * kLog2e);
            float t = a;
            if (p.entropy_term) t = fmaf(b, lp + H, a);
            float y = -pi * t;
            if (i == tok) y += a;
            g[i] = (keep >> i) & 1u ? y * xs : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) packed[i] = pack_bf16(g[2 * i], g[2 * i + 1]);
    }
    uint16_t* o = p.dz + (uint64_t)row * p.dz_pitch + col;
    stg32(o, packed);
    stg32(o + 16, packed + 8);
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

template <int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kHgThreads, 1) head_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ HeadGemm p) {
    extern __shared__ uint8_t smem_raw[];
    constexpr bool kI8 = EPI == kEpiInt8;
    constexpr uint32_t kKStep = kI8 ? 128 : 64;  // elements of K per stage (128 bytes)
    const uint32_t smem_base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t b_bytes = (p.bn / 2) * 128, stage_bytes = kHgABytes + b_bytes;
    const uint32_t bars = smem_base + kHgSmemTiles;
    const uint32_t bar_full = bars, bar_empty = bars + 8 * kHgMaxStages, bar_acc_full = bars + 16 * kHgMaxStages, bar_acc_empty = bar_acc_full + 16, bar_done = bar_acc_empty + 16;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t mm = p.m_count ? min(*p.m_count, p.m) : p.m, kk = p.k_count ? min(*p.k_count, p.k) : p.k;
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
        const uint32_t r_in_block = quarter * 32u + (uint32_t)lane;
        const uint32_t half_cols = p.bn / 2;  // this warp's columns: [half · bn/2, + bn/2), a multiple of 16
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
            const uint32_t row = w.tm * 2 * kHgBM + rank * kHgBM + r_in_block;
            const bool live = row < mm;
            const uint32_t taddr = tmem + ((quarter * 32u) << 16) + acc * 256 + half * half_cols;
            float4 cf = make_float4(0.f, 0.f, 0.f, 0.f), mo = cf;
            uint64_t caller_row = 0;
            float scale = alpha;
            if constexpr (EPI == kEpiGrad) {
                if (live) {
                    cf = __ldg(p.coef + row);
                    mo = __ldg(p.more + row);
                    caller_row = p.rows_at[row];
                }
            }
            if constexpr (EPI == kEpiHidden) {
                if (live && !p.acc_out) {
                    caller_row = p.rows_at[row];
                    scale = alpha * __ldg(p.more + row).z;
                }
            }
            if constexpr (EPI == kEpiInt8) scale = live ? __ldg(p.m_scale + row) : 0.f;
            if constexpr (EPI != kEpiInt8) {
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
                    const uint32_t col = w.tn * p.bn + half * half_cols + c;
                    if constexpr (EPI == kEpiGrad) {
                        epi_grad(p, row, live, col, y, cf, mo, caller_row);
                    } else {
                        if (live && col < p.n) {
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
                                const uint64_t orow = EPI == kEpiHidden ? caller_row : (uint64_t)p.out_row0 + row;
                                store_row32(p.out, orow * p.out_pitch + p.out_col0 + col, p.out_f32, p.out_add, p.wide, p.n - col, y);
                            }
                        }
                    }
                }
            } else {
                // thread = vocabulary entry, registers = tokens: a warp's store covers 32 consecutive entries of a row
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
                    const uint32_t col = w.tn * p.bn + half * half_cols + c;
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

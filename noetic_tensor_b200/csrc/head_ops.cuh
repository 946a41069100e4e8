// The small kernels around the products of head_gemm.cuh: which rows carry a gradient and with what
// coefficients, the scored rows' hidden states brought together, the ranges of a split sum added up,
// and rows quantised to 8-bit integers and back.
#pragma once
#include "head_gemm.cuh"

namespace nrl {

struct HeadRows {
    uint64_t rows;
    uint32_t d;
    uint32_t per_block;       // rows a block owns
    // which rows are scored: backward, those with an upstream; forward, those whose mask is not 0
    const float* g_logp;      // [rows] or null
    const float* g_ent;       // [rows] or null
    const float* scored;      // [rows] or null (forward)
    // backward: the rows' coefficients
    const float* rowstats;    // [rows, 4]: (m, ln Z, ·, ·)
    const float* entropy;     // [rows], with g_ent
    const int32_t* tokens;    // [rows], with g_logp
    float tau;
    float* alpha;             // out: the common factor of the coefficients
    float4* coef;             // out [rows]
    float4* more;             // out [rows]
    const void* hidden;       // bf16 [rows, d], or int8 [rows, pitch]
    uint64_t pitch;           // of int8 rows
    const float* scales;      // [rows] of int8 rows, or null: bf16
    uint32_t* count;          // out: scored rows
    uint32_t* rows_at;        // out [rows]: the scored rows in order
    uint16_t* x;              // out bf16 [rows rounded up to 256, d]
    // rows that are not scored: zeros into d_hidden (backward, unless null) or into the results (forward)
    void* d_hidden;
    uint32_t d_hidden_f32;
    float* logp;
    float* out_entropy;
    float4* out_rowstats;
    uint8_t* status;
};

constexpr int kRowsThreads = 256;

// A row without an upstream (a mask) is not scored: nothing of it is read, so whatever a padded position holds stays out of the sums.
__device__ __forceinline__ bool head_scored(const HeadRows& p, uint64_t r) {
    if (p.scored) return p.scored[r] != 0.f;
    const float a = p.g_logp ? p.g_logp[r] : 0.f, b = p.g_ent ? p.g_ent[r] : 0.f;
    return a != 0.f || b != 0.f;  // a NaN counts as scored
}

// Brings the scored rows together: their hidden states (8-bit integers as bf16, exactly), with zeros up to the next multiple of 256
// rows because the products read whole tiles; their places; and, backward, their coefficients. One launch: every block looks at all
// rows' upstreams (a few KB out of L2) to know where its own rows go, which costs less than a second launch.
//
// The coefficients are divided by c = the largest finite |upstream| of the call, which goes into alpha = c / τ and is applied to the
// f32 sums at the end: dz is rounded to bf16 before the products, and with equal upstreams (a mean) the target's entry −(1 − π)
// then keeps the precision it would lose as −(1 − π) / N in every row alike.
__global__ void __launch_bounds__(kRowsThreads) head_rows_kernel(HeadRows p) {
    constexpr int kW = kRowsThreads / 32;
    __shared__ uint32_t sum_before[kW], sum_all[kW], wcount[kW];
    __shared__ float wmax[kW];
    __shared__ uint32_t place_of[kRowsThreads];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t first = (uint64_t)blockIdx.x * p.per_block, last = min(first + p.per_block, p.rows);
    uint32_t before = 0, total = 0;
    float c = 0.f;
#pragma unroll 4
    for (uint64_t r = threadIdx.x; r < p.rows; r += kRowsThreads) {
        const float a = p.scored ? fabsf(p.scored[r]) : p.g_logp ? fabsf(p.g_logp[r]) : 0.f, b = p.g_ent ? fabsf(p.g_ent[r]) : 0.f;
        const uint32_t on = (a != 0.f || b != 0.f) ? 1u : 0u;
        total += on;
        before += r < first ? on : 0u;
        if (a <= FLT_MAX) c = fmaxf(c, a);
        if (b <= FLT_MAX) c = fmaxf(c, b);
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, k);
        total += __shfl_xor_sync(0xffffffffu, total, k);
        c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, k));
    }
    if (lane == 0) { sum_before[warp] = before; sum_all[warp] = total; wmax[warp] = c; }
    __syncthreads();
    before = total = 0;
    for (int w = 0; w < kW; w++) { before += sum_before[w]; total += sum_all[w]; c = fmaxf(c, wmax[w]); }
    if (!(c > 0.f)) c = 1.f;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *p.count = total;
        if (p.alpha) *p.alpha = c / p.tau;
    }
    const uint32_t pieces = p.d / 8;
    for (uint64_t r0 = first; r0 < last; r0 += kRowsThreads) {
        const uint64_t r = r0 + threadIdx.x;
        const bool mine = r < last, on = mine && head_scored(p, r);
        const uint32_t ballot = __ballot_sync(0xffffffffu, on);
        if (lane == 0) wcount[warp] = __popc(ballot);
        __syncthreads();
        uint32_t place = before + __popc(ballot & ((1u << lane) - 1u)), here = 0;
        for (int w = 0; w < kW; w++) {
            if (w < warp) place += wcount[w];
            here += wcount[w];
        }
        place_of[threadIdx.x] = on ? place : 0xffffffffu;
        if (on) {
            p.rows_at[place] = (uint32_t)r;
            if (p.coef) {
                const float4 st = reinterpret_cast<const float4*>(p.rowstats)[r];
                float a = p.g_logp ? p.g_logp[r] / c : 0.f;
                const float b = p.g_ent ? p.g_ent[r] / c : 0.f, H = p.g_ent ? p.entropy[r] : 0.f;
                if (!(fabsf(st.x) <= FLT_MAX && fabsf(st.y) <= FLT_MAX)) a = __int_as_float(0x7fc00000);  // a row the forward refused: its gradient is NaN
                float s = p.scales ? p.scales[r] : 1.f;
                if (fabsf(s) < 0x1p-100f) s = 1.f;  // a row of zeros (it is gathered as zeros)
                p.coef[place] = make_float4(a * s, b * s, (st.x + st.y) * kLog2e, a * s + b * s * H);
                p.more[place] = make_float4(s, 1.f / s, __int_as_float(p.tokens && p.g_logp ? p.tokens[r] : -1), 0.f);
            }
        } else if (mine) {
            if (p.logp) p.logp[r] = 0.f;
            if (p.out_entropy) p.out_entropy[r] = 0.f;
            if (p.out_rowstats) p.out_rowstats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.status) p.status[r] = 0;
        }
        __syncthreads();
        const uint32_t n = (uint32_t)min((uint64_t)kRowsThreads, last - r0);
        for (uint32_t j = warp; j < n; j += kW) {  // a warp per row
            const uint64_t row = r0 + j;
            const uint32_t at = place_of[j];
            if (at == 0xffffffffu) {
                if (p.d_hidden) {
                    const uint32_t n16 = pieces * (p.d_hidden_f32 ? 2u : 1u);
                    uint4* o = reinterpret_cast<uint4*>(p.d_hidden) + row * n16;
                    for (uint32_t i = lane; i < n16; i += 32) o[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                continue;
            }
            uint4* o = reinterpret_cast<uint4*>(p.x + (uint64_t)at * p.d);
            if (p.scales && fabsf(p.scales[row]) < 0x1p-100f) {
                for (uint32_t i = lane; i < pieces; i += 32) o[i] = make_uint4(0u, 0u, 0u, 0u);
            } else if (p.scales) {
                const uint2* q = reinterpret_cast<const uint2*>(reinterpret_cast<const int8_t*>(p.hidden) + row * p.pitch);
#pragma unroll 4
                for (uint32_t i = lane; i < pieces; i += 32) {
                    const uint2 v = q[i];
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t two = (k < 2 ? v.x : v.y) >> (16 * (k & 1));
                        w[k] = pack_bf16((float)(int8_t)(two & 0xffu), (float)(int8_t)((two >> 8) & 0xffu));
                    }
                    o[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
                const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.hidden) + row * p.d);
#pragma unroll 8
                for (uint32_t i = lane; i < pieces; i += 32) o[i] = q[i];
            }
        }
        before += here;
        __syncthreads();
    }
    for (uint64_t i = total + (uint64_t)blockIdx.x * kW + warp; i < ((total + 255u) & ~255u); i += (uint64_t)gridDim.x * kW) {
        uint4* o = reinterpret_cast<uint4*>(p.x + i * p.d);
        for (uint32_t k = lane; k < pieces; k += 32) o[k] = make_uint4(0u, 0u, 0u, 0u);
    }
}

// The partial statistics of a row merged: a warp per scored row, lane l taking the partials l, l + 32, …, f64 sums, a butterfly.
struct HeadFinish {
    uint32_t rows;              // of this launch
    const uint32_t* count;      // device: scored rows in all, or null
    uint32_t first;             // this launch's first among them
    const uint32_t* rows_at;    // from `first` on, or null: the caller's order
    const float* scored;        // with rows_at null: rows that are not scored get zeros
    const float4* parts;
    uint32_t nparts;
    const int32_t* tokens;
    float* logp;
    float* entropy;
    float4* rowstats;
    uint8_t* status;
};
__global__ void __launch_bounds__(256) head_finish_kernel(HeadFinish p) {
    const uint32_t i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= p.rows || (p.count && p.first + i >= *p.count)) return;
    const uint64_t row = p.rows_at ? p.rows_at[i] : i;
    if (!p.rows_at && p.scored && p.scored[row] == 0.f) {
        if (lane == 0) {
            if (p.logp) p.logp[row] = 0.f;
            if (p.entropy) p.entropy[row] = 0.f;
            if (p.rowstats) p.rowstats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.status) p.status[row] = 0;
        }
        return;
    }
    const float4* q = p.parts + (uint64_t)i * p.nparts;
    float m = -FLT_MAX, ztok = __int_as_float(0x7fc00000);
    uint32_t gave_up = 0u;
#pragma unroll 4
    for (uint32_t j = lane; j < p.nparts; j += 32) {
        const float4 a = q[j];
        m = fmax_nan(m, a.x);
        gave_up |= a.y < 0.f ? 1u : 0u;
        if (a.w == a.w) ztok = a.w;
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, k));
    double Z = 0.0, W = 0.0;
#pragma unroll 4
    for (uint32_t j = lane; j < p.nparts; j += 32) {
        const float4 a = q[j];
        if (a.y > 0.f) {
            const float dm = a.x - m;
            const double c = (double)expf(dm);
            Z += c * (double)a.y;
            W += c * ((double)a.z + (double)a.y * (double)dm);
        }
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) {
        Z += __shfl_xor_sync(0xffffffffu, Z, k);
        W += __shfl_xor_sync(0xffffffffu, W, k);
    }
    const uint32_t has = __ballot_sync(0xffffffffu, ztok == ztok);
    if (has) ztok = __shfl_sync(0xffffffffu, ztok, __ffs(has) - 1);
    gave_up = __any_sync(0xffffffffu, gave_up);
    if (lane) return;
    uint32_t st = gave_up ? 4u : 0u;
    if (m != m) st |= 2u;
    else if (m <= -FLT_MAX) st |= 1u;
    const float nan = __int_as_float(0x7fc00000), lnZ = (float)log(Z);
    if (p.rowstats) p.rowstats[row] = st ? make_float4(nan, nan, nan, nan) : make_float4(m, lnZ, 0.f, 0.f);
    if (p.entropy) p.entropy[row] = st ? nan : (float)(log(Z) - W / Z);
    // a token outside [0, V) has no logit: NaN; an excluded one has log-prob −inf
    if (p.logp) p.logp[row] = st ? nan : ztok <= -FLT_MAX ? NRL_NEG_INF : (ztok - m) - lnZ;
    if (p.status) p.status[row] = (uint8_t)st;
}

// A block per seed: value = Σ keep·(−logp) / max(Σ keep, 1) and its gradient upstream·(−keep / max(Σ keep, 1)). Positions with
// keep = 0 are not looked at.
__global__ void __launch_bounds__(512) ce_mean_kernel(uint64_t n, const float* logp, const float* keep, const float* upstream, float* out, float* g_logp) {
    __shared__ double sv[16], sc[16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t base = (uint64_t)blockIdx.x * n;
    double v = 0.0, c = 0.0;
#pragma unroll 4
    for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const float k = keep ? keep[base + i] : 1.f;
        c += (double)k;
        if (out && k != 0.f) v -= (double)(logp[base + i] * k);
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, k);
        c += __shfl_xor_sync(0xffffffffu, c, k);
    }
    if (lane == 0) { sv[warp] = v; sc[warp] = c; }
    __syncthreads();
    v = c = 0.0;
    for (int w = 0; w < 16; w++) { v += sv[w]; c += sc[w]; }
    const double count = c > 1.0 ? c : 1.0;
    if (out && threadIdx.x == 0) out[blockIdx.x] = (float)(v / count);
    if (!g_logp) return;
    const float g = (float)((upstream ? (double)upstream[blockIdx.x] : 1.0) / count);
    for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) g_logp[base + i] = keep ? -(keep[base + i] * g) : -g;
}

// d_hidden of the scored rows from the ranges of a split sum, added in range order.
__global__ void __launch_bounds__(128) head_fold_kernel(const uint32_t* count, const float* alpha, const float4* more, const uint32_t* rows_at, const float* acc, uint64_t acc_rows, uint32_t nsplit,
                                                        uint32_t d, void* out, uint32_t out_f32, uint32_t add) {
    const uint32_t i = blockIdx.x;
    if (i >= *count) return;
    const float scale = *alpha * more[i].y;
    const uint64_t r = rows_at[i];
    for (uint32_t c = threadIdx.x * 4; c < d; c += blockDim.x * 4) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t s = 0; s < nsplit; s++) {
            const float4 q = *reinterpret_cast<const float4*>(acc + ((uint64_t)s * acc_rows + i) * d + c);
            y.x += q.x; y.y += q.y; y.z += q.z; y.w += q.w;
        }
        y.x *= scale; y.y *= scale; y.z *= scale; y.w *= scale;
        if (out_f32) {
            float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + r * d + c);
            if (add) {
                const float4 q = *o;
                y.x += q.x; y.y += q.y; y.z += q.z; y.w += q.w;
            }
            *o = y;
        } else {
            uint2* o = reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + r * d + c);
            if (add) {
                const uint2 q = *o;
                y.x += bf16_lo(q.x); y.y += bf16_hi(q.x); y.z += bf16_lo(q.y); y.w += bf16_hi(q.y);
            }
            *o = make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
        }
    }
}

// ---- 8-bit rows -----------------------------------------------------------------------------------
//
// q = rint(127·x / max|x|) (ties to even) and the scale max|x| / 127 in f32, so x ≈ q·scale. 127·x is exact for bf16 x and the
// division is correctly rounded, so q is the integer of exact arithmetic: x / (max|x| / 127) would fall on either side of the
// ties that x = max|x| / 2 produces. A row with an infinity or a NaN gets a non-finite scale and zeros.
__device__ __forceinline__ int32_t quantise(float x, float big) {
    const float q = __fdiv_rn(x * 127.f, big);
    return big > 0.f ? max(-127, min(127, __float2int_rn(q))) : 0;
}
template <int DT>
__device__ __forceinline__ float load_x(const void* x, uint64_t i) {
    if (DT == NRL_BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(x)[i] << 16);
    return reinterpret_cast<const float*>(x)[i];
}
template <int DT>
__device__ __forceinline__ void load_x8(const void* x, uint64_t i, float z[8]) {
    if (DT == NRL_BF16) {
        const uint4 q = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + i);
        z[0] = bf16_lo(q.x); z[1] = bf16_hi(q.x); z[2] = bf16_lo(q.y); z[3] = bf16_hi(q.y);
        z[4] = bf16_lo(q.z); z[5] = bf16_hi(q.z); z[6] = bf16_lo(q.w); z[7] = bf16_hi(q.w);
    } else {
        const float4 a = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + i)[0], b = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + i)[1];
        z[0] = a.x; z[1] = a.y; z[2] = a.z; z[3] = a.w; z[4] = b.x; z[5] = b.y; z[6] = b.z; z[7] = b.w;
    }
}
// the block's maximum, a NaN winning; `sm` holds 33 floats
__device__ __forceinline__ float block_max_nan(float m, float* sm) {
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, k));
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < blockDim.x >> 5; w++) m = fmax_nan(m, sm[w]);
        sm[32] = m;
    }
    __syncthreads();
    return sm[32];
}

// A block per row; `vec`: the row starts are 16-byte aligned and d is a multiple of 8. Up to 8192 elements stay in registers
// between the maximum and the rounding; what a longer row has beyond them is read a second time.
template <int DT>
__global__ void __launch_bounds__(256) quantise_rows_kernel(const void* x, uint32_t d, uint64_t pitch, int8_t* q, float* scales, bool vec) {
    __shared__ float sm[33];
    const uint64_t row = blockIdx.x, at = row * d;
    constexpr int kHeld = 4;
    float z[kHeld][8];
    float big = 0.f;
    if (vec) {
#pragma unroll
        for (int k = 0; k < kHeld; k++) {
            const uint32_t c = (threadIdx.x + k * 256) * 8;
            if (c < d) load_x8<DT>(x, at + c, z[k]);
        }
#pragma unroll
        for (int k = 0; k < kHeld; k++)
            if ((threadIdx.x + k * 256) * 8 < d) {
#pragma unroll
                for (int i = 0; i < 8; i++) big = fmax_nan(big, fabsf(z[k][i]));
            }
        for (uint32_t c = (threadIdx.x + kHeld * 256) * 8; c < d; c += 256 * 8) {
            float t[8];
            load_x8<DT>(x, at + c, t);
#pragma unroll
            for (int i = 0; i < 8; i++) big = fmax_nan(big, fabsf(t[i]));
        }
    } else {
        for (uint32_t c = threadIdx.x; c < d; c += blockDim.x) big = fmax_nan(big, fabsf(load_x<DT>(x, at + c)));
    }
    big = block_max_nan(big, sm);
    int8_t* o = q + row * pitch;
    auto store8 = [&](const float t[8], uint32_t c) {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; i++) w[i >> 2] |= ((uint32_t)quantise(t[i], big) & 0xffu) << (8 * (i & 3));
        *reinterpret_cast<uint2*>(o + c) = make_uint2(w[0], w[1]);
    };
    if (vec) {
#pragma unroll
        for (int k = 0; k < kHeld; k++) {
            const uint32_t c = (threadIdx.x + k * 256) * 8;
            if (c < d) store8(z[k], c);
        }
        for (uint32_t c = (threadIdx.x + kHeld * 256) * 8; c < d; c += 256 * 8) {
            float t[8];
            load_x8<DT>(x, at + c, t);
            store8(t, c);
        }
    } else {
        for (uint32_t c = threadIdx.x; c < d; c += blockDim.x) o[c] = (int8_t)quantise(load_x<DT>(x, at + c), big);
    }
    for (uint64_t c = d + threadIdx.x; c < pitch; c += blockDim.x) o[c] = 0;
    if (threadIdx.x == 0) scales[row] = __fdiv_rn(big, 127.f);
}

// Columns of a bf16 [d, V] weight as rows [V, pitch] of integers: a block takes 64 columns, finds their maxima over d and then
// turns 64 × 64 tiles over in shared memory. Bound by HBM: the second read of the block's columns (64·d·2 bytes) hits L2.
__global__ void __launch_bounds__(256) quantise_columns_kernel(const uint16_t* w, uint32_t d, uint32_t V, uint64_t pitch, int8_t* q, float* scales) {
    __shared__ float part[4][64];
    __shared__ float big[64];
    __shared__ int8_t tile[64][68];
    const uint32_t c = threadIdx.x & 63, part_of = threadIdx.x >> 6;
    const uint32_t v = blockIdx.x * 64 + c;
    float m = 0.f;
    if (v < V)
        for (uint32_t k = part_of; k < d; k += 4) m = fmax_nan(m, fabsf(load_x<NRL_BF16>(w, (uint64_t)k * V + v)));
    part[part_of][c] = m;
    __syncthreads();
    if (threadIdx.x < 64) {
        m = fmax_nan(fmax_nan(part[0][c], part[1][c]), fmax_nan(part[2][c], part[3][c]));
        big[c] = m;
        if (v < V) scales[v] = __fdiv_rn(m, 127.f);
    }
    __syncthreads();
    const float b = big[c];
    for (uint32_t k0 = 0; k0 < pitch; k0 += 64) {
        for (uint32_t k = part_of; k < 64; k += 4) tile[c][k] = v < V && k0 + k < d ? (int8_t)quantise(load_x<NRL_BF16>(w, (uint64_t)(k0 + k) * V + v), b) : (int8_t)0;
        __syncthreads();
        // 64 rows of 64 bytes, four bytes a thread and step
        for (uint32_t i = threadIdx.x; i < 64 * 16; i += 256) {
            const uint32_t r = i >> 4, k = (i & 15) * 4;
            if (blockIdx.x * 64 + r < V && k0 + k < pitch) *reinterpret_cast<uint32_t*>(q + (uint64_t)(blockIdx.x * 64 + r) * pitch + k0 + k) = *reinterpret_cast<const uint32_t*>(&tile[r][k]);
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) dequantise_rows_kernel(const int8_t* q, const float* scales, uint32_t d, uint64_t pitch, void* out, uint32_t out_f32) {
    const uint64_t row = blockIdx.x;
    const float s = scales[row];
    for (uint32_t c = threadIdx.x; c < d; c += blockDim.x) {
        const float y = (float)q[row * pitch + c] * s;
        if (out_f32) reinterpret_cast<float*>(out)[row * d + c] = y;
        else reinterpret_cast<uint16_t*>(out)[row * d + c] = (uint16_t)pack_bf16(y, 0.f);
    }
}

}  // namespace nrl

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
    uint16_t* x;              // out bf16 [rows rounded up to 256, x_pitch]
    uint32_t x_pitch;         // d rounded up to 128 bytes: TMA reads then cover whole lines
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
    next_kernel_may_start();
    after_previous_kernel();
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
            uint4* o = reinterpret_cast<uint4*>(p.x + (uint64_t)at * p.x_pitch);
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
        uint4* o = reinterpret_cast<uint4*>(p.x + i * p.x_pitch);
        for (uint32_t k = lane; k < pieces; k += 32) o[k] = make_uint4(0u, 0u, 0u, 0u);
    }
}

// Per seed: out = Σ keep·(−logp) / max(Σ keep, 1) and its gradient g_logp = upstream·(−keep / max(Σ keep, 1)), by one block: thread t
// takes the positions t, t + blockDim, …, f64 sums, a butterfly, the warps in order. Positions with keep = 0 are not looked at. With
// `weights` it is the policy-gradient loss: the kept positions' −logp·weight over the same count, keep itself not a factor.
struct CeMean {
    uint64_t seeds, n;
    const float* logp;
    const float* keep;
    const float* weights;
    const float* upstream;
    float* out;
    float* g_logp;
};
constexpr int kMeanThreads = 1024;
// one seed, by all threads of the block; sh: a pair per warp
__device__ __forceinline__ void ce_mean_seed(const CeMean& p, uint64_t seed, double (*sh)[2]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t base = seed * p.n;
    double v = 0.0, c = 0.0;
#pragma unroll 8
    for (uint64_t i = threadIdx.x; i < p.n; i += blockDim.x) {
        const float k = p.keep ? p.keep[base + i] : 1.f, lp = p.out ? __ldcg(p.logp + base + i) : 0.f, w = p.weights ? p.weights[base + i] : k;
        c += (double)k;
        if (k != 0.f) v -= (double)(lp * w);
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, k);
        c += __shfl_xor_sync(0xffffffffu, c, k);
    }
    __syncthreads();
    if (lane == 0) { sh[warp][0] = v; sh[warp][1] = c; }
    __syncthreads();
    v = c = 0.0;
#pragma unroll 8
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) { v += sh[w][0]; c += sh[w][1]; }
    const double count = c > 1.0 ? c : 1.0;
    if (p.out && threadIdx.x == 0) p.out[seed] = (float)(v / count);
    if (!p.g_logp) return;
    const float g = (float)((p.upstream ? (double)p.upstream[seed] : 1.0) / count);
#pragma unroll 8
    for (uint64_t i = threadIdx.x; i < p.n; i += blockDim.x) {
        const float k = p.keep ? p.keep[base + i] : 1.f, w = p.weights ? p.weights[base + i] : k;
        p.g_logp[base + i] = k != 0.f ? -(w * g) : 0.f;
    }
}
__global__ void __launch_bounds__(kMeanThreads) ce_mean_kernel(CeMean p) {
    __shared__ double sh[kMeanThreads / 32][2];
    next_kernel_may_start();
    after_previous_kernel();
    ce_mean_seed(p, blockIdx.x, sh);
}

// The partial statistics of a row merged by kW warps (one when there are many rows, eight when there are few): thread t takes the
// partials t, t + 32·kW, …, f64 sums, a butterfly, then the warps in order.
struct HeadFinish {
    uint32_t rows;              // of this launch
    const uint32_t* count;      // device: scored rows in all, or null
    uint32_t first;             // this launch's first among them
    const uint32_t* rows_at;    // from `first` on, or null: the caller's order
    const float* scored;        // with rows_at null: rows that are not scored get zeros
    const float4* parts;
    uint32_t nparts;
    float* logp;
    float* entropy;
    float4* rowstats;
    uint8_t* status;
    // the means of a few seeds of a small call, by the last block to finish: which one that is changes no sum
    CeMean ce;                  // ce.seeds = 0: not here
    uint32_t* done;
};
template <int kW>
__device__ __forceinline__ void head_finish_row(const HeadFinish& p) {
    __shared__ float sm[8], st_[8];
    __shared__ double sz[8], sw[8];
    __shared__ uint32_t sg[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t i = kW == 1 ? blockIdx.x * 8 + warp : blockIdx.x, t = kW == 1 ? lane : threadIdx.x;
    if (i >= p.rows || (p.count && p.first + i >= *p.count)) return;
    const uint64_t row = p.rows_at ? p.rows_at[i] : i;
    if (!p.rows_at && p.scored && p.scored[row] == 0.f) {
        if (t == 0) {
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
    for (uint32_t j = t; j < p.nparts; j += 32 * kW) {
        const float4 a = q[j];
        m = fmax_nan(m, a.x);
        gave_up |= a.y < 0.f ? 1u : 0u;
        if (a.w == a.w) ztok = a.w;
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, k));
    const uint32_t has = __ballot_sync(0xffffffffu, ztok == ztok);
    if (has) ztok = __shfl_sync(0xffffffffu, ztok, __ffs(has) - 1);
    gave_up = __any_sync(0xffffffffu, gave_up);
    if (kW > 1) {
        if (lane == 0) { sm[warp] = m; st_[warp] = ztok; sg[warp] = gave_up; }
        __syncthreads();
        for (int w = 0; w < kW; w++) {
            m = fmax_nan(m, sm[w]);
            gave_up |= sg[w];
            if (st_[w] == st_[w]) ztok = st_[w];
        }
    }
    double Z = 0.0, W = 0.0;
#pragma unroll 4
    for (uint32_t j = t; j < p.nparts; j += 32 * kW) {
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
    if (kW > 1) {
        if (lane == 0) { sz[warp] = Z; sw[warp] = W; }
        __syncthreads();
        Z = W = 0.0;
        for (int w = 0; w < kW; w++) { Z += sz[w]; W += sw[w]; }
    }
    if (t) return;
    uint32_t st = gave_up ? 4u : 0u;
    if (m != m) st |= 2u;
    else if (m <= -FLT_MAX) st |= 1u;
    const float nan = __int_as_float(0x7fc00000);
    const double lnZ = log(Z);
    if (p.rowstats) p.rowstats[row] = st ? make_float4(nan, nan, nan, nan) : make_float4(m, (float)lnZ, 0.f, 0.f);
    if (p.entropy) p.entropy[row] = st ? nan : (float)(lnZ - W / Z);
    // a token outside [0, V) has no logit: NaN; an excluded one has log-prob −inf
    if (p.logp) p.logp[row] = st ? nan : ztok <= -FLT_MAX ? NRL_NEG_INF : (ztok - m) - (float)lnZ;
    if (p.status) p.status[row] = (uint8_t)st;
}

template <int kW>
__global__ void __launch_bounds__(256) head_finish_kernel(HeadFinish p) {
    next_kernel_may_start();
    after_previous_kernel();
    head_finish_row<kW>(p);
    if (!p.ce.seeds) return;
    __shared__ double sh[8][2];
    __shared__ uint32_t last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(p.done, 1u) == gridDim.x - 1 ? 1u : 0u;
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (uint64_t s = 0; s < p.ce.seeds; s++) ce_mean_seed(p.ce, s, sh);
}

// d_hidden of the scored rows from the ranges of a split sum; nothing to do where K was not split. 32 threads take 128 columns of a row,
// four each, with up to eight groups of them where there are many ranges: group g of G adds the ranges g, g + G, … in order, then the
// groups are added in order. With few ranges (many rows) the block's eight groups take eight rows instead (three ranges of 1536 × 2048:
// 29 us cold with eight groups to a row, bound by its barriers; 30 us less in a backward call). The grid goes on with its stride (the
// host does not know the number of rows).
__global__ void __launch_bounds__(256) head_fold_kernel(const uint32_t* count, const float* alpha, const float4* more, const uint32_t* rows_at, const float* acc, uint32_t chunks, uint32_t side_by_side, uint32_t bn, uint32_t d, void* out,
                                                        uint32_t out_f32, uint32_t add) {
    __shared__ float4 part[8][32];
    next_kernel_may_start();
    after_previous_kernel();
    const uint32_t n = *count, tiles_m = (n + 255) / 256, nsplit = hidden_split(tiles_m * ((d + bn - 1) / bn), chunks, side_by_side), across = (d + 127) / 128;
    if (nsplit == 1) return;
    const float common = *alpha;
    const uint64_t range = (uint64_t)HeadGemm::acc_rows(n) * d;
    const uint32_t t = threadIdx.x & 31, warp = threadIdx.x >> 5, G = nsplit >= 16 ? 8u : nsplit >= 8 ? 4u : 1u, g = warp & (G - 1), rows = 8 / G;
    for (uint32_t b = blockIdx.x; b < (n + rows - 1) / rows * across; b += gridDim.x) {
        const uint32_t i = b / across * rows + warp / G, c = (b % across * 32 + t) * 4;
        const bool mine = i < n && c < d;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mine) {
            const float* q0 = acc + (uint64_t)i * d + c;
#pragma unroll 8
            for (uint32_t s = g; s < nsplit; s += G) {
                const float4 q = *reinterpret_cast<const float4*>(q0 + s * range);
                y.x += q.x; y.y += q.y; y.z += q.z; y.w += q.w;
            }
        }
        if (G > 1) {
            part[warp][t] = y;
            __syncthreads();
            if (g == 0)
                for (uint32_t k = 1; k < G; k++) { y.x += part[warp + k][t].x; y.y += part[warp + k][t].y; y.z += part[warp + k][t].z; y.w += part[warp + k][t].w; }
        }
        if (g == 0 && mine) {
            const float scale = common * more[i].y;
            const uint64_t r = rows_at[i];
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
        if (G > 1) __syncthreads();
    }
}

// ---- 8-bit rows -----------------------------------------------------------------------------------
//
// q = rint(127·x / max|x|) (ties to even) and the scale max|x| / 127 in f32, so x ≈ q·scale. 127·x is exact for bf16 x and the
// division is correctly rounded, so q is the integer of exact arithmetic: x / (max|x| / 127) would fall on either side of the
// ties that x = max|x| / 2 produces. A row with an infinity or a NaN gets a non-finite scale and zeros.
// The division is a product with 127 / max|x| wherever that cannot change the integer, which is unless the quotient lies within 1e-4
// of a tie (the product's error is below 127·2^-22), and the rounding is an addition of 1.5·2^23, whose low byte then is the integer:
// with the IEEE division and the conversion instructions the kernel was bound by arithmetic (39 us for 8192 × 4096 bf16).
struct Quantiser {
    float big, c;
    __device__ __forceinline__ explicit Quantiser(float b) : big(b) { c = b >= 0x1p-100f && b <= FLT_MAX ? 127.f * __frcp_rn(b) : __int_as_float(0x7fc00000); }
    // the integer in the low byte, and how far the quotient is from it
    __device__ __forceinline__ uint32_t near(float x, float& off) const {
        const float a = x * c, r = a + 12582912.f;
        off = fabsf(a - (r - 12582912.f));
        return __float_as_uint(r);
    }
    __device__ __forceinline__ uint32_t exact(float x) const {
        const float k = big > 0x1p100f ? 0x1p-32f : 1.f;  // 127·x stays finite (what becomes subnormal here rounds to 0 either way)
        return big > 0.f ? (uint32_t)max(-127, min(127, __float2int_rn(__fdiv_rn(x * k * 127.f, big * k)))) : 0u;
    }
    __device__ __forceinline__ uint32_t operator()(float x) const {
        float off;
        const uint32_t q = near(x, off);
        return off <= 0.4999f ? q : exact(x);
    }
    __device__ __forceinline__ uint2 eight(const float z[8]) const {
        uint32_t q[8];
        float worst = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float off;
            q[i] = near(z[i], off);
            worst = fmax_nan(worst, off);
        }
        if (!(worst <= 0.4999f)) {
#pragma unroll
            for (int i = 0; i < 8; i++) q[i] = exact(z[i]);
        }
        return make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410), __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
    }
};
template <int DT>
__device__ __forceinline__ float load_x(const void* x, uint64_t i) {
    if (DT == NRL_BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(x)[i] << 16);
    return reinterpret_cast<const float*>(x)[i];
}
// eight elements as they lie in memory
template <int DT>
struct RawX {
    uint4 q[DT == NRL_BF16 ? 1 : 2];
    __device__ __forceinline__ void load(const void* x, uint64_t i) {
        const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(x) + i * (DT == NRL_BF16 ? 2 : 4));
#pragma unroll
        for (int k = 0; k < (DT == NRL_BF16 ? 1 : 2); k++) q[k] = s[k];
    }
    __device__ __forceinline__ void unpack(float z[8]) const {
        if constexpr (DT == NRL_BF16) {
            z[0] = bf16_lo(q[0].x); z[1] = bf16_hi(q[0].x); z[2] = bf16_lo(q[0].y); z[3] = bf16_hi(q[0].y);
            z[4] = bf16_lo(q[0].z); z[5] = bf16_hi(q[0].z); z[6] = bf16_lo(q[0].w); z[7] = bf16_hi(q[0].w);
        } else {
            z[0] = __uint_as_float(q[0].x); z[1] = __uint_as_float(q[0].y); z[2] = __uint_as_float(q[0].z); z[3] = __uint_as_float(q[0].w);
            z[4] = __uint_as_float(q[1].x); z[5] = __uint_as_float(q[1].y); z[6] = __uint_as_float(q[1].z); z[7] = __uint_as_float(q[1].w);
        }
    }
};

// kW warps per row (eight, or one when there are rows enough to fill the device: no barrier then, and eight rows to a block); `vec`:
// the row starts are 16-byte aligned and d is a multiple of 8. The second look at a row hits the caches. Keeping the row in registers
// instead took 16 unrolled copies of the rounding per warp, and the kernel waited for instructions (50 us for 8192 × 4096 bf16).
template <int DT, int kW>
__global__ void __launch_bounds__(256) quantise_rows_kernel(const void* x, uint64_t rows, uint32_t d, uint64_t pitch, int8_t* q, float* scales, bool vec) {
    __shared__ float sm[8];
    next_kernel_may_start();
    after_previous_kernel();
    constexpr uint32_t kT = 32 * kW;  // threads per row
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t row = kW == 1 ? (uint64_t)blockIdx.x * 8 + warp : blockIdx.x;
    const uint32_t t = kW == 1 ? (uint32_t)lane : threadIdx.x;
    if (row >= rows) return;
    const uint64_t at = row * d;
    float big = 0.f;
    if (vec) {
#pragma unroll 4
        for (uint32_t c = t * 8; c < d; c += kT * 8) {
            RawX<DT> r;
            float z[8];
            r.load(x, at + c);
            r.unpack(z);
#pragma unroll
            for (int i = 0; i < 8; i++) z[i] = fabsf(z[i]);
            big = fmax3_nan(big, fmax3_nan(z[0], z[1], z[2]), fmax3_nan(fmax3_nan(z[3], z[4], z[5]), z[6], z[7]));
        }
    } else {
#pragma unroll 4
        for (uint32_t c = t; c < d; c += kT) big = fmax_nan(big, fabsf(load_x<DT>(x, at + c)));
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) big = fmax_nan(big, __shfl_xor_sync(0xffffffffu, big, k));
    if (kW > 1) {
        if (lane == 0) sm[warp] = big;
        __syncthreads();
        for (int w = 0; w < kW; w++) big = fmax_nan(big, sm[w]);
    }
    const Quantiser quantise(big);
    int8_t* o = q + row * pitch;
    if (vec) {
#pragma unroll 2
        for (uint32_t c = t * 8; c < d; c += kT * 8) {
            RawX<DT> r;
            float z[8];
            r.load(x, at + c);
            r.unpack(z);
            *reinterpret_cast<uint2*>(o + c) = quantise.eight(z);
        }
    } else {
#pragma unroll 4
        for (uint32_t c = t; c < d; c += kT) o[c] = (int8_t)quantise(load_x<DT>(x, at + c));
    }
    for (uint64_t c = d + t; c < pitch; c += kT) o[c] = 0;
    if (t == 0) scales[row] = __fdiv_rn(big, 127.f);
}

// Columns of a bf16 [d, V] weight as rows [V, pitch] of integers: a block takes 64 columns, finds their maxima over d and then
// turns 64 × 64 tiles over in shared memory. Bound by the latency of its two-byte loads and the two barriers per tile, not by HBM
// (2048 × 151 936: 870 us, 1.24 GB read, each column twice since the blocks' columns do not stay in L2, 0.28 GB written); a weight is
// laid out once. A [V, d] weight goes through the row kernel (197 us).
__global__ void __launch_bounds__(256) quantise_columns_kernel(const uint16_t* w, uint32_t d, uint32_t V, uint64_t pitch, int8_t* q, float* scales) {
    __shared__ float part[4][64];
    __shared__ float big[64];
    __shared__ uint32_t tile[64][17];  // 64 bytes a row and one word more: written by bytes down a column, read by words
    next_kernel_may_start();
    after_previous_kernel();
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
    const Quantiser quantise(big[c]);
    int8_t* mine = reinterpret_cast<int8_t*>(tile[c]);
    for (uint32_t k0 = 0; k0 < pitch; k0 += 64) {
        for (uint32_t k = part_of; k < 64; k += 4) mine[k] = v < V && k0 + k < d ? (int8_t)quantise(load_x<NRL_BF16>(w, (uint64_t)(k0 + k) * V + v)) : (int8_t)0;
        __syncthreads();
        // 64 rows of 64 bytes, four bytes a thread and step
        for (uint32_t i = threadIdx.x; i < 64 * 16; i += 256) {
            const uint32_t r = i >> 4, k = (i & 15) * 4;
            if (blockIdx.x * 64 + r < V && k0 + k < pitch) *reinterpret_cast<uint32_t*>(q + (uint64_t)(blockIdx.x * 64 + r) * pitch + k0 + k) = tile[r][i & 15];
        }
        __syncthreads();
    }
}

// A block per row, a value per thread and step: bound by its narrow loads and stores (151 936 × 2048 as bf16: 578 us, 1.6 TB/s).
__global__ void __launch_bounds__(256) dequantise_rows_kernel(const int8_t* q, const float* scales, uint32_t d, uint64_t pitch, void* out, uint32_t out_f32) {
    next_kernel_may_start();
    after_previous_kernel();
    const uint64_t row = blockIdx.x;
    const float s = scales[row];
    for (uint32_t c = threadIdx.x; c < d; c += blockDim.x) {
        const float y = (float)q[row * pitch + c] * s;
        if (out_f32) reinterpret_cast<float*>(out)[row * d + c] = y;
        else reinterpret_cast<uint16_t*>(out)[row * d + c] = (uint16_t)pack_bf16(y, 0.f);
    }
}

}  // namespace nrl

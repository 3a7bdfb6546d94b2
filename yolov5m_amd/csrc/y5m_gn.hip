// Group normalisation + activation over channels-last rows, forward and backward, with the input optionally kept in 8 bits.
//
//   forward   per (sample n, group g of D = C / G channels), K = S * D values:  mean, rstd = 1 / sqrt(var + eps)
//             xhat = (x - mean) rstd,  t = gamma_c xhat + beta_c,  z = t or t sigmoid(t);  optionally the 8-bit form of x (y5m_act8.h)
//   backward  from x or its 8-bit form:  dt = dz act'(t),  dbeta_c = sum dt,  dgamma_c = sum dt xhat  (over n and rows)
//             dx = rstd (gamma dt - A - xhat B),  A = sum_group(gamma dt) / K,  B = sum_group(gamma dt xhat) / K
//
// All of it is bound by bytes. The statistics of a group must be complete before its first output, so either the values stay on the
// chip between the two (not here) or they are read twice:
//   split form: a reduce pass over row chunks (partial sums per channel and chunk, f32), a small launch that joins the chunks in a
//   fixed order in f64, and an apply pass. No atomics: the result does not depend on the order in which workgroups run.
// A thread owns 8 channels of a row (16 bytes of bf16) for the whole launch, so gamma / beta / mean / rstd sit in registers and
// consecutive lanes read consecutive pieces of consecutive rows, whatever D is: groups are cut out when the channel sums are joined,
// never by the loads (at 96 channels in 32 groups a group is 6 bytes wide).
// Sums of squares are taken about a pivot per (n, channel), the median of three of its rows: sum (x - p)^2 - (sum (x - p))^2 / S
// cancels only by how far p lies from the mean, and the median keeps a single outlier row from becoming the pivot.
#include "y5m_act8.h"

#define GN_THREADS 256

struct GnParams {
    const void* x;                 // input rows (null in the backward when q is read)
    const void* dz;                // backward
    void* out;                     // z, or dx
    const float *gamma, *beta;     // null: 1, 0
    float *mean, *rstd;            // [N][G]
    uint8_t *q, *scale;            // 8-bit form
    float* part;                   // [N][chunks][2][C] channel sums of the reduce pass
    float* nc;                     // backward: [N][2][C] channel sums
    float* ab;                     // backward: [N][G][2] A, B
    float *dgamma, *dbeta;
    int64_t N, xn, xr, zn, zr, on, orow;
    int S, C, G, D, ldq, CB, act;
    float eps;
    int CV, ct, tiles, RP, chunks, rpc;      // pieces per row / per column tile, column tiles, rows side by side, row chunks, rows per chunk
    unsigned main_blocks;                    // backward apply: blocks beyond these reduce dgamma / dbeta
};

template <int DT> __device__ __forceinline__ float gn_sigmoid(float t) {
    const float a = -t;
    float e;
    if constexpr (DT == Y5M_F32) {
        // exp2 of the product a log2(e) carried to twice the precision: the hardware exp2 is within 1 ulp, the rounded product is
        // not (its error grows with |t|); outputs of 16 bits do not see it
        const float h = a * 1.44269502f, l = fmaf(a, 1.44269502f, -h) + a * 1.92596299e-8f;
        e = __builtin_amdgcn_exp2f(fminf(h, 126.0f));
        e = fmaf(e, l * 0.693147182f, e);
    } else {
        e = __builtin_amdgcn_exp2f(a * 1.44269502f);
    }
    return __builtin_amdgcn_rcpf(1.0f + e);
}
__device__ __forceinline__ float gn_pivot(float a, float b, float c) {
    return fmaxf(fminf(a, b), fminf(fmaxf(a, b), c));
}

// sums over the RP rows that a workgroup holds side by side: v[16] = two sums of 8 channels per thread -> dst[which * C + c]
__device__ __forceinline__ void gn_join_rows(const float* v, float* red, int lr, int lc, int ct, int RP, bool in, int c0, int C, float* __restrict__ dst) {
    const int w = ct * 16;
    if (in) {
#pragma unroll
        for (int k = 0; k < 16; ++k) red[lr * w + (k >> 3) * (ct * 8) + lc * 8 + (k & 7)] = v[k];
    }
    __syncthreads();
    for (int j = threadIdx.x; j < w; j += GN_THREADS) {
        const int which = j / (ct * 8), c = c0 + j - which * (ct * 8);
        if (c >= C) continue;
        float a = 0.f;
        for (int r = 0; r < RP; ++r) a += red[r * w + j];
        dst[(size_t)which * C + c] = a;
    }
}

struct GnPlace { int64_t n; int lr, lc, piece, c, nv, r0, r1, chunk; bool in; };
__device__ __forceinline__ GnPlace gn_place(const GnParams& P, unsigned blk) {
    GnPlace w;
    const int tile = (int)(blk % (unsigned)P.tiles);
    blk /= (unsigned)P.tiles;
    w.chunk = (int)(blk % (unsigned)P.chunks);
    w.n = blk / (unsigned)P.chunks;
    w.lr = (int)threadIdx.x / P.ct;
    w.lc = (int)threadIdx.x - w.lr * P.ct;
    w.piece = tile * P.ct + w.lc;
    w.c = w.piece * 8;
    w.nv = P.C - w.c;
    w.in = w.lr < P.RP && w.piece < P.CV && w.nv > 0;
    w.r0 = w.chunk * P.rpc;
    w.r1 = w.r0 + P.rpc < P.S ? w.r0 + P.rpc : P.S;
    return w;
}

// three rows whose median is a channel's pivot
template <int DT, bool AL> __device__ __forceinline__ void gn_pivots(const GnParams& P, int64_t n, int c, int nv, float p[8]) {
    typedef typename RowElem<DT>::T T;
    const T* b = static_cast<const T*>(P.x) + n * P.xn + c;
    float u[8], v[8], w[8];
    load8<DT, AL>(b, nv, u);
    load8<DT, AL>(b + (int64_t)(P.S / 2) * P.xr, nv, v);
    load8<DT, AL>(b + (int64_t)(P.S - 1) * P.xr, nv, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) p[k] = gn_pivot(u[k], v[k], w[k]);
}

template <int DT, bool AL>
__global__ __launch_bounds__(GN_THREADS) void gn_stats_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    __shared__ float red[GN_THREADS * 16];
    const GnPlace w = gn_place(P, blockIdx.x);
    float a[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) a[k] = 0.f;
    if (w.in) {
        float p[8];
        gn_pivots<DT, AL>(P, w.n, w.c, w.nv, p);
        const T* b = static_cast<const T*>(P.x) + w.n * P.xn + w.c;
        auto add = [&](const Raw8<DT>& raw) __attribute__((always_inline)) {
            float v[8];
            unpack8<DT>(raw, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float d = v[k] - p[k];
                a[k] += d;
                a[8 + k] = fmaf(d, d, a[8 + k]);
            }
        };
        int r = w.r0 + w.lr;
        for (; r + 3 * P.RP < w.r1; r += 4 * P.RP) {
            Raw8<DT> raw[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) raw[u] = load_raw8<DT, AL>(b + (int64_t)(r + u * P.RP) * P.xr, w.nv);
#pragma unroll
            for (int u = 0; u < 4; ++u) add(raw[u]);
        }
        for (; r < w.r1; r += P.RP) add(load_raw8<DT, AL>(b + (int64_t)r * P.xr, w.nv));
    }
    gn_join_rows(a, red, w.lr, w.lc, P.ct, P.RP, w.in, (w.piece - w.lc) * 8, P.C, P.part + ((size_t)w.n * P.chunks + w.chunk) * 2 * P.C);
}

// one wave per (n, group); lane = (chunk slot, channel of the group)
__device__ __forceinline__ double gn_shfl_xor(double v, int o) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const unsigned lo = (unsigned)__shfl_xor((int)(unsigned)u, o, 64), hi = (unsigned)__shfl_xor((int)(unsigned)(u >> 32), o, 64);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double gn_wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += gn_shfl_xor(v, o);
    return v;
}
struct GnSlots { int p2, d0, slot, slots; };
__device__ __forceinline__ GnSlots gn_slots(int D, int lane) {
    GnSlots s;
    s.p2 = 1;
    while (s.p2 < D && s.p2 < 64) s.p2 <<= 1;
    s.slots = 64 / s.p2;
    s.slot = lane / s.p2;
    s.d0 = lane - s.slot * s.p2;
    return s;
}
// sums of one channel over the row chunks, joined over the slots: every lane of the channel gets both
__device__ __forceinline__ void gn_channel_sums(const GnParams& P, int64_t n, int c, bool in, const GnSlots& s, double& a, double& b) {
    a = b = 0.0;
    if (in)
        for (int ch = s.slot; ch < P.chunks; ch += s.slots) {
            const float* p = P.part + ((size_t)n * P.chunks + ch) * 2 * P.C + c;
            a += (double)p[0];
            b += (double)p[P.C];
        }
    for (int o = 32; o >= s.p2; o >>= 1) {
        a += gn_shfl_xor(a, o);
        b += gn_shfl_xor(b, o);
    }
}

template <int DT>
__global__ __launch_bounds__(GN_THREADS) void gn_stats_join_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    const int lane = threadIdx.x & 63;
    const int64_t ng = (int64_t)blockIdx.x * (GN_THREADS / 64) + (threadIdx.x >> 6);
    if (ng >= P.N * P.G) return;                                   // (whole waves)
    const int64_t n = ng / P.G;
    const int g = (int)(ng - n * P.G);
    const GnSlots s = gn_slots(P.D, lane);
    const double S = (double)P.S;
    double m1 = 0.0, m2 = 0.0, mm = 0.0, ref = 0.0;                // sum of channel means (about ref), of M2, of squared means (about ref)
    for (int db = 0; db < P.D; db += s.p2) {
        const int d = db + s.d0, c = g * P.D + d;
        const bool in = d < P.D;
        double a, b;
        gn_channel_sums(P, n, c, in, s, a, b);
        double cm = 0.0;
        if (in) {
            float u, v, w;
            const T* x = static_cast<const T*>(P.x) + n * P.xn + c;
            if constexpr (DT == Y5M_F32) { u = x[0]; v = x[(int64_t)(P.S / 2) * P.xr]; w = x[(int64_t)(P.S - 1) * P.xr]; }
            else if constexpr (DT == Y5M_BF16) { u = bf16_to_f32(x[0]); v = bf16_to_f32(x[(int64_t)(P.S / 2) * P.xr]); w = bf16_to_f32(x[(int64_t)(P.S - 1) * P.xr]); }
            else { u = f16_to_f32(x[0]); v = f16_to_f32(x[(int64_t)(P.S / 2) * P.xr]); w = f16_to_f32(x[(int64_t)(P.S - 1) * P.xr]); }
            cm = (double)gn_pivot(u, v, w) + a / S;
        }
        if (db == 0) {                                             // about the first channel's mean: its lane is lane 0
            const uint64_t u = __builtin_bit_cast(uint64_t, cm);
            const unsigned lo = (unsigned)__shfl((int)(unsigned)u, 0, 64), hi = (unsigned)__shfl((int)(unsigned)(u >> 32), 0, 64);
            ref = __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
        }
        if (in && s.slot == 0) {
            m1 += cm - ref;
            mm += (cm - ref) * (cm - ref);
            m2 += b - a * a / S;
        }
    }
    m1 = gn_wave_sum(m1);
    m2 = gn_wave_sum(m2);
    mm = gn_wave_sum(mm);
    const double D = (double)P.D;
    double var = m2 / (S * D) + mm / D - (m1 / D) * (m1 / D);
    if (!(var > 0.0) && var == var) var = 0.0;                     // (a NaN stays)
    if (lane == 0) {
        P.mean[ng] = (float)(ref + m1 / D);
        P.rstd[ng] = (float)(1.0 / sqrt(var + (double)P.eps));
    }
}

struct GnCoef { float mean[8], rstd[8], gamma[8], beta[8]; };
__device__ __forceinline__ void gn_coef(const GnParams& P, const GnPlace& w, GnCoef& k) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = w.c + i < P.C ? w.c + i : P.C - 1, g = c / P.D;
        k.mean[i] = P.mean[w.n * P.G + g];
        k.rstd[i] = P.rstd[w.n * P.G + g];
        k.gamma[i] = P.gamma ? P.gamma[c] : 1.0f;
        k.beta[i] = P.beta ? P.beta[c] : 0.0f;
    }
}

template <int DT, bool AL, int FMT>
__global__ __launch_bounds__(GN_THREADS) void gn_apply_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    const GnPlace w = gn_place(P, blockIdx.x);
    GnCoef k;
    if (w.in) {
        gn_coef(P, w, k);
#pragma unroll
        for (int i = 0; i < 8; ++i) k.rstd[i] *= k.gamma[i];
    }
    const bool silu = P.act == Y5M_ACT_SILU;
    const T* b = static_cast<const T*>(P.x) + w.n * P.xn + w.c;
    T* o = static_cast<T*>(P.out) + w.n * P.on + w.c;
    // Every lane runs the same trips (the four lanes of a block must meet in the encoder): rows and pieces beyond the end are read
    // from the last row / the first piece instead, which is in bounds, and not stored.
    const T* bl = w.in ? b : static_cast<const T*>(P.x) + w.n * P.xn;
    const int nvl = w.in ? w.nv : P.C;
    auto finish = [&](const Raw8<DT>& raw, int r) __attribute__((always_inline)) {
        const bool live = w.in && r < w.r1;
        float v[8], z[8];
        unpack8<DT>(raw, v);
        if constexpr (FMT != Y5M_KEEP_NONE) {
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = w.in ? v[i] : 0.f;
            unsigned sb;
            const act8_u32x2 q = act8_encode8<FMT, DT>(z, sb);
            if (live) {
                const int64_t row = w.n * P.S + r;
                *reinterpret_cast<act8_u32x2*>(P.q + row * P.ldq + w.c) = q;
                if ((w.piece & 3) == 0) P.scale[row * P.CB + (w.piece >> 2)] = (uint8_t)sb;
            }
        }
        if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = fmaf(v[i] - k.mean[i], k.rstd[i], k.beta[i]);
                z[i] = silu ? t * gn_sigmoid<DT>(t) : t;
            }
            store8<DT, AL>(o + (int64_t)r * P.orow, w.nv, z);
        }
    };
    const int lr = w.lr < P.RP ? w.lr : 0;
    for (int rb = w.r0; rb < w.r1; rb += 4 * P.RP) {
        Raw8<DT> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = rb + lr + u * P.RP;
            raw[u] = load_raw8<DT, AL>(bl + (int64_t)(r < w.r1 ? r : w.r1 - 1) * P.xr, nvl);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) finish(raw[u], rb + lr + u * P.RP);
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------------
// the kept input of one row piece: x itself or its 8-bit form
template <int DT, int FMT> struct GnKept {
    Raw8<DT> raw;
};
template <int DT> struct GnKept<DT, Y5M_KEEP_E4M3> { act8_u32x2 q; unsigned s; };
template <int DT> struct GnKept<DT, Y5M_KEEP_INT8> { act8_u32x2 q; unsigned s; };
template <int DT, bool AL, int FMT>
__device__ __forceinline__ GnKept<DT, FMT> gn_kept(const GnParams& P, const GnPlace& w, int r) {
    typedef typename RowElem<DT>::T T;
    GnKept<DT, FMT> k;
    if constexpr (FMT == Y5M_KEEP_NONE) {
        k.raw = load_raw8<DT, AL>(static_cast<const T*>(P.x) + w.n * P.xn + (int64_t)r * P.xr + w.c, w.nv);
    } else {
        const int64_t row = w.n * P.S + r;
        k.q = *reinterpret_cast<const act8_u32x2*>(P.q + row * P.ldq + w.c);
        k.s = P.scale[row * P.CB + (w.piece >> 2)];
    }
    return k;
}
template <int DT, int FMT> __device__ __forceinline__ void gn_kept_values(const GnKept<DT, FMT>& k, float v[8]) {
    if constexpr (FMT == Y5M_KEEP_NONE) unpack8<DT>(k.raw, v);
    else act8_decode8<FMT>(k.q, act8_scale(k.s), v);
}
template <int DT> __device__ __forceinline__ float gn_act_grad(bool silu, float t) {
    const float s = gn_sigmoid<DT>(t);
    return silu ? s * fmaf(t, 1.0f - s, 1.0f) : 1.0f;
}

template <int DT, bool AL, int FMT>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_reduce_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    __shared__ float red[GN_THREADS * 16];
    const GnPlace w = gn_place(P, blockIdx.x);
    float a[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) a[k] = 0.f;
    if (w.in) {
        GnCoef k;
        gn_coef(P, w, k);
        const bool silu = P.act == Y5M_ACT_SILU;
        const T* d = static_cast<const T*>(P.dz) + w.n * P.zn + w.c;
        auto add = [&](const GnKept<DT, FMT>& kept, const Raw8<DT>& graw) __attribute__((always_inline)) {
            float v[8], g[8];
            gn_kept_values<DT, FMT>(kept, v);
            unpack8<DT>(graw, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float xh = (v[i] - k.mean[i]) * k.rstd[i];
                const float dt = g[i] * gn_act_grad<DT>(silu, fmaf(xh, k.gamma[i], k.beta[i]));
                a[i] += dt;
                a[8 + i] = fmaf(dt, xh, a[8 + i]);
            }
        };
        int r = w.r0 + w.lr;
        for (; r + P.RP < w.r1; r += 2 * P.RP) {
            GnKept<DT, FMT> kept[2];
            Raw8<DT> graw[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                kept[u] = gn_kept<DT, AL, FMT>(P, w, r + u * P.RP);
                graw[u] = load_raw8<DT, AL>(d + (int64_t)(r + u * P.RP) * P.zr, w.nv);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) add(kept[u], graw[u]);
        }
        for (; r < w.r1; r += P.RP) add(gn_kept<DT, AL, FMT>(P, w, r), load_raw8<DT, AL>(d + (int64_t)r * P.zr, w.nv));
    }
    gn_join_rows(a, red, w.lr, w.lc, P.ct, P.RP, w.in, (w.piece - w.lc) * 8, P.C, P.part + ((size_t)w.n * P.chunks + w.chunk) * 2 * P.C);
}

__global__ __launch_bounds__(GN_THREADS) void gn_bwd_join_kernel(const GnParams P) {
    const int lane = threadIdx.x & 63;
    const int64_t ng = (int64_t)blockIdx.x * (GN_THREADS / 64) + (threadIdx.x >> 6);
    if (ng >= P.N * P.G) return;
    const int64_t n = ng / P.G;
    const int g = (int)(ng - n * P.G);
    const GnSlots s = gn_slots(P.D, lane);
    double A = 0.0, B = 0.0;
    for (int db = 0; db < P.D; db += s.p2) {
        const int d = db + s.d0, c = g * P.D + d;
        const bool in = d < P.D;
        double a, b;
        gn_channel_sums(P, n, c, in, s, a, b);
        if (in && s.slot == 0) {
            const double ga = P.gamma ? (double)P.gamma[c] : 1.0;
            A += ga * a;
            B += ga * b;
            P.nc[((size_t)n * 2 + 0) * P.C + c] = (float)a;
            P.nc[((size_t)n * 2 + 1) * P.C + c] = (float)b;
        }
    }
    A = gn_wave_sum(A);
    B = gn_wave_sum(B);
    if (lane == 0) {
        const double K = (double)P.S * (double)P.D;
        P.ab[ng * 2 + 0] = (float)(A / K);
        P.ab[ng * 2 + 1] = (float)(B / K);
    }
}

template <int DT, bool AL, int FMT>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_apply_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    if (blockIdx.x >= P.main_blocks) {
        // dbeta / dgamma: 16 channels x 16 sample slots per block, joined in a fixed order in f64
        __shared__ double acc[2][16][17];
        const int c = (int)(blockIdx.x - P.main_blocks) * 16 + (threadIdx.x & 15), slot = threadIdx.x >> 4;
        double a = 0.0, b = 0.0;
        if (c < P.C)
            for (int64_t n = slot; n < P.N; n += 16) {
                a += (double)P.nc[((size_t)n * 2 + 0) * P.C + c];
                b += (double)P.nc[((size_t)n * 2 + 1) * P.C + c];
            }
        acc[0][slot][threadIdx.x & 15] = a;
        acc[1][slot][threadIdx.x & 15] = b;
        __syncthreads();
        if (slot < 2 && c < P.C) {
            double t = 0.0;
#pragma unroll
            for (int i = 0; i < 16; ++i) t += acc[slot][i][threadIdx.x & 15];
            float* dst = slot == 0 ? P.dbeta : P.dgamma;
            if (dst) dst[c] = (float)t;
        }
        return;
    }
    const GnPlace w = gn_place(P, blockIdx.x);
    if (!w.in) return;
    GnCoef k;
    gn_coef(P, w, k);
    float ra[8], rb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = w.c + i < P.C ? w.c + i : P.C - 1, g = c / P.D;
        ra[i] = P.ab[(w.n * P.G + g) * 2 + 0];
        rb[i] = P.ab[(w.n * P.G + g) * 2 + 1];
    }
    const bool silu = P.act == Y5M_ACT_SILU;
    const T* d = static_cast<const T*>(P.dz) + w.n * P.zn + w.c;
    T* o = static_cast<T*>(P.out) + w.n * P.on + w.c;
    auto finish = [&](const GnKept<DT, FMT>& kept, const Raw8<DT>& graw, int r) __attribute__((always_inline)) {
        float v[8], g[8];
        gn_kept_values<DT, FMT>(kept, v);
        unpack8<DT>(graw, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float xh = (v[i] - k.mean[i]) * k.rstd[i];
            const float dt = g[i] * gn_act_grad<DT>(silu, fmaf(xh, k.gamma[i], k.beta[i]));
            g[i] = k.rstd[i] * (fmaf(k.gamma[i], dt, -ra[i]) - xh * rb[i]);
        }
        store8<DT, AL>(o + (int64_t)r * P.orow, w.nv, g);
    };
    int r = w.r0 + w.lr;
    for (; r + P.RP < w.r1; r += 2 * P.RP) {
        GnKept<DT, FMT> kept[2];
        Raw8<DT> graw[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            kept[u] = gn_kept<DT, AL, FMT>(P, w, r + u * P.RP);
            graw[u] = load_raw8<DT, AL>(d + (int64_t)(r + u * P.RP) * P.zr, w.nv);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) finish(kept[u], graw[u], r + u * P.RP);
    }
    for (; r < w.r1; r += P.RP) finish(gn_kept<DT, AL, FMT>(P, w, r), load_raw8<DT, AL>(d + (int64_t)r * P.zr, w.nv), r);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// column tiles of at most GN_THREADS pieces; row chunks so that about 4096 workgroups run and a thread still has 8 rows where there are
static void gn_geometry(GnParams& P, bool quads) {
    P.CB = (P.C + 31) / 32;
    P.CV = quads ? P.CB * 4 : (P.C + 7) / 8;
    P.tiles = (int)ceil_div(P.CV, GN_THREADS);
    P.ct = (int)ceil_div(P.CV, P.tiles);
    if (quads) P.ct = (P.ct + 3) / 4 * 4;
    P.RP = GN_THREADS / P.ct;
    const int64_t most = ceil_div(P.S, (int64_t)P.RP * 8), want = ceil_div(4096, P.N * P.tiles);
    int64_t chunks = want < most ? want : most;
    if (chunks < 1) chunks = 1;
    P.rpc = (int)ceil_div(ceil_div(P.S, chunks), P.RP) * P.RP;
    P.chunks = (int)ceil_div(P.S, P.rpc);
}

static int gn_check(int64_t N, int64_t S, int C, int G, int act, int dtype) {
    Y5M_REQUIRE(dtype == Y5M_F32 || dtype == Y5M_BF16 || dtype == Y5M_F16, "dtype");
    Y5M_REQUIRE(act == Y5M_ACT_NONE || act == Y5M_ACT_SILU, "activation");
    Y5M_REQUIRE(C > 0 && G > 0 && C % G == 0, "the groups must divide the channels");
    Y5M_REQUIRE(N >= 0 && S >= 0 && S < (1ll << 30) && N < (1ll << 30), "sizes");
    return Y5M_OK;
}
static void gn_sizes(GnParams& P, int64_t N, int64_t S, int C, int G) {
    P.N = N; P.S = (int)S; P.C = C; P.G = G; P.D = C / G;
}

extern "C" size_t y5m_gn_act_workspace_bytes(int64_t N, int64_t S, int C, int G) {
    if (N <= 0 || S <= 0 || C <= 0 || G <= 0 || C % G || S >= (1ll << 30)) return 0;
    GnParams P = {};
    gn_sizes(P, N, S, C, G);
    gn_geometry(P, true);
    const int64_t a = P.chunks;
    gn_geometry(P, false);
    return (size_t)(N * (a > P.chunks ? a : P.chunks)) * 2 * C * sizeof(float);
}

#define GN_DT(GO)                                                                    \
    do {                                                                             \
        if (dtype == Y5M_F32) GO(Y5M_F32);                                           \
        else if (dtype == Y5M_BF16) GO(Y5M_BF16);                                    \
        else GO(Y5M_F16);                                                            \
    } while (0)
#define GN_LAUNCH(K, blocks) hipLaunchKernelGGL(K, dim3((unsigned)(blocks)), dim3(GN_THREADS), 0, y5m_stream(stream), P)

extern "C" int y5m_gn_act(const void* x, int64_t x_batch_stride, int64_t x_row_stride, const float* gamma, const float* beta, int64_t N, int64_t S,
                          int C, int G, float eps, int act, void* z, int64_t z_batch_stride, int64_t z_row_stride, float* mean, float* rstd,
                          void* q, int ldq, void* scale, int fmt, void* ws, size_t ws_bytes, int dtype, void* stream) {
    int rc = gn_check(N, S, C, G, act, dtype);
    if (rc != Y5M_OK) return rc;
    Y5M_REQUIRE(fmt >= Y5M_KEEP_NONE && fmt <= Y5M_KEEP_INT8, "8-bit format");
    if (N == 0 || S == 0) return Y5M_OK;
    Y5M_REQUIRE(x && z && mean && rstd, "null pointer");
    Y5M_REQUIRE(z != x || (z_batch_stride == x_batch_stride && z_row_stride == x_row_stride), "in place needs equal strides");
    Y5M_REQUIRE((S == 1 || z_row_stride >= C) && (N == 1 || z_batch_stride >= (S - 1) * z_row_stride + C), "rows of the output overlap");
    if (fmt != Y5M_KEEP_NONE) Y5M_REQUIRE(q && scale && ldq >= C && ldq % 8 == 0 && ((uintptr_t)q & 7) == 0, "8-bit form: ldq % 8 == 0, at least C, codes 8-byte aligned");
    Y5M_REQUIRE(ws && ws_bytes >= y5m_gn_act_workspace_bytes(N, S, C, G), "workspace too small");
    GnParams P = {};
    gn_sizes(P, N, S, C, G);
    P.x = x; P.out = z; P.gamma = gamma; P.beta = beta; P.mean = mean; P.rstd = rstd; P.eps = eps; P.act = act;
    P.xn = x_batch_stride; P.xr = x_row_stride; P.on = z_batch_stride; P.orow = z_row_stride;
    P.q = static_cast<uint8_t*>(q); P.scale = static_cast<uint8_t*>(scale); P.ldq = ldq;
    P.part = static_cast<float*>(ws);
    gn_geometry(P, fmt != Y5M_KEEP_NONE);
    Y5M_REQUIRE(P.N * P.chunks * P.tiles < (1ll << 31) && P.N * P.G < (1ll << 31), "too many workgroups");
    const bool al = rows_aligned16(x, x_batch_stride, x_row_stride, N, S, C, dtype) && rows_aligned16(z, z_batch_stride, z_row_stride, N, S, C, dtype);
    const int64_t blocks = P.N * P.chunks * P.tiles;
#define GO(DT)                                                                                                                   \
    do {                                                                                                                         \
        if (al) GN_LAUNCH((gn_stats_kernel<DT, true>), blocks); else GN_LAUNCH((gn_stats_kernel<DT, false>), blocks);            \
        GN_LAUNCH((gn_stats_join_kernel<DT>), ceil_div(P.N * P.G, GN_THREADS / 64));                                             \
        if (fmt == Y5M_KEEP_NONE) { if (al) GN_LAUNCH((gn_apply_kernel<DT, true, Y5M_KEEP_NONE>), blocks); else GN_LAUNCH((gn_apply_kernel<DT, false, Y5M_KEEP_NONE>), blocks); } \
        else if (fmt == Y5M_KEEP_E4M3) { if (al) GN_LAUNCH((gn_apply_kernel<DT, true, Y5M_KEEP_E4M3>), blocks); else GN_LAUNCH((gn_apply_kernel<DT, false, Y5M_KEEP_E4M3>), blocks); } \
        else { if (al) GN_LAUNCH((gn_apply_kernel<DT, true, Y5M_KEEP_INT8>), blocks); else GN_LAUNCH((gn_apply_kernel<DT, false, Y5M_KEEP_INT8>), blocks); } \
    } while (0)
    GN_DT(GO);
#undef GO
    Y5M_CHECK_LAUNCH("gn_act");
    return Y5M_OK;
}

extern "C" size_t y5m_gn_act_bwd_workspace_bytes(int64_t N, int64_t S, int C, int G) {
    if (N <= 0 || S <= 0 || C <= 0 || G <= 0 || C % G || S >= (1ll << 30)) return 0;
    return y5m_gn_act_workspace_bytes(N, S, C, G) + ((size_t)N * 2 * C + (size_t)N * G * 2) * sizeof(float);
}

extern "C" int y5m_gn_act_bwd(const void* dz, int64_t dz_batch_stride, int64_t dz_row_stride, const void* x, int64_t x_batch_stride, int64_t x_row_stride,
                              const void* q, int ldq, const void* scale, int fmt, const float* gamma, const float* beta, const float* mean,
                              const float* rstd, int64_t N, int64_t S, int C, int G, int act, void* dx, int64_t dx_batch_stride, int64_t dx_row_stride,
                              float* dgamma, float* dbeta, void* ws, size_t ws_bytes, int dtype, void* stream) {
    int rc = gn_check(N, S, C, G, act, dtype);
    if (rc != Y5M_OK) return rc;
    Y5M_REQUIRE(fmt >= Y5M_KEEP_NONE && fmt <= Y5M_KEEP_INT8, "8-bit format");
    if (N == 0 || S == 0) {                                       // no rows: the parameter gradients are zero
        if (dgamma && (rc = y5m_fill32(dgamma, 0, C, y5m_stream(stream))) != Y5M_OK) return rc;
        if (dbeta && (rc = y5m_fill32(dbeta, 0, C, y5m_stream(stream))) != Y5M_OK) return rc;
        return Y5M_OK;
    }
    Y5M_REQUIRE(dz && dx && mean && rstd, "null pointer");
    Y5M_REQUIRE((S == 1 || dx_row_stride >= C) && (N == 1 || dx_batch_stride >= (S - 1) * dx_row_stride + C), "rows of the output overlap");
    if (fmt == Y5M_KEEP_NONE) Y5M_REQUIRE(x, "the input, or its 8-bit form");
    else Y5M_REQUIRE(q && scale && ldq >= C && ldq % 8 == 0 && ((uintptr_t)q & 7) == 0, "8-bit form: ldq % 8 == 0, at least C, codes 8-byte aligned");
    Y5M_REQUIRE(ws && ws_bytes >= y5m_gn_act_bwd_workspace_bytes(N, S, C, G), "workspace too small");
    GnParams P = {};
    gn_sizes(P, N, S, C, G);
    P.x = x; P.dz = dz; P.out = dx; P.gamma = gamma; P.beta = beta; P.mean = const_cast<float*>(mean); P.rstd = const_cast<float*>(rstd); P.act = act;
    P.xn = x_batch_stride; P.xr = x_row_stride; P.zn = dz_batch_stride; P.zr = dz_row_stride; P.on = dx_batch_stride; P.orow = dx_row_stride;
    P.q = static_cast<uint8_t*>(const_cast<void*>(q)); P.scale = static_cast<uint8_t*>(const_cast<void*>(scale)); P.ldq = ldq;
    P.dgamma = dgamma; P.dbeta = dbeta;
    gn_geometry(P, false);
    P.part = static_cast<float*>(ws);
    P.nc = P.part + (size_t)P.N * P.chunks * 2 * C;
    P.ab = P.nc + (size_t)P.N * 2 * C;
    Y5M_REQUIRE(P.N * P.chunks * P.tiles + C < (1ll << 31) && P.N * P.G < (1ll << 31), "too many workgroups");
    const bool al = rows_aligned16(dz, dz_batch_stride, dz_row_stride, N, S, C, dtype) && rows_aligned16(dx, dx_batch_stride, dx_row_stride, N, S, C, dtype) &&
                    (fmt != Y5M_KEEP_NONE || rows_aligned16(x, x_batch_stride, x_row_stride, N, S, C, dtype));
    const int64_t blocks = P.N * P.chunks * P.tiles;
    P.main_blocks = (unsigned)blocks;
    const int64_t extra = (dgamma || dbeta) ? (C + 15) / 16 : 0;
#define GO2(DT, FMT)                                                                                                             \
    do {                                                                                                                         \
        if (al) GN_LAUNCH((gn_bwd_reduce_kernel<DT, true, FMT>), blocks); else GN_LAUNCH((gn_bwd_reduce_kernel<DT, false, FMT>), blocks); \
        GN_LAUNCH(gn_bwd_join_kernel, ceil_div(P.N * P.G, GN_THREADS / 64));                                                     \
        if (al) GN_LAUNCH((gn_bwd_apply_kernel<DT, true, FMT>), blocks + extra); else GN_LAUNCH((gn_bwd_apply_kernel<DT, false, FMT>), blocks + extra); \
    } while (0)
#define GO(DT)                                                                                                                   \
    do {                                                                                                                         \
        if (fmt == Y5M_KEEP_NONE) GO2(DT, Y5M_KEEP_NONE);                                                                        \
        else if (fmt == Y5M_KEEP_E4M3) GO2(DT, Y5M_KEEP_E4M3);                                                                   \
        else GO2(DT, Y5M_KEEP_INT8);                                                                                             \
    } while (0)
    GN_DT(GO);
#undef GO
#undef GO2
    Y5M_CHECK_LAUNCH("gn_act_bwd");
    return Y5M_OK;
}

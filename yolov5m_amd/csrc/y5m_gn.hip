// Group normalisation + activation over channels-last rows, forward and backward, with the input optionally kept in 8 bits.
//
//   forward   per (sample n, group g of D = C / G channels), K = S * D values:  mean, rstd = 1 / sqrt(var + eps)
//             xhat = (x - mean) rstd,  t = gamma_c xhat + beta_c,  z = t or t sigmoid(t);  optionally the 8-bit form of x (y5m_act8.h)
//   backward  from x or its 8-bit form:  dt = dz act'(t),  dbeta_c = sum dt,  dgamma_c = sum dt xhat  (over n and rows)
//             dx = rstd (gamma dt - A - xhat B),  A = sum_group(gamma dt) / K,  B = sum_group(gamma dt xhat) / K
//
// All of it is bound by bytes; the statistics of a group must be complete before its first output. Two forms:
//   held (gn_held_*): a workgroup loads all rows of a slice of whole groups of one sample into registers, reduces, applies, stores: every
//     byte is touched once, one launch (the backward's sums over the samples take a second, small one). For small maps, where launches
//     are what costs;
//   split: a reduce pass over row chunks, a small launch that joins the chunks in f64 (few of them: the apply pass does it), an apply
//     pass that reads the rows again.
// Neither uses atomics: the result does not depend on the order in which workgroups run. What else was built and measured, at
// 64 x 160 x 160 x 96 in bf16 with the int8 form (forward + backward): one launch whose workgroups wait for each other's sums (their
// round trips past the L2s and the registers of the join cost more than the second read: 604 us at best), batches of samples whose
// rows fit the memory-side cache between the two reads (653 us: the apply pass is bound by its writes), 300 KB slices held at 40 rows
// a thread (spills: 186 us for the forward at 40 x 40 x 384, split 69).
// A thread owns 8 channels of a row (16 bytes of bf16), so gamma / beta / mean / rstd sit in registers, and consecutive lanes read
// consecutive pieces of consecutive rows, whatever D is: groups are cut out when the channel sums are joined, never by the loads (at 96
// channels in 32 groups a group is 6 bytes wide).
#include "y5m_act8.h"

#define GN_THREADS 256

struct GnParams {
    const void* x;                 // input rows (null in the backward when q is read)
    const void* dz;                // backward
    void* out;                     // z, or dx
    const float *gamma, *beta;     // null: 1, 0
    float *mean, *rstd;            // [N][G]
    uint8_t *q, *scale;            // 8-bit form
    float* part;                   // split: [N][chunks][C][2] of a channel in a chunk: mean and deviation; backward: sum dt, sum dt xhat
    float* nc;                     // backward: [N][C][2] channel sums
    float* ab;                     // backward, split: [N][G][2] A, B
    float *dgamma, *dbeta;
    int64_t N, xn, xr, zn, zr, on, orow;
    int S, C, G, D, ldq, CB, act;
    float eps;
    double inv_k;                            // 1 / (S D)
    int CV, ct, tiles, RP, chunks, rpc;      // split: pieces per row / per column tile, column tiles, rows side by side, row chunks, rows per chunk
    int achunks, arpc;                       // the apply pass's chunks
    unsigned ctm, dm;                        // ceil(2^32 / ct), ceil(2^32 / D): quotients of threads and channels by one multiply
    int sc, slices;                          // held: channels per slice, slices (ct pieces, RP rows side by side)
};

// ---- arithmetic -----------------------------------------------------------------------------------------------------------------
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

// ---- places -----------------------------------------------------------------------------------------------------------------------
struct GnPlace { int64_t n; int lr, lc, piece, c, nv, r0, r1, chunk; bool in; };
// (exact: numerator * divisor < 2^32; the launcher keeps C below 2^16)
__device__ __forceinline__ int gn_div(int a, unsigned magic) { return magic ? (int)__umulhi((unsigned)a, magic) : a; }
static unsigned gn_magic(int d) { return d == 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d); }
// grid: (chunks * tiles, samples folded over y and z). The apply pass takes the samples from the last to the first: what the reduce pass
// read last is still in the memory-side cache
template <bool BACK> __device__ __forceinline__ GnPlace gn_place(const GnParams& P, int rpc) {
    GnPlace w;
    const int tile = P.tiles > 1 ? (int)(blockIdx.x % (unsigned)P.tiles) : 0;
    w.chunk = P.tiles > 1 ? (int)(blockIdx.x / (unsigned)P.tiles) : (int)blockIdx.x;
    w.n = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
    if (BACK) w.n = P.N - 1 - w.n;                                 // (below 0: beyond the last, as w.n >= N)
    w.lr = gn_div((int)threadIdx.x, P.ctm);
    w.lc = (int)threadIdx.x - w.lr * P.ct;
    w.piece = tile * P.ct + w.lc;
    w.c = w.piece * 8;
    w.nv = P.C - w.c;
    w.in = w.lr < P.RP && w.piece < P.CV && w.nv > 0;
    w.r0 = w.chunk * rpc;
    w.r1 = w.r0 + rpc < P.S ? w.r0 + rpc : P.S;
    return w;
}
// group of each of the thread's 8 channels
struct GnGroups { int g[8]; };
__device__ __forceinline__ GnGroups gn_groups(const GnParams& P, int c) {
    GnGroups k;
    int g = c < P.C ? gn_div(c, P.dm) : 0, left = (g + 1) * P.D - c;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        k.g[i] = g < P.G ? g : P.G - 1;
        if (--left == 0) { ++g; left = P.D; }
    }
    return k;
}

// sums over the RP rows that a workgroup holds side by side: v[16] = two sums of 8 channels per thread. f(channel, sum, sum) for each
// channel, one thread per channel
template <typename A, typename F>
__device__ __forceinline__ void gn_join_rows(const A* v, A* red, const GnPlace& w, int ct, int RP, int C, F f) {
    typedef A V __attribute__((ext_vector_type(16 / sizeof(A))));
    constexpr int NV = 16 / (int)sizeof(A);
    const int wd = ct * 8, c0 = (w.piece - w.lc) * 8;
    A* red2 = red + GN_THREADS * 8;
    if (w.in) {
        V *d = reinterpret_cast<V*>(red + w.lr * wd + w.lc * 8), *d2 = reinterpret_cast<V*>(red2 + w.lr * wd + w.lc * 8);
#pragma unroll
        for (int i = 0; i < 8 / NV; ++i) {
            V t, t2;
#pragma unroll
            for (int k = 0; k < NV; ++k) { t[k] = v[i * NV + k]; t2[k] = v[8 + i * NV + k]; }
            d[i] = t;
            d2[i] = t2;
        }
    }
    __syncthreads();
    const int parts = GN_THREADS / wd;
    if (parts < 2) {
        for (int j = threadIdx.x; j < wd; j += GN_THREADS) {
            A a = 0, b = 0;
            for (int r = 0; r < RP; ++r) {
                a += red[r * wd + j];
                b += red2[r * wd + j];
            }
            if (c0 + j < C) f(c0 + j, a, b);
        }
        return;
    }
    // spare threads take every parts-th row; their sums meet in LDS
    const int part = (int)threadIdx.x / wd, j = (int)threadIdx.x - part * wd;
    A a = 0, b = 0;
    if (part < parts) {
        int r = part;
        for (; r + 3 * parts < RP; r += 4 * parts) {
            A u[4], v4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) { u[k] = red[(r + k * parts) * wd + j]; v4[k] = red2[(r + k * parts) * wd + j]; }
#pragma unroll
            for (int k = 0; k < 4; ++k) { a += u[k]; b += v4[k]; }
        }
        for (; r < RP; r += parts) {
            a += red[r * wd + j];
            b += red2[r * wd + j];
        }
    }
    __syncthreads();
    if (part < parts) {
        red[threadIdx.x] = a;
        red2[threadIdx.x] = b;
    }
    __syncthreads();
    if (part == 0 && c0 + j < C) {
        for (int k = 1; k < parts; ++k) {
            a += red[k * wd + j];
            b += red2[k * wd + j];
        }
        f(c0 + j, a, b);
    }
}
// (with a channel's chunks next to each other the join is 1 us shorter and the reduce pass, whose 8-byte stores then scatter, 3 to 8 longer)
__device__ __forceinline__ float2* gn_part(const GnParams& P, const GnPlace& w, int c) { return reinterpret_cast<float2*>(P.part) + ((size_t)w.n * P.chunks + w.chunk) * P.C + c; }

// ---- forward, split ---------------------------------------------------------------------------------------------------------------
// Values and squares are summed in f64, where the square of an f32 is exact: M2 = sum x^2 - (sum x)^2 / R loses mean^2 / var of 2^-53, whichever
// row comes first and however many share a chunk. (In f32 about the chunk's first row an outlier there cost up to R of 2^-24, R = 4096 rows at 8
// channels. The pass over 32 x 160 x 160 x 96 takes 27.5 us instead of 25.0, behind whose end the call does not show it; over 35 x 530 x 758,
// rows from any start, 14.3 instead of 12.0.) A chunk leaves its mean and sqrt(M2 / R),
// which f32 holds for every input, where M2 overflows from deviations of 2^60 on. Chunks are joined by the pairwise formula, in f64.
template <int DT, int AL>
__global__ __launch_bounds__(GN_THREADS) void gn_stats_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    __shared__ __attribute__((aligned(16))) double red[GN_THREADS * 16];
    const GnPlace w = gn_place<false>(P, P.rpc);
    if (w.n >= P.N) return;
    double a[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) a[k] = 0.0;
    if (w.in) {
        auto add = [&](const Raw8<DT>& raw) __attribute__((always_inline)) {
            float v[8];
            unpack8<DT>(raw, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const double d = (double)v[k];
                a[k] += d;
                a[8 + k] = fma(d, d, a[8 + k]);
            }
        };
        constexpr int U = 4;                                       // rows in flight (8: five waves per SIMD instead of eight, no faster)
        const int64_t step = (int64_t)P.RP * P.xr;
        int r = w.r0 + w.lr;
        const T* p = static_cast<const T*>(P.x) + w.n * P.xn + w.c + (int64_t)r * P.xr;
        for (; r + (U - 1) * P.RP < w.r1; r += U * P.RP) {
            Raw8<DT> raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                raw[u] = load_raw8<DT, AL>(p, w.nv);
                p += step;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) add(raw[u]);
        }
        for (; r < w.r1; r += P.RP) {
            add(load_raw8<DT, AL>(p, w.nv));
            p += step;
        }
    }
    // -> the chunk's mean and deviation
    const double R = (double)(w.r1 - w.r0), inv = 1.0 / R;
    gn_join_rows(a, red, w, P.ct, P.RP, P.C, [&](int c, double s1, double s2) __attribute__((always_inline)) {
        const double m = s1 * inv, m2 = fma(-s1, m, s2);
        *gn_part(P, w, c) = make_float2((float)m, (float)sqrt(m2 < 0.0 ? 0.0 : m2 * inv));          // (a NaN stays)
    });
}

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
// a workgroup's sum of NV doubles per thread, in a fixed order; every thread gets it
template <int NV, int T> __device__ __forceinline__ void gn_block_sum(double* v, double* red) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = gn_wave_sum(v[i]);
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) red[i * (T / 64) + (threadIdx.x >> 6)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        v[i] = 0.0;
        for (int k = 0; k < T / 64; k += 4) v[i] += (red[i * (T / 64) + k] + red[i * (T / 64) + k + 1]) + (red[i * (T / 64) + k + 2] + red[i * (T / 64) + k + 3]);
    }
    __syncthreads();
}
// One workgroup of T threads per (sample, group): its chunks x D channels are walked over in pieces of w = min(D, T) channels, T / w
// chunks side by side. (Latency is all there is: four loads in flight per thread, 4 us where one wave per group took 7.) T = 1024 where a
// group has many channels and chunks.
struct GnWalk { int w, slots, slot, d; };
template <int T> __device__ __forceinline__ GnWalk gn_walk(int D) {
    GnWalk k;
    k.w = D < T ? D : T;
    k.slots = T / k.w;
    k.slot = (int)threadIdx.x / k.w;
    k.d = (int)threadIdx.x - k.slot * k.w;
    return k;
}

// 1 / sqrt(v): in f32 where v is well inside its range, which is where the other way's time would be noticed
__device__ __forceinline__ float gn_rsqrt(double v) {
    const float f = (float)v;
    return f > 1e-30f && f < 1e30f ? 1.0f / sqrtf(f) : (float)(1.0 / sqrt(v));
}
// a group's mean and rstd from its chunks' sums about ref: sum R (m - ref), sum R (m - ref)^2, sum M2
__device__ __forceinline__ float2 gn_group_stat(const GnParams& P, const double* v, double ref) {
    const double off = v[0] * P.inv_k;
    double var = (v[2] + v[1]) * P.inv_k - off * off;
    if (!(var > 0.0) && var == var) var = 0.0;                     // (a NaN stays)
    return make_float2((float)(ref + off), gn_rsqrt(var + (double)P.eps));
}
__device__ __forceinline__ void gn_add_chunk(const GnParams& P, const float2& m, int ch, double ref, double* v) {
    const double R = (double)(ch + 1 < P.chunks ? P.rpc : P.S - ch * P.rpc), e = (double)m.x - ref;
    v[0] += R * e;
    v[1] += R * e * e;
    v[2] += R * (double)m.y * (double)m.y;
}

template <int T> __global__ __launch_bounds__(T) void gn_stats_join_kernel(const GnParams P) {
    __shared__ double red[3 * T / 64];
    const int64_t b = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
    const int g = (int)blockIdx.x;
    if (b >= P.N) return;
    const float* part = P.part + (size_t)b * P.chunks * 2 * P.C + 2 * g * P.D;
    const GnWalk k = gn_walk<T>(P.D);
    const double ref = (double)part[0];
    double v[3] = {0.0, 0.0, 0.0};
    if (k.slot < k.slots)
        for (int d = k.d; d < P.D; d += T) {
            auto add = [&](const float2& m, int ch) __attribute__((always_inline)) { gn_add_chunk(P, m, ch, ref, v); };
            int ch = k.slot;
            for (; ch + 3 * k.slots < P.chunks; ch += 4 * k.slots) {
                float2 m[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) m[u] = *reinterpret_cast<const float2*>(part + (size_t)(ch + u * k.slots) * 2 * P.C + 2 * d);
#pragma unroll
                for (int u = 0; u < 4; ++u) add(m[u], ch + u * k.slots);
            }
            for (; ch < P.chunks; ch += k.slots) add(*reinterpret_cast<const float2*>(part + (size_t)ch * 2 * P.C + 2 * d), ch);
        }
    gn_block_sum<3, T>(v, red);
    if (threadIdx.x == 0) {
        const float2 st = gn_group_stat(P, v, ref);
        const int64_t ng = b * P.G + g;
        P.mean[ng] = st.x;
        P.rstd[ng] = st.y;
    }
}

// The same in the prologue of the apply passes, where the sums are few (gn_inline): every workgroup joins the groups that its tile
// touches, k lanes a group, and saves the launch. val(g, chunk, channel of the group, pair of sums, v) adds, f(g, v) takes the result.
template <int NV, typename V, typename F> __device__ __forceinline__ void gn_tile_groups(const GnParams& P, const GnPlace& w, int g0, int g1, V val, F f) {
    int k = 64;
    while ((g1 - g0 + 1) * k > GN_THREADS && k > 1) k >>= 1;
    const int sub = threadIdx.x & (k - 1), pairs = P.chunks * P.D;
    const float2* part = reinterpret_cast<const float2*>(P.part) + (size_t)w.n * P.chunks * P.C;
    for (int b = g0; b <= g1; b += GN_THREADS / k) {               // (every lane runs the same trips: they meet in the shuffles)
        const int at = b + (int)threadIdx.x / k, g = at < g1 ? at : g1;
        double v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = 0.0;
        for (int i = sub; i < pairs; i += 4 * k) {
            float2 m[4];
            int ch[4], d[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = i + u * k < pairs ? i + u * k : pairs - 1;
                ch[u] = gn_div(j, P.dm);
                d[u] = j - ch[u] * P.D;
                m[u] = part[(size_t)ch[u] * P.C + g * P.D + d[u]];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * k < pairs) val(g, ch[u], d[u], m[u], v);
        }
        for (int o = k >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += gn_shfl_xor(v[i], o);
        if (sub == 0 && at <= g1) f(g, v);
    }
}

// 8 values of a per-channel parameter (absent: `none`)
__device__ __forceinline__ void gn_param8(const float* __restrict__ p, int c, int nv, float none, float* v) {
    if (p && nv >= 8) {
        __builtin_memcpy(v, p + c, 32);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p ? p[c + (i < nv ? i : nv - 1)] : none;
    }
}
// coefficients of a thread's 8 channels
struct GnCoef { float mean[8], rstd[8], gamma[8], beta[8]; };
__device__ __forceinline__ void gn_stat8(const GnParams& P, const GnPlace& w, const GnGroups& gr, GnCoef& k) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        k.mean[i] = P.mean[w.n * P.G + gr.g[i]];
        k.rstd[i] = P.rstd[w.n * P.G + gr.g[i]];
    }
}
__device__ __forceinline__ void gn_param(const GnParams& P, const GnPlace& w, GnCoef& k) {
    const int c = w.in ? w.c : 0, nv = w.in ? w.nv : P.C;
    gn_param8(P.gamma, c, nv, 1.0f, k.gamma);
    gn_param8(P.beta, c, nv, 0.0f, k.beta);
}
__device__ __forceinline__ void gn_coef(const GnParams& P, const GnPlace& w, const GnGroups& gr, GnCoef& k) {
    gn_stat8(P, w, gr, k);
    gn_param(P, w, k);
}

// t = gamma xhat + beta. f32: (x - mean) first, exact where x is near the mean. 16 bits: one fma, x a + b -- its rounding of |mean| a
// is 2^-24 where x's own type already cost 2^-9 or 2^-12 of the same
template <int DT> struct GnAffine {
    float a[8], b[8], m[DT == Y5M_F32 ? 8 : 1];
    __device__ __forceinline__ void set(const GnCoef& k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = k.rstd[i] * k.gamma[i];
            if constexpr (DT == Y5M_F32) {
                m[i] = k.mean[i];
                b[i] = k.beta[i];
            } else {
                // above 2^27 the group's values are all the same: 16-bit ones that differ spread over 2^-11 / sqrt(K) of the mean at least,
                // K < 2^31. xhat is 0 then, and mean a would only leave its rounding, or infinity
                const bool same = fabsf(k.mean[i]) * k.rstd[i] > 0x1p27f;
                if (same) a[i] = 0.f;
                b[i] = same ? k.beta[i] : fmaf(-k.mean[i], a[i], k.beta[i]);
            }
        }
    }
    __device__ __forceinline__ float operator()(float v, int i) const {
        if constexpr (DT == Y5M_F32) return fmaf(v - m[i], a[i], b[i]);
        else return fmaf(v, a[i], b[i]);
    }
};

template <int DT, int AL, int FMT, bool INL>
__global__ __launch_bounds__(GN_THREADS) void gn_apply_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    const GnPlace w = gn_place<true>(P, P.arpc);
    if (w.n < 0) return;
    const GnGroups gr = gn_groups(P, w.c);
    GnAffine<DT> af;
    {
        GnCoef k;
        if constexpr (INL) {
            __shared__ float2 stat[GN_THREADS];
            const int c0 = (w.piece - w.lc) * 8, c1 = c0 + P.ct * 8 < P.C ? c0 + P.ct * 8 : P.C, g0 = gn_div(c0, P.dm), g1 = gn_div(c1 - 1, P.dm);
            const float* ref = P.part + (size_t)w.n * P.chunks * 2 * P.C;
            gn_tile_groups<3>(P, w, g0, g1, [&](int g, int ch, int, const float2& m, double* v) __attribute__((always_inline)) {
                gn_add_chunk(P, m, ch, (double)ref[2 * g * P.D], v);
            }, [&](int g, const double* v) __attribute__((always_inline)) {
                const float2 st = gn_group_stat(P, v, (double)ref[2 * g * P.D]);
                stat[g - g0] = st;
                if (w.chunk == 0) {
                    P.mean[w.n * P.G + g] = st.x;
                    P.rstd[w.n * P.G + g] = st.y;
                }
            });
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int g = gr.g[i] < g0 ? g0 : gr.g[i] > g1 ? g1 : gr.g[i];
                k.mean[i] = stat[g - g0].x;
                k.rstd[i] = stat[g - g0].y;
            }
            gn_param(P, w, k);
        } else {
            gn_coef(P, w, gr, k);
        }
        af.set(k);
    }
    const bool silu = P.act == Y5M_ACT_SILU;
    const T* b = static_cast<const T*>(P.x) + w.n * P.xn + (w.in ? w.c : 0);
    T* o = static_cast<T*>(P.out) + w.n * P.on + w.c;
    // Every lane runs the same trips (the four lanes of a block must meet in the encoder): rows and pieces beyond the end are read
    // from the last row / the first piece instead, which is in bounds, and not stored.
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
                const float t = af(v[i], i);
                z[i] = silu ? t * gn_sigmoid<DT>(t) : t;
            }
            store8<DT, AL>(o + (int64_t)r * P.orow, w.nv, z);
        }
    };
    const int lr = w.lr < P.RP ? w.lr : 0;
    const int64_t step = (int64_t)P.RP * P.xr;
    const T *p = b + (int64_t)(w.r0 + lr) * P.xr, *end = b + (int64_t)(w.r1 - 1) * P.xr;
    for (int rb = w.r0; rb < w.r1; rb += 4 * P.RP) {
        Raw8<DT> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            raw[u] = load_raw8<DT, AL>(rb + lr + u * P.RP < w.r1 ? p : end, nvl);
            p += step;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) finish(raw[u], rb + lr + u * P.RP);
    }
}

// ---- backward, split ---------------------------------------------------------------------------------------------------------------
// the kept input of one row piece: x itself or its 8-bit form
template <int DT, int FMT> struct GnKept {
    Raw8<DT> raw;
};
template <int DT> struct GnKept<DT, Y5M_KEEP_E4M3> { act8_u32x2 q; unsigned s; };
template <int DT> struct GnKept<DT, Y5M_KEEP_INT8> { act8_u32x2 q; unsigned s; };
template <int DT, int AL, int FMT>
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
// a thread's rows r, r + RP, ...: what was kept and the incoming gradient, by pointers that step
template <int DT, int AL, int FMT> struct GnCursor {
    typedef typename RowElem<DT>::T T;
    const T *x, *d;
    const uint8_t *q, *s;
    int64_t xs, ds, qs, ss;
    int nv;
    __device__ __forceinline__ GnCursor(const GnParams& P, const GnPlace& w, int r, const T* dz) {
        nv = w.nv;
        d = dz + (int64_t)r * P.zr;
        ds = (int64_t)P.RP * P.zr;
        if constexpr (FMT == Y5M_KEEP_NONE) {
            x = static_cast<const T*>(P.x) + w.n * P.xn + (int64_t)r * P.xr + w.c;
            xs = (int64_t)P.RP * P.xr;
        } else {
            const int64_t row = w.n * P.S + r;
            q = P.q + row * P.ldq + w.c;
            s = P.scale + row * P.CB + (w.piece >> 2);
            qs = (int64_t)P.RP * P.ldq;
            ss = (int64_t)P.RP * P.CB;
        }
    }
    __device__ __forceinline__ void next(GnKept<DT, FMT>& k, Raw8<DT>& g) {
        if constexpr (FMT == Y5M_KEEP_NONE) {
            k.raw = load_raw8<DT, AL>(x, nv);
            x += xs;
        } else {
            k.q = *reinterpret_cast<const act8_u32x2*>(q);
            k.s = *s;
            q += qs;
            s += ss;
        }
        g = load_raw8<DT, AL>(d, nv);
        d += ds;
    }
};
template <int DT> __device__ __forceinline__ float gn_act_grad(bool silu, float t) {
    const float s = gn_sigmoid<DT>(t);
    return silu ? s * fmaf(t, 1.0f - s, 1.0f) : 1.0f;
}
// xhat = (x - mean) rstd, for 16-bit types as one fma (GnAffine says why)
template <int DT> __device__ __forceinline__ float gn_xhat(float v, const GnCoef& k, int i) {
    if constexpr (DT == Y5M_F32) return (v - k.mean[i]) * k.rstd[i];
    else return fmaf(v, k.rstd[i], k.mean[i]);
}
template <int DT> __device__ __forceinline__ void gn_coef_xhat(GnCoef& k) {
    if constexpr (DT != Y5M_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) k.mean[i] = -k.mean[i] * k.rstd[i];
    }
}

// dt = dz act'(t) of one piece. f32: through xhat, which comes back in v. 16 bits: v stays the kept value and u = -t log2(e) is one
// fma of it (GnAffine says why that is enough): act'(t) = s (1 + t (1 - s)), s = 1 / (1 + 2^u), t (1 - s) = u (ln2 s - ln2)
template <int DT> struct GnGrad {
    float a[8], b[8], m[DT == Y5M_F32 ? 8 : 1], r[DT == Y5M_F32 ? 8 : 1];
    __device__ __forceinline__ void set(const GnCoef& k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DT == Y5M_F32) {
                a[i] = k.gamma[i];
                b[i] = k.beta[i];
                m[i] = k.mean[i];
                r[i] = k.rstd[i];
            } else {
                a[i] = k.gamma[i] * k.rstd[i];
                b[i] = -1.44269502f * fmaf(-k.mean[i], a[i], k.beta[i]);
                a[i] *= -1.44269502f;
            }
        }
    }
    template <bool SILU> __device__ __forceinline__ void operator()(float* v, float* g) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DT == Y5M_F32) {
                v[i] = (v[i] - m[i]) * r[i];
                if constexpr (SILU) g[i] *= gn_act_grad<DT>(true, fmaf(v[i], a[i], b[i]));
            } else if constexpr (SILU) {
                const float u = fmaf(v[i], a[i], b[i]);
                const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u));
                // (2^u past the largest f32: s = 0 and u may be large, never infinite for finite x)
                g[i] *= s * fmaf(u, fmaf(s, 0.693147182f, -0.693147182f), 1.0f);
            }
        }
    }
};

// bf16 reaches as far as f32: where a group's values do, sums of dt x (they come out infinite or NaN) and products with rstd^2 (gn_far) leave
// f32's range. Such channels are taken one by one through xhat: rare, and small enough to leave the usual way its registers. (xhat for all
// of bf16: 16 registers more, and with the waves they cost 526 us instead of 450 for a step over 64 x 160 x 160 x 96 in int8.)
template <int DT> __device__ __forceinline__ bool gn_far(const GnCoef& k) {
    bool far = false;
    if constexpr (DT == Y5M_BF16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) far |= k.rstd[i] < 0x1p-30f || fabsf(k.mean[i]) > 0x1p40f;
    }
    return far;
}
// f(row, dt, xhat) of channel c over the thread's rows
template <int FMT, typename F> __device__ __forceinline__ void gn_far_rows(const GnParams& P, const GnPlace& w, int c, F f) {
    const int64_t ng = w.n * P.G + gn_div(c, P.dm);
    const float mean = P.mean[ng], rstd = P.rstd[ng], gamma = P.gamma ? P.gamma[c] : 1.0f, beta = P.beta ? P.beta[c] : 0.0f;
#pragma unroll 1
    for (int r = w.r0 + w.lr; r < w.r1; r += P.RP) {
        const int64_t row = w.n * P.S + r;
        float v;
        if constexpr (FMT == Y5M_KEEP_NONE) {
            v = bf16_to_f32(static_cast<const bf16_t*>(P.x)[w.n * P.xn + (int64_t)r * P.xr + c]);
        } else {
            const uint8_t q = P.q[row * P.ldq + c];
            const float scale = act8_scale(P.scale[row * P.CB + (c >> 5)]);
            if constexpr (FMT == Y5M_KEEP_E4M3) v = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false)[0] * scale;
            else v = (float)(int8_t)q * scale;
        }
        const float xh = (v - mean) * rstd, dz = bf16_to_f32(static_cast<const bf16_t*>(P.dz)[w.n * P.zn + (int64_t)r * P.zr + c]);
        f(r, dz * gn_act_grad<Y5M_BF16>(P.act == Y5M_ACT_SILU, fmaf(xh, gamma, beta)), xh);
    }
}

template <int DT, int AL, int FMT, bool SILU>
__device__ __forceinline__ void gn_bwd_sums(const GnParams& P, const GnPlace& w, const GnGroups& gr, float* a) {
    typedef typename RowElem<DT>::T T;
    GnGrad<DT> grad;
    {
        GnCoef k;
        gn_coef(P, w, gr, k);
        grad.set(k);
    }
    auto add = [&](const GnKept<DT, FMT>& kept, const Raw8<DT>& graw) __attribute__((always_inline)) {
        float v[8], g[8];
        gn_kept_values<DT, FMT>(kept, v);
        unpack8<DT>(graw, g);
        grad.template operator()<SILU>(v, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] += g[i];
            a[8 + i] = fmaf(g[i], v[i], a[8 + i]);
        }
    };
    int r = w.r0 + w.lr;
    GnCursor<DT, AL, FMT> at(P, w, r, static_cast<const T*>(P.dz) + w.n * P.zn + w.c);
    // (two rows in flight: four cost a quarter of the waves and 30 % of the time)
    for (; r + P.RP < w.r1; r += 2 * P.RP) {
        GnKept<DT, FMT> kept[2];
        Raw8<DT> graw[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) at.next(kept[u], graw[u]);
#pragma unroll
        for (int u = 0; u < 2; ++u) add(kept[u], graw[u]);
    }
    for (; r < w.r1; r += P.RP) {
        GnKept<DT, FMT> kept;
        Raw8<DT> graw;
        at.next(kept, graw);
        add(kept, graw);
    }
    if constexpr (DT != Y5M_F32) {
        // sum dt x -> sum dt xhat
        GnCoef k;
        gn_stat8(P, w, gr, k);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[8 + i] = k.rstd[i] * fmaf(-k.mean[i], a[i], a[8 + i]);
    }
}

template <int DT, int AL, int FMT>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_reduce_kernel(const GnParams P) {
    __shared__ __attribute__((aligned(16))) float red[GN_THREADS * 16];
    __shared__ int far;
    const GnPlace w = gn_place<false>(P, P.rpc);
    if (w.n >= P.N) return;
    if (DT == Y5M_BF16 && threadIdx.x == 0) far = 0;
    float a[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) a[k] = 0.f;
    if (w.in) {
        const GnGroups gr = gn_groups(P, w.c);
        if (P.act == Y5M_ACT_SILU) gn_bwd_sums<DT, AL, FMT, true>(P, w, gr, a);
        else gn_bwd_sums<DT, AL, FMT, false>(P, w, gr, a);
    }
    gn_join_rows(a, red, w, P.ct, P.RP, P.C, [&](int c, float s0, float s1) __attribute__((always_inline)) {
        *gn_part(P, w, c) = make_float2(s0, s1);
        if (DT == Y5M_BF16 && !(fabsf(s1) < INFINITY)) far = 1;
    });
    if constexpr (DT == Y5M_BF16) {
        // (asked last, where nothing of the loop is held any more: a step over 64 x 160 x 160 x 96 in int8 takes 448 us, 493 with the statistics
        // asked in front of the rows, 455 to 460 between the loop and the join)
        __syncthreads();
        if (__builtin_expect(far, 0)) {
            for (int i = 0; i < 8; ++i) {
                float s0 = 0.f, s1 = 0.f;
                if (w.in && i < w.nv)
                    gn_far_rows<FMT>(P, w, w.c + i, [&](int, float dt, float xh) __attribute__((always_inline)) {
                        s0 += dt;
                        s1 = fmaf(dt, xh, s1);
                    });
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    a[j] = i == j ? s0 : a[j];
                    a[8 + j] = i == j ? s1 : a[8 + j];
                }
            }
            gn_join_rows(a, red, w, P.ct, P.RP, P.C, [&](int c, float s0, float s1) __attribute__((always_inline)) { *gn_part(P, w, c) = make_float2(s0, s1); });
        }
    }
}

// channel sums of a sample and A, B of its groups, one workgroup per (sample, group)
template <int T> __global__ __launch_bounds__(T) void gn_bwd_join_kernel(const GnParams P) {
    __shared__ double red[2 * T];
    const int64_t n = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
    const int g = (int)blockIdx.x;
    if (n >= P.N) return;
    const float* part = P.part + (size_t)n * P.chunks * 2 * P.C + 2 * g * P.D;
    const GnWalk k = gn_walk<T>(P.D);
    double v[2] = {0.0, 0.0};
    for (int d0 = 0; d0 < P.D; d0 += T) {                 // (uniform: every thread meets at the barriers)
        const int d = d0 + k.d;
        const bool in = k.slot < k.slots && d < P.D;
        double s0 = 0.0, s1 = 0.0;
        if (in) {
            int ch = k.slot;
            for (; ch + 3 * k.slots < P.chunks; ch += 4 * k.slots) {
                float2 m[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) m[u] = *reinterpret_cast<const float2*>(part + (size_t)(ch + u * k.slots) * 2 * P.C + 2 * d);
#pragma unroll
                for (int u = 0; u < 4; ++u) { s0 += (double)m[u].x; s1 += (double)m[u].y; }
            }
            for (; ch < P.chunks; ch += k.slots) {
                const float2 m = *reinterpret_cast<const float2*>(part + (size_t)ch * 2 * P.C + 2 * d);
                s0 += (double)m.x;
                s1 += (double)m.y;
            }
        }
        red[threadIdx.x] = s0;
        red[T + threadIdx.x] = s1;
        __syncthreads();
        if (in && k.slot == 0) {
            for (int sl = 1; sl < k.slots; ++sl) {
                s0 += red[sl * k.w + k.d];
                s1 += red[T + sl * k.w + k.d];
            }
            const int c = g * P.D + d;
            *reinterpret_cast<float2*>(P.nc + ((size_t)n * P.C + c) * 2) = make_float2((float)s0, (float)s1);
            const double ga = P.gamma ? (double)P.gamma[c] : 1.0;
            v[0] += ga * s0;
            v[1] += ga * s1;
        }
        __syncthreads();
    }
    gn_block_sum<2, T>(v, red);
    if (threadIdx.x == 0) {
        *reinterpret_cast<float2*>(P.ab + (n * P.G + g) * 2) = make_float2((float)(v[0] * P.inv_k), (float)(v[1] * P.inv_k));
    }
}

// dbeta / dgamma: the samples' channel sums, 16 channels x 16 sample slots per workgroup, joined in a fixed order in f64
__global__ __launch_bounds__(GN_THREADS) void gn_param_grad_kernel(const GnParams P) {
    __shared__ double acc[2][16][17];
    const int cl = threadIdx.x & 15, c = (int)blockIdx.x * 16 + cl, slot = threadIdx.x >> 4;
    double a = 0.0, b = 0.0;
    if (c < P.C) {
        const float* p = P.nc + ((size_t)slot * P.C + c) * 2;
        const size_t st = (size_t)P.C * 32;
        int64_t n = slot;
        for (; n + 48 < P.N; n += 64, p += 4 * st) {
            float2 m[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) m[u] = *reinterpret_cast<const float2*>(p + u * st);
#pragma unroll
            for (int u = 0; u < 4; ++u) { a += (double)m[u].x; b += (double)m[u].y; }
        }
        for (; n < P.N; n += 16, p += st) {
            const float2 m = *reinterpret_cast<const float2*>(p);
            a += (double)m.x;
            b += (double)m.y;
        }
    }
    acc[0][slot][cl] = a;
    acc[1][slot][cl] = b;
    __syncthreads();
    if (slot < 2 && c < P.C) {
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += acc[slot][i][cl];
        float* dst = slot == 0 ? P.dbeta : P.dgamma;
        if (dst) dst[c] = (float)t;
    }
}

template <int DT, int AL, int FMT, bool SILU, bool INL>
__device__ __forceinline__ void gn_bwd_rows(const GnParams& P, const GnPlace& w, const float2* lab, int g0) {
    typedef typename RowElem<DT>::T T;
    // dx = r gamma dt - r A - r B xhat = c1 dt + (c2 v + c3), v = xhat in f32, the kept value in 16 bits
    GnGrad<DT> grad;
    float c1[8], c2[8], c3[8];
    {
        const GnGroups gr = gn_groups(P, w.c);
        GnCoef k;
        gn_coef(P, w, gr, k);
        if (__builtin_expect(gn_far<DT>(k), 0)) {
            const float2* ab = INL ? lab - g0 : reinterpret_cast<const float2*>(P.ab) + w.n * P.G;
#pragma unroll 1
            for (int i = 0; i < 8 && i < w.nv; ++i) {
                const int c = w.c + i, g = gn_div(c, P.dm);
                const float r = P.rstd[w.n * P.G + g], A = ab[g].x, B = ab[g].y, ga = P.gamma ? P.gamma[c] : 1.0f;
                gn_far_rows<FMT>(P, w, c, [&](int row, float dt, float xh) __attribute__((always_inline)) {
                    static_cast<bf16_t*>(P.out)[w.n * P.on + (int64_t)row * P.orow + c] = f32_to_bf16(r * (ga * dt - A - xh * B));
                });
            }
            return;
        }
        grad.set(k);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // (channels behind the last: any of the tile's groups)
            const int g = gr.g[i];
            const float2 ab = INL ? lab[g - g0] : *reinterpret_cast<const float2*>(P.ab + (w.n * P.G + g) * 2);
            c1[i] = k.rstd[i] * k.gamma[i];
            c2[i] = -k.rstd[i] * ab.y;
            c3[i] = -k.rstd[i] * ab.x;
            if constexpr (DT != Y5M_F32) {
                c2[i] *= k.rstd[i];
                c3[i] = fmaf(-c2[i], k.mean[i], c3[i]);
            }
        }
    }
    auto finish = [&](const GnKept<DT, FMT>& kept, const Raw8<DT>& graw, T* to) __attribute__((always_inline)) {
        float v[8], g[8];
        gn_kept_values<DT, FMT>(kept, v);
        unpack8<DT>(graw, g);
        grad.template operator()<SILU>(v, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = fmaf(c1[i], g[i], fmaf(c2[i], v[i], c3[i]));
        store8<DT, AL>(to, w.nv, g);
    };
    int r = w.r0 + w.lr;
    GnCursor<DT, AL, FMT> at(P, w, r, static_cast<const T*>(P.dz) + w.n * P.zn + w.c);
    T* op = static_cast<T*>(P.out) + w.n * P.on + (int64_t)r * P.orow + w.c;
    const int64_t ostep = (int64_t)P.RP * P.orow;
    for (; r + P.RP < w.r1; r += 2 * P.RP) {
        GnKept<DT, FMT> kept[2];
        Raw8<DT> graw[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) at.next(kept[u], graw[u]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            finish(kept[u], graw[u], op);
            op += ostep;
        }
    }
    if (r < w.r1) {
        GnKept<DT, FMT> kept;
        Raw8<DT> graw;
        at.next(kept, graw);
        finish(kept, graw, op);
    }
}

template <int DT, int AL, int FMT, bool INL>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_apply_kernel(const GnParams P) {
    const GnPlace w = gn_place<true>(P, P.arpc);
    if (w.n < 0) return;
    const float2* lab = nullptr;
    int g0 = 0;
    if constexpr (INL) {
        __shared__ float2 ab[GN_THREADS];
        const int c0 = (w.piece - w.lc) * 8, c1 = c0 + P.ct * 8 < P.C ? c0 + P.ct * 8 : P.C, g1 = gn_div(c1 - 1, P.dm);
        g0 = gn_div(c0, P.dm);
        gn_tile_groups<2>(P, w, g0, g1, [&](int g, int, int d, const float2& m, double* v) __attribute__((always_inline)) {
            const double ga = P.gamma ? (double)P.gamma[g * P.D + d] : 1.0;
            v[0] += ga * (double)m.x;
            v[1] += ga * (double)m.y;
        }, [&](int g, const double* v) __attribute__((always_inline)) { ab[g - g0] = make_float2((float)(v[0] * P.inv_k), (float)(v[1] * P.inv_k)); });
        if (w.chunk == 0) {                                        // the sample's channel sums, for the parameters' gradients
            const float2* part = reinterpret_cast<const float2*>(P.part) + (size_t)w.n * P.chunks * P.C;
            for (int c = c0 + (int)threadIdx.x; c < c1; c += GN_THREADS) {
                double a = 0.0, b = 0.0;
                for (int ch = 0; ch < P.chunks; ++ch) {
                    const float2 m = part[(size_t)ch * P.C + c];
                    a += (double)m.x;
                    b += (double)m.y;
                }
                *reinterpret_cast<float2*>(P.nc + ((size_t)w.n * P.C + c) * 2) = make_float2((float)a, (float)b);
            }
        }
        lab = ab;
        __syncthreads();
    }
    if (!w.in) return;
    if (P.act == Y5M_ACT_SILU) gn_bwd_rows<DT, AL, FMT, true, INL>(P, w, lab, g0);
    else gn_bwd_rows<DT, AL, FMT, false, INL>(P, w, lab, g0);
}

// ---- held -------------------------------------------------------------------------------------------------------------------------
// A workgroup of up to 512 threads (256 registers each) holds a slice of `sc` channels (whole groups; whole 32-channel blocks where the 8-bit form is
// written) of one sample: NR row pieces per thread, RP rows side by side, two plain passes over registers for mean and variance.
// Slices of a sample follow each other on one XCD (the hardware deals workgroups round the 8 XCDs): a row's cache lines, which several
// slices share, are fetched once.
#define GN_HELD_THREADS 512

struct GnSlice { int64_t n; int c0, nc, lr, lc, c, nv; bool in; };
__device__ __forceinline__ GnSlice gn_slice(const GnParams& P) {
    const unsigned q8 = gridDim.x >> 3, r8 = gridDim.x & 7, xcd = blockIdx.x & 7;
    const unsigned b = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
    GnSlice w;
    w.n = b / (unsigned)P.slices;
    w.c0 = (int)(b - (unsigned)w.n * (unsigned)P.slices) * P.sc;
    w.nc = P.C - w.c0 < P.sc ? P.C - w.c0 : P.sc;
    w.lr = gn_div((int)threadIdx.x, P.ctm);
    w.lc = (int)threadIdx.x - w.lr * P.ct;
    w.c = w.c0 + w.lc * 8;
    w.nv = w.c0 + w.nc - w.c;
    w.in = w.lr < P.RP && w.nv > 0;
    return w;
}
// NS sums of 8 channels per thread -> tot[which][channel of the slice] in LDS. red: NS * 8 * threads floats, sub: threads floats,
// tot: NS * sc floats
template <int NS> __device__ __forceinline__ void gn_slice_sums(const GnParams& P, const GnSlice& w, const float* v, float* red, float* sub, float* tot) {
    const int T = (int)blockDim.x, wd = P.ct * 8, cols = NS * wd;
    __syncthreads();
    if (w.in) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            float4* d = reinterpret_cast<float4*>(red + w.lr * cols + s * wd + w.lc * 8);
            d[0] = make_float4(v[s * 8], v[s * 8 + 1], v[s * 8 + 2], v[s * 8 + 3]);
            d[1] = make_float4(v[s * 8 + 4], v[s * 8 + 5], v[s * 8 + 6], v[s * 8 + 7]);
        }
    }
    __syncthreads();
    const int rows = P.RP < P.S ? P.RP : P.S, parts = T / cols > 0 ? T / cols : 1;
    for (int j = threadIdx.x; j < cols * parts; j += T) {
        const int part = j / cols, c = j - part * cols;
        float a = 0.f;
        for (int r = part; r < rows; r += parts) a += red[r * cols + c];
        if (parts > 1) sub[j] = a;
        else tot[c] = a;
    }
    __syncthreads();
    if (parts > 1) {
        for (int c = threadIdx.x; c < cols; c += T) {
            float a = 0.f;
            for (int p = 0; p < parts; ++p) a += sub[p * cols + c];
            tot[c] = a;
        }
        __syncthreads();
    }
}
// f(group of the slice, sums over its channels of val(channel of the slice, i) in f64): a thread per narrow group, a wave per wide one
template <int NV, typename V, typename F> __device__ __forceinline__ void gn_slice_groups(const GnParams& P, const GnSlice& w, V val, F f) {
    const int groups = gn_div(w.nc, P.dm);
    double a[NV];
    if (P.D <= 32) {
        for (int g = threadIdx.x; g < groups; g += (int)blockDim.x) {
#pragma unroll
            for (int i = 0; i < NV; ++i) a[i] = 0.0;
            for (int d = 0; d < P.D; ++d)
#pragma unroll
                for (int i = 0; i < NV; ++i) a[i] += val(g * P.D + d, i);
            f(g, a);
        }
        return;
    }
    const int lane = threadIdx.x & 63;
    for (int g = threadIdx.x >> 6; g < groups; g += (int)blockDim.x >> 6) {
#pragma unroll
        for (int i = 0; i < NV; ++i) a[i] = 0.0;
        for (int d = lane; d < P.D; d += 64)
#pragma unroll
            for (int i = 0; i < NV; ++i) a[i] += val(g * P.D + d, i);
#pragma unroll
        for (int i = 0; i < NV; ++i) a[i] = gn_wave_sum(a[i]);
        if (lane == 0) f(g, a);
    }
}

// The statistics in f64, for a slice whose f32 sums may have left their range (deviations from 1e15 on, or values that are not finite
// themselves). A thread a channel, the rows read again: rare, and small enough not to cost the usual way registers. (f64 for every slice:
// 39 us instead of 15 for 32 x 768 x 20 x 20.) lds: 16 * ct doubles, over all that the kernel has
template <int DT> __device__ __forceinline__ void gn_held_far(const GnParams& P, const GnSlice& w, float* lds, float* gm, float* gr) {
    typedef typename RowElem<DT>::T T;
    const int wd = P.ct * 8, groups = gn_div(w.nc, P.dm);
    double* tot = reinterpret_cast<double*>(lds);
    const int64_t ng = w.n * P.G + gn_div(w.c0, P.dm);
    const T* x = static_cast<const T*>(P.x) + w.n * P.xn + w.c0;
#pragma unroll 1
    for (int c = threadIdx.x; c < w.nc; c += (int)blockDim.x) {
        double a = 0.0, b = 0.0;
#pragma unroll 1
        for (int r = 0; r < P.S; ++r) {
            const T e = x[(int64_t)r * P.xr + c];
            double d;
            if constexpr (DT == Y5M_F32) d = (double)e;
            else if constexpr (DT == Y5M_BF16) d = (double)bf16_to_f32(e);
            else d = (double)f16_to_f32(e);
            a += d;
            b = fma(d, d, b);
        }
        tot[c] = a;
        tot[wd + c] = b;
    }
    __syncthreads();
    gn_slice_groups<2>(P, w, [&](int c, int i) __attribute__((always_inline)) { return tot[i * wd + c]; }, [&](int g, const double* s) __attribute__((always_inline)) {
        const double md = s[0] * P.inv_k, var = fma(-md, md, s[1] * P.inv_k);
        P.mean[ng + g] = (float)md;
        P.rstd[ng + g] = gn_rsqrt((var < 0.0 ? 0.0 : var) + (double)P.eps);          // (a NaN stays)
    });
    __syncthreads();                                               // (gm and gr may lie where the sums were)
    for (int g = threadIdx.x; g < groups; g += (int)blockDim.x) {
        gm[g] = P.mean[ng + g];
        gr[g] = P.rstd[ng + g];
    }
    __syncthreads();
}

template <int DT, int AL, int FMT, int NR>
__global__ __launch_bounds__(GN_HELD_THREADS) void gn_held_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float *red = lds, *sub = red + 16 * blockDim.x, *tot = sub + blockDim.x, *gm = tot + P.ct * 16, *gr = gm + P.ct * 8;
    int& far = *reinterpret_cast<int*>(gr + P.ct * 8);              // did sums leave f32?
    if (threadIdx.x == 0) far = 0;
    const GnSlice w = gn_slice(P);
    const T* b = static_cast<const T*>(P.x) + w.n * P.xn + (w.in ? w.c : w.c0);
    const int nvl = w.in ? w.nv : w.nc, lr = w.lr < P.RP ? w.lr : 0;
    Raw8<DT> raw[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = lr + i * P.RP;
        raw[i] = load_raw8<DT, AL>(b + (int64_t)(r < P.S ? r : P.S - 1) * P.xr, nvl);
    }
    float a[16], m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const bool ok = lr + i * P.RP < P.S;
        float v[8];
        unpack8<DT>(raw[i], v);
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] += ok ? v[k] : 0.f;
    }
    gn_slice_sums<1>(P, w, a, red, sub, tot);
    gn_slice_groups<1>(P, w, [&](int c, int) __attribute__((always_inline)) { return (double)tot[c]; },
                       [&](int g, const double* s) __attribute__((always_inline)) { gm[g] = (float)(s[0] * P.inv_k); });
    __syncthreads();
    const GnGroups gi = gn_groups(P, w.in ? w.lc * 8 : 0);         // (groups of the slice)
    const int glast = gn_div(w.nc, P.dm) - 1;
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = gm[gi.g[k] < glast ? gi.g[k] : glast];
#pragma unroll
    for (int k = 0; k < 16; ++k) a[k] = 0.f;
    // about that mean: the squares, and the rest of the mean (what the first sum's rounding lost)
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const bool ok = lr + i * P.RP < P.S;
        float v[8];
        unpack8<DT>(raw[i], v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float d = ok ? v[k] - m[k] : 0.f;
            a[k] += d;
            a[8 + k] = fmaf(d, d, a[8 + k]);
        }
    }
    gn_slice_sums<2>(P, w, a, red, sub, tot);
    const int wd = P.ct * 8;
    gn_slice_groups<2>(P, w, [&](int c, int i) __attribute__((always_inline)) { return (double)tot[i * wd + c]; }, [&](int g, const double* s) __attribute__((always_inline)) {
        const double off = s[0] * P.inv_k, var = s[1] * P.inv_k - off * off;
        const float mean = (float)((double)gm[g] + off), v = (float)((var < 0.0 ? 0.0 : var) + (double)P.eps), rs = 1.0f / sqrtf(v);          // (a NaN stays)
        if (!(v > 1e-30f && v < 1e30f)) far = 1;
        gm[g] = mean;
        gr[g] = rs;
        const int64_t ng = w.n * P.G + gn_div(w.c0, P.dm) + g;
        P.mean[ng] = mean;
        P.rstd[ng] = rs;
    });
    __syncthreads();
    if (__builtin_expect(far, 0)) gn_held_far<DT>(P, w, red, gm, gr);
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = gm[gi.g[k] < glast ? gi.g[k] : glast];
    GnAffine<DT> af;
    {
        GnCoef k;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k.mean[i] = m[i];
            k.rstd[i] = gr[gi.g[i] < glast ? gi.g[i] : glast];
            const int c = w.in && i < w.nv ? w.c + i : w.c0;
            k.gamma[i] = P.gamma ? P.gamma[c] : 1.0f;
            k.beta[i] = P.beta ? P.beta[c] : 0.0f;
        }
        af.set(k);
    }
    const bool silu = P.act == Y5M_ACT_SILU;
    T* o = static_cast<T*>(P.out) + w.n * P.on + w.c;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = lr + i * P.RP;
        const bool live = w.in && r < P.S;
        float v[8], z[8];
        unpack8<DT>(raw[i], v);
        if constexpr (FMT != Y5M_KEEP_NONE) {
#pragma unroll
            for (int k = 0; k < 8; ++k) z[k] = w.in ? v[k] : 0.f;
            unsigned sb;
            const act8_u32x2 q = act8_encode8<FMT, DT>(z, sb);
            if (live) {
                const int64_t row = w.n * P.S + r;
                *reinterpret_cast<act8_u32x2*>(P.q + row * P.ldq + w.c) = q;
                if ((w.lc & 3) == 0) P.scale[row * P.CB + (w.c >> 5)] = (uint8_t)sb;
            }
        }
        if (live) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float t = af(v[k], k);
                z[k] = silu ? t * gn_sigmoid<DT>(t) : t;
            }
            store8<DT, AL>(o + (int64_t)r * P.orow, w.nv, z);
        }
    }
}

template <int DT, int AL, int FMT, int NR>
__global__ __launch_bounds__(GN_HELD_THREADS) void gn_bwd_held_kernel(const GnParams P) {
    typedef typename RowElem<DT>::T T;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float *red = lds, *sub = red + 16 * blockDim.x, *tot = sub + blockDim.x, *gA = tot + P.ct * 16, *gB = gA + P.ct * 8;
    const GnSlice w = gn_slice(P);
    const int lr = w.lr < P.RP ? w.lr : 0;
    GnPlace at;                                                    // where gn_kept reads
    at.n = w.n;
    at.c = w.in ? w.c : w.c0;
    at.nv = w.in ? w.nv : w.nc;
    at.piece = at.c >> 3;
    const T* d = static_cast<const T*>(P.dz) + w.n * P.zn + at.c;
    GnKept<DT, FMT> kept[NR];
    Raw8<DT> graw[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = lr + i * P.RP < P.S ? lr + i * P.RP : P.S - 1;
        kept[i] = gn_kept<DT, AL, FMT>(P, at, r);
        graw[i] = load_raw8<DT, AL>(d + (int64_t)r * P.zr, at.nv);
    }
    const GnGroups gi = gn_groups(P, w.in ? w.lc * 8 : 0);
    const int glast = gn_div(w.nc, P.dm) - 1;
    GnCoef k;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = w.in && i < w.nv ? w.c + i : w.c0;
        const int64_t ng = w.n * P.G + gn_div(w.c0, P.dm) + (gi.g[i] < glast ? gi.g[i] : glast);
        k.mean[i] = P.mean[ng];
        k.rstd[i] = P.rstd[ng];
        k.gamma[i] = P.gamma ? P.gamma[c] : 1.0f;
        k.beta[i] = P.beta ? P.beta[c] : 0.0f;
    }
    float c1[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c1[i] = k.rstd[i];
    gn_coef_xhat<DT>(k);
    const bool silu = P.act == Y5M_ACT_SILU;
    auto grad = [&](const GnKept<DT, FMT>& kp, const Raw8<DT>& gw, float* xh, float* dt) __attribute__((always_inline)) {
        gn_kept_values<DT, FMT>(kp, xh);
        unpack8<DT>(gw, dt);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            xh[i] = gn_xhat<DT>(xh[i], k, i);
            dt[i] *= gn_act_grad<DT>(silu, fmaf(xh[i], k.gamma[i], k.beta[i]));
        }
    };
    float a[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) a[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        if (lr + i * P.RP < P.S) {
            float xh[8], dt[8];
            grad(kept[i], graw[i], xh, dt);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                a[j] += dt[j];
                a[8 + j] = fmaf(dt[j], xh[j], a[8 + j]);
            }
        }
    }
    gn_slice_sums<2>(P, w, a, red, sub, tot);
    const int wd = P.ct * 8;
    for (int c = threadIdx.x; c < w.nc; c += (int)blockDim.x) {
        *reinterpret_cast<float2*>(P.nc + ((size_t)w.n * P.C + w.c0 + c) * 2) = make_float2(tot[c], tot[wd + c]);
        if (P.gamma) {
            tot[c] *= P.gamma[w.c0 + c];
            tot[wd + c] *= P.gamma[w.c0 + c];
        }
    }
    __syncthreads();
    gn_slice_groups<2>(P, w, [&](int c, int i) __attribute__((always_inline)) { return (double)tot[i * wd + c]; }, [&](int g, const double* s) __attribute__((always_inline)) {
        gA[g] = (float)(s[0] * P.inv_k);
        gB[g] = (float)(s[1] * P.inv_k);
    });
    __syncthreads();
    // dx = r gamma dt - r A - r B xhat = c1 dt + (c2 xhat + c3)
    float c2[8], c3[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int g = gi.g[i] < glast ? gi.g[i] : glast;
        c2[i] = -c1[i] * gB[g];
        c3[i] = -c1[i] * gA[g];
        c1[i] *= k.gamma[i];
    }
    T* o = static_cast<T*>(P.out) + w.n * P.on + w.c;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = lr + i * P.RP;
        if (w.in && r < P.S) {
            float xh[8], dt[8];
            grad(kept[i], graw[i], xh, dt);
#pragma unroll
            for (int j = 0; j < 8; ++j) dt[j] = fmaf(c1[j], dt[j], fmaf(c2[j], xh[j], c3[j]));
            store8<DT, AL>(o + (int64_t)r * P.orow, w.nv, dt);
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// split: column tiles of at most GN_THREADS pieces; row chunks of 16 rows a thread in the reduce pass (whose sums are then joined), of 8
// in the apply pass (short workgroups: 10000 of them stream at 6 TB/s, 2048 long ones at 5). 8 / 16, 12 / 12, 24 / 24 and 16 / 48 were 2 to
// 9 % slower over the 40 x 40, 80 x 80 and 160 x 160 training steps at batch 64. At most 65536 chunks in all, so that the sums stay small
// against the rows. Below two workgroups per CU the chunks are shorter, down to 4 rows a thread (what a thread does in turn is all the
// time there is: the backward of one 80 x 80 x 96 map 20.7 -> 16.1 us, of four 22.5 -> 19.7; 2 rows gain where one map is small, 15.1,
// and lose at two to eight), unless the joins would grow beyond 4096 pairs a group (2 groups of 693 channels, 155 rows: 24.5 -> 29).
// A group of GN_WIDE pairs or more is joined by 1024 threads (one group of 768 channels, 2500 rows: forward 38 -> 24.5).
#define GN_ROWS 16
#define GN_APPLY_ROWS 8
#define GN_WIDE 4096
static void gn_geometry(GnParams& P, bool quads, int rows, int arows) {
    P.CB = (P.C + 31) / 32;
    P.CV = quads ? P.CB * 4 : (P.C + 7) / 8;
    P.tiles = (int)ceil_div(P.CV, GN_THREADS);
    P.ct = (int)ceil_div(P.CV, P.tiles);
    if (quads) P.ct = (P.ct + 3) / 4 * 4;
    P.RP = GN_THREADS / P.ct;
    auto cut = [&](int rows, int& chunks, int& rpc) {
        while (rows > 4 && P.N * P.tiles * ceil_div(P.S, (int64_t)P.RP * rows) < 512 && ceil_div(P.S, (int64_t)P.RP * rows / 2) * P.D <= 4096) rows /= 2;
        int64_t c = ceil_div(P.S, (int64_t)P.RP * rows), cap = ceil_div(65536, P.N);
        if (c > cap) c = cap;
        rpc = (int)(ceil_div(ceil_div(P.S, c), P.RP) * P.RP);
        chunks = (int)ceil_div(P.S, rpc);
    };
    cut(rows, P.chunks, P.rpc);
    cut(arows, P.achunks, P.arpc);
    P.ctm = gn_magic(P.ct);
}

// held: threads and rows per thread that hold a slice, NR = 0 where it does not fit or pays. `nrs`: the row counts that are compiled,
// ascending; `most`: elements in all, above which the split form is faster -- except for samples of few rows, whose chunks would be
// scraps. Held against split, 20 x 20 x 768 bf16 in 32 groups: forward of 1 / 16 / 32 / 64 images 9 / 14 / 17 / 30 us against 14 / 18 / 23 / 32,
// of 256 165 against 105; backward of 1 / 8 / 16 / 32 images 13 / 14 / 23 / 39 against 21 / 24 / 29 / 36. 16384 x 768 tokens (one row
// each): forward 92 against 940. 16 rows a thread pay from 128 workgroups on: 64 / 128 / 256 of them (40 x 40, 96 and 192 channels) 13.4 /
// 14.6 / 17.4 against 12.1 / 14.4 / 24.1; three of one channel per group, 7623 rows: 28.4 against 10.6.
struct GnHeld { int threads, nr; };
static GnHeld gn_held(GnParams& P, bool blocks, bool aligned, const int* nrs, int64_t most) {
    // whole groups, whole blocks or pieces; rows that start anywhere may be cut anywhere (at 8 channels or more: load_raw8)
    const int cut = blocks ? 32 : 8;
    int a = P.D, b = cut;
    while (b) { const int t = a % b; a = b; b = t; }               // gcd
    const int64_t lcm = blocks || aligned ? (int64_t)P.D / a * cut : ceil_div(8, P.D) * P.D;
    const int unit = lcm < P.C ? (int)lcm : P.C, units = (int)ceil_div(P.C, unit);
    auto pieces = [&](int sc) { const int p = (sc + 7) / 8; return blocks ? (p + 3) / 4 * 4 : p; };
    auto fit = [&](int k) {
        GnHeld h = {0, 0};
        const int sc = (int64_t)unit * k < P.C ? unit * k : P.C, ct = pieces(sc);
        for (int i = 0; nrs[i]; ++i)                               // (few rows a thread before few threads: what is serial is what counts)
            for (int t = 64; t <= GN_HELD_THREADS; t *= 2) {
                if (ct > t || ceil_div(P.S, t / ct) > nrs[i]) continue;
                h.threads = t;
                h.nr = nrs[i];
                return h;
            }
        return h;
    };
    // wider slices (longer runs of a row, fewer idle threads) while 512 workgroups remain
    int k = 1;
    GnHeld h = fit(1);
    while (h.nr && k < units && P.N * ceil_div(units, k + 1) >= 512 && (int64_t)P.S * pieces(unit * k) < 2048) {
        const GnHeld w = fit(k + 1);
        if (!w.nr) break;
        h = w;
        ++k;
    }
    if (h.nr == 0 || (P.N * P.S * P.C > most && P.S >= 128)) return {0, 0};
    if (h.nr > 4 && P.N * ceil_div(units, k) < 128) return {0, 0};
    if (P.N * ceil_div(units, k) * h.threads >= (1ll << 32)) return {0, 0};          // (the launch's threads are counted in 32 bits)
    P.sc = (int64_t)unit * k < P.C ? unit * k : P.C;
    P.slices = (int)ceil_div(P.C, P.sc);
    P.ct = pieces(P.sc);
    P.RP = h.threads / P.ct;
    P.ctm = gn_magic(P.ct);
    P.CB = (P.C + 31) / 32;
    return h;
}
static const int GN_FWD_ROWS[] = {4, 16, 0}, GN_BWD_ROWS[] = {4, 0};
#define GN_HELD_FWD (24ll << 20)
#define GN_HELD_BWD (6ll << 20)

static int gn_check(int64_t N, int64_t S, int C, int G, int act, int dtype) {
    Y5M_REQUIRE(dtype == Y5M_F32 || dtype == Y5M_BF16 || dtype == Y5M_F16, "dtype");
    Y5M_REQUIRE(act == Y5M_ACT_NONE || act == Y5M_ACT_SILU, "activation");
    Y5M_REQUIRE(C > 0 && G > 0 && C % G == 0, "the groups must divide the channels");
    Y5M_REQUIRE(N >= 0 && S >= 0 && S < (1ll << 30) && N < (1ll << 30) && C < (1 << 16), "sizes");
    return Y5M_OK;
}
static void gn_sizes(GnParams& P, int64_t N, int64_t S, int C, int G) {
    P.N = N; P.S = (int)S; P.C = C; P.G = G; P.D = C / G; P.dm = gn_magic(P.D);
    P.inv_k = 1.0 / ((double)S * (double)P.D);
}

static bool gn_no_sizes(int64_t N, int64_t S, int C, int G) {
    return N <= 0 || S <= 0 || C <= 0 || C >= (1 << 16) || G <= 0 || C % G || S >= (1ll << 30) || N >= (1ll << 30);
}
// the split form's sums, for the alignment and 8-bit form that need most
static size_t gn_part_bytes(GnParams P) {
    gn_geometry(P, true, GN_ROWS, GN_APPLY_ROWS);
    const int64_t a = P.chunks;
    gn_geometry(P, false, GN_ROWS, GN_APPLY_ROWS);
    return (size_t)P.N * (size_t)(a > P.chunks ? a : P.chunks) * 2 * P.C * sizeof(float);
}
// does the held form run whatever the alignment and the 8-bit form are?
static bool gn_always_held(GnParams P, bool forward) {
    const int* nrs = forward ? GN_FWD_ROWS : GN_BWD_ROWS;
    const int64_t most = forward ? GN_HELD_FWD : GN_HELD_BWD;
    return gn_held(P, false, false, nrs, most).nr && gn_held(P, false, true, nrs, most).nr && (!forward || gn_held(P, true, true, nrs, most).nr);
}
extern "C" size_t y5m_gn_act_workspace_bytes(int64_t N, int64_t S, int C, int G) {
    if (gn_no_sizes(N, S, C, G)) return 0;
    GnParams P = {};
    gn_sizes(P, N, S, C, G);
    return gn_always_held(P, true) ? 0 : gn_part_bytes(P);
}

#define GN_DT(GO)                                                                    \
    do {                                                                             \
        if (dtype == Y5M_F32) GO(Y5M_F32);                                           \
        else if (dtype == Y5M_BF16) GO(Y5M_BF16);                                    \
        else GO(Y5M_F16);                                                            \
    } while (0)
#define GN_LAUNCH(K, blocks) hipLaunchKernelGGL(K, dim3((unsigned)(blocks)), dim3(GN_THREADS), 0, st, P)

// a grid of (x, samples): the samples folded over y and z
static dim3 gn_grid(int64_t x, int64_t N) {
    const int64_t y = N < 32768 ? N : 32768;
    return dim3((unsigned)x, (unsigned)y, (unsigned)ceil_div(N, y));
}
// (at most 65536 chunks of 32 tiles, or 65535 groups: every dimension is below 2^24 workgroups = 2^32 threads)
#define GN_JOINS(K)                                                                                                          \
    do {                                                                                                                     \
        if ((int64_t)P.chunks * P.D >= GN_WIDE) hipLaunchKernelGGL(K<1024>, gn_grid(P.G, P.N), dim3(1024), 0, st, P);        \
        else hipLaunchKernelGGL(K<GN_THREADS>, gn_grid(P.G, P.N), dim3(GN_THREADS), 0, st, P);                               \
    } while (0)
#define GN_LAUNCH2(K, x) hipLaunchKernelGGL(K, gn_grid((int64_t)(x), P.N), dim3(GN_THREADS), 0, st, P)

// may the apply pass join the sums itself? At most 16 pairs a lane, outputs that stay in the caches (5 x 21 x 37 x 36 fp16 with the 8-bit
// form, 12 groups: forward 12.9 -> 11.1 us, backward 18.5 -> 14.9; backward of 64 x 40 x 40 x 96 36 -> 30; at 64 pairs a lane one 80 x 80 x 96
// map takes 12.6 and 26.3 where the launch of its own takes 11.3 and 16.4)
static bool gn_inline(const GnParams& P) {
    const int ng = (P.ct * 8 < P.C ? P.ct * 8 : P.C) / P.D + 2;    // groups that a tile touches, at most
    if (ng > GN_THREADS) return false;
    int k = 64;
    while (ng * k > GN_THREADS && k > 1) k >>= 1;
    return (int64_t)P.chunks * P.D <= 16ll * k;
}

template <int DT, int AL, int FMT> static int gn_fwd_split(GnParams& P, hipStream_t st) {
    gn_geometry(P, FMT != Y5M_KEEP_NONE, GN_ROWS, GN_APPLY_ROWS);
    GN_LAUNCH2((gn_stats_kernel<DT, AL>), P.chunks * P.tiles);
    const bool past = rows_past_caches(P.N * P.S, P.C, DT);
    if (!past && gn_inline(P)) {
        GN_LAUNCH2((gn_apply_kernel<DT, AL, FMT, true>), P.achunks * P.tiles);
    } else {
        GN_JOINS(gn_stats_join_kernel);
        if constexpr (AL > 0) {
            if (past) GN_LAUNCH2((gn_apply_kernel<DT, 2, FMT, false>), P.achunks * P.tiles);
            else GN_LAUNCH2((gn_apply_kernel<DT, AL, FMT, false>), P.achunks * P.tiles);
        } else {
            GN_LAUNCH2((gn_apply_kernel<DT, AL, FMT, false>), P.achunks * P.tiles);
        }
    }
    Y5M_CHECK_LAUNCH("gn_apply_kernel");
    return Y5M_OK;
}
#define GN_HELD_LAUNCH(K, lds)                                                                                                   \
    do {                                                                                                                         \
        static std::atomic<uint64_t> asked{0};                                                                                   \
        if (!lds_ask(reinterpret_cast<const void*>(K), lds, 160 * 1024, asked)) return Y5M_ELAUNCH;                              \
        hipLaunchKernelGGL(K, dim3((unsigned)(P.N * P.slices)), dim3(h.threads), lds, st, P);                                    \
    } while (0)
template <int DT, int AL, int FMT> static int gn_fwd(GnParams& P, hipStream_t st) {
    const GnHeld h = gn_held(P, FMT != Y5M_KEEP_NONE, AL > 0, GN_FWD_ROWS, GN_HELD_FWD);
    if (h.nr == 0) return gn_fwd_split<DT, AL, FMT>(P, st);
    const int lds = (17 * h.threads + 4 * P.ct * 8 + 4) * (int)sizeof(float);
    if (h.nr == 4) GN_HELD_LAUNCH((gn_held_kernel<DT, AL, FMT, 4>), lds);
    else GN_HELD_LAUNCH((gn_held_kernel<DT, AL, FMT, 16>), lds);
    Y5M_CHECK_LAUNCH("gn_held_kernel");
    return Y5M_OK;
}
template <int DT, int AL> static int gn_fwd_fmt(GnParams& P, int fmt, hipStream_t st) {
    return fmt == Y5M_KEEP_NONE ? gn_fwd<DT, AL, Y5M_KEEP_NONE>(P, st) : fmt == Y5M_KEEP_E4M3 ? gn_fwd<DT, AL, Y5M_KEEP_E4M3>(P, st) : gn_fwd<DT, AL, Y5M_KEEP_INT8>(P, st);
}

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
    const size_t need = y5m_gn_act_workspace_bytes(N, S, C, G);
    Y5M_REQUIRE(need == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= need), "workspace too small or not 16-byte aligned");
    GnParams P = {};
    gn_sizes(P, N, S, C, G);
    P.x = x; P.out = z; P.gamma = gamma; P.beta = beta; P.mean = mean; P.rstd = rstd; P.eps = eps; P.act = act;
    P.xn = x_batch_stride; P.xr = x_row_stride; P.on = z_batch_stride; P.orow = z_row_stride;
    P.q = static_cast<uint8_t*>(q); P.scale = static_cast<uint8_t*>(scale); P.ldq = ldq;
    P.part = static_cast<float*>(ws);
    const int al = rows_mode(rows_aligned16(x, x_batch_stride, x_row_stride, N, S, C, dtype) && rows_aligned16(z, z_batch_stride, z_row_stride, N, S, C, dtype), C);
    hipStream_t st = y5m_stream(stream);
#define GO(DT) rc = al > 0 ? gn_fwd_fmt<DT, 1>(P, fmt, st) : al == 0 ? gn_fwd_fmt<DT, 0>(P, fmt, st) : gn_fwd_fmt<DT, -1>(P, fmt, st)
    GN_DT(GO);
#undef GO
    return rc;
}

extern "C" size_t y5m_gn_act_bwd_workspace_bytes(int64_t N, int64_t S, int C, int G) {
    if (gn_no_sizes(N, S, C, G)) return 0;
    GnParams P = {};
    gn_sizes(P, N, S, C, G);
    const size_t nc = (size_t)N * 2 * C * sizeof(float);
    return gn_always_held(P, false) ? nc : nc + (size_t)N * G * 2 * sizeof(float) + gn_part_bytes(P);
}

template <int DT, int AL, int FMT> static int gn_bwd(GnParams& P, hipStream_t st) {
    const GnHeld h = gn_held(P, false, AL > 0 || FMT != Y5M_KEEP_NONE, GN_BWD_ROWS, GN_HELD_BWD);
    if (h.nr) {
        const int lds = (17 * h.threads + 4 * P.ct * 8) * (int)sizeof(float);
        GN_HELD_LAUNCH((gn_bwd_held_kernel<DT, AL, FMT, 4>), lds);
        Y5M_CHECK_LAUNCH("gn_bwd_held_kernel");
    } else {
        gn_geometry(P, false, GN_ROWS, GN_APPLY_ROWS);
        GN_LAUNCH2((gn_bwd_reduce_kernel<DT, AL, FMT>), P.chunks * P.tiles);
        const bool past = rows_past_caches(P.N * P.S, P.C, DT);
        if (!past && gn_inline(P)) {
            GN_LAUNCH2((gn_bwd_apply_kernel<DT, AL, FMT, true>), P.achunks * P.tiles);
        } else {
            GN_JOINS(gn_bwd_join_kernel);
            if constexpr (AL > 0) {
                if (past) GN_LAUNCH2((gn_bwd_apply_kernel<DT, 2, FMT, false>), P.achunks * P.tiles);
                else GN_LAUNCH2((gn_bwd_apply_kernel<DT, AL, FMT, false>), P.achunks * P.tiles);
            } else {
                GN_LAUNCH2((gn_bwd_apply_kernel<DT, AL, FMT, false>), P.achunks * P.tiles);
            }
        }
        Y5M_CHECK_LAUNCH("gn_bwd_apply_kernel");
    }
    // (as workgroups of the apply pass the parameters' gradients cost it more, in registers, than this launch)
    if (P.dgamma || P.dbeta) {
        GN_LAUNCH(gn_param_grad_kernel, (P.C + 15) / 16);
        Y5M_CHECK_LAUNCH("gn_param_grad_kernel");
    }
    return Y5M_OK;
}
template <int DT, int AL> static int gn_bwd_fmt(GnParams& P, int fmt, hipStream_t st) {
    return fmt == Y5M_KEEP_NONE ? gn_bwd<DT, AL, Y5M_KEEP_NONE>(P, st) : fmt == Y5M_KEEP_E4M3 ? gn_bwd<DT, AL, Y5M_KEEP_E4M3>(P, st) : gn_bwd<DT, AL, Y5M_KEEP_INT8>(P, st);
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
    Y5M_REQUIRE(dx != dz || (dx_batch_stride == dz_batch_stride && dx_row_stride == dz_row_stride), "in place needs equal strides");
    Y5M_REQUIRE(dx != x || (dx_batch_stride == x_batch_stride && dx_row_stride == x_row_stride), "in place needs equal strides");
    if (fmt == Y5M_KEEP_NONE) Y5M_REQUIRE(x, "the input, or its 8-bit form");
    else Y5M_REQUIRE(q && scale && ldq >= C && ldq % 8 == 0 && ((uintptr_t)q & 7) == 0, "8-bit form: ldq % 8 == 0, at least C, codes 8-byte aligned");
    Y5M_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= y5m_gn_act_bwd_workspace_bytes(N, S, C, G), "workspace too small or not 16-byte aligned");
    GnParams P = {};
    gn_sizes(P, N, S, C, G);
    P.x = x; P.dz = dz; P.out = dx; P.gamma = gamma; P.beta = beta; P.mean = const_cast<float*>(mean); P.rstd = const_cast<float*>(rstd); P.act = act;
    P.xn = x_batch_stride; P.xr = x_row_stride; P.zn = dz_batch_stride; P.zr = dz_row_stride; P.on = dx_batch_stride; P.orow = dx_row_stride;
    P.q = static_cast<uint8_t*>(const_cast<void*>(q)); P.scale = static_cast<uint8_t*>(const_cast<void*>(scale)); P.ldq = ldq;
    P.dgamma = dgamma; P.dbeta = dbeta;
    P.nc = static_cast<float*>(ws);
    P.ab = P.nc + (size_t)N * 2 * C;
    P.part = P.ab + (size_t)N * 2 * G;
    const int al = rows_mode(rows_aligned16(dz, dz_batch_stride, dz_row_stride, N, S, C, dtype) && rows_aligned16(dx, dx_batch_stride, dx_row_stride, N, S, C, dtype) &&
                             (fmt != Y5M_KEEP_NONE || rows_aligned16(x, x_batch_stride, x_row_stride, N, S, C, dtype)), C);
    hipStream_t st = y5m_stream(stream);
#define GO(DT) rc = al > 0 ? gn_bwd_fmt<DT, 1>(P, fmt, st) : al == 0 ? gn_bwd_fmt<DT, 0>(P, fmt, st) : gn_bwd_fmt<DT, -1>(P, fmt, st)
    GN_DT(GO);
#undef GO
    return rc;
}

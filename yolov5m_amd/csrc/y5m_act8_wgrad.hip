// Weight gradient of a pointwise convolution from its input in 8 bits:  dW[n][c] = sum_m dY[m][n] X8[m][c],  db[n] = sum_m dY[m][n].
//
// GEMM with K = rows (up to millions) and both operands row-major along K, as they lie in memory. Arithmetic: an 8-bit value times its
// power-of-two scale has at most 8 significant bits, so it IS a bf16 value; dY in bf16 is one, in fp16 (11 bits) the exact sum of two
// and in f32 (24 bits) of three bf16 values. Products of bf16 MFMAs are exact in f32, so every type runs on the bf16 matrix cores
// with f32 accumulation, and nothing is rounded before the sum (f32 MFMA: 1/16 of the rate).
//
// A workgroup (4 waves) owns a 128 x 128 tile of dW and a range of rows; per step 64 rows of dY and of the codes go through registers
// (the codes become bf16 there) into LDS as [32 rows][16 channels] sub-tiles, and the fragments come back through
// ds_read_b64_tr_b16, which transposes 4 x 16 blocks: 4 rows of one channel per lane. Row ranges are joined from f32 partial tiles by
// a second launch in a fixed order (no atomics: one result per input).
#include "y5m_act8.h"

#define AW_THREADS 256
#define AW_T 128                  // tile edge (channels of dY, channels of X)
#define AW_K 64                   // rows per step
#define AW_SUB 1088               // [32][16] bf16 sub-tile: 1024 bytes + 64 so that neighbouring sub-tiles start on other banks
#define AW_TILE ((AW_K / 32) * (AW_T / 16) * AW_SUB)

typedef __bf16 aw_bf16x8 __attribute__((ext_vector_type(8)));
typedef float aw_f32x4 __attribute__((ext_vector_type(4)));
typedef short aw_s16x4 __attribute__((ext_vector_type(4)));

struct AwParams {
    const void* dy;
    const uint8_t *q, *scale;
    float *part, *dbpart;          // [ranges][N][C], [ranges][N]
    float *dw, *db;
    int64_t M, S, dn, dr;
    int N, C, ldq, CB, tiles_n, tiles_c, ranges;
    int64_t per;                   // rows per range, a multiple of AW_K
};

__device__ __forceinline__ aw_s16x4 aw_tr(const unsigned char* sub, int lane_off, int rowblk) {
    const unsigned char* p = sub + lane_off + rowblk * 512;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((aw_s16x4 __attribute__((address_space(3)))*)(p));
}
__device__ __forceinline__ aw_bf16x8 aw_frag(const unsigned char* sub, int lane_off) {
    const aw_s16x4 lo = aw_tr(sub, lane_off, 0), hi = aw_tr(sub, lane_off, 1);
    const uint4 v = make_uint4(((const unsigned*)&lo)[0], ((const unsigned*)&lo)[1], ((const unsigned*)&hi)[0], ((const unsigned*)&hi)[1]);
    return __builtin_bit_cast(aw_bf16x8, v);
}
// byte offset of the 8-channel piece pc of row r inside a tile
__device__ __forceinline__ int aw_off(int r, int pc) {
    return ((r >> 5) * (AW_T / 16) + (pc >> 1)) * AW_SUB + (r & 31) * 32 + (pc & 1) * 16;
}

template <int DT> struct AwPieces { static constexpr int n = DT == Y5M_BF16 ? 1 : DT == Y5M_F16 ? 2 : 3; };
// dY values as NP bf16 summands, highest first; the last one takes what is left (exact: 8 bits each)
template <int DT, int NP> __device__ __forceinline__ void aw_split(const Raw8<DT>& raw, act8_u32x4 out[NP]) {
    if constexpr (NP == 1) {
        out[0] = raw.r[0];
    } else {
        float v[8];
        unpack8<DT>(raw, v);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t w = f32x2_to_bf16x2(v[2 * k], v[2 * k + 1]);
                out[p][k] = w;
                if (p + 1 < NP) {
                    v[2 * k] -= __uint_as_float(w << 16);
                    v[2 * k + 1] -= __uint_as_float(w & 0xffff0000u);
                }
            }
    }
}

template <int DT, int FMT, bool AL>
__global__ __launch_bounds__(AW_THREADS) void act8_wgrad_kernel(const AwParams P) {
    typedef typename RowElem<DT>::T T;
    constexpr int NP = AwPieces<DT>::n;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    unsigned char* Xs = smem + NP * AW_TILE;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wn = wid & 1, wc = wid >> 1;
    unsigned b = blockIdx.x;
    const int ct = (int)(b % (unsigned)P.tiles_c);
    b /= (unsigned)P.tiles_c;
    const int nt = (int)(b % (unsigned)P.tiles_n), range = (int)(b / (unsigned)P.tiles_n);
    const int n0 = nt * AW_T, c0 = ct * AW_T;
    const int64_t m0 = range * P.per, m1 = m0 + P.per < P.M ? m0 + P.per : P.M;

    aw_f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (aw_f32x4){0.f, 0.f, 0.f, 0.f};
    float bias[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) bias[k] = 0.f;
    const bool want_db = P.dbpart && ct == 0;

    // loader: 16 threads per row (8 channels each), 16 rows at once, 4 times
    const int pc = tid & 15, rl = tid >> 4;
    const int yc = n0 + pc * 8, xc = c0 + pc * 8;
    const bool yin = yc < P.N, xin = xc < P.C;
    const int lane_off = (4 * (lane >> 4) + ((lane & 15) >> 2)) * 32 + (lane & 3) * 8;

    for (int64_t m = m0; m < m1; m += AW_K) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = u * 16 + rl;
            const int64_t row = m + r;
            Raw8<DT> y = {};
            act8_u32x2 q = {0u, 0u};
            float sc = 1.0f;
            if (row < m1) {
                const int64_t n = row / P.S;
                if (yin) y = load_raw8<DT, AL>(static_cast<const T*>(P.dy) + n * P.dn + (row - n * P.S) * P.dr + yc, P.N - yc);
                if (xin) {
                    q = *reinterpret_cast<const act8_u32x2*>(P.q + row * P.ldq + xc);
                    sc = act8_scale(P.scale[row * P.CB + (xc >> 5)]);
                }
            }
            act8_u32x4 yp[NP];
            aw_split<DT, NP>(y, yp);
#pragma unroll
            for (int p = 0; p < NP; ++p) *reinterpret_cast<act8_u32x4*>(smem + p * AW_TILE + aw_off(r, pc)) = yp[p];
            if (want_db) {
                float v[8];
                unpack8<DT>(y, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) bias[k] += v[k];
            }
            float xv[8];
            act8_decode8<FMT>(q, sc, xv);
            act8_u32x4 xp;
#pragma unroll
            for (int k = 0; k < 4; ++k) xp[k] = f32x2_to_bf16x2(xv[2 * k], xv[2 * k + 1]);
            *reinterpret_cast<act8_u32x4*>(Xs + aw_off(r, pc)) = xp;
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < AW_K / 32; ++ks) {
            aw_bf16x8 xf[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) xf[j] = aw_frag(Xs + (ks * (AW_T / 16) + wc * 4 + j) * AW_SUB, lane_off);
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const aw_bf16x8 yf = aw_frag(smem + p * AW_TILE + (ks * (AW_T / 16) + wn * 4 + i) * AW_SUB, lane_off);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yf, xf[j], acc[i][j], 0, 0, 0);
                }
        }
    }
    // D[n][c]: lane holds n = 4 (lane >> 4) + r, c = lane & 15
    float* part = P.part + (size_t)range * P.N * P.C;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + (wc * 4 + j) * 16 + (lane & 15);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + (wn * 4 + i) * 16 + 4 * (lane >> 4) + r;
                if (n < P.N && c < P.C) part[(size_t)n * P.C + c] = acc[i][j][r];
            }
        }
    if (P.dbpart) {                                            // (uniform over the launch)
        float* red = reinterpret_cast<float*>(smem);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) red[rl * AW_T + pc * 8 + k] = bias[k];
        __syncthreads();
        if (want_db && tid < AW_T && n0 + tid < P.N) {
            float t = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) t += red[r * AW_T + tid];
            P.dbpart[(size_t)range * P.N + n0 + tid] = t;
        }
    }
}

// dW = sum of the ranges' tiles, in order
__global__ __launch_bounds__(AW_THREADS) void act8_wgrad_join_kernel(const AwParams P) {
    const int64_t i = (int64_t)blockIdx.x * AW_THREADS + threadIdx.x, nw = (int64_t)P.N * P.C;
    if (i < nw) {
        double t = 0.0;
        for (int r = 0; r < P.ranges; ++r) t += (double)P.part[(size_t)r * nw + i];
        P.dw[i] = (float)t;
    } else if (P.db && i - nw < P.N) {
        double t = 0.0;
        for (int r = 0; r < P.ranges; ++r) t += (double)P.dbpart[(size_t)r * P.N + (i - nw)];
        P.db[i - nw] = (float)t;
    }
}

static void aw_geometry(AwParams& P, int64_t M, int N, int C) {
    P.M = M; P.N = N; P.C = C; P.CB = (C + 31) / 32;
    P.tiles_n = (N + AW_T - 1) / AW_T;
    P.tiles_c = (C + AW_T - 1) / AW_T;
    const int64_t tiles = (int64_t)P.tiles_n * P.tiles_c, steps = (M + AW_K - 1) / AW_K;
    int64_t want = (1024 + tiles - 1) / tiles, most = (steps + 3) / 4;     // about 4 workgroups per CU, at least 4 steps each
    if (want > most) want = most;
    if (want < 1) want = 1;
    P.per = (steps + want - 1) / want * AW_K;
    P.ranges = (int)((M + P.per - 1) / P.per);
}

extern "C" size_t y5m_act8_wgrad_workspace_bytes(int64_t M, int Cout, int C) {
    if (M <= 0 || Cout <= 0 || C <= 0) return 0;
    AwParams P = {};
    aw_geometry(P, M, Cout, C);
    return (size_t)P.ranges * ((size_t)Cout * C + Cout) * sizeof(float);
}

extern "C" int y5m_act8_wgrad(const void* dy, int64_t dy_batch_stride, int64_t dy_row_stride, int64_t N, int64_t S, int Cout, const void* q, int ldq,
                              const void* scale, int C, int fmt, float* dw, float* db, void* ws, size_t ws_bytes, int dtype, void* stream) {
    Y5M_REQUIRE(dtype == Y5M_F32 || dtype == Y5M_BF16 || dtype == Y5M_F16, "dtype");
    Y5M_REQUIRE(fmt == Y5M_KEEP_E4M3 || fmt == Y5M_KEEP_INT8, "8-bit format");
    Y5M_REQUIRE(N >= 0 && S >= 0 && Cout > 0 && C > 0 && (double)N * (double)S < 1e12, "sizes");
    Y5M_REQUIRE((double)Cout * (double)C < 1e9, "weight too large");
    Y5M_REQUIRE(dw, "null pointer");
    if (N * S == 0) {
        const int rc = y5m_fill32(dw, 0, (size_t)Cout * C, y5m_stream(stream));
        return rc != Y5M_OK || !db ? rc : y5m_fill32(db, 0, Cout, y5m_stream(stream));
    }
    Y5M_REQUIRE(dy && q && scale, "null pointer");
    Y5M_REQUIRE(ldq >= C && ldq % 8 == 0 && ((uintptr_t)q & 7) == 0, "8-bit form: ldq % 8 == 0, at least C, codes 8-byte aligned");
    Y5M_REQUIRE(ws && ws_bytes >= y5m_act8_wgrad_workspace_bytes(N * S, Cout, C), "workspace too small");
    AwParams P = {};
    aw_geometry(P, N * S, Cout, C);
    P.dy = dy; P.dn = dy_batch_stride; P.dr = dy_row_stride; P.S = S;
    P.q = static_cast<const uint8_t*>(q); P.scale = static_cast<const uint8_t*>(scale); P.ldq = ldq;
    P.part = static_cast<float*>(ws);
    P.dbpart = db ? P.part + (size_t)P.ranges * Cout * C : nullptr;
    P.dw = dw; P.db = db;
    const int64_t blocks = (int64_t)P.tiles_n * P.tiles_c * P.ranges;
    Y5M_REQUIRE(blocks < (1ll << 31), "too many workgroups");
    const bool al = rows_aligned16(dy, dy_batch_stride, dy_row_stride, N, S, Cout, dtype);
#define GO(DT, FMT, AL)                                                                                                          \
    do {                                                                                                                         \
        constexpr int lds = (AwPieces<DT>::n + 1) * AW_TILE;                                                                     \
        static bool set = false;                                                                                                 \
        if (!set && hipFuncSetAttribute(reinterpret_cast<const void*>(act8_wgrad_kernel<DT, FMT, AL>), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) { \
            y5m_set_error("act8_wgrad_kernel: %d bytes of LDS refused", lds);                                                    \
            return Y5M_ELAUNCH;                                                                                                  \
        }                                                                                                                        \
        set = true;                                                                                                              \
        hipLaunchKernelGGL((act8_wgrad_kernel<DT, FMT, AL>), dim3((unsigned)blocks), dim3(AW_THREADS), lds, y5m_stream(stream), P); \
    } while (0)
#define GO2(DT)                                                                                                                  \
    do {                                                                                                                         \
        if (fmt == Y5M_KEEP_E4M3) { if (al) GO(DT, Y5M_KEEP_E4M3, true); else GO(DT, Y5M_KEEP_E4M3, false); }                    \
        else { if (al) GO(DT, Y5M_KEEP_INT8, true); else GO(DT, Y5M_KEEP_INT8, false); }                                         \
    } while (0)
    if (dtype == Y5M_F32) GO2(Y5M_F32);
    else if (dtype == Y5M_BF16) GO2(Y5M_BF16);
    else GO2(Y5M_F16);
#undef GO2
#undef GO
    Y5M_CHECK_LAUNCH("act8_wgrad_kernel");
    const int64_t items = (int64_t)Cout * C + (db ? Cout : 0);
    hipLaunchKernelGGL(act8_wgrad_join_kernel, dim3((unsigned)((items + AW_THREADS - 1) / AW_THREADS)), dim3(AW_THREADS), 0, y5m_stream(stream), P);
    Y5M_CHECK_LAUNCH("act8_wgrad_join_kernel");
    return Y5M_OK;
}

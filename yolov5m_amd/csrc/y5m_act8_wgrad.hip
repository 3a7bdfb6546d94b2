// Weight gradient of a pointwise convolution from its input in 8 bits:  dW[n][c] = sum_m dY[m][n] X8[m][c],  db[n] = sum_m dY[m][n].
//
// GEMM with K = rows (up to millions) and both operands row-major along K, as they lie in memory. Arithmetic: an 8-bit value times its
// power-of-two scale has at most 8 significant bits, so it IS a bf16 value; dY in bf16 is one, in fp16 (11 bits) the exact sum of two
// and in f32 (24 bits) of three bf16 values (infinities and what rounds to one are taken again, in limited pieces). Products of bf16 MFMAs are exact in f32, so every type runs on the bf16 matrix cores
// with f32 accumulation, and nothing is rounded before the sum (f32 MFMA: 1/16 of the rate).
//
// An MFMA operand wants 8 consecutive k (rows) of ONE channel per lane, memory has 8 channels of one row next to each other. No LDS
// is needed for that transpose: the order of rows and channels inside a tile is free as long as both operands agree on the rows. Lane
// (i = lane & 15, g = lane >> 4) loads rows 8 g .. 8 g + 7 of its OWN P channels (16 bytes of bf16, 8 of codes: a 16-lane group reads
// 256 consecutive bytes of a row), and byte permutes (one per two values) turn the 8 x P block into P operands. Operand ja of lane i is
// then channel P i + ja: the product of operands (ja, jb) is the 16 x 16 block of dW at rows P i + ja, columns P i' + jb, and the P x P
// products of one 32-row step fill a (16 P)^2 tile (P = 8: 128 x 128, 64 MFMAs, 256 accumulators a lane), no barrier in the loop.
// A lane ends up with P consecutive columns of a row of dW: 16-byte stores.
// The four waves of a workgroup are WN x WC tiles side by side (they share operands through L1) times WK interleaved parts of the
// rows, added in LDS; row ranges of different workgroups are joined from f32 partial tiles by a second launch in a fixed order (no
// atomics: one result per input).
#include "y5m_act8.h"

#define AW_THREADS 256
#define AW_K 32                   // rows per step of a wave

typedef __bf16 aw_bf16x8 __attribute__((ext_vector_type(8)));
typedef float aw_f32x4 __attribute__((ext_vector_type(4)));

struct AwParams {
    const void* dy;
    const uint8_t *q, *scale;
    float *part, *dbpart;          // [ranges][N][C], [ranges][N]
    float *dw, *db;
    int64_t M, S, dn, dr;
    int N, C, ldq, CB, tiles_n, tiles_c, ranges, slots;
    int64_t per;                   // rows per range, a multiple of AW_K
};

template <int DT> struct AwPieces { static constexpr int n = DT == Y5M_BF16 ? 1 : DT == Y5M_F16 ? 2 : 3; };

// one step's data of a lane: 8 rows of PA channels of dY (raw) and of PC codes, and the rows' scales
template <int DT, int PA, int PC> struct AwStage {
    static constexpr int AD = DT == Y5M_F32 ? PA : PA / 2;
    unsigned a[8][AD];
    unsigned q[8][PC / 4];
    unsigned s, s2;                          // scale bytes of row 8 g + (i & 7), blocks (i >> 3) and (i >> 3) + 2 of the tile
};

// n dwords at byte offset `off` of a buffer resource: zero beyond its last byte, in hardware
template <int ND> __device__ __forceinline__ void aw_buffer(__amdgpu_buffer_rsrc_t rs, unsigned off, unsigned* d) {
    if constexpr (ND == 1) {
        d[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
    } else if constexpr (ND == 2) {
        const act8_u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0);
        d[0] = v[0];
        d[1] = v[1];
    } else {
        const act8_u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0);
        d[0] = v[0];
        d[1] = v[1];
        d[2] = v[2];
        d[3] = v[3];
        if constexpr (ND == 8) aw_buffer<4>(rs, off + 16, d + 4);
    }
}

// How rows are read.
// AW_PIECES: rows at one distance, in whole pieces through buffer resources that end with the range (the launcher keeps a range below
// 2 GiB): rows beyond the range and channels beyond the last read as zero, the loop has no tail.
// AW_ROWS: rows at one distance that start at any element (codes and scales as above). A row's last piece is the PA values that END with
// the row: its lane then holds `aw_shift` channels of its neighbour's as well, which are not stored. (Values shifted and masked
// in the loop, rows addressed in 64 bits: 69 x 659 over 64152 rows in fp16 with the store of X 194 us, 84 so.)
// AW_FEW: the same for fewer than PA channels, by elements (2 x 189 over 540676 rows in fp16 with the store: 224 us through AW_ANY, 115).
// AW_ANY: any strides, any size.
enum { AW_ANY = 0, AW_FEW = 1, AW_ROWS = 2, AW_PIECES = 3 };
template <int MODE, int PA> __device__ __forceinline__ int aw_shift(int n, int N) {
    return MODE != AW_PIECES && N >= PA && n < N && n + PA > N ? n + PA - N : 0;
}
template <int DT, int PA, int PC, int MODE> struct AwLoader {
    typedef typename RowElem<DT>::T T;
    static constexpr unsigned OOB = 0x80000000u;
    const AwParams& P;
    int64_t m0, m1;
    int n, c, g, nl;
    bool nin, cin;
    __amdgpu_buffer_rsrc_t ry, rq, rs;
    unsigned ao, qo, so, as;                 // byte offsets of row 8 g (scales: of this lane's row) of the range, bytes from row to row of dY
    int sr, sb;                              // the row and block of the tile whose scale this lane fetches
    bool sin, sin2;
    __device__ __forceinline__ AwLoader(const AwParams& P_, int64_t m0_, int64_t m1_, int n_, int c_, int g_, int c0, int i16)
        : P(P_), m0(m0_), m1(m1_), n(n_), c(c_), g(g_) {
        nin = n < P.N;
        cin = c < P.C;
        nl = nin && MODE != AW_FEW ? n - aw_shift<MODE, PA>(n, P.N) : 0;
        sr = 8 * g + (i16 & 7);
        sb = (c0 >> 5) + (i16 >> 3);
        sin = sb < P.CB;
        sin2 = PC == 8 && sb + 2 < P.CB;
        if constexpr (MODE != AW_ANY) {
            as = (unsigned)(P.dr * (int64_t)sizeof(T));
            const unsigned rows = (unsigned)(m1 - m0);
            if constexpr (MODE == AW_PIECES) ry = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(static_cast<const T*>(P.dy) + m0 * P.dr), 0, (rows - 1) * as + (unsigned)P.N * (unsigned)sizeof(T), 0x00020000);
            rq = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(P.q + m0 * P.ldq), 0, rows * (unsigned)P.ldq, 0x00020000);
            rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(P.scale + m0 * P.CB), 0, rows * (unsigned)P.CB, 0x00020000);
            ao = MODE != AW_PIECES ? (unsigned)nl * (unsigned)sizeof(T) : nin ? (unsigned)(8 * g) * as + (unsigned)n * (unsigned)sizeof(T) : OOB;
            qo = cin ? (unsigned)(8 * g) * (unsigned)P.ldq + (unsigned)c : OOB;
            so = (unsigned)sr * (unsigned)P.CB + (unsigned)sb;
        }
    }
    __device__ __forceinline__ void load(AwStage<DT, PA, PC>& st, unsigned step) const {       // step: rows from m0
        constexpr int AD = AwStage<DT, PA, PC>::AD;
        if constexpr (MODE != AW_ANY) {
            const unsigned a = ao + step * as, q = qo + step * (unsigned)P.ldq, s = so + step * (unsigned)P.CB;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (MODE == AW_PIECES) {
                    aw_buffer<AD>(ry, a + (unsigned)j * as, st.a[j]);
                } else {
                    const unsigned r = step + (unsigned)(8 * g + j);
                    const bool in = r < (unsigned)(m1 - m0);
                    const char* p = reinterpret_cast<const char*>(static_cast<const T*>(P.dy) + m0 * P.dr) + ((in ? r : 0u) * as + ao);
                    if constexpr (MODE == AW_ROWS) {
                        __builtin_memcpy(st.a[j], p, sizeof(st.a[j]));
                    } else {
                        T e[PA];
#pragma unroll
                        for (int k = 0; k < PA; ++k) e[k] = reinterpret_cast<const T*>(p)[k < P.N ? k : P.N - 1];
                        __builtin_memcpy(st.a[j], e, sizeof(e));
                    }
#pragma unroll
                    for (int k = 0; k < AD; ++k) st.a[j][k] = in ? st.a[j][k] : 0u;
                }
                aw_buffer<PC / 4>(rq, q + (unsigned)(j * P.ldq), st.q[j]);
            }
            st.s = __builtin_amdgcn_raw_buffer_load_b8(rs, sin ? s : OOB, 0, 0);
            if constexpr (PC == 8) st.s2 = __builtin_amdgcn_raw_buffer_load_b8(rs, sin2 ? s + 2 : OOB, 0, 0);
        } else {
            // N < PA by elements. P.S = 0: the rows at one distance
            const bool small = P.N < PA;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t row = m0 + step + 8 * g + j;
                const bool in = row < m1;
                const int64_t r = in ? row : m0, nb = P.S ? r / P.S : 0;
                const T* p = static_cast<const T*>(P.dy) + nb * P.dn + (r - nb * P.S) * P.dr;
                T e[PA];
                if (small) {
#pragma unroll
                    for (int k = 0; k < PA; ++k) e[k] = p[n + k < P.N ? n + k : P.N - 1];
                } else {
                    __builtin_memcpy(e, p + nl, sizeof(e));
                }
                if constexpr (DT == Y5M_F32) {
#pragma unroll
                    for (int k = 0; k < PA; ++k) st.a[j][k] = in ? __float_as_uint(e[k]) : 0u;
                } else {
#pragma unroll
                    for (int k = 0; k < PA / 2; ++k) st.a[j][k] = in ? (unsigned)e[2 * k] | (unsigned)e[2 * k + 1] << 16 : 0u;
                }
                const uint8_t* q = P.q + r * P.ldq + (cin ? c : 0);
#pragma unroll
                for (int k = 0; k < PC / 4; ++k) {
                    const unsigned w = *reinterpret_cast<const unsigned*>(q + 4 * k);
                    st.q[j][k] = in && cin ? w : 0u;
                }
            }
            const int64_t row = m0 + step + sr;
            const bool in = row < m1;
            const uint8_t* sp = P.scale + (in ? row : m0) * P.CB;
            const unsigned a = sp[sin ? sb : 0], b = PC == 8 ? sp[sin2 ? sb + 2 : 0] : 0u;
            st.s = in && sin ? a : 0u;
            if constexpr (PC == 8) st.s2 = in && sin2 ? b : 0u;
        }
    }
};

// low or high halves of two dwords: [lo.h, hi.h]
__device__ __forceinline__ unsigned aw_pair(unsigned lo, unsigned hi, int h) {
    return __builtin_amdgcn_perm(hi, lo, h ? 0x07060302u : 0x05040100u);
}
template <bool LIM, bool FIRST> struct AwPass { static constexpr bool lim = LIM, first = FIRST; };
// bits of v within bf16's finite values (a NaN: any of them)
__device__ __forceinline__ unsigned aw_limit(float v) { return __float_as_uint(__builtin_amdgcn_fmed3f(v, -0x1.fep127f, 0x1.fep127f)); }
// two codes (bytes 2 h, 2 h + 1 of w) times their scale as a pair of bf16 (exact)
template <int FMT> __device__ __forceinline__ unsigned aw_decode2(unsigned w, float scale, int h) {
    if constexpr (FMT == Y5M_KEEP_E4M3) {
        return __builtin_bit_cast(unsigned, h ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
    } else {
        // (a signed byte converts in one instruction; as (b + 128) * scale - 128 * scale in one fma the offset left f32 at the largest scale)
        return f32x2_to_bf16x2((float)(int8_t)(w >> (16 * h)) * scale, (float)(int8_t)(w >> (16 * h + 8)) * scale);
    }
}

template <int DT, int FMT, int PA, int PC, int WN, int WC, int WK, int MODE, bool DB>
__global__ __launch_bounds__(AW_THREADS, PA * PC <= 32 ? 2 : 1) void act8_wgrad_kernel(const AwParams P) {
    static_assert(WN * WC * WK == AW_THREADS / 64, "four waves");
    constexpr int NP = AwPieces<DT>::n;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, i16 = lane & 15, g = lane >> 4;
    const int wn = wid % WN, wc = (wid / WN) % WC, wk = wid / (WN * WC);
    // workgroups go round the 8 XCDs: give each XCD a contiguous stretch of the range-major order, so that the tiles that read the
    // same rows share its L2
    const unsigned q8 = gridDim.x >> 3, r8 = gridDim.x & 7, xcd = blockIdx.x & 7;
    unsigned b = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
    const int ct = (int)(b % (unsigned)P.tiles_c);
    b /= (unsigned)P.tiles_c;
    const int nt = (int)(b % (unsigned)P.tiles_n), range = (int)(b / (unsigned)P.tiles_n);
    const int n0 = (nt * WN + wn) * 16 * PA, c0 = (ct * WC + wc) * 16 * PC;
    const int64_t m0 = range * P.per, m1 = m0 + P.per < P.M ? m0 + P.per : P.M;

    aw_f32x4 acc[PA][PC];
#pragma unroll
    for (int i = 0; i < PA; ++i)
#pragma unroll
        for (int j = 0; j < PC; ++j) acc[i][j] = (aw_f32x4){0.f, 0.f, 0.f, 0.f};
    float bias[PA];
#pragma unroll
    for (int k = 0; k < PA; ++k) bias[k] = 0.f;

    const AwLoader<DT, PA, PC, MODE> L(P, m0, m1, n0 + PA * i16, c0 + PC * i16, g, c0, i16);
    // pass: are the pieces before the last limited to bf16's finite values, are these rows taken for the first time
    auto compute = [&](AwStage<DT, PA, PC>& st, auto pass) __attribute__((always_inline)) {
        constexpr bool LIM = decltype(pass)::lim, BIAS = DB && decltype(pass)::first;
        // (rows and channels beyond the last: codes 0, scale byte 0 = 0.0)
        aw_bf16x8 xf[PC];
        float sc[8];
        const int blk = PC * i16 >> 5;                             // this lane's block of the tile
        // (opaque here: combined where they are loaded, the two would be waited for there)
        unsigned pair = st.s, high = PC == 8 ? st.s2 : 0u;
        asm volatile("" : "+v"(pair));
        asm volatile("" : "+v"(high));
        pair |= high << 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned w = (unsigned)__shfl((int)pair, 16 * g + j + 8 * (blk & 1), 64);
            sc[j] = act8_scale((w >> (8 * (blk >> 1))) & 255u);
        }
#pragma unroll
        for (int w = 0; w < PC / 2; ++w) {
            unsigned v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = aw_decode2<FMT>(st.q[j][w >> 1], sc[j], w & 1);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                xf[2 * w + h] = __builtin_bit_cast(aw_bf16x8, (act8_u32x4){aw_pair(v[0], v[1], h), aw_pair(v[2], v[3], h), aw_pair(v[4], v[5], h), aw_pair(v[6], v[7], h)});
        }
#pragma unroll
        for (int ja = 0; ja < PA; ++ja) {
            act8_u32x4 yf[NP];
            if constexpr (DT == Y5M_BF16) {
#pragma unroll
                for (int p = 0; p < 4; ++p) yf[0][p] = aw_pair(st.a[2 * p][ja >> 1], st.a[2 * p + 1][ja >> 1], ja & 1);
                if constexpr (BIAS) {
#pragma unroll
                    for (int p = 0; p < 4; ++p) bias[ja] += __uint_as_float(yf[0][p] << 16) + __uint_as_float(yf[0][p] & 0xffff0000u);
                }
            } else {
                // the value as a sum of NP bf16, highest first; what is left after the others fits the last one
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    float lo, hi;
                    if constexpr (DT == Y5M_F32) {
                        lo = __uint_as_float(st.a[2 * p][ja]);
                        hi = __uint_as_float(st.a[2 * p + 1][ja]);
                    } else {
                        lo = f16_to_f32((uint16_t)(st.a[2 * p][ja >> 1] >> (16 * (ja & 1))));
                        hi = f16_to_f32((uint16_t)(st.a[2 * p + 1][ja >> 1] >> (16 * (ja & 1))));
                    }
                    if constexpr (BIAS) bias[ja] += lo + hi;
#pragma unroll
                    for (int e = 0; e < NP; ++e) {
                        // (limited pieces are truncated: rounded, the first two of the largest f32 would pass it in the sum)
                        const unsigned w = LIM && e + 1 < NP ? aw_pair(aw_limit(lo), aw_limit(hi), 1) : f32x2_to_bf16x2(lo, hi);
                        yf[e][p] = w;
                        lo -= __uint_as_float(w << 16);
                        hi -= __uint_as_float(w & 0xffff0000u);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < NP; ++e)
#pragma unroll
                for (int jb = 0; jb < PC; ++jb)
                    acc[ja][jb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(aw_bf16x8, yf[e]), xf[jb], acc[ja][jb], 0, 0, 0);
        }
    };

    // this wave's steps are rows 32 (wk + WK t) of the range; the next step's loads are in flight under the current one's products.
    // Steps are taken in pairs: one beyond the end reads zeros.
    auto steps = [&](auto pass) __attribute__((always_inline)) {
        const unsigned rows = (unsigned)(m1 - m0), stride = AW_K * WK;
        AwStage<DT, PA, PC> s0, s1;
        L.load(s0, AW_K * wk);
        for (unsigned t = AW_K * wk; t < rows; t += 2 * stride) {
            // (the loads stay ahead of the products: left to itself the scheduler sinks each to its use and waits for it there)
            L.load(s1, t + stride);
            __builtin_amdgcn_sched_barrier(0);
            compute(s0, pass);
            __builtin_amdgcn_sched_barrier(0);
            L.load(s0, t + 2 * stride);
            __builtin_amdgcn_sched_barrier(0);
            compute(s1, pass);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr bool ONCE = NP == 3 && MODE == AW_ANY && DB;
    steps(AwPass<ONCE, true>());
    if constexpr (NP > 1 && !ONCE) {
        // A dY that is infinite, or finite above bf16's largest value, left an infinite first piece and an opposite or NaN rest: every sum of its
        // channel is NaN. Then, and where a NaN is the right result, the wave takes its rows again with limited pieces (an infinity is left for the
        // last one). Limiting always would cost every call 4 (fp16) to 9 % (f32). (ONCE: limited
        // at once where a second loop would spill 39 registers: 255 x 100 over 1200 rows 18.1 us instead of 19.3.)
        bool nan = false;
#pragma unroll
        for (int i = 0; i < PA; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) nan |= acc[i][0][r] != acc[i][0][r];
        if (__any(nan)) {
#pragma unroll
            for (int i = 0; i < PA; ++i)
#pragma unroll
                for (int j = 0; j < PC; ++j) acc[i][j] = (aw_f32x4){0.f, 0.f, 0.f, 0.f};
            steps(AwPass<true, false>());
        }
    }

    // bias: the four row groups of the wave
    if constexpr (DB) {
#pragma unroll
        for (int k = 0; k < PA; ++k) {
            bias[k] += __shfl_xor(bias[k], 16, 64);
            bias[k] += __shfl_xor(bias[k], 32, 64);
        }
    }
    // the WK parts of a tile are added in LDS, PA / 2 operands' worth at a time
    constexpr int HALF = PA / 2 * PC * 4;                      // floats of a lane
    float* red = reinterpret_cast<float*>(smem);               // [WK - 1][WN * WC][HALF][64], then [WK][WN][16 PA]
    float* redb = red + (WK > 1 ? (size_t)(WK - 1) * WN * WC * HALF * 64 : 0);
    if constexpr (WK > 1) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            __syncthreads();
            if (wk > 0) {
                float* d = red + ((size_t)(wk - 1) * WN * WC + wid % (WN * WC)) * HALF * 64 + lane;
#pragma unroll
                for (int i = 0; i < PA / 2; ++i)
#pragma unroll
                    for (int j = 0; j < PC; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) d[((i * PC + j) * 4 + r) * 64] = acc[half * (PA / 2) + i][j][r];
            }
            __syncthreads();
            if (wk == 0) {
#pragma unroll
                for (int o = 1; o < WK; ++o) {
                    const float* d = red + ((size_t)(o - 1) * WN * WC + wid % (WN * WC)) * HALF * 64 + lane;
#pragma unroll
                    for (int i = 0; i < PA / 2; ++i)
#pragma unroll
                        for (int j = 0; j < PC; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[half * (PA / 2) + i][j][r] += d[((i * PC + j) * 4 + r) * 64];
                }
            }
        }
    }
    if constexpr (DB) {
        __syncthreads();
        if (ct == 0 && wc == 0 && g == 0) {
            const int sh = aw_shift<MODE, PA>(n0 + PA * i16, P.N);
#pragma unroll
            for (int k = 0; k < PA; ++k)
                if (k >= sh) redb[(wk * WN + wn) * 16 * PA + PA * i16 + k - sh] = bias[k];
        }
        __syncthreads();
        const int nn = nt * WN * 16 * PA + tid;
        if (ct == 0 && tid < WN * 16 * PA && nn < P.N) {
            float t = 0.f;
#pragma unroll
            for (int o = 0; o < WK; ++o) t += redb[o * WN * 16 * PA + tid];
            P.dbpart[(size_t)range * P.N + nn] = t;
        }
    }
    if (wk == 0) {
        // lane: rows n0 + PA (4 g + r) + ja, columns c0 + PC i16 .. + PC - 1
        float* part = P.part + (size_t)range * P.N * P.C;
        const int c = c0 + PC * i16;
        const bool vec = (P.C & 3) == 0;
#pragma unroll
        for (int ja = 0; ja < PA; ++ja)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int np = n0 + PA * (4 * g + r), sh = aw_shift<MODE, PA>(np, P.N), n = np + ja - sh;
                if (n >= P.N || ja < sh) continue;
                float* d = part + (size_t)n * P.C + c;
#pragma unroll
                for (int h = 0; h < PC / 4; ++h) {
                    if (vec && c + 4 * h < P.C) {
                        *reinterpret_cast<aw_f32x4*>(d + 4 * h) = (aw_f32x4){acc[ja][4 * h][r], acc[ja][4 * h + 1][r], acc[ja][4 * h + 2][r], acc[ja][4 * h + 3][r]};
                    } else if (!vec) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (c + 4 * h + k < P.C) d[4 * h + k] = acc[ja][4 * h + k][r];
                    }
                }
            }
    }
}

// dW = sum of the ranges' tiles: `slots` threads share an output, each takes every slots-th range; joined in order, in f64
__global__ __launch_bounds__(AW_THREADS) void act8_wgrad_join_kernel(const AwParams P) {
    __shared__ double red[AW_THREADS];
    const int per = AW_THREADS / P.slots, o = threadIdx.x % per, slot = threadIdx.x / per;
    const int64_t i = (int64_t)blockIdx.x * per + o, nw = (int64_t)P.N * P.C;
    const bool isw = i < nw, in = isw || (P.db && i - nw < P.N);
    const float* src = isw ? P.part + i : P.dbpart + (i - nw);
    const size_t step = isw ? (size_t)nw : (size_t)P.N;
    double t = 0.0;
    if (in) {
        int r = slot;
        for (; r + 7 * P.slots < P.ranges; r += 8 * P.slots) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = src[(size_t)(r + u * P.slots) * step];
#pragma unroll
            for (int u = 0; u < 8; ++u) t += (double)v[u];
        }
        for (; r < P.ranges; r += P.slots) t += (double)src[(size_t)r * step];
    }
    if (P.slots > 1) {
        red[threadIdx.x] = t;
        __syncthreads();
        if (slot != 0) return;
        t = 0.0;
        for (int s = 0; s < P.slots; ++s) t += red[s * per + o];
    }
    if (in) (isw ? P.dw : P.db)[isw ? i : i - nw] = (float)t;
}

// Tiles. bf16 in whole pieces: 128 x 128 at one wave per SIMD; 64 x 128 / 64 x 64 at two where the weight is no wider (half the wasted
// products). (64 x 128 for all: 120 us instead of 112 for store + gradient at 768 x 1536 over 25600 rows; the second wave fills the
// waits, but every byte goes through L1 half as often again.) fp16 / f32 (two or three products per value, twice the raw registers) and
// rows read from any start: 64 x 64. Waves: two tiles of dY channels (else of X channels) side by side where there are two, so that a
// workgroup's partial tiles are joined in LDS only twice; else all four waves split the rows of one tile.
struct AwShape { int pa, pc, wn, wc, wk; };
static AwShape aw_shape(int N, int C, bool wide) {
    AwShape s;
    s.pc = !wide || C <= 64 ? 4 : 8;
    s.pa = s.pc == 4 || N <= 64 ? 4 : 8;
    const int tn = (N + 16 * s.pa - 1) / (16 * s.pa), tc = (C + 16 * s.pc - 1) / (16 * s.pc);
    s.wn = s.pa == 8 && tn % 2 == 0 ? 2 : 1;
    s.wc = s.pa == 8 && s.wn == 1 && tc % 2 == 0 ? 2 : 1;
    s.wk = 4 / (s.wn * s.wc);
    return s;
}
static void aw_geometry(AwParams& P, const AwShape& s, int64_t M, int N, int C) {
    P.M = M; P.N = N; P.C = C; P.CB = (C + 31) / 32;
    P.tiles_n = (N + 16 * s.pa * s.wn - 1) / (16 * s.pa * s.wn);
    P.tiles_c = (C + 16 * s.pc * s.wc - 1) / (16 * s.pc * s.wc);
    // ranges: as many workgroups as fit the CUs at once, at least a step per wave, and less than 2 GiB of rows each
    const int64_t tiles = (int64_t)P.tiles_n * P.tiles_c, steps = (M + AW_K - 1) / AW_K, most = (steps + s.wk - 1) / s.wk;
    int64_t want = (s.pa == 8 ? 256 : 512) / tiles;
    if (want > most) want = most;
    if (want < 1) want = 1;
    int64_t per = (steps + want - 1) / want * AW_K;
    const int64_t cap = (1ll << 30) / (4ll * (N > C + 8 ? N : C + 8)) / AW_K * AW_K;
    if (per > cap) per = cap > AW_K ? cap : AW_K;
    P.per = per;
    P.ranges = (int)((M + P.per - 1) / P.per);
    P.slots = P.ranges > 64 ? 16 : P.ranges > 16 ? 4 : 1;
}

extern "C" size_t y5m_act8_wgrad_workspace_bytes(int64_t M, int Cout, int C) {
    if (M <= 0 || Cout <= 0 || C <= 0) return 0;
    AwParams P = {};
    aw_geometry(P, aw_shape(Cout, C, true), M, Cout, C);
    const int a = P.ranges;
    aw_geometry(P, aw_shape(Cout, C, false), M, Cout, C);
    return (size_t)(a > P.ranges ? a : P.ranges) * ((size_t)Cout * C + Cout) * sizeof(float);
}

template <int DT, int FMT, int PA, int PC, int WN, int WC, int MODE, bool DB>
static int aw_launch_db(const AwParams& P, hipStream_t st) {
    constexpr int WK = 4 / (WN * WC), lds = ((WK - 1) * WN * WC * (PA / 2 * PC * 4) * 64 + WK * WN * 16 * PA) * (int)sizeof(float);
    static_assert(lds <= 160 * 1024, "LDS");
    static std::atomic<uint64_t> asked{0};
    if (!lds_ask(reinterpret_cast<const void*>(act8_wgrad_kernel<DT, FMT, PA, PC, WN, WC, WK, MODE, DB>), lds, lds, asked)) return Y5M_ELAUNCH;
    hipLaunchKernelGGL((act8_wgrad_kernel<DT, FMT, PA, PC, WN, WC, WK, MODE, DB>), dim3((unsigned)((int64_t)P.tiles_n * P.tiles_c * P.ranges)), dim3(AW_THREADS), lds, st, P);
    Y5M_CHECK_LAUNCH("act8_wgrad_kernel");
    return Y5M_OK;
}
template <int DT, int FMT, int PA, int PC, int WN, int WC, int MODE> static int aw_launch(const AwParams& P, hipStream_t st) {
    return P.dbpart ? aw_launch_db<DT, FMT, PA, PC, WN, WC, MODE, true>(P, st) : aw_launch_db<DT, FMT, PA, PC, WN, WC, MODE, false>(P, st);
}
template <int DT, int FMT> static int aw_small(const AwParams& P, int mode, hipStream_t st) {
    return mode == AW_PIECES ? aw_launch<DT, FMT, 4, 4, 1, 1, AW_PIECES>(P, st) : mode == AW_ROWS ? aw_launch<DT, FMT, 4, 4, 1, 1, AW_ROWS>(P, st)
           : mode == AW_FEW ? aw_launch<DT, FMT, 4, 4, 1, 1, AW_FEW>(P, st) : aw_launch<DT, FMT, 4, 4, 1, 1, AW_ANY>(P, st);
}
template <int FMT> static int aw_dispatch(const AwParams& P, const AwShape& s, int dtype, int mode, hipStream_t st) {
    constexpr int B = Y5M_BF16;
    if (s.pa == 4 && s.pc == 4) return dtype == Y5M_F32 ? aw_small<Y5M_F32, FMT>(P, mode, st) : dtype == Y5M_F16 ? aw_small<Y5M_F16, FMT>(P, mode, st) : aw_small<B, FMT>(P, mode, st);
    if (s.pa == 4) return aw_launch<B, FMT, 4, 8, 1, 1, AW_PIECES>(P, st);
    if (s.wn == 2) return aw_launch<B, FMT, 8, 8, 2, 1, AW_PIECES>(P, st);
    return s.wc == 2 ? aw_launch<B, FMT, 8, 8, 1, 2, AW_PIECES>(P, st) : aw_launch<B, FMT, 8, 8, 1, 1, AW_PIECES>(P, st);
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
    Y5M_REQUIRE(ldq >= C && ldq % 8 == 0 && ldq <= (1 << 26) && ((uintptr_t)q & 7) == 0, "8-bit form: ldq % 8 == 0, at least C, codes 8-byte aligned");
    Y5M_REQUIRE(((uintptr_t)ws & 15) == 0 && ws && ws_bytes >= y5m_act8_wgrad_workspace_bytes(N * S, Cout, C), "workspace too small or not 16-byte aligned");
    // rows of all samples at one distance in whole vector pieces, and a range of them within a buffer resource's 32-bit offsets
    const int64_t pitch = S == 1 && N > 1 ? dy_batch_stride : dy_row_stride;      // (one row per sample: the samples are the rows)
    const bool flat = N == 1 || S == 1 || dy_batch_stride == S * dy_row_stride;
    const bool near = flat && pitch >= 0 && pitch < (1 << 24);
    int mode = near && pitch >= Cout && rows_aligned16(dy, dy_batch_stride, dy_row_stride, N, S, Cout, dtype) ? AW_PIECES : near ? (Cout >= 4 ? AW_ROWS : AW_FEW) : AW_ANY;
    AwParams P = {};
    AwShape s = aw_shape(Cout, C, mode == AW_PIECES && dtype == Y5M_BF16);
    aw_geometry(P, s, N * S, Cout, C);
    if (mode != AW_ANY && (P.per + 4 * AW_K * s.wk) * (pitch > ldq ? pitch : ldq) * (dtype == Y5M_F32 ? 4 : 2) >= (1ll << 31)) {
        mode = AW_ANY;
        s = aw_shape(Cout, C, false);
        aw_geometry(P, s, N * S, Cout, C);
    }
    P.dy = dy; P.dn = dy_batch_stride; P.dr = flat ? pitch : dy_row_stride; P.S = flat ? 0 : S;
    P.q = static_cast<const uint8_t*>(q); P.scale = static_cast<const uint8_t*>(scale); P.ldq = ldq;
    P.part = static_cast<float*>(ws);
    P.dbpart = db ? P.part + (size_t)P.ranges * Cout * C : nullptr;
    P.dw = dw; P.db = db;
    Y5M_REQUIRE((int64_t)P.tiles_n * P.tiles_c * P.ranges < (1ll << 24) && (int64_t)Cout * C * P.slots < (1ll << 31), "too many workgroups");
    const int rc = fmt == Y5M_KEEP_E4M3 ? aw_dispatch<Y5M_KEEP_E4M3>(P, s, dtype, mode, y5m_stream(stream)) : aw_dispatch<Y5M_KEEP_INT8>(P, s, dtype, mode, y5m_stream(stream));
    if (rc != Y5M_OK) return rc;
    const int64_t items = (int64_t)Cout * C + (db ? Cout : 0), per = AW_THREADS / P.slots;
    hipLaunchKernelGGL(act8_wgrad_join_kernel, dim3((unsigned)((items + per - 1) / per)), dim3(AW_THREADS), 0, y5m_stream(stream), P);
    Y5M_CHECK_LAUNCH("act8_wgrad_join_kernel");
    return Y5M_OK;
}

// An activation written in 8 bits with one power-of-two scale per 32 channels of a row, and read back (y5m_act8.h: the form).
// Both are pure streams: bytes are all there is (bf16: 2 read + 1.03 written per element, and the reverse).
// A thread holds 8 channels of a row, four lanes a block; consecutive lanes take consecutive pieces of consecutive rows, so a wave
// reads 1 KB runs where the rows lie densely.
#include "y5m_act8.h"

#define A8_THREADS 256

struct Act8Params {
    const void* x;
    void* y;
    uint8_t* q;
    uint8_t* scale;
    int64_t N, S, sn, sr, M;
    int C, ldq, CB, CV;          // CB = ceil(C / 32) blocks, CV = 4 * CB pieces of 8 channels per row
};

// item = (row, piece); the four pieces of a block sit in lanes 4k .. 4k+3 because CV is a multiple of 4
template <int DT, int FMT, bool AL>
__global__ __launch_bounds__(A8_THREADS) void act8_store_kernel(const Act8Params P) {
    typedef typename RowElem<DT>::T T;
    const int64_t items = P.M * P.CV, step = (int64_t)gridDim.x * A8_THREADS;
    for (int64_t i0 = (int64_t)blockIdx.x * A8_THREADS; i0 < items; i0 += step) {       // (uniform: every lane meets in quad_max)
        const int64_t i = i0 + threadIdx.x;
        const bool in = i < items;
        const int64_t row = in ? i / P.CV : 0;
        const int pc = in ? (int)(i - row * P.CV) : 0, c = pc * 8;
        const int64_t n = row / P.S, s = row - n * P.S;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const bool live = in && c < P.C;
        if (live) load8<DT, AL>(static_cast<const T*>(P.x) + n * P.sn + s * P.sr + c, P.C - c, v);
        unsigned sb;
        const act8_u32x2 q = act8_encode8<FMT, DT>(v, sb);
        if (live) {
            *reinterpret_cast<act8_u32x2*>(P.q + row * P.ldq + c) = q;
            if ((pc & 3) == 0) P.scale[row * P.CB + (pc >> 2)] = (uint8_t)sb;
        }
    }
}

template <int DT, int FMT, bool AL>
__global__ __launch_bounds__(A8_THREADS) void act8_load_kernel(const Act8Params P) {
    typedef typename RowElem<DT>::T T;
    const int64_t items = P.M * P.CV, step = (int64_t)gridDim.x * A8_THREADS;
    for (int64_t i = (int64_t)blockIdx.x * A8_THREADS + threadIdx.x; i < items; i += step) {
        const int64_t row = i / P.CV;
        const int pc = (int)(i - row * P.CV), c = pc * 8;
        if (c >= P.C) continue;
        float v[8];
        act8_decode8<FMT>(*reinterpret_cast<const act8_u32x2*>(P.q + row * P.ldq + c), act8_scale(P.scale[row * P.CB + (pc >> 2)]), v);
        store8<DT, AL>(static_cast<T*>(P.y) + row * P.sr + c, P.C - c, v);
    }
}

static int act8_check(const void* x, const void* q, const void* scale, int64_t N, int64_t S, int C, int ldq, int fmt, int dtype) {
    Y5M_REQUIRE(dtype == Y5M_F32 || dtype == Y5M_BF16 || dtype == Y5M_F16, "dtype");
    Y5M_REQUIRE(fmt == Y5M_KEEP_E4M3 || fmt == Y5M_KEEP_INT8, "8-bit format");
    Y5M_REQUIRE(N >= 0 && S >= 0 && C > 0 && (double)N * (double)S < 1e15, "sizes");
    Y5M_REQUIRE(ldq >= C && ldq % 8 == 0, "ldq must be a multiple of 8, at least C");
    if (N * S > 0) {
        Y5M_REQUIRE(x && q && scale, "null pointer");
        Y5M_REQUIRE(((uintptr_t)q & 7) == 0, "the codes must be 8-byte aligned");
        Y5M_REQUIRE(((uintptr_t)x & (dtype == Y5M_F32 ? 3 : 1)) == 0, "the rows must be aligned to their element");
    }
    return Y5M_OK;
}

static unsigned act8_grid(int64_t items) {
    const int64_t b = (items + A8_THREADS - 1) / A8_THREADS;
    return (unsigned)(b < 8192 ? b : 8192);
}

#define ACT8_DISPATCH(KERN)                                                                                                       \
    do {                                                                                                                          \
        if (dtype == Y5M_F32) ACT8_D2(KERN, Y5M_F32);                                                                             \
        else if (dtype == Y5M_BF16) ACT8_D2(KERN, Y5M_BF16);                                                                      \
        else ACT8_D2(KERN, Y5M_F16);                                                                                              \
    } while (0)
#define ACT8_D2(KERN, DT)                                                                                                         \
    do {                                                                                                                          \
        if (fmt == Y5M_KEEP_E4M3) { if (al) ACT8_GO((KERN<DT, Y5M_KEEP_E4M3, true>)); else ACT8_GO((KERN<DT, Y5M_KEEP_E4M3, false>)); } \
        else { if (al) ACT8_GO((KERN<DT, Y5M_KEEP_INT8, true>)); else ACT8_GO((KERN<DT, Y5M_KEEP_INT8, false>)); }                \
    } while (0)
#define ACT8_GO(K) hipLaunchKernelGGL(K, dim3(act8_grid(P.M * P.CV)), dim3(A8_THREADS), 0, y5m_stream(stream), P)

extern "C" int y5m_act8_store(const void* x, int64_t x_batch_stride, int64_t x_row_stride, int64_t N, int64_t S, int C, void* q, int ldq,
                              void* scale, int fmt, int dtype, void* stream) {
    const int rc = act8_check(x, q, scale, N, S, C, ldq, fmt, dtype);
    if (rc != Y5M_OK) return rc;
    if (N * S == 0) return Y5M_OK;
    Act8Params P = {};
    P.x = x; P.q = static_cast<uint8_t*>(q); P.scale = static_cast<uint8_t*>(scale);
    P.N = N; P.S = S; P.sn = x_batch_stride; P.sr = x_row_stride; P.M = N * S;
    P.C = C; P.ldq = ldq; P.CB = (C + 31) / 32; P.CV = 4 * P.CB;
    const bool al = rows_aligned16(x, x_batch_stride, x_row_stride, N, S, C, dtype);
    ACT8_DISPATCH(act8_store_kernel);
    Y5M_CHECK_LAUNCH("act8_store_kernel");
    return Y5M_OK;
}

extern "C" int y5m_act8_load(const void* q, int ldq, const void* scale, int64_t M, int C, void* x, int64_t x_row_stride, int fmt, int dtype,
                             void* stream) {
    const int rc = act8_check(x, q, scale, 1, M, C, ldq, fmt, dtype);
    if (rc != Y5M_OK) return rc;
    if (M == 0) return Y5M_OK;
    Y5M_REQUIRE(M == 1 || x_row_stride >= C, "rows of the output overlap");
    Act8Params P = {};
    P.y = x; P.q = static_cast<uint8_t*>(const_cast<void*>(q)); P.scale = static_cast<uint8_t*>(const_cast<void*>(scale));
    P.N = 1; P.S = M; P.sr = x_row_stride; P.M = M;
    P.C = C; P.ldq = ldq; P.CB = (C + 31) / 32; P.CV = 4 * P.CB;
    const bool al = rows_aligned16(x, 0, x_row_stride, 1, M, C, dtype);
    ACT8_DISPATCH(act8_load_kernel);
    Y5M_CHECK_LAUNCH("act8_load_kernel");
    return Y5M_OK;
}

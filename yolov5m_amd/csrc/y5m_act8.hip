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
    int C, ldq, CB, CV, RP, rpc;         // CB = ceil(C / 32) blocks, CV = 4 * CB pieces of 8 channels per row (at most 256 side by side), rows
    int ct, tiles;                       // side by side and per workgroup
};
// A workgroup takes rpc consecutive rows of a column tile; a thread one piece of every RP-th of them, four in flight. (Short workgroups
// that end: a grid that strides over the whole tensor reads at 4.3 to 5.3 TB/s here, these at 6; and no division per piece.)
struct Act8Place { int64_t row, end; int pc, c, lr; bool in; };
__device__ __forceinline__ Act8Place act8_place(const Act8Params& P) {
    Act8Place w;
    const int tile = P.tiles > 1 ? (int)(blockIdx.x % (unsigned)P.tiles) : 0;
    const int64_t chunk = P.tiles > 1 ? blockIdx.x / (unsigned)P.tiles : blockIdx.x;
    w.lr = (int)threadIdx.x / P.ct;
    w.pc = tile * P.ct + ((int)threadIdx.x - w.lr * P.ct);
    w.c = w.pc * 8;
    w.in = w.lr < P.RP && w.c < P.C;
    w.row = chunk * P.rpc;
    w.end = w.row + P.rpc < P.M ? w.row + P.rpc : P.M;
    return w;
}

// the four pieces of a block sit in lanes 4k .. 4k+3 because ct is a multiple of 4
template <int DT, int FMT, int AL>
__global__ __launch_bounds__(A8_THREADS) void act8_store_kernel(const Act8Params P) {
    typedef typename RowElem<DT>::T T;
    const Act8Place w = act8_place(P);
    // every lane runs the same trips and meets in the encoder: pieces and rows beyond the end are read from the first and the last instead
    const int c = w.in ? w.c : 0, nv = P.C - c, lr = w.lr < P.RP ? w.lr : 0;
    const T* x = static_cast<const T*>(P.x) + c;
    for (int64_t r0 = w.row; r0 < w.end; r0 += 4 * P.RP) {
        Raw8<DT> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            int64_t r = r0 + lr + u * P.RP;
            if (r >= w.end) r = w.end - 1;
            const int64_t n = P.S ? r / P.S : 0;                   // (S = 0: one distance throughout)
            raw[u] = load_raw8<DT, AL>(x + n * P.sn + (r - n * P.S) * P.sr, nv);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t r = r0 + lr + u * P.RP;
            float v[8];
            unpack8<DT>(raw[u], v);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = w.in ? v[k] : 0.f;
            unsigned sb;
            const act8_u32x2 q = act8_encode8<FMT, DT>(v, sb);
            if (w.in && r < w.end) {
                *reinterpret_cast<act8_u32x2*>(P.q + r * P.ldq + w.c) = q;
                if ((w.pc & 3) == 0) P.scale[r * P.CB + (w.pc >> 2)] = (uint8_t)sb;
            }
        }
    }
}

template <int DT, int FMT, int AL>
__global__ __launch_bounds__(A8_THREADS) void act8_load_kernel(const Act8Params P) {
    typedef typename RowElem<DT>::T T;
    const Act8Place w = act8_place(P);
    if (!w.in) return;
    for (int64_t r0 = w.row + w.lr; r0 < w.end; r0 += 4 * P.RP) {
        act8_u32x2 q[4];
        unsigned s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t r = r0 + u * P.RP < w.end ? r0 + u * P.RP : w.end - 1;
            q[u] = *reinterpret_cast<const act8_u32x2*>(P.q + r * P.ldq + w.c);
            s[u] = P.scale[r * P.CB + (w.pc >> 2)];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t r = r0 + u * P.RP;
            if (r >= w.end) break;
            float v[8];
            act8_decode8<FMT>(q[u], act8_scale(s[u]), v);
            store8<DT, AL>(static_cast<T*>(P.y) + r * P.sr + w.c, P.C - w.c, v);
        }
    }
}

static int act8_check(const void* x, const void* q, const void* scale, int64_t N, int64_t S, int C, int ldq, int fmt, int dtype) {
    Y5M_REQUIRE(dtype == Y5M_F32 || dtype == Y5M_BF16 || dtype == Y5M_F16, "dtype");
    Y5M_REQUIRE(fmt == Y5M_KEEP_E4M3 || fmt == Y5M_KEEP_INT8, "8-bit format");
    Y5M_REQUIRE(N >= 0 && S >= 0 && C > 0 && (double)N * (double)S < 1e12, "sizes");
    Y5M_REQUIRE(ldq >= C && ldq % 8 == 0, "ldq must be a multiple of 8, at least C");
    if (N * S > 0) {
        Y5M_REQUIRE(x && q && scale, "null pointer");
        Y5M_REQUIRE(((uintptr_t)q & 7) == 0, "the codes must be 8-byte aligned");
        Y5M_REQUIRE(((uintptr_t)x & (dtype == Y5M_F32 ? 3 : 1)) == 0, "the rows must be aligned to their element");
    }
    return Y5M_OK;
}

static void act8_geometry(Act8Params& P) {
    P.CB = (P.C + 31) / 32;
    P.CV = 4 * P.CB;
    P.tiles = (P.CV + A8_THREADS - 1) / A8_THREADS;
    P.ct = ((P.CV + P.tiles - 1) / P.tiles + 3) / 4 * 4;
    P.RP = A8_THREADS / P.ct;
    // 8 rows a thread; more where the grid would not fit
    int64_t rpc = (int64_t)P.RP * 8;
    while ((P.M + rpc - 1) / rpc * P.tiles >= (1ll << 24)) rpc *= 2;
    P.rpc = (int)rpc;
}

// NT: the kernel's AL for a call that stores rows past the caches
#define ACT8_DISPATCH(KERN, NT)                                                                                                   \
    do {                                                                                                                          \
        if (dtype == Y5M_F32) ACT8_D2(KERN, Y5M_F32, NT);                                                                         \
        else if (dtype == Y5M_BF16) ACT8_D2(KERN, Y5M_BF16, NT);                                                                  \
        else ACT8_D2(KERN, Y5M_F16, NT);                                                                                          \
    } while (0)
#define ACT8_D2(KERN, DT, NT)                                                                                                     \
    do {                                                                                                                          \
        if (fmt == Y5M_KEEP_E4M3) ACT8_D3(KERN, DT, Y5M_KEEP_E4M3, NT);                                                           \
        else ACT8_D3(KERN, DT, Y5M_KEEP_INT8, NT);                                                                                \
    } while (0)
#define ACT8_D3(KERN, DT, FMT, NT)                                                                                                \
    do {                                                                                                                          \
        if (al < 0) ACT8_GO((KERN<DT, FMT, -1>));                                                                                 \
        else if (al == 0) ACT8_GO((KERN<DT, FMT, 0>));                                                                            \
        else if (nt) ACT8_GO((KERN<DT, FMT, NT>));                                                                                \
        else ACT8_GO((KERN<DT, FMT, 1>));                                                                                         \
    } while (0)
#define ACT8_GO(K) hipLaunchKernelGGL(K, dim3((unsigned)((P.M + P.rpc - 1) / P.rpc * P.tiles)), dim3(A8_THREADS), 0, y5m_stream(stream), P)

extern "C" int y5m_act8_store(const void* x, int64_t x_batch_stride, int64_t x_row_stride, int64_t N, int64_t S, int C, void* q, int ldq,
                              void* scale, int fmt, int dtype, void* stream) {
    const int rc = act8_check(x, q, scale, N, S, C, ldq, fmt, dtype);
    if (rc != Y5M_OK) return rc;
    if (N * S == 0) return Y5M_OK;
    Act8Params P = {};
    P.x = x; P.q = static_cast<uint8_t*>(q); P.scale = static_cast<uint8_t*>(scale);
    P.N = N; P.S = S; P.sn = x_batch_stride; P.sr = x_row_stride; P.M = N * S;
    P.C = C; P.ldq = ldq;
    act8_geometry(P);
    if (N == 1 || S == 1 || x_batch_stride == S * x_row_stride) {
        if (S == 1 && N > 1) P.sr = x_batch_stride;
        P.S = 0;
    }
    const int al = rows_mode(rows_aligned16(x, x_batch_stride, x_row_stride, N, S, C, dtype), C);
    const bool nt = false;
    ACT8_DISPATCH(act8_store_kernel, 1);
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
    P.C = C; P.ldq = ldq;
    const bool nt = rows_past_caches(M, C, dtype);
    act8_geometry(P);
    const int al = rows_mode(rows_aligned16(x, 0, x_row_stride, 1, M, C, dtype), C);
    ACT8_DISPATCH(act8_load_kernel, 2);
    Y5M_CHECK_LAUNCH("act8_load_kernel");
    return Y5M_OK;
}

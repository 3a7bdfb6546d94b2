// Channels-last rows in f32 / bf16 / fp16 and the 8-bit kept form of an activation: what y5m_act8*.hip and y5m_gn.hip share.
//
// The 8-bit form. A row of C channels is cut into blocks of 32 (the last may be shorter). One block has one scale 2^e, stored as the
// byte e + 127, and 32 codes:  e = the smallest integer with max|x| <= TOP * 2^e, at least -117;  code = rne(x * 2^-e), an e4m3
// value (TOP 448) or an int8 (TOP 127). Why a power of two: x * 2^-e is exact, so the only rounding is the one to the code, the
// result does not depend on the order or the unit that computes it, and code * 2^e is exact in f32 and bf16 (at most 8 significant
// bits) -- the weight gradient feeds it to bf16 MFMAs without another rounding. It costs up to one bit of an int8 against a scale of
// max / 127. Why 32 channels of one row: four lanes that hold 8 channels each, so the block maximum is two DPP steps, and 3 % extra
// bytes. e >= -117 keeps the smallest code (2^-9 * 2^-117) a normal f32. x is limited to 15/8 * 2^E first (E: the type's largest
// exponent): the largest values round to a code that stays finite when read back. A block holding a NaN or an infinity gets scale
// byte 255 and reads back as NaN throughout: an overflow in a training step must reach the gradients, and int8 has no NaN code.
#pragma once
#include <atomic>
#include "y5m_common.h"

typedef _Float16 y5m_f16;
typedef unsigned act8_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned act8_u32x2 __attribute__((ext_vector_type(2)));

template <int DT> struct RowElem { typedef uint16_t T; };
template <> struct RowElem<Y5M_F32> { typedef float T; };

// 8 consecutive channels of a row as they lie in memory (16 bytes, f32: 32)
template <int DT> struct Raw8 { act8_u32x4 r[DT == Y5M_F32 ? 2 : 1]; };

__device__ __forceinline__ float f16_to_f32(uint16_t h) { return (float)__builtin_bit_cast(y5m_f16, h); }
__device__ __forceinline__ uint16_t f32_to_f16(float f) { return __builtin_bit_cast(uint16_t, (y5m_f16)f); }

// AL = 1: 16-byte pieces (the launcher checks base, strides and C).
// AL = 0: pieces that start at any element, C >= 8. A row's last piece (nv < 8) is read as the 8 elements that END with the row and
// shifted down, zeros behind: every lane does the same, so the loads of an unrolled loop stay in flight together (a branch for the
// short piece makes each load wait for the one before: 12 rows held in registers took 21 us of such waits).
// AL = -1: C < 8, element by element; elements beyond the row are read as its last one and zeroed.
template <int DT, int AL>
__device__ __forceinline__ Raw8<DT> load_raw8(const typename RowElem<DT>::T* __restrict__ p, int nv) {
    Raw8<DT> w;
    if constexpr (AL > 0) {
        w.r[0] = *reinterpret_cast<const act8_u32x4*>(p);
        if constexpr (DT == Y5M_F32) w.r[1] = *reinterpret_cast<const act8_u32x4*>(p + 4);
    } else if constexpr (AL == 0) {
        const int sh = nv < 8 ? 8 - nv : 0;
        __builtin_memcpy(&w, p - sh, sizeof(w));
        if constexpr (DT == Y5M_F32) {
            unsigned v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = w.r[k >> 2][k & 3];
#pragma unroll
            for (int s = 4; s > 0; s >>= 1)
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = (sh & s) ? (k + s < 8 ? v[k + s < 8 ? k + s : 0] : 0u) : v[k];
#pragma unroll
            for (int k = 0; k < 8; ++k) w.r[k >> 2][k & 3] = v[k];
        } else {
            unsigned v[5] = {w.r[0][0], w.r[0][1], w.r[0][2], w.r[0][3], 0u};
#pragma unroll
            for (int s = 4; s > 1; s >>= 1)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = (sh & s) ? (k + s / 2 < 4 ? v[k + s / 2 < 4 ? k + s / 2 : 0] : 0u) : v[k];
#pragma unroll
            for (int k = 0; k < 4; ++k) w.r[0][k] = (sh & 1) ? (v[k] >> 16) | (v[k + 1] << 16) : v[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const typename RowElem<DT>::T e = p[k < nv ? k : nv - 1];
            if constexpr (DT == Y5M_F32) {
                w.r[k >> 2][k & 3] = k < nv ? __float_as_uint(e) : 0u;
            } else {
                const unsigned x = k < nv ? (unsigned)e : 0u;
                if (k & 1) w.r[0][k >> 1] |= x << 16;
                else w.r[0][k >> 1] = x;
            }
        }
    }
    return w;
}
template <int DT> __device__ __forceinline__ void unpack8(const Raw8<DT>& w, float v[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if constexpr (DT == Y5M_F32) v[k] = __uint_as_float(w.r[k >> 2][k & 3]);
        else if constexpr (DT == Y5M_BF16) v[k] = __uint_as_float((k & 1) ? (w.r[0][k >> 1] & 0xffff0000u) : (w.r[0][k >> 1] << 16));
        else v[k] = f16_to_f32((uint16_t)(w.r[0][k >> 1] >> (16 * (k & 1))));
    }
}
template <int DT, int AL>
__device__ __forceinline__ void load8(const typename RowElem<DT>::T* __restrict__ p, int nv, float v[8]) {
    unpack8<DT>(load_raw8<DT, AL>(p, nv), v);
}
// AL = 2: 16-byte pieces stored past the caches. For outputs too large to be read back from the memory-side cache by whoever comes next: stored there
// they would only push out the rows that this operator reads twice, or whose rest is still to be read
template <int DT, int AL>
__device__ __forceinline__ void store8(typename RowElem<DT>::T* __restrict__ p, int nv, const float v[8]) {
    Raw8<DT> w;
    if constexpr (DT == Y5M_F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) w.r[k >> 2][k & 3] = __float_as_uint(v[k]);
    } else if constexpr (DT == Y5M_BF16) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w.r[0][k] = f32x2_to_bf16x2(v[2 * k], v[2 * k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) w.r[0][k] = (unsigned)f32_to_f16(v[2 * k]) | ((unsigned)f32_to_f16(v[2 * k + 1]) << 16);
    }
    if constexpr (AL > 0) {
        act8_u32x4* q = reinterpret_cast<act8_u32x4*>(p);
#pragma unroll
        for (int h = 0; h < (DT == Y5M_F32 ? 2 : 1); ++h) {
            if constexpr (AL == 2) __builtin_nontemporal_store(w.r[h], q + h);
            else q[h] = w.r[h];
        }
    } else if (nv >= 8) {
        __builtin_memcpy(p, &w, sizeof(w));
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < nv) {
                if constexpr (DT == Y5M_F32) p[k] = v[k];
                else p[k] = (uint16_t)(w.r[0][k >> 1] >> (16 * (k & 1)));
            }
    }
}
// host: does an output of this size go past the caches? (256 MB memory-side cache; 64 x 80 x 80 x 192 in bf16, a forward and backward
// whose outputs are 157 MB each: 226 us with, 257 without; at 79 MB 125 against 134)
static inline bool rows_past_caches(int64_t rows, int C, int dtype) { return rows * C * (dtype == Y5M_F32 ? 4 : 2) > (64ll << 20); }

// ---- the 8-bit form ---------------------------------------------------------------------------------------------------------
template <int DT> __device__ __forceinline__ float act8_limit() {
    return DT == Y5M_F16 ? 61440.0f : __uint_as_float(0x7f700000u);          // 15/8 * 2^15, 15/8 * 2^127
}
// maximum over the four lanes 4k .. 4k+3 that hold one block (quad_perm DPP: no LDS)
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
    v = v > o ? v : o;
    o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);
    return v > o ? v : o;
}
// scale byte of a block from the bits of its largest |x| (>= 0x7f800000: a value that is not finite). Adding the distance of TOP's
// mantissa from the next binade carries into the exponent exactly when the mantissa is above TOP's: 448 = 1.75 * 2^8 (0x600000),
// 127 = 1.984375 * 2^6 (0x7e0000)
template <int FMT, int DT> __device__ __forceinline__ unsigned act8_scale_byte(unsigned amax) {
    const unsigned lim = __float_as_uint(act8_limit<DT>());
    const unsigned a = amax < lim ? amax : lim;
    const unsigned ex = (a + (FMT == Y5M_KEEP_E4M3 ? 0x1fffffu : 0x1ffffu)) >> 23;
    const unsigned sub = FMT == Y5M_KEEP_E4M3 ? 8u : 6u;
    const unsigned b = ex > sub + 10u ? ex - sub : 10u;
    return amax >= 0x7f800000u ? 255u : b;
}
// codes of 8 channels (this lane's quarter of the block); every lane of the quad calls it
template <int FMT, int DT> __device__ __forceinline__ act8_u32x2 act8_encode8(const float v[8], unsigned& sbyte) {
    unsigned a = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const unsigned u = __float_as_uint(v[k]) & 0x7fffffffu;
        a = a > u ? a : u;
    }
    a = quad_max(a);
    sbyte = act8_scale_byte<FMT, DT>(a);
    // 2^-e = bits (254 - byte) << 23; a block that is not finite is multiplied by 0 and its NaNs dropped: codes 0, scale 255
    const float inv = __uint_as_float(sbyte == 255u ? 0u : (254u - sbyte) << 23);
    const float lim = act8_limit<DT>();
    float t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = fminf(fmaxf(v[k], -lim), lim) * inv;
    act8_u32x2 q;
    if constexpr (FMT == Y5M_KEEP_E4M3) {
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[4], t[5], 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[6], t[7], hi, true);
        q[0] = (unsigned)lo;
        q[1] = (unsigned)hi;
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            unsigned w = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) w |= ((unsigned)(int)rintf(t[4 * h + k]) & 0xffu) << (8 * k);
            q[h] = w;
        }
    }
    return q;
}
__device__ __forceinline__ float act8_scale(unsigned sbyte) {
    return __uint_as_float(sbyte == 255u ? 0x7fc00000u : sbyte << 23);
}
template <int FMT> __device__ __forceinline__ void act8_decode8(act8_u32x2 q, float scale, float v[8]) {
    if constexpr (FMT == Y5M_KEEP_E4M3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const y5m_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
            v[4 * h] = a[0] * scale;
            v[4 * h + 1] = a[1] * scale;
            v[4 * h + 2] = b[0] * scale;
            v[4 * h + 3] = b[1] * scale;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)(int8_t)(q[k >> 2] >> (8 * (k & 3))) * scale;
    }
}

// host: the AL of kernels for these rows
static inline int rows_mode(bool aligned, int C) { return aligned ? 1 : C >= 8 ? 0 : -1; }
// host: may rows at p (batch stride sn, row stride sr, in elements) be read in 16-byte pieces?
static inline bool rows_aligned16(const void* p, int64_t sn, int64_t sr, int64_t N, int64_t S, int C, int dtype) {
    const int per = dtype == Y5M_F32 ? 4 : 8;
    return ((uintptr_t)p & 15) == 0 && C % 8 == 0 && (S <= 1 || sr % per == 0) && (N <= 1 || sn % per == 0);
}
// host: dynamic LDS above 64 KB has to be asked for, per kernel and device; `asked`: one bit for each of the first 64 devices
static inline bool lds_ask(const void* kernel, int need, int most, std::atomic<uint64_t>& asked) {
    if (need <= 64 * 1024) return true;
    int dev = 64;
    (void)hipGetDevice(&dev);
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (asked.load(std::memory_order_relaxed) & bit) return true;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, most) != hipSuccess) {
        (void)hipGetLastError();
        y5m_set_error("%d bytes of LDS refused", most);
        return false;
    }
    asked.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

// int8_store.h -- the end of the 8-bit products' kernels: sums to scaled
// results, and where a tile of them stands.
#pragma once

#include "common.h"
#include "int8.h"

namespace terhip {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <int C>
using Words = unsigned int __attribute__((ext_vector_type(C / 2)));

// C (4 or 8) scaled sums in 16 bits.
template <int YT, int C>
__device__ __forceinline__ Words<C> words_of(const int (&sum)[C], float xs, const float (&ws)[C]) {
#pragma clang fp contract(off)
    Words<C> o;
#pragma unroll
    for (int i = 0; i < C; i += 2) {
        unsigned w = 0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float f = (float)sum[i + k] * (xs * ws[i + k]);
            w |= (unsigned)(YT == TER_HIP_T_F16 ? float_to_half_bits(f) : __builtin_bit_cast(uint16_t, (__bf16)f)) << (16 * k);
        }
        o[i / 2] = w;
    }
    return o;
}

// C results of 16 bits from element `at` of y on, `left` of which exist.
template <int C>
__device__ __forceinline__ void store_words(char* y, long long at, int left, Words<C> o, bool wide) {
    TER_GLOBAL uint16_t* p = gptr(reinterpret_cast<uint16_t*>(y)) + at;
    if (wide && left >= C) {
        *reinterpret_cast<TER_GLOBAL Words<C>*>(p) = o;
    } else {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (i < left) p[i] = (uint16_t)(o[i / 2] >> (16 * (i & 1)));
    }
}

// Scaled results of C (4 or 8) consecutive channels of one token, `left` of
// which exist.  wide: groups of 8 are 16-byte aligned in y.
template <int YT, int C>
__device__ __forceinline__ void store_run(char* y, long long at, int left, const int (&sum)[C], float xs,
                                          const float (&ws)[C], bool wide) {
#pragma clang fp contract(off)
    if constexpr (YT == TER_HIP_T_I32 || YT == TER_HIP_T_F32) {
        unsigned v[C];
#pragma unroll
        for (int i = 0; i < C; ++i)
            v[i] = YT == TER_HIP_T_I32 ? (unsigned)sum[i] : __builtin_bit_cast(unsigned, (float)sum[i] * (xs * ws[i]));
        TER_GLOBAL unsigned* p = gptr(reinterpret_cast<unsigned*>(y)) + at;
        if (wide && left >= C) {
#pragma unroll
            for (int i = 0; i < C; i += 4)
                *reinterpret_cast<TER_GLOBAL u32x4*>(p + i) = u32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (i < left) p[i] = v[i];
        }
    } else {
        store_words<C>(y, at, left, words_of<YT, C>(sum, xs, ws), wide);
    }
}

__device__ __forceinline__ bool wide_rows(const Int8MmArgs& a) {
    return a.ldy % 8 == 0 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0;
}

// A wave's sums: MB blocks of 16 rows from m0 on, S strips (an even number)
// from channel n0 on (a multiple of 32).
template <int MB, int S, int YT>
__device__ __forceinline__ void store_tile(const Int8MmArgs& a, int m0, int n0, const i32x4 (&acc)[MB][S], int lane) {
    const int j = lane & 15, g = lane >> 4;
    const bool wide = wide_rows(a);
#pragma unroll
    for (int p = 0; p < S / 2; ++p) {
        const int n = n0 + 32 * p + 8 * g;
        if (n >= a.N) continue;
        float ws[8];
        if constexpr (YT != TER_HIP_T_I32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) ws[i] = gptr(a.ws)[n + i];
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int m = m0 + 16 * i + j;
            if (m >= a.M) continue;
            const i32x4 u = acc[i][2 * p], v = acc[i][2 * p + 1];
            const int sum[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
            store_run<YT, 8>(a.y, (long long)m * a.ldy + n, a.N - n, sum, YT == TER_HIP_T_I32 ? 0.f : gptr(a.xs)[m], ws, wide);
        }
    }
}

// The tile of a workgroup.  Workgroups go to the 8 XCDs in turn, so those of one
// XCD take a run of tiles, by groups of 4 rows of tiles: the ones that run at
// a time on an XCD share their operands in its L2.
__device__ __forceinline__ void tile_of(int id, int mt, int nt, int& tm, int& tn) {
    const int total = mt * nt, per = total / 8, rest = total % 8;
    const int x = id % 8, k = id / 8;
    const int t = x * per + (x < rest ? x : rest) + k;
    const int group = t / (4 * nt), in = t - group * 4 * nt;
    const int height = mt - group * 4 < 4 ? mt - group * 4 : 4;
    tm = group * 4 + in % height;
    tn = in / height;
}

}  // namespace terhip

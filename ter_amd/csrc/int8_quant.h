// int8_quant.h -- the steps from a row to 8 bits (include/ter_hip_int8.h), for the
// kernels that take them.
#pragma once

#include "common.h"
#include "int8.h"

namespace terhip {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

template <int TYPE>
struct Elem;
template <>
struct Elem<TER_HIP_T_F16> {
    typedef uint16_t T;
    static __device__ float get(T v) { return half_bits_to_float(v); }
};
template <>
struct Elem<TER_HIP_T_BF16> {
    typedef uint16_t T;
    static __device__ float get(T v) { return __builtin_bit_cast(float, (unsigned)v << 16); }
};
template <>
struct Elem<TER_HIP_T_F32> {
    typedef float T;
    static __device__ float get(T v) { return v; }
};

struct Quant {
    float s, inv;
};

// The steps of quant_rows_kernel (pack.hip), binary32, each rounded.
__device__ __forceinline__ Quant quant_of(unsigned amax_bits) {
#pragma clang fp contract(off)
    Quant q;
    q.s = 127.0f / (__builtin_bit_cast(float, amax_bits) + 1e-9f);
    q.inv = 1.0f / q.s;
    if (amax_bits >= 0x7F800000u) {  // an infinity or NaN in the row
        q.s = 0.f;
        q.inv = __builtin_nanf("");
    }
    return q;
}

__device__ __forceinline__ int quantize(float v, float s) {
#pragma clang fp contract(off)
    return (int)__builtin_fminf(__builtin_fmaxf(__builtin_rintf(v * s), -128.f), 127.f);  // (of NaN -128)
}

// Elements k .. k + 7 of a row of K (zeros behind it).  vec: rows are 16-byte
// aligned.
template <int TYPE>
__device__ __forceinline__ void row8(const TER_GLOBAL typename Elem<TYPE>::T* row, int k, int K, bool vec, float (&v)[8]) {
    typedef typename Elem<TYPE>::T E;
    constexpr int PER = 16 / (int)sizeof(E);
    if (vec && k + 8 <= K) {
#pragma unroll
        for (int h = 0; h < 8 / PER; ++h) {
            const u32x4 w = *reinterpret_cast<const TER_GLOBAL u32x4*>(row + k + h * PER);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const unsigned d = w[e * (int)sizeof(E) / 4];
                if constexpr (sizeof(E) == 4)
                    v[h * PER + e] = Elem<TYPE>::get(__builtin_bit_cast(float, d));
                else
                    v[h * PER + e] = Elem<TYPE>::get((uint16_t)(d >> (16 * (e & 1))));
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < K ? Elem<TYPE>::get(row[k + e]) : 0.f;
    }
}

__device__ __forceinline__ u32x2 quantize8(const float (&v)[8], float s) {
    u32x2 d = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e >> 2] |= ((unsigned)quantize(v[e], s) & 255u) << (8 * (e & 3));
    return d;
}

}  // namespace terhip

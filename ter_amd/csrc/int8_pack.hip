// int8_pack.hip -- weights in 8 bits to and from the tiles of int8.h, and the
// rows of a product in 8 bits: quantized by their largest magnitude, or
// integers laid out at 16-byte alignment.
//
// Quantizing is by one workgroup a row.  Weights, and rows of more than 16384
// values, are read twice (their largest magnitude, then their values).
//
// Measured: 1021 x 2048 bf16 rows 3.3 to 5 us, 96 x 2560 fp16 3.8 to 5 and 23 x
// 6912 bf16 3.7, all of it the launch and two trips to memory; 8000 x 6911
// integers at odd addresses 19 us, 5.7 TB/s read and written.  Once for a weight, at
// 128256 x 2560: integers to tiles 243 us, 2.7 TB/s; fp16 or bf16 quantized 1020 and
// fp32 1364, 1.0 and 1.2 TB/s, of elements read one by one and twice; back to integers
// 762, one byte a thread.
#include "common.h"
#include "int8.h"
#include "int8_quant.h"

namespace terhip {
namespace {

// The largest magnitude of a workgroup's values as bits (an infinity or NaN is
// larger than any number), to every thread.
__device__ unsigned block_max(unsigned v, unsigned* red) {
    for (int s = 32; s; s >>= 1) {
        const unsigned o = (unsigned)__shfl_xor((int)v, s);
        v = o > v ? o : v;
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < (int)(blockDim.x >> 6); ++i) v = red[i] > v ? red[i] : v;
    __syncthreads();
    return v;
}

// Largest magnitude of row `row` of K elements.
template <int TYPE>
__device__ unsigned row_amax(const typename Elem<TYPE>::T* row, int K, unsigned* red) {
    unsigned m = 0;
    for (int k = threadIdx.x; k < K; k += blockDim.x) {
        const unsigned b = __builtin_bit_cast(unsigned, Elem<TYPE>::get(gptr(row)[k])) & 0x7FFFFFFFu;
        m = b > m ? b : m;
    }
    return block_max(m, red);
}

// One workgroup of T threads a row, held in registers: 8 NC values a thread,
// read once.  VEC: rows are 16-byte aligned.
template <int TYPE, int T, int NC, bool VEC>
__global__ __launch_bounds__(T) void rows8_quant_kernel(const void* __restrict__ x, long long stride, int K,
                                                        int8_t* __restrict__ q, long long ldq,
                                                        float* __restrict__ scale) {
    typedef typename Elem<TYPE>::T E;
    __shared__ unsigned red[T / 64];
    const TER_GLOBAL E* row = gptr(static_cast<const E*>(x) + (long long)blockIdx.x * stride);
    float v[NC][8];
    unsigned m = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        row8<TYPE>(row, 8 * (threadIdx.x + T * c), K, VEC, v[c]);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned b = __builtin_bit_cast(unsigned, v[c][e]) & 0x7FFFFFFFu;
            m = b > m ? b : m;
        }
    const Quant z = quant_of(block_max(m, red));
    if (threadIdx.x == 0) gptr(scale)[blockIdx.x] = z.inv;
    TER_GLOBAL int8_t* out = gptr(q) + (long long)blockIdx.x * ldq;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int k = 8 * (threadIdx.x + T * c);
        if (k >= ldq) continue;  // (zeros up to ldq, a multiple of 8)
        *reinterpret_cast<TER_GLOBAL u32x2*>(out + k) = quantize8(v[c], z.s);
    }
}

// The same for rows of any length, read twice.
template <int TYPE>
__global__ __launch_bounds__(256) void rows8_long_kernel(const void* __restrict__ x, long long stride, int K,
                                                         int8_t* __restrict__ q, long long ldq,
                                                         float* __restrict__ scale) {
    typedef typename Elem<TYPE>::T T;
    __shared__ unsigned red[4];
    const T* row = static_cast<const T*>(x) + (long long)blockIdx.x * stride;
    const Quant z = quant_of(row_amax<TYPE>(row, K, red));
    if (threadIdx.x == 0) gptr(scale)[blockIdx.x] = z.inv;
    int8_t* out = q + (long long)blockIdx.x * ldq;
    for (int k = threadIdx.x * 4; k < ldq; k += 1024) {
        unsigned v = 0;
        for (int i = 0; i < 4; ++i)
            if (k + i < K) v |= ((unsigned)quantize(Elem<TYPE>::get(gptr(row)[k + i]), z.s) & 255u) << (8 * i);
        *reinterpret_cast<TER_GLOBAL unsigned*>(gptr(out) + k) = v;
    }
}

// Integer rows at any alignment to aligned ones, 16 bytes a thread, from the aligned
// words that hold them where those lie within the row.
__global__ __launch_bounds__(256) void rows8_copy_kernel(const int8_t* __restrict__ x, long long stride, int K,
                                                         int8_t* __restrict__ q, long long ldq, int chunks,
                                                         long long total) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += 256ll * gridDim.x) {
        const long long m = i / chunks;
        const int k0 = (int)(i - m * chunks) * 16;
        const int8_t* row = x + m * stride;
        const int off = (int)(reinterpret_cast<uintptr_t>(row + k0) & 3);
        u32x4 v;
        if (k0 >= off && k0 - off + 20 <= K) {
            const TER_GLOBAL unsigned* w = reinterpret_cast<const TER_GLOBAL unsigned*>(gptr(row) + (k0 - off));
            const unsigned d[5] = {w[0], w[1], w[2], w[3], w[4]};
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __builtin_amdgcn_alignbyte(d[j + 1], d[j], (unsigned)off);
        } else {
            for (int j = 0; j < 4; ++j) {
                unsigned e = 0;
                for (int b = 0; b < 4; ++b) {
                    const int k = k0 + 4 * j + b;
                    if (k < K) e |= (unsigned)(uint8_t)gptr(row)[k] << (8 * b);
                }
                v[j] = e;
            }
        }
        *reinterpret_cast<TER_GLOBAL u32x4*>(gptr(q) + m * ldq + k0) = v;
    }
}

// Chunk c (16 values of K) of channel n within the tiles.
__device__ __forceinline__ long long chunk_at(int n, int c, int Ku) {
    const int strip = 2 * (n >> 5) + ((n >> 2) & 1), row = 4 * ((n >> 3) & 3) + (n & 3);
    return ((long long)strip * (2 * Ku) + (c >> 2)) * 1024 + ((c & 3) * 16 + row) * 16;
}

// One workgroup a channel (those that pad the last strip are zero).
template <int TYPE>
__global__ __launch_bounds__(256) void w8_quantize_kernel(const void* __restrict__ src, long long stride, int K, int N,
                                                          int Ku, uint8_t* __restrict__ tiles,
                                                          float* __restrict__ scale) {
    typedef typename Elem<TYPE>::T T;
    __shared__ unsigned red[4];
    const int n = blockIdx.x;
    const T* row = static_cast<const T*>(src) + (long long)(n < N ? n : 0) * stride;
    Quant z{};
    if (n < N) z = quant_of(row_amax<TYPE>(row, K, red));  // (by workgroups)
    if (threadIdx.x == 0) gptr(scale)[n] = z.inv;
    for (int c = threadIdx.x; c < 8 * Ku; c += 256) {
        u32x4 v;
        for (int j = 0; j < 4; ++j) {
            unsigned d = 0;
            for (int b = 0; b < 4; ++b) {
                const int k = c * 16 + 4 * j + b;
                if (n < N && k < K) d |= ((unsigned)quantize(Elem<TYPE>::get(gptr(row)[k]), z.s) & 255u) << (8 * b);
            }
            v[j] = d;
        }
        *reinterpret_cast<TER_GLOBAL u32x4*>(gptr(tiles) + chunk_at(n, c, Ku)) = v;
    }
}

// One thread a chunk.
__global__ __launch_bounds__(256) void w8_pack_kernel(const int8_t* __restrict__ q, long long stride,
                                                      const float* __restrict__ src_scale, int K, int N, int Ku,
                                                      uint8_t* __restrict__ tiles, float* __restrict__ scale,
                                                      bool vec, long long total) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += 256ll * gridDim.x) {
        const int n = (int)(i / (8 * Ku)), c = (int)(i % (8 * Ku));
        if (c == 0) gptr(scale)[n] = n < N ? gptr(src_scale)[n] : 0.f;
        const int8_t* row = q + (long long)n * stride;
        u32x4 v = {};
        if (n >= N || c * 16 >= K) {
        } else if (vec && c * 16 + 16 <= K) {
            v = *reinterpret_cast<const TER_GLOBAL u32x4*>(gptr(row) + c * 16);
        } else {
            for (int j = 0; j < 4; ++j) {
                unsigned d = 0;
                for (int b = 0; b < 4; ++b) {
                    const int k = c * 16 + 4 * j + b;
                    if (k < K) d |= (unsigned)(uint8_t)gptr(row)[k] << (8 * b);
                }
                v[j] = d;
            }
        }
        *reinterpret_cast<TER_GLOBAL u32x4*>(gptr(tiles) + chunk_at(n, c, Ku)) = v;
    }
}

__global__ __launch_bounds__(256) void w8_unpack_kernel(const uint8_t* __restrict__ tiles,
                                                        const float* __restrict__ scale, int K, int N, int Ku,
                                                        int8_t* __restrict__ q, float* __restrict__ out_scale,
                                                        long long total) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += 256ll * gridDim.x) {
        const int n = (int)(i / K), k = (int)(i % K);
        if (q) gptr(q)[i] = (int8_t)gptr(tiles)[chunk_at(n, k >> 4, Ku) + (k & 15)];
        if (out_scale && k == 0) gptr(out_scale)[n] = gptr(scale)[n];
    }
}

inline unsigned grid_of(long long n) { return (unsigned)(n < (1ll << 30) ? (n + 255) / 256 : 1 << 22); }

// (a launch has fewer than 2^32 threads)
template <int TYPE, int T, int NC>
hipError_t launch_rows_as(const void* x, long long stride, int M, int K, int8_t* q, long long ldq, float* scale,
                          hipStream_t st) {
    typedef typename Elem<TYPE>::T E;
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (stride * (int)sizeof(E) % 16 == 0 || M == 1);
    constexpr int kRows = 1 << 21;
    for (int m = 0; m < M; m += kRows) {
        const dim3 grid(M - m < kRows ? M - m : kRows);
        const E* rows = static_cast<const E*>(x) + m * stride;
        if (vec)
            hipLaunchKernelGGL((rows8_quant_kernel<TYPE, T, NC, true>), grid, dim3(T), 0, st, rows, stride, K, q + m * ldq,
                               ldq, scale + m);
        else
            hipLaunchKernelGGL((rows8_quant_kernel<TYPE, T, NC, false>), grid, dim3(T), 0, st, rows, stride, K, q + m * ldq,
                               ldq, scale + m);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int TYPE>
hipError_t launch_rows_quant(const void* x, long long stride, int M, int K, int8_t* q, long long ldq, float* scale,
                             hipStream_t st) {
    if (ldq <= 2048) return launch_rows_as<TYPE, 256, 1>(x, stride, M, K, q, ldq, scale, st);
    if (ldq <= 4096) return launch_rows_as<TYPE, 512, 1>(x, stride, M, K, q, ldq, scale, st);
    if (ldq <= 8192) return launch_rows_as<TYPE, 1024, 1>(x, stride, M, K, q, ldq, scale, st);
    if (ldq <= 16384) return launch_rows_as<TYPE, 1024, 2>(x, stride, M, K, q, ldq, scale, st);
    hipLaunchKernelGGL(rows8_long_kernel<TYPE>, dim3(M), dim3(256), 0, st, x, stride, K, q, ldq, scale);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_w8_pack(const int8_t* q, long long stride, const float* scale, uint8_t* tiles, float* out_scale,
                          int K, int N, hipStream_t st) {
    const int Ku = i8_units(K);
    const long long n = (long long)i8_pairs(N) * 32 * 8 * Ku;
    hipLaunchKernelGGL(w8_pack_kernel, dim3(grid_of(n)), dim3(256), 0, st, q, stride, scale, K, N, Ku, tiles, out_scale,
                       reinterpret_cast<uintptr_t>(q) % 16 == 0 && stride % 16 == 0, n);
    return hipGetLastError();
}

hipError_t launch_w8_quantize(const void* src, int type, long long stride, uint8_t* tiles, float* out_scale, int K,
                              int N, hipStream_t st) {
    const dim3 grid(i8_pairs(N) * 32);
    const int Ku = i8_units(K);
    if (type == TER_HIP_T_F16)
        hipLaunchKernelGGL(w8_quantize_kernel<TER_HIP_T_F16>, grid, dim3(256), 0, st, src, stride, K, N, Ku, tiles,
                           out_scale);
    else if (type == TER_HIP_T_BF16)
        hipLaunchKernelGGL(w8_quantize_kernel<TER_HIP_T_BF16>, grid, dim3(256), 0, st, src, stride, K, N, Ku, tiles,
                           out_scale);
    else
        hipLaunchKernelGGL(w8_quantize_kernel<TER_HIP_T_F32>, grid, dim3(256), 0, st, src, stride, K, N, Ku, tiles,
                           out_scale);
    return hipGetLastError();
}

hipError_t launch_w8_unpack(const uint8_t* tiles, const float* scale, int8_t* q, float* out_scale, int K, int N,
                            hipStream_t st) {
    const long long n = (long long)N * K;
    hipLaunchKernelGGL(w8_unpack_kernel, dim3(grid_of(n)), dim3(256), 0, st, tiles, scale, K, N, i8_units(K), q,
                       out_scale, n);
    return hipGetLastError();
}

hipError_t launch_rows8(const void* x, int type, long long stride, int M, int K, int8_t* q, long long ldq, float* scale,
                        hipStream_t st) {
    if (type == TER_HIP_T_F16) return launch_rows_quant<TER_HIP_T_F16>(x, stride, M, K, q, ldq, scale, st);
    if (type == TER_HIP_T_BF16) return launch_rows_quant<TER_HIP_T_BF16>(x, stride, M, K, q, ldq, scale, st);
    if (type == TER_HIP_T_F32) return launch_rows_quant<TER_HIP_T_F32>(x, stride, M, K, q, ldq, scale, st);
    const int chunks = (int)(ldq / 16);
    const long long n = (long long)M * chunks;
    hipLaunchKernelGGL(rows8_copy_kernel, dim3(grid_of(n)), dim3(256), 0, st, static_cast<const int8_t*>(x), stride, K, q,
                       ldq, chunks, n);
    return hipGetLastError();
}

}  // namespace terhip

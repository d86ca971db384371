// int8.h -- shared definitions of the 8-bit products (include/ter_hip_int8.h).
//
// Weight layout.  Channels are cut into strips of 16 and K into units of 128
// (zero-padded).  A tile is one strip x 64 values of K in the order in which
// v_mfma_i32_16x16x64_i8 takes an operand: lane l's 16 bytes, row l % 16 of
// the strip, k = 16 * (l / 16) .. + 15, at byte 16 * l of 1024.  Tile (strip
// s, k-tile t) is at (s * 2 Ku + t) * 1024, Ku = ceil(K / 128): one wave reads
// an operand with one 16-byte load a lane over 1 KiB without gaps, from memory
// straight to registers or, past LDS, without bank conflicts.
//
// Two strips hold 32 channels, dealt to them by fours: row 4 g + r of strip
// 2 p + t is channel 32 p + 8 g + 4 t + r.  The weights are the product's A
// operand, so a lane's sums are rows 4 g .. 4 g + 3 (g = l / 16) of token
// l % 16: of the two strips together, 8 consecutive channels of one token,
// which are one 16-byte store in 16 bits, 64 contiguous bytes a token and wave.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "int8_rows.h"
#include "ter_hip_int8.h"

namespace terhip {

__host__ __device__ inline int i8_units(int K) { return (K + kI8Unit - 1) / kI8Unit; }
__host__ __device__ inline int i8_pairs(int N) { return (N + 31) / 32; }  // of strips
inline size_t i8_tile_bytes(int K, int N) { return (size_t)i8_pairs(N) * i8_units(K) * 4096; }

// Weights that are read by one workgroup each pass the caches by where they are
// a good part of the memory-side cache or more (128 MiB of 256): by the next call
// they would be gone.  Smaller ones may still be there (16 x 8192 x 8192 12.5
// against 13.5 us, called again and again).
inline bool i8_past_caches(int N, int Ku) { return (long long)N * Ku * kI8Unit >= 1ll << 27; }

struct Int8MmArgs {
    const uint8_t* w;     // tiles
    const float* ws;      // [32 pairs] (zero behind N)
    const int8_t* x;      // [M] rows, 16-byte aligned, a multiple of 16 values each
    const float* xs;      // [M], or null (y_type I32)
    char* y;
    long long ldx, ldy;   // bytes, elements
    int M, N, Kx, Ku;     // Kx: values of a row of x (a multiple of 16; those from K on meet zero weights)
    int y_type;
    int x_type;           // TER_HIP_T_I8, or rows quantized by the product's kernel: x, ldx and Kx are those of its elements
    int vec;              // such rows are 16-byte aligned
    int* sums;            // [parts][M][i8_sums_stride(N)] where tiles take a part of K each (parts > 1)
    int parts;
};

// Parts of K that the tiles of a call take (1: all of it), by sizes alone, and
// the stride of their sums.
int i8_parts(int M, int N, int Ku);
__host__ __device__ inline int i8_sums_stride(int N) { return (N + 7) / 8 * 8; }

// Rows that the product's kernel quantizes itself: a team of waves holds one
// in registers, at most kI8Chunks of 8 values a lane where 4 waves work
// together, fewer where 8 or 16 do.
constexpr int kI8Chunks = 8;
__host__ __device__ inline int i8_team(int M, int waves) {
    return M == 1 ? waves : M == 2 ? waves / 2 : M <= 4 ? waves / 4 : 1;
}
inline bool i8_quant_within(int M, int Ku) {
    return M <= 4 && Ku * 128 <= kI8Chunks * 512 * i8_team(M, 4) && M * Ku <= 128;
}

hipError_t launch_w8_pack(const int8_t* q, long long stride, const float* scale, uint8_t* tiles, float* out_scale,
                          int K, int N, hipStream_t st);
hipError_t launch_w8_quantize(const void* src, int type, long long stride, uint8_t* tiles, float* out_scale, int K,
                              int N, hipStream_t st);
hipError_t launch_w8_unpack(const uint8_t* tiles, const float* scale, int8_t* q, float* out_scale, int K, int N,
                            hipStream_t st);
// Rows to int8 rows ldq bytes apart (a multiple of 16) with zeros behind K;
// scales [M] for types other than TER_HIP_T_I8.
hipError_t launch_rows8(const void* x, int type, long long stride, int M, int K, int8_t* q, long long ldq, float* scale,
                        hipStream_t st);
// Whether a call is computed in tiles.
inline bool i8_in_tiles(int M, int N) { return M > 64 || (M > 16 && i8_pairs(N) > 300); }
hipError_t launch_int8_mm(const Int8MmArgs& a, hipStream_t st);
hipError_t launch_int8_gemm(const Int8MmArgs& a, hipStream_t st);  // many rows

}  // namespace terhip

// int8_mm.hip -- y[m][n] = (sum_k x[m][k] w[n][k]) * (xs[m] * ws[n]) on
// v_mfma_i32_16x16x64_i8, exact sums in int32: few rows, bound by the read of
// the weights.
//
// A workgroup computes S strips of 16 channels for 16 MB rows, its KS waves
// take every KS-th unit of 128 values of K.  Weights go from memory straight to
// the matrix units' registers (a tile of int8.h is an operand, 1 KiB a load
// without gaps), D units ahead; rows come from the L2, where all workgroups
// read the same ones.  The waves' sums are joined in LDS, each wave joining
// and storing a part of the results.
//
// Measured: 1 x 2048 x 128256 (rows, K, channels) 38.8 to 39.5 us, 6.7 to 6.8 TB/s
// (a pure read of as many bytes 39.2 to 40.4); 16 x 2560 x 128256 62 us, 5.3 TB/s
// and every workgroup's read of the rows; 23 x 6912 x 2560 8.8 to 9.1 us, 2.0 TB/s:
// 160 workgroups of 8 waves, a wave with two units in flight of the 7 it takes in
// turn.  One token of 2560 x 2560 takes 5.4 us, of which the weights' bytes are 1.
#include "common.h"
#include "int8.h"
#include "int8_quant.h"
#include "int8_store.h"

namespace terhip {
namespace {

__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* p, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}

// past: the data pass the caches by.
__device__ __forceinline__ i32x4 load16(__amdgpu_buffer_rsrc_t r, unsigned v, unsigned s, bool past = false) {
    return __builtin_bit_cast(i32x4, past ? __builtin_amdgcn_raw_buffer_load_b128(r, (int)v, (int)s, 2)
                                          : __builtin_amdgcn_raw_buffer_load_b128(r, (int)v, (int)s, 0));
}

// The rows in 8 bits to LDS: teams of waves, one a row, a row held in registers.
template <int XT, int KS>
__device__ __forceinline__ void quantize_rows(const Int8MmArgs& a, unsigned char* out, int ldl, float* scale, unsigned* red) {
    typedef typename Elem<XT>::T E;
    constexpr int NC = kI8Chunks * 4 / KS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int team = i8_team(a.M, KS), teams = KS / team, member = wave % team * 64 + lane;
    for (int m0 = 0; m0 < a.M; m0 += teams) {
        const int m = m0 + wave / team;
        const bool here = m < a.M;
        const TER_GLOBAL E* row = gptr(reinterpret_cast<const E*>(a.x)) + (long long)(here ? m : 0) * a.ldx;
        float v[NC][8];
        unsigned amax = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int k = 8 * (member + team * 64 * c);
            if (8 * team * 64 * c >= a.Ku * 128) break;
            row8<XT>(row, k, here ? a.Kx : 0, a.vec, v[c]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned b = __builtin_bit_cast(unsigned, v[c][e]) & 0x7FFFFFFFu;
                amax = b > amax ? b : amax;
            }
        }
        for (int s = 32; s; s >>= 1) {
            const unsigned o = (unsigned)__shfl_xor((int)amax, s);
            amax = o > amax ? o : amax;
        }
        __syncthreads();  // (red of the rows before)
        if (lane == 0) red[wave] = amax;
        __syncthreads();
        for (int i = 0; i < team; ++i) {
            const unsigned o = red[wave / team * team + i];
            amax = o > amax ? o : amax;
        }
        const Quant z = quant_of(amax);
        if (here && member == 0) scale[m] = z.inv;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int k = 8 * (member + team * 64 * c);
            if (8 * team * 64 * c >= a.Ku * 128) break;
            if (here && k < a.Ku * 128) *reinterpret_cast<u32x2*>(out + m * ldl + k) = quantize8(v[c], z.s);
        }
    }
    __syncthreads();
}

// XT: the type of rows that the workgroup quantizes itself, or TER_HIP_T_I8.
// Such rows are few and short (i8_quant_within): every workgroup does it again,
// under its first loads of weights, which is less than another launch takes.
template <int MB, int S, int KS, int D, int YT, int XT, bool PAST>
__global__ __launch_bounds__(64 * KS) void int8_stream_kernel(Int8MmArgs a, int groups) {
    constexpr bool kQuant = XT != TER_HIP_T_I8;
    __shared__ __align__(16) i32x4 part[KS][MB * S][64];
    extern __shared__ __align__(16) unsigned char rows8[];  // kQuant: [M][Ku * 128 + 16]
    __shared__ float row_scale[16];
    __shared__ unsigned red[KS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, g = lane >> 4;
    const int nb = blockIdx.x % groups, m0 = blockIdx.x / groups * (16 * MB);
    const int rows = a.M - m0 < 16 * MB ? a.M - m0 : 16 * MB;
    // units past the last are past the range by the vector offset: zeros
    const __amdgpu_buffer_rsrc_t wr = resource(a.w + (long long)nb * S * a.Ku * 2048, (unsigned)(S * a.Ku * 2048));
    const __amdgpu_buffer_rsrc_t xr =
        resource(a.x + (kQuant ? 0 : (long long)m0 * a.ldx), kQuant ? 0u : i8_rows_size(rows, (int)a.ldx, a.Kx));
    const int ldl = a.Ku * 128 + 16;
    unsigned xo[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) xo[i] = i8_stream_lane(16 * i + j, g, rows, kQuant ? ldl : (int)a.ldx);
    i32x4 acc[MB][S] = {};
    i32x4 w[D][2][S], x[kQuant ? 1 : D][2][MB];
    auto load = [&](int d, int u) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                // (the end of a strip is not the end of the range)
                w[d][t][s] = load16(wr, u < a.Ku ? lane * 16 : 0x7FFFFFFFu,
                                    (unsigned)((s * a.Ku + (u < a.Ku ? u : 0)) * 2048 + t * 1024), PAST);
            if constexpr (!kQuant) {
#pragma unroll
                for (int i = 0; i < MB; ++i) x[d][t][i] = load16(xr, i8_rows_at(xo[i], u, t), 0);
            }
        }
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, wave + d * KS);
    if constexpr (kQuant) quantize_rows<XT, KS>(a, rows8, ldl, row_scale, red);
    for (int u0 = wave; u0 < a.Ku; u0 += KS * D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if constexpr (kQuant) {
                const int u = u0 + d * KS < a.Ku ? u0 + d * KS : a.Ku - 1;  // (past the last the weights are zeros)
#pragma unroll
                for (int t = 0; t < 2; ++t) x[0][t][0] = *reinterpret_cast<const i32x4*>(rows8 + i8_rows_at(xo[0], u, t));
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int s = 0; s < S; ++s)
                        acc[i][s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d][t][s], x[kQuant ? 0 : d][t][i], acc[i][s], 0, 0, 0);
            if (u0 + KS * D < a.Ku) load(d, u0 + (D + d) * KS);
        }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int s = 0; s < S; ++s) part[wave][i * S + s][lane] = acc[i][s];
    __syncthreads();
    // results: strip s of row block i by wave (i S + s) / S, the strips of a pair by one
    const bool wide = wide_rows(a);
    for (int i = wave; i < MB; i += KS) {
        i32x4 sum[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            sum[s] = part[0][i * S + s][lane];
#pragma unroll
            for (int k = 1; k < KS; ++k) sum[s] += part[k][i * S + s][lane];
        }
        const int m = m0 + 16 * i + j;
        if (m >= a.M) continue;
        const float xs = YT == TER_HIP_T_I32 ? 0.f : kQuant ? row_scale[m - m0] : gptr(a.xs)[m];
        if constexpr (S == 2) {
            const int n = nb * 32 + 8 * g;
            if (n >= a.N) continue;
            float ws[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) ws[c] = YT == TER_HIP_T_I32 ? 0.f : gptr(a.ws)[n + c];
            const int v[8] = {sum[0][0], sum[0][1], sum[0][2], sum[0][3], sum[1][0], sum[1][1], sum[1][2], sum[1][3]};
            store_run<YT, 8>(a.y, (long long)m * a.ldy + n, a.N - n, v, xs, ws, wide);
        } else {
            const int n = nb / 2 * 32 + 8 * g + 4 * (nb & 1);
            if (n >= a.N) continue;
            float ws[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) ws[c] = YT == TER_HIP_T_I32 ? 0.f : gptr(a.ws)[n + c];
            const int v[4] = {sum[0][0], sum[0][1], sum[0][2], sum[0][3]};
            store_run<YT, 4>(a.y, (long long)m * a.ldy + n, a.N - n, v, xs, ws, wide);
        }
    }
}

template <int MB, int S, int KS, int D, int XT, bool PAST = false>
hipError_t launch(const Int8MmArgs& a, hipStream_t st) {
    const int groups = i8_pairs(a.N) * 2 / S, mb = (a.M + 16 * MB - 1) / (16 * MB);
    const dim3 grid((unsigned)((long long)groups * mb)), block(64 * KS);
    const int lds = XT != TER_HIP_T_I8 ? a.M * (a.Ku * 128 + 16) : 0;
    if (a.y_type == TER_HIP_T_F16)
        hipLaunchKernelGGL((int8_stream_kernel<MB, S, KS, D, TER_HIP_T_F16, XT, PAST>), grid, block, lds, st, a, groups);
    else if (a.y_type == TER_HIP_T_BF16)
        hipLaunchKernelGGL((int8_stream_kernel<MB, S, KS, D, TER_HIP_T_BF16, XT, PAST>), grid, block, lds, st, a, groups);
    else if (a.y_type == TER_HIP_T_F32)
        hipLaunchKernelGGL((int8_stream_kernel<MB, S, KS, D, TER_HIP_T_F32, XT, PAST>), grid, block, lds, st, a, groups);
    else if constexpr (XT == TER_HIP_T_I8)
        hipLaunchKernelGGL((int8_stream_kernel<MB, S, KS, D, TER_HIP_T_I32, XT, PAST>), grid, block, lds, st, a, groups);
    return hipGetLastError();
}

// Strips of a workgroup and waves that split K: enough waves for the GPU where
// there are few channels, few joins where there are many.  Measured (us; a
// call's host time is 7.3): 16 x 6912 x 2560 rows, K, channels 7.5 with 8 or 16
// waves; 32 x 2560 x 6912 8.4 with one strip and 8 waves, 7.3 with two and 4;
// 64 x 2048 x 8192 10.4 and 7.2; 48 x 6912 x 2560 13.8 and 14.8; 16 x 2048 x
// 128256 41.5 and 38.8.
template <int MB, int XT>
hipError_t launch_rows(const Int8MmArgs& a, hipStream_t st) {
    const int strips = 2 * i8_pairs(a.N);
    if constexpr (MB == 1) {
        if (strips <= 256) return launch<1, 1, 16, 4, XT>(a, st);
        if (strips <= 1024) return launch<1, 1, 8, 4, XT>(a, st);
        // (16 x 2560 x 128256 69 -> 62 us, 4 rows 56 -> 51)
        if (i8_past_caches(a.N, a.Ku)) return launch<1, 2, 4, 4, XT, true>(a, st);
        return launch<1, 2, 4, 4, XT>(a, st);
    } else {
        if (strips <= 256) return launch<MB, 1, 8, 2, XT>(a, st);
        return launch<MB, 2, 4, 2, XT>(a, st);
    }
}

}  // namespace

hipError_t launch_int8_mm(const Int8MmArgs& a, hipStream_t st) {
    if (a.x_type == TER_HIP_T_F16) return launch_rows<1, TER_HIP_T_F16>(a, st);
    if (a.x_type == TER_HIP_T_BF16) return launch_rows<1, TER_HIP_T_BF16>(a, st);
    if (a.x_type == TER_HIP_T_F32) return launch_rows<1, TER_HIP_T_F32>(a, st);
    // From 17 rows on and many channels the rows' reads by every workgroup weigh
    // more than the tiles' way over LDS: 32 x 2560 x 128256 78.6 us here, 62.1 in
    // tiles; 64 rows 111 and 70.  At 64 x 2048 x 8192 7.2 and 7.9.
    if (i8_in_tiles(a.M, a.N)) return launch_int8_gemm(a, st);
    if (a.M <= 16) return launch_rows<1, TER_HIP_T_I8>(a, st);
    if (a.M <= 32) return launch_rows<2, TER_HIP_T_I8>(a, st);
    return launch_rows<4, TER_HIP_T_I8>(a, st);
}

}  // namespace terhip

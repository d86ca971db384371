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
#include "common.h"
#include "int8.h"
#include "int8_store.h"

namespace terhip {
namespace {

__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* p, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ i32x4 load16(__amdgpu_buffer_rsrc_t r, unsigned v, unsigned s) {
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)v, (int)s, 0));
}

template <int MB, int S, int KS, int D, int YT>
__global__ __launch_bounds__(64 * KS) void int8_stream_kernel(Int8MmArgs a, int groups) {
    __shared__ __align__(16) i32x4 part[KS][MB * S][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, g = lane >> 4;
    const int nb = blockIdx.x % groups, m0 = blockIdx.x / groups * (16 * MB);
    const int rows = a.M - m0 < 16 * MB ? a.M - m0 : 16 * MB;
    // units past the last are past the range: zeros
    const __amdgpu_buffer_rsrc_t wr = resource(a.w + (long long)nb * S * a.Ku * 2048, (unsigned)(S * a.Ku * 2048));
    const __amdgpu_buffer_rsrc_t xr = resource(a.x + (long long)m0 * a.ldx, (unsigned)((rows - 1) * (int)a.ldx + a.Kx));
    unsigned xo[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int m = 16 * i + j;  // (rows behind the last: the last one's loads, whose sums nobody stores)
        xo[i] = (unsigned)((m < rows ? m : rows - 1) * (int)a.ldx + g * 16);
    }
    i32x4 acc[MB][S] = {};
    i32x4 w[D][2][S], x[D][2][MB];
    auto load = [&](int d, int u) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                // (the end of a strip is not the end of the range)
                w[d][t][s] = load16(wr, u < a.Ku ? lane * 16 : 0x7FFFFFFFu, (unsigned)((s * a.Ku + (u < a.Ku ? u : 0)) * 2048 + t * 1024));
#pragma unroll
            for (int i = 0; i < MB; ++i) x[d][t][i] = load16(xr, xo[i], (unsigned)(u * 128 + t * 64));
        }
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, wave + d * KS);
    for (int u0 = wave; u0 < a.Ku; u0 += KS * D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int s = 0; s < S; ++s)
                        acc[i][s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d][t][s], x[d][t][i], acc[i][s], 0, 0, 0);
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
        const float xs = YT == TER_HIP_T_I32 ? 0.f : gptr(a.xs)[m];
        if constexpr (S == 2) {
            const int n = nb * 32 + 8 * g;
            if (n >= a.N) continue;
            float ws[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) ws[c] = YT == TER_HIP_T_I32 ? 0.f : gptr(a.ws)[n + c];
            const int v[8] = {sum[0][0], sum[0][1], sum[0][2], sum[0][3], sum[1][0], sum[1][1], sum[1][2], sum[1][3]};
            store8<YT>(a.y, (long long)m * a.ldy + n, a.N - n, v, xs, ws, wide);
        } else {
            const int n = nb / 2 * 32 + 8 * g + 4 * (nb & 1);
            if (n >= a.N) continue;
            float ws[8];
#pragma unroll
            for (int c = 0; c < 4; ++c) ws[c] = YT == TER_HIP_T_I32 ? 0.f : gptr(a.ws)[n + c];
            const int v[8] = {sum[0][0], sum[0][1], sum[0][2], sum[0][3]};
            store8<YT>(a.y, (long long)m * a.ldy + n, a.N - n < 4 ? a.N - n : 4, v, xs, ws, false);
        }
    }
}

template <int MB, int S, int KS, int D>
hipError_t launch(const Int8MmArgs& a, hipStream_t st) {
    const int groups = i8_pairs(a.N) * 2 / S, mb = (a.M + 16 * MB - 1) / (16 * MB);
    const dim3 grid((unsigned)((long long)groups * mb)), block(64 * KS);
    if (a.y_type == TER_HIP_T_F16)
        hipLaunchKernelGGL((int8_stream_kernel<MB, S, KS, D, TER_HIP_T_F16>), grid, block, 0, st, a, groups);
    else if (a.y_type == TER_HIP_T_BF16)
        hipLaunchKernelGGL((int8_stream_kernel<MB, S, KS, D, TER_HIP_T_BF16>), grid, block, 0, st, a, groups);
    else if (a.y_type == TER_HIP_T_F32)
        hipLaunchKernelGGL((int8_stream_kernel<MB, S, KS, D, TER_HIP_T_F32>), grid, block, 0, st, a, groups);
    else
        hipLaunchKernelGGL((int8_stream_kernel<MB, S, KS, D, TER_HIP_T_I32>), grid, block, 0, st, a, groups);
    return hipGetLastError();
}

template <int MB>
hipError_t launch_rows(const Int8MmArgs& a, hipStream_t st) {
    constexpr int D = MB == 1 ? 4 : 2;
    if (i8_pairs(a.N) >= 512) return launch<MB, 2, 4, D>(a, st);
    return launch<MB, 1, 8, D>(a, st);
}

}  // namespace

hipError_t launch_int8_mm(const Int8MmArgs& a, hipStream_t st) {
    if (a.M > 64) return launch_int8_gemm(a, st);
    if (a.M <= 16) return launch_rows<1>(a, st);
    if (a.M <= 32) return launch_rows<2>(a, st);
    return launch_rows<4>(a, st);
}

}  // namespace terhip

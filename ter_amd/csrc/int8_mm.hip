// int8_mm.hip -- y[m][n] = (sum_k x[m][k] w[n][k]) * (xs[m] * ws[n]) on
// v_mfma_i32_16x16x64_i8, exact sums in int32.
#include "common.h"
#include "int8.h"
#include "int8_store.h"

namespace terhip {
namespace {

// A workgroup: 64 rows x 4 strip pairs, one pair a wave, operands straight
// from memory.
template <int YT>
__global__ __launch_bounds__(256) void int8_mm_kernel(Int8MmArgs a, int n_blocks) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nb = blockIdx.x % n_blocks, mb = blockIdx.x / n_blocks;
    const int pair = nb * 4 + wave, m0 = mb * 64, j = lane & 15, g = lane >> 4;
    if (pair * 32 >= a.N) return;
    i32x4 acc[4][2] = {};
    const uint8_t* w0 = a.w + (long long)pair * a.Ku * 4096 + lane * 16;
    const uint8_t* w1 = w0 + (long long)a.Ku * 2048;
    const int8_t* x[4];
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + 16 * i + j;
        x[i] = a.x + (long long)(m < a.M ? m : a.M - 1) * a.ldx;
    }
    for (int t = 0; t < 2 * a.Ku; ++t) {
        const i32x4 wa = *reinterpret_cast<const TER_GLOBAL i32x4*>(gptr(w0) + t * 1024);
        const i32x4 wb = *reinterpret_cast<const TER_GLOBAL i32x4*>(gptr(w1) + t * 1024);
        const int k = t * 64 + g * 16;
        for (int i = 0; i < 4; ++i) {
            i32x4 b = {};
            if (k < a.Kx) b = *reinterpret_cast<const TER_GLOBAL i32x4*>(gptr(x[i]) + k);
            acc[i][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wa, b, acc[i][0], 0, 0, 0);
            acc[i][1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wb, b, acc[i][1], 0, 0, 0);
        }
    }
    const int n = pair * 32 + 8 * g;
    float ws[8];
    for (int i = 0; i < 8; ++i) ws[i] = gptr(a.ws)[n + i];
    const bool wide = a.ldy % 8 == 0 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0;
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + 16 * i + j;
        if (m >= a.M || n >= a.N) continue;
        const int sum[8] = {acc[i][0][0], acc[i][0][1], acc[i][0][2], acc[i][0][3],
                            acc[i][1][0], acc[i][1][1], acc[i][1][2], acc[i][1][3]};
        store8<YT>(a.y, (long long)m * a.ldy + n, a.N - n, sum, YT == TER_HIP_T_I32 ? 0.f : gptr(a.xs)[m], ws, wide);
    }
}

template <int YT>
hipError_t launch(const Int8MmArgs& a, hipStream_t st) {
    const int nb = (i8_pairs(a.N) + 3) / 4, mb = (a.M + 63) / 64;
    hipLaunchKernelGGL(int8_mm_kernel<YT>, dim3((unsigned)((long long)nb * mb)), dim3(256), 0, st, a, nb);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_int8_mm(const Int8MmArgs& a, hipStream_t st) {
    if (a.M > 64) return launch_int8_gemm(a, st);
    switch (a.y_type) {
        case TER_HIP_T_F16: return launch<TER_HIP_T_F16>(a, st);
        case TER_HIP_T_BF16: return launch<TER_HIP_T_BF16>(a, st);
        case TER_HIP_T_F32: return launch<TER_HIP_T_F32>(a, st);
        default: return launch<TER_HIP_T_I32>(a, st);
    }
}

}  // namespace terhip

// int8_gemm.hip -- the 8-bit product of many rows: tiles of rows x channels in
// LDS, v_mfma_i32_16x16x64_i8.
//
// A workgroup of 8 waves (RW x CW) computes BM x BN results.  Per unit of 128
// values of K both operands come to LDS straight from memory (buffer_load ...
// lds, 1 KiB an instruction, no registers), two stages, the next unit's loads
// in flight under the products of the one at hand.
//
// LDS.  Weights keep their tiles (int8.h): an operand is one ds_read_b128 at 16
// * lane.  A row of x is 128 bytes, its 16-byte chunk c at position c ^ g(row),
// g(row) = (row & 7) ^ (row >> 3 & 1): the 16 rows that an operand reads at one
// chunk fall on 16 different positions of 256 bytes, 8 of them on 8 of 128.
// A load's lanes cover whole 128-byte lines of 8 rows in any case.
//
// Rows behind the last and values behind K are zeros by the buffer's range, or
// meet the zeros that pad the weights.
#include "common.h"
#include "int8.h"
#include "int8_store.h"

namespace terhip {
namespace {

#define TER_LDS __attribute__((address_space(3)))

// MBW row blocks of 16 and SW strips of 16 a wave, RW x CW waves.
template <int MBW_, int SW_, int RW_, int CW_>
struct GCfg {
    static constexpr int MBW = MBW_, SW = SW_, RW = RW_, CW = CW_, WAVES = RW * CW, THREADS = 64 * WAVES;
    static constexpr int BM = 16 * MBW * RW, BN = 16 * SW * CW;
    static constexpr int XB = BM * 128, WB = BN * 128, STAGE = XB + WB;
    static constexpr int XL = XB / 1024 / WAVES, WL = WB / 1024 / WAVES;  // loads of a wave and stage
    static_assert(XB % (1024 * WAVES) == 0 && WB % (1024 * WAVES) == 0 && SW % 2 == 0 && SW <= MBW, "");
    static_assert(2 * STAGE <= kLdsMax, "");
};

// 16 bytes a lane from memory to LDS at lds + 16 * lane.  Inline asm without
// outputs: behind the builtin the compiler makes every LDS read wait for the
// loads of the next stage; the waits are explicit instead.  (Also for the
// scalar registers, which a buffer load reads five wait states or more after a
// lane read wrote them.)
__device__ __forceinline__ void load_to_lds(u32x4 rsrc, unsigned voff, unsigned soff, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory", "m0");
}

__device__ __forceinline__ u32x4 resource(const void* p, unsigned bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a),
                 (unsigned)__builtin_amdgcn_readfirstlane((int)((unsigned)(a >> 32) & 0xFFFFu)),
                 (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

// Until at most N of this wave's loads are in flight.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ int swizzle(int row) { return (row & 7) ^ (row >> 3 & 1); }

template <class C, int YT>
__global__ __launch_bounds__(C::THREADS) void int8_gemm_kernel(Int8MmArgs a, int mt, int nt) {
    extern __shared__ __align__(1024) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, g = lane >> 4;
    int tm, tn;
    tile_of(blockIdx.x, mt, nt, tm, tn);
    const int m0 = tm * C::BM, s0 = tn * (C::BN / 16);
    const int rows = a.M - m0 < C::BM ? a.M - m0 : C::BM;
    const int strips = 2 * i8_pairs(a.N) - s0;
    const u32x4 xr = resource(a.x + (long long)m0 * a.ldx, (unsigned)((rows - 1) * (int)a.ldx + a.Kx));
    const u32x4 wr = resource(a.w + (long long)s0 * a.Ku * 2048,
                              (unsigned)((strips < C::BN / 16 ? strips : C::BN / 16) * a.Ku * 2048));
    const unsigned base = (unsigned)reinterpret_cast<uintptr_t>((TER_LDS unsigned char*)lds);
    // loads of this wave: X runs of 8 rows, W runs of a tile
    unsigned xo[C::XL], wo[C::WL];
#pragma unroll
    for (int i = 0; i < C::XL; ++i) {
        const int row = (wave * C::XL + i) * 8 + (lane >> 3);
        xo[i] = (unsigned)(row * (int)a.ldx + ((lane & 7) ^ swizzle(row)) * 16);
    }
#pragma unroll
    for (int i = 0; i < C::WL; ++i) {
        const int run = wave * C::WL + i;  // strip run / 2, k-tile run % 2
        wo[i] = (unsigned)((run >> 1) * a.Ku * 2048 + (run & 1) * 1024 + lane * 16);
    }
    auto issue = [&](int u, int buf) {
        const unsigned at = base + buf * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::XL; ++i) load_to_lds(xr, xo[i], u * 128, at + (wave * C::XL + i) * 1024);
#pragma unroll
        for (int i = 0; i < C::WL; ++i) load_to_lds(wr, wo[i], u * 2048, at + C::XB + (wave * C::WL + i) * 1024);
    };
    const int rw = wave / C::CW, cw = wave % C::CW;
    const int xat = (rw * C::MBW * 16 + j) * 128, wat = C::XB + cw * C::SW * 2048 + lane * 16;
    auto read_x = [&](const unsigned char* st, int q) {  // step q of a stage: k-tile q / MBW, row block q % MBW
        // (rows 16 apart have the same swizzle)
        return *reinterpret_cast<const i32x4*>(st + xat + q % C::MBW * 2048 + ((q / C::MBW * 4 + g) ^ swizzle(j)) * 16);
    };
    auto read_w = [&](const unsigned char* st, int t, int s) {
        return *reinterpret_cast<const i32x4*>(st + wat + s * 2048 + t * 1024);
    };
    // A stage is 2 MBW steps of SW products.  Operands are read kAhead steps
    // before their products; the stage's reads are over kAhead steps before its
    // end.  There the wave waits for its loads of the next stage and for the
    // other waves: then the stage's place is free for the loads of the one after
    // the next, and the next one's operands are read under the last products.
    constexpr int STEPS = 2 * C::MBW, kAhead = 3;
    i32x4 acc[C::MBW][C::SW] = {};
    i32x4 x[kAhead + 1], w[2][C::SW];
    issue(0, 0);
    if (a.Ku > 1) {
        issue(1, 1);
        wait_loads<C::XL + C::WL>();
    } else {
        wait_loads<0>();
    }
    barrier();
#pragma unroll
    for (int s = 0; s < C::SW; ++s) w[0][s] = read_w(lds, 0, s);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) x[q] = read_x(lds, q);
    for (int u = 0; u < a.Ku; ++u) {
        const unsigned char* st = lds + (u & 1) * C::STAGE;
        const unsigned char* next = lds + ((u + 1) & 1) * C::STAGE;
#pragma unroll
        for (int q = 0; q < STEPS; ++q) {
            const int t = q / C::MBW, i = q % C::MBW;
            if (q + kAhead < STEPS)
                x[(q + kAhead) % (kAhead + 1)] = read_x(st, q + kAhead);
            else
                x[(q + kAhead) % (kAhead + 1)] = read_x(next, q + kAhead - STEPS);
            // weights of the second k-tile: during the first; of the next stage's first: at the end
            if (t == 0 && i < C::SW) w[1][i] = read_w(st, 1, i);
            if (q == STEPS - kAhead) {
#pragma unroll
                for (int s = 0; s < C::SW; ++s) w[0][s] = read_w(next, 0, s);
            }
#pragma unroll
            for (int s = 0; s < C::SW; ++s)
                acc[i][s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t][s], x[q % (kAhead + 1)], acc[i][s], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (q == STEPS - kAhead - 1) {
                // (the step's reads were the stage's last)
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                wait_loads<0>();
                barrier();
                if (u + 2 < a.Ku) issue(u + 2, u & 1);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    store_tile<C::MBW, C::SW, YT>(a, m0 + rw * C::MBW * 16, (s0 + cw * C::SW) * 16, acc, lane);
}

template <class C, int YT>
hipError_t launch(const Int8MmArgs& a, hipStream_t st) {
    static LdsLimit limit;
    const hipError_t e = limit.allow(2 * C::STAGE, {reinterpret_cast<const void*>(&int8_gemm_kernel<C, YT>)});
    if (e != hipSuccess) return e;
    const int mt = (a.M + C::BM - 1) / C::BM, nt = (a.N + C::BN - 1) / C::BN;
    hipLaunchKernelGGL((int8_gemm_kernel<C, YT>), dim3((unsigned)((long long)mt * nt)), dim3(C::THREADS), 2 * C::STAGE, st, a,
                       mt, nt);
    return hipGetLastError();
}

template <class C>
hipError_t launch_type(const Int8MmArgs& a, hipStream_t st) {
    switch (a.y_type) {
        case TER_HIP_T_F16: return launch<C, TER_HIP_T_F16>(a, st);
        case TER_HIP_T_BF16: return launch<C, TER_HIP_T_BF16>(a, st);
        case TER_HIP_T_F32: return launch<C, TER_HIP_T_F32>(a, st);
        default: return launch<C, TER_HIP_T_I32>(a, st);
    }
}

}  // namespace

hipError_t launch_int8_gemm(const Int8MmArgs& a, hipStream_t st) {
    return launch_type<GCfg<8, 4, 2, 4>>(a, st);
}

}  // namespace terhip

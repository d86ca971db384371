// int8_gemm.hip -- the 8-bit product of many rows: tiles of rows x channels in
// LDS, v_mfma_i32_16x16x64_i8.
//
// A workgroup of 8 waves (RW x CW) computes BM x BN results, tile after tile of
// its share.  Per unit of 128 values of K both operands come to LDS straight
// from memory (buffer_load ... lds, 1 KiB an instruction, no registers), NST
// stages, the next units' loads in flight under the products of the one at
// hand.  The units of a workgroup's tiles are one sequence: the next tile's
// first ones are loaded under the last products of a tile and its stores.
//
// LDS.  Weights keep their tiles (int8.h): an operand is one ds_read_b128 at 16
// * lane.  A row of x is 128 bytes, its 16-byte chunk c at position c ^ g(row),
// g(row) = (row & 7) ^ (row >> 3 & 1): the 16 rows that an operand reads at one
// chunk fall on 16 different positions of 256 bytes, 8 of them on 8 of 128.
// A load's lanes cover whole 128-byte lines of 8 rows in any case.
//
// Rows behind the last, and the last row's values behind K, are zeros by the
// buffer's range, which covers a load's vector offset and not its scalar one: a
// row's whole offset is in the former (int8_rows.h).  Other rows' values behind K
// meet the zeros that pad the weights, whose unit is the scalar offset: behind the
// last strip the vector offset alone is out of range.
//
// Measured: 8192 x 8192 x 8192 395 to 412 us, 2.67 to 2.79 P op/s (the library's
// product 464); 8192 x 2560 x 6912 127 to 150 us by the machine, 1.9 to 2.3 (177).
// Of a unit's 1.59 us in the largest tile the products alone are 1.03, the loads
// alone 1.02: LDS serves both, and the barrier's wait is not all hidden.  Products
// of 32 x 32 x 32 instead of 16 x 16 x 64 (8192 cubed 475 against 441 us then)
// and 4 waves of 128 x 128 instead of 8 were slower.
#include "common.h"
#include "int8.h"
#include "int8_store.h"

namespace terhip {
namespace {

#define TER_LDS __attribute__((address_space(3)))

// MBW row blocks of 16 and SW strips of 16 a wave, RW x CW waves, NST stages;
// a unit's loads are issued over SPREAD steps.
template <int MBW_, int SW_, int RW_, int CW_, int NST_, int SPREAD_>
struct GCfg {
    static constexpr int MBW = MBW_, SW = SW_, RW = RW_, CW = CW_, NST = NST_, SPREAD = SPREAD_, WAVES = RW * CW, THREADS = 64 * WAVES;
    static constexpr int BM = 16 * MBW * RW, BN = 16 * SW * CW;
    static constexpr int XB = BM * 128, WB = BN * 128, STAGE = XB + WB, LDS = NST * STAGE;
    // loads of a wave and stage: X runs (the first XR waves one more), W runs
    static constexpr int XL = XB / 1024 / WAVES, XR = XB / 1024 % WAVES, WL = WB / 1024 / WAVES;
    static_assert(WB % (1024 * WAVES) == 0 && SW % 2 == 0 && SW <= MBW * 2, "");
    static_assert(LDS <= kLdsMax && NST >= 2 && (NST - 2) * (XL + 1 + WL) < 64, "");
};

// 16 bytes a lane from memory to LDS at lds + 16 * lane.  Inline asm without
// outputs: behind the builtin the compiler makes every LDS read wait for the
// loads of the next stage; the waits are explicit instead.  (Also for the
// scalar registers, which a buffer load reads five wait states or more after a
// lane read wrote them.)
__device__ __forceinline__ void load_rows(u32x4 rsrc, unsigned voff, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(rsrc)
                 : "memory", "m0");
}

// once: read by nobody else, so not kept in the caches.
__device__ __forceinline__ void load_weights(u32x4 rsrc, unsigned voff, unsigned soff, unsigned lds, bool once) {
    if (once)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds"
                     :
                     : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
                     : "memory", "m0");
    else
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

// Until the loads of the units behind the next one are all that is in flight.
template <class C, int BEHIND>
__device__ __forceinline__ void wait_unit(int behind, bool more) {
    if constexpr (BEHIND == 0) {
        wait_loads<0>();
    } else if (behind >= BEHIND) {
        if (C::XR != 0 && more)
            wait_loads<BEHIND*(C::XL + 1 + C::WL)>();
        else
            wait_loads<BEHIND*(C::XL + C::WL)>();
    } else {
        wait_unit<C, BEHIND - 1>(behind, more);
    }
}

// SPLIT: a tile is computed by a.parts workgroups, `per` units of K each, whose
// bare sums int8_join_kernel joins; the grid is all of them.
template <class C, int YT, bool SPLIT>
__global__ __launch_bounds__(C::THREADS) void int8_gemm_kernel(Int8MmArgs a, int mt, int nt, bool once, int per) {
    extern __shared__ __align__(1024) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, g = lane >> 4;
    const bool more = wave < C::XR;
    const unsigned base = (unsigned)reinterpret_cast<uintptr_t>((TER_LDS unsigned char*)lds);
    // loads of this wave: X runs of 8 rows, W runs of a tile
    const int run0 = wave * C::XL + (more ? wave : C::XR);
    unsigned xo[C::XL + 1], wo[C::WL];
#pragma unroll
    for (int i = 0; i < C::XL + (C::XR != 0); ++i) xo[i] = i8_tile_lane((run0 + i) * 8 + (lane >> 3), lane, (int)a.ldx);
#pragma unroll
    for (int i = 0; i < C::WL; ++i) {
        const int run = wave * C::WL + i;  // strip run / 2, k-tile run % 2
        wo[i] = (unsigned)((run >> 1) * a.Ku * 2048 + (run & 1) * 1024 + lane * 16);
    }
    // what is loaded: unit iu of tile it.  Large weights that one tile needs pass
    // the caches by: 96 x 2560 x 128256 75.1 -> 66.3 us (8192 x 2560 x 6912, where
    // they are needed again, 134 -> 161).
    const int tiles = mt * nt, part = SPLIT ? (int)blockIdx.x / tiles : 0, tile0 = (int)blockIdx.x - part * tiles;
    const int first = SPLIT ? part * per : 0, last = SPLIT && first + per < a.Ku ? first + per : a.Ku;
    int it = tile0, iu = first, place = 0;
    u32x4 xr, wr;
    auto aim = [&] {
        int tm, tn;
        tile_of(it, mt, nt, tm, tn);
        const int m0 = tm * C::BM, s0 = tn * (C::BN / 16);
        const int rows = a.M - m0 < C::BM ? a.M - m0 : C::BM;
        const int strips = 2 * i8_pairs(a.N) - s0;
        xr = resource(a.x + (long long)m0 * a.ldx, i8_rows_size(rows, (int)a.ldx, a.Kx));
        wr = resource(a.w + (long long)s0 * a.Ku * 2048,
                      (unsigned)((strips < C::BN / 16 ? strips : C::BN / 16) * a.Ku * 2048));
    };
    constexpr int RUNS = C::XL + (C::XR != 0) + C::WL;
    auto issue = [&](int i) {  // load i of the next unit, to its place
        if (it >= tiles) return;
        const unsigned at = base + place * C::STAGE;
        if (i < C::XL)
            load_rows(xr, i8_rows_at(xo[i], iu, 0), at + (run0 + i) * 1024);
        else if (i >= C::XL + C::WL)
            if (more) load_rows(xr, i8_rows_at(xo[C::XL], iu, 0), at + (run0 + C::XL) * 1024);
        if (i >= C::XL && i < C::XL + C::WL)
            load_weights(wr, wo[i - C::XL], iu * 2048, at + C::XB + (wave * C::WL + i - C::XL) * 1024, once);
        if (i == RUNS - 1) {
            place = place + 1 == C::NST ? 0 : place + 1;
            if (++iu == last) {
                iu = first;
                it += gridDim.x;
                if (it < tiles) aim();
            }
        }
    };
    const int rw = wave / C::CW, cw = wave % C::CW;
    const int xat = (rw * C::MBW * 16 + j) * 128, wat = C::XB + cw * C::SW * 2048 + lane * 16;
    auto read_x = [&](const unsigned char* st, int q) {  // step q of a stage: k-tile q / MBW, row block q % MBW
        // (rows 16 apart have the same swizzle)
        return *reinterpret_cast<const i32x4*>(st + xat + q % C::MBW * 2048 + ((q / C::MBW * 4 + g) ^ i8_swizzle(j)) * 16);
    };
    auto read_w = [&](const unsigned char* st, int t, int s) {
        return *reinterpret_cast<const i32x4*>(st + wat + s * 2048 + t * 1024);
    };
    // A stage is 2 MBW steps of SW products.  Operands are read kAhead steps
    // before their products; the stage's reads are over kAhead steps before its
    // end.  There the wave waits for its loads of the next unit and for the
    // other waves: then the stage's place is free for the loads of a later one,
    // and the next one's operands are read under the last products.
    // (kRing operands of x in turn, a divisor of STEPS)
    constexpr int STEPS = 2 * C::MBW, kRing = C::MBW == 2 ? 2 : C::MBW % 2 ? C::MBW : 4, kAhead = kRing - 1;
    constexpr int kW = (C::SW + C::MBW - 1) / C::MBW;
    static_assert(STEPS % kRing == 0 && STEPS - kAhead > C::MBW, "weights of the second k-tile before the stage is free");
    i32x4 x[kRing], w[2][C::SW];
    aim();
#pragma unroll
    for (int k = 0; k < C::NST; ++k)
#pragma unroll
        for (int i = 0; i < RUNS; ++i) issue(i);
    int left = SPLIT ? last - first : ((tiles - 1 - tile0) / (int)gridDim.x + 1) * a.Ku;  // units, the one at hand included
    wait_unit<C, C::NST - 1>(left - 1, more);
    barrier();
    int cur = 0;
#pragma unroll
    for (int s = 0; s < C::SW; ++s) w[0][s] = read_w(lds, 0, s);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) x[q] = read_x(lds, q);
    constexpr int kSlots = C::SPREAD < STEPS ? C::SPREAD : STEPS - 1;
    bool loading = false;
    if (SPLIT) {
        a.ldy = i8_sums_stride(a.N);
        a.y = reinterpret_cast<char*>(a.sums + (long long)part * a.M * a.ldy);
    }
    for (int tile = tile0; tile < tiles; tile += gridDim.x) {
        i32x4 acc[C::MBW][C::SW] = {};
        for (int u = first; u < last; ++u) {
            const unsigned char* st = lds + cur * C::STAGE;
            cur = cur + 1 == C::NST ? 0 : cur + 1;
            const unsigned char* next = lds + cur * C::STAGE;
            --left;
#pragma unroll
            for (int q = 0; q < STEPS; ++q) {
                const int t = q / C::MBW, i = q % C::MBW;
                if (q + kAhead < STEPS)
                    x[(q + kAhead) % kRing] = read_x(st, q + kAhead);
                else
                    x[(q + kAhead) % kRing] = read_x(next, q + kAhead - STEPS);
                // weights of the second k-tile: during the first; of the next unit's first: at the end
                if (t == 0) {
#pragma unroll
                    for (int s = i * kW; s < i * kW + kW && s < C::SW; ++s) w[1][s] = read_w(st, 1, s);
                }
                if (q == STEPS - kAhead) {
#pragma unroll
                    for (int s = 0; s < C::SW; ++s) w[0][s] = read_w(next, 0, s);
                }
#pragma unroll
                for (int s = 0; s < C::SW; ++s)
                    acc[i][s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t][s], x[q % kRing], acc[i][s], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                if (q == STEPS - kAhead - 1) {
                    // (the step's reads were the stage's last)
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    wait_unit<C, C::NST - 2>(left - 1, more);
                    barrier();
                    loading = true;
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    // the loads of a later unit, a few a step: their issue then runs under the products
                    constexpr int PER = (RUNS + kSlots - 1) / kSlots;
                    const int slot = (q - (STEPS - kAhead) + STEPS) % STEPS;
                    if (slot < kSlots && loading) {
#pragma unroll
                        for (int i = slot * PER; i < slot * PER + PER && i < RUNS; ++i) issue(i);
                        if (slot == kSlots - 1) loading = false;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        int tm, tn;
        tile_of(tile, mt, nt, tm, tn);
        store_tile<C::MBW, C::SW, YT>(a, tm * C::BM + rw * C::MBW * 16, tn * C::BN + cw * C::SW * 16, acc, lane);
    }
}

// Eight results of one row a thread: the parts' sums, scaled.
template <int YT>
__global__ __launch_bounds__(256) void int8_join_kernel(Int8MmArgs a) {
    const int stride = i8_sums_stride(a.N), chunks = stride / 8;
    const int i = blockIdx.x * 256 + threadIdx.x, m = i / chunks, n = (i - m * chunks) * 8;
    if (m >= a.M) return;
    i32x4 s[2] = {};
    for (int p = 0; p < a.parts; ++p) {
        const TER_GLOBAL i32x4* from = reinterpret_cast<const TER_GLOBAL i32x4*>(gptr(a.sums) + ((long long)p * a.M + m) * stride + n);
        s[0] += from[0];
        s[1] += from[1];
    }
    float ws[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) ws[c] = YT == TER_HIP_T_I32 ? 0.f : gptr(a.ws)[n + c];
    const int v[8] = {s[0][0], s[0][1], s[0][2], s[0][3], s[1][0], s[1][1], s[1][2], s[1][3]};
    store_run<YT, 8>(a.y, (long long)m * a.ldy + n, a.N - n, v, YT == TER_HIP_T_I32 ? 0.f : gptr(a.xs)[m], ws, wide_rows(a));
}

template <class C, int YT>
hipError_t launch(const Int8MmArgs& a, int cus, hipStream_t st) {
    static LdsLimit limit;
    const hipError_t e = limit.allow(C::LDS, {reinterpret_cast<const void*>(&int8_gemm_kernel<C, YT, false>)});
    if (e != hipSuccess) return e;
    const int mt = (a.M + C::BM - 1) / C::BM, nt = (a.N + C::BN - 1) / C::BN;
    const int fit = kLdsMax / C::LDS > 1 ? 2 : 1;
    const int grid = mt * nt < cus * fit ? mt * nt : cus * fit;
    hipLaunchKernelGGL((int8_gemm_kernel<C, YT, false>), dim3(grid), dim3(C::THREADS), C::LDS, st, a, mt, nt,
                       mt == 1 && i8_past_caches(a.N, a.Ku), 0);
    return hipGetLastError();
}

using Small = GCfg<2, 2, 2, 2, 5, 4>;

hipError_t launch_parts(const Int8MmArgs& a, hipStream_t st) {
    static LdsLimit limit;
    const auto kernel = &int8_gemm_kernel<Small, TER_HIP_T_I32, true>;
    hipError_t e = limit.allow(Small::LDS, {reinterpret_cast<const void*>(kernel)});
    if (e != hipSuccess) return e;
    const int mt = (a.M + Small::BM - 1) / Small::BM, nt = (a.N + Small::BN - 1) / Small::BN;
    hipLaunchKernelGGL(kernel, dim3(mt * nt * a.parts), dim3(Small::THREADS), Small::LDS, st, a, mt, nt, false,
                       (a.Ku + a.parts - 1) / a.parts);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    const dim3 grid((a.M * (i8_sums_stride(a.N) / 8) + 255) / 256), block(256);
    switch (a.y_type) {
        case TER_HIP_T_F16: hipLaunchKernelGGL(int8_join_kernel<TER_HIP_T_F16>, grid, block, 0, st, a); break;
        case TER_HIP_T_BF16: hipLaunchKernelGGL(int8_join_kernel<TER_HIP_T_BF16>, grid, block, 0, st, a); break;
        case TER_HIP_T_F32: hipLaunchKernelGGL(int8_join_kernel<TER_HIP_T_F32>, grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL(int8_join_kernel<TER_HIP_T_I32>, grid, block, 0, st, a); break;
    }
    return hipGetLastError();
}

template <class C>
hipError_t launch_type(const Int8MmArgs& a, int cus, hipStream_t st) {
    switch (a.y_type) {
        case TER_HIP_T_F16: return launch<C, TER_HIP_T_F16>(a, cus, st);
        case TER_HIP_T_BF16: return launch<C, TER_HIP_T_BF16>(a, cus, st);
        case TER_HIP_T_F32: return launch<C, TER_HIP_T_F32>(a, cus, st);
        default: return launch<C, TER_HIP_T_I32>(a, cus, st);
    }
}

}  // namespace

// The variants.  A call takes the one whose estimate is the least: rounds of
// the GPU times (units times `unit` + `tile`), in us, measured on calls that fill
// it once to many times; `few` is a unit where a CU holds one workgroup of two.
// 8192 x 8192 x 8192: 789, 531, 493, 463, 493, 466, 437 and 407 us in the order
// of the table; 128 rows x 2560 channels, K 6912: 17.8, 36, 46, 42, 51, 55, 58,
// 67; 1021 x 8192, K 2048: 32.5, 29.7, 23, 22.2, 26, 27.6, 28.8, 31.
namespace {
struct Variant {
    int bm, bn, fit;
    float few, unit, tile;
};
constexpr Variant kVariants[] = {
    {64, 64, 2, 0.28f, 0.39f, 3.f},    {96, 256, 1, 0.75f, 0.75f, 4.f},  {128, 256, 1, 0.93f, 0.93f, 4.5f},
    {256, 128, 1, 0.90f, 0.90f, 4.5f}, {160, 256, 1, 1.10f, 1.10f, 5.f}, {192, 256, 1, 1.21f, 1.21f, 6.f},
    {224, 256, 1, 1.37f, 1.37f, 7.f},  {256, 256, 1, 1.59f, 1.59f, 8.f},
};

// The variant of the least estimate, and that estimate.
int best_variant(int M, int N, int Ku, int cus, float* us) {
    int best = 0;
    for (int i = 0; i < (int)(sizeof(kVariants) / sizeof(kVariants[0])); ++i) {
        const Variant& v = kVariants[i];
        const long long tiles = (long long)((M + v.bm - 1) / v.bm) * ((N + v.bn - 1) / v.bn);
        const long long rounds = (tiles + (long long)cus * v.fit - 1) / ((long long)cus * v.fit);
        const float t = (float)rounds * ((float)Ku * (tiles <= cus ? v.few : v.unit) + v.tile);
        if (i == 0 || t < *us) {
            *us = t;
            best = i;
        }
    }
    return best;
}
}  // namespace

// Few tiles of a long K leave most of the GPU idle: parts of it then, as many
// workgroups as fit at once, and their sums joined by one launch more, whose host
// time counts too (us, rows x channels x K, all of K and parts): 380 x 512 x 8192
// 24.6 and 13.3, 128 x 2560 x 6912 20.8 and 14.7, 300 x 2560 x 16384 44.3 and
// 31.9, 256 x 2560 x 6912 21.3 and 16.1; 128 x 640 x 2560 9.6 and 13.3: not in parts.
// The parts are those of a whole GPU's 256 CUs, so that the workspace is one size on
// every device; on a partition of one they are more than fit at once.
int i8_parts(int M, int N, int Ku) {
    constexpr int kCus = 256;
    constexpr float kJoin = 5.f, kJoinBytes = 1.f / 3e6f;  // us a launch, us a byte of sums
    float least;
    best_variant(M, N, Ku, kCus, &least);
    const long long tiles = (long long)((M + 63) / 64) * ((N + 63) / 64);
    int best = 1;
    for (int parts = 2; parts <= 8 && parts * tiles <= 2 * kCus && parts * 4 <= Ku; ++parts) {
        const int per = (Ku + parts - 1) / parts;
        if (per * (parts - 1) >= Ku) continue;  // (each part has units)
        const float us = (float)per * (parts * tiles <= kCus ? kVariants[0].few : kVariants[0].unit) + kVariants[0].tile +
                         kJoin + kJoinBytes * 4.f * (float)parts * (float)M * (float)N;
        if (us < least) {
            least = us;
            best = parts;
        }
    }
    return best;
}

hipError_t launch_int8_gemm(const Int8MmArgs& a, hipStream_t st) {
    if (a.parts > 1) return launch_parts(a, st);
    int dev = 0;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const int cus = device_cu_count(dev);
    if (cus <= 0) return hipErrorInvalidDevice;
    float us;
    switch (best_variant(a.M, a.N, a.Ku, cus, &us)) {
        case 0: return launch_type<Small>(a, cus, st);
        case 1: return launch_type<GCfg<3, 4, 2, 4, 3, 8>>(a, cus, st);
        case 2: return launch_type<GCfg<4, 4, 2, 4, 3, 4>>(a, cus, st);
        case 3: return launch_type<GCfg<4, 4, 4, 2, 3, 4>>(a, cus, st);
        case 4: return launch_type<GCfg<5, 4, 2, 4, 3, 4>>(a, cus, st);
        case 5: return launch_type<GCfg<6, 4, 2, 4, 2, 4>>(a, cus, st);
        case 6: return launch_type<GCfg<7, 4, 2, 4, 2, 8>>(a, cus, st);
        default: return launch_type<GCfg<8, 4, 2, 4, 2, 4>>(a, cus, st);
    }
}

}  // namespace terhip

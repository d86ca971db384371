// paged_attend.hip -- causal attention of the new rows of a batch of sequences
// over a paged cache: prompts, pieces of prompts and single tokens in one
// launch, and a prefix that all sequences share multiplied once.
//
// For a row with query q that sees positions s < lim:
//   x_s = scale log2(e) q . K_s,  out = sum_s 2^(x_s + o) V_s / sum_s 2^(x_s + o)
// for any offset o.  One pass over the positions holds the running sums in
// binary32 with an o near minus the largest x so far; where that grows by
// enough, sums are multiplied by 2^(new o - old o).  Partial results (sums and
// their o) of different ranges of positions are joined the same way.
//
// Scores, sums and statistics are binary32.  For the second product the matrix
// cores take weights of the element type: of few rows, which wait for memory,
// each is the sum of two (so results are as near to the formula as with binary32
// weights: relative error 0.00021 in fp16, 0.0016 in bf16, the rounding of the
// result itself); of many rows, which wait for the matrix cores, it is rounded
// to one, half a step as the inputs are (0.00026-0.00029 and 0.0023).  Two there
// make 5,600 rows of prompts 148 us instead of 118, one prompt of 16,384 2.0 ms
// instead of 1.5, single tokens behind a shared prefix 40.5 us instead of 36;
// of few rows they cost nothing that shows.  Rounded weights are what their sum
// adds up, too: a result lies between the values whatever the rounding.
//
// What bounds it, on an MI355X whose large copies run at 4.85 TB/s and whose
// large matrix products at 1,150 (fp16) to 1,210 (bf16) TFLOP/s:
//   single tokens: memory.  96 sequences of up to 4,095 positions (32 heads on
//     8 of 64, 421 MB of keys and values) 86 us, 4.9 TB/s; one sequence of
//     65,521 positions (20 on 5 of 128, 168 MB) 31 us, 5.4 TB/s, and 8 to join.
//   prompts: a SIMD's matrix and vector work, which overlap in part only (two
//     waves that alternate them take the matrix time and 0.4 of the vector
//     time).  One prompt of 16,384 tokens (20 on 5 of 128, bf16) 1.47 to 1.55
//     ms, 890 to 935 TFLOP/s; in a run of 1.64 ms with counters (838 TFLOP/s)
//     the matrix cores were busy 42% of the cycles, at 1.9 GHz.  A workgroup of
//     256 rows, twice the rows a wave and half the LDS reads a product, took
//     1.70 ms: one wave a SIMD hides less.
//   small calls: latency.  A workgroup needs 3 to 5 us to find its range and
//     have its first tiles, two launches 9 us of the host.
#include "common.h"
#include "paged.h"
#include "paged_plan.h"

namespace terhip {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
#define TER_LDS __attribute__((address_space(3)))

// Uniform reads: of tables in memory through the scalar cache (nothing in the
// launch writes them), of LDS into a scalar register.
struct ConstInts {
    const int32_t* p;
    __device__ int operator[](long long i) const {
        return *(const __attribute__((address_space(4))) int32_t*)(size_t)(p + i);
    }
};
// What a workgroup keeps of the batch in LDS: units before each sequence, row
// boundaries (within [0, n_rows]) and PagedSeq::base.
struct Seqs {
    int *before, *row0, *base;
    int n;
    __device__ Seqs(int* p, int n_seq) : before(p), row0(p + n_seq + 1), base(p + 2 * n_seq + 2), n(n_seq) {}
    static __device__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
    __device__ PagedSeq operator[](int b) const {
        const int r0 = row0[b], r1 = row0[b + 1], k = base[b];
        return {uniform(r0), max(uniform(r1) - uniform(r0), 0), uniform(k)};
    }
    // The first sequence whose units end behind u: 64 looked at together.
    __device__ int find(int u) const {
        const int lane = threadIdx.x & 63;
        int lo = 0, step = 1;
        if (n > 64) {
            step = (n + 63) / 64;
            const int i = (lane + 1) * step;
            lo = step * __builtin_popcountll(__ballot(i < n && before[min(i, n)] <= u));
        } else {
            step = 64;
        }
        lo += __builtin_popcountll(__ballot(lane < step && lo + lane + 1 < n && before[min(lo + lane + 1, n)] <= u));
        return uniform(lo);
    }
};

template <typename T>
struct Elem;
template <>
struct Elem<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    // Weights below 2^-14 lose bits in fp16: with this added to the exponent
    // the largest weight is 2^8 .. 2^15 (paged_tile's kSlack) and those 2^-22
    // of it are still exact to 11 bits.
    static constexpr float kOffset = 8.f;
    static __device__ f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ f32x4 mma16k16(v4 a, v4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
    static __device__ float add(v2 e, float l) { return __builtin_amdgcn_fdot2(e, v2{1, 1}, l, false); }
    static __device__ v4 read_tr(const TER_LDS char* p) {
        typedef __fp16 h4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((TER_LDS h4*)p));
    }
    static constexpr unsigned kExp = 0x7C00u;  // exponent bits: all set in infinities and NaN
};
template <>
struct Elem<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    typedef short s4 __attribute__((ext_vector_type(4)));
    // Values may be near binary32's largest: with weights of at most 2^-25 no
    // sum of 2^20 of them leaves it, and weights have 2^-94 to go.
    static constexpr float kOffset = -32.f;
    static __device__ f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ f32x4 mma16k16(v4 a, v4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
    }
    static __device__ float add(v2 e, float l) { return __builtin_amdgcn_fdot2_f32_bf16(e, v2{1, 1}, l, false); }
    static __device__ v4 read_tr(const TER_LDS char* p) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((TER_LDS v4*)p);
    }
    static constexpr unsigned kExp = 0x7F80u;
};

// 16 bytes a lane from memory straight to LDS at lds_off + 16 * lane.  Inline
// asm without outputs: the compiler's own wait insertion would make every LDS
// read wait for the loads of the next tile; the waits are explicit instead.
// (Also the one that hardware does not enforce: a buffer load reads its
// descriptor five wait states or more after a lane read wrote a part of it.
// Behind fewer it may be bounded by the size of another load.)
// kOnce: read by nobody else, so not kept in the caches.
template <bool kOnce>
__device__ __forceinline__ void load_to_lds(u32x4 rsrc, unsigned voff, unsigned lds_off) {
    if constexpr (kOnce)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
                     :
                     : "s"(lds_off), "v"(voff), "s"(rsrc)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(lds_off), "v"(voff), "s"(rsrc)
                     : "memory", "m0");
}
// Waits until at most N loads are in flight, and for this wave's LDS reads.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier_only() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// One key tile in LDS: 64 rows of K, then 64 of V, HD * 2 bytes each, their
// 16-byte pieces permuted within the row so that the operand reads below hit
// all banks: piece p of row r is at p ^ swizzle(r).
template <int HD>
struct Tile {
    static constexpr int ROW = HD * 2;
    static constexpr int V = kPagedKeys * ROW;
    static constexpr int BYTES = 2 * V;
    static constexpr int RPI = 1024 / ROW;   // rows a load instruction fills
    static constexpr int NI = 16 / RPI;      // instructions for a wave's 16 rows of K or V
    static constexpr int PIECES = ROW / 16;
    // K operands: 16 or 32 rows, one piece of each
    static __device__ int swizzle_k(int r) { return HD == 128 ? r & 15 : (r >> 1) & 7; }
    // V operands: 64 bytes of each of four rows (transposing reads)
    static __device__ int swizzle_v(int r) { return HD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }
};

// The sign bits of the halves of y that hold infinities or NaN (all exponent
// bits set: adding the lowest one carries into the sign), and y without them.
template <typename T>
__device__ __forceinline__ unsigned odd_halves(unsigned y) {
    constexpr unsigned E1 = Elem<T>::kExp, E2 = E1 | E1 << 16, one = E1 & (0u - E1);
    return ((y & E2) + (one | one << 16)) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ unsigned without_odd(unsigned y) {
    const unsigned s = odd_halves<T>(y);
    return y & ~((s - (s >> 15)) | s);
}

// Adds the odd ones of four values to four sums, where the row sees them.
template <typename T, class V>
__device__ __forceinline__ void add_odd(V& sums, int i, u32x2 y, bool sees) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const unsigned short u = (unsigned short)(y[m >> 1] >> (16 * (m & 1)));
        if (sees && (u & Elem<T>::kExp) == Elem<T>::kExp) sums[i + m] += (float)__builtin_bit_cast(T, u);
    }
}
// What sums are multiplied by when their offset changes by x <= 0: never zero,
// which would turn infinite ones into NaN.
__device__ __forceinline__ float shrink(float x) { return fmaxf(__builtin_amdgcn_exp2f(x), 1.17549435e-38f); }

// An MFMA's result may be read by another kind of instruction only some wait
// states later (up to 20), which hardware does not enforce and the compiler
// fills.  It has left out the wait where the reader is the first instruction
// behind a branch (an element of the scores read as it was before), so scores
// pass through here before their maximum, and sums before they are multiplied
// or stored.  (tests/test_paged_waits.py checks the built code.)
template <class V>
__device__ __forceinline__ void settle(V& x) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(x));
}
// (one wait for all of them)
template <class V, int N>
__device__ __forceinline__ void settle_all(V (&x)[N]) {
    static_assert(N == 2 || N == 4 || N == 8, "sums of a row");
    if constexpr (N == 2)
        asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(x[0]), "+v"(x[1]));
    else if constexpr (N == 4)
        asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
    else
        asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"
                     : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]));
}

// Whether all sums are finite.
template <class V, int N>
__device__ __forceinline__ bool all_finite(const V (&x)[N]) {
    float m = 0.f;
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int i = 0; i < (int)(sizeof(V) / 4); i += 2)
            m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(x[d][i]), fabsf(x[d][i + 1])), m);
    return m < __builtin_inff();
}

__device__ __forceinline__ bool minus_zero(float x) { return __builtin_bit_cast(unsigned, x) == 0x80000000u; }

// Four elements of a row's partial results, added up.  Beside its sums one has
// their offset and the sum of their weights, or (a far level, see there) the
// score that was subtracted and minus that sum.  An infinite offset: it has no
// weights, and -0 as their sum if the row sees no position of the range at all
// (such sums add up to -0 among themselves only).
template <typename T>
struct PartSum {
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    float l = -0.f, ref = 0.f, off = __builtin_inff();
    __device__ __forceinline__ void add(f32x4 v, f32x2 st, float scale2) {
        const float inf = __builtin_inff();
        // (a sum that is NaN has any sign; the result is NaN with either)
        const bool far = __builtin_signbit(st[1]) && st[0] != inf;
        const float r = far ? st[0] : 0.f, o = far ? Elem<T>::kOffset : st[0], lv = far ? -st[1] : st[1];
        // 2^d takes sums to the new level; the larger level's stay.  (Never
        // less than 2^-126, as in shrink, of which no finite sum is left.)
        float d = __builtin_fmaf(ref - r, scale2, -off) + o;
        d = off == inf ? -inf : d;
        const float f = __builtin_amdgcn_exp2f(fmaxf(-fabsf(d), -126.f)), f0 = d < 0.f ? f : 1.f, f1 = d < 0.f ? 1.f : f;
        l = l * f0 + lv * f1;
        y = y * f0 + v * f1;
        ref = d < 0.f ? r : ref;
        off = d < 0.f ? o : off;
    }
    __device__ __forceinline__ f32x2 stats() const { return ref != 0.f ? f32x2{ref, -l} : f32x2{off, l}; }
    __device__ __forceinline__ typename Elem<T>::v4 result() const {
        const float inv = minus_zero(l) ? 0.f : 1.f / l;
        return {(T)(y[0] * inv), (T)(y[1] * inv), (T)(y[2] * inv), (T)(y[3] * inv)};
    }
};

// What is computed from x behind here is not moved in front of it.  Rows of
// either kind start so: with the places of their lanes in LDS computed once for
// all segments, the kernels kept both kinds' in registers, and at head_dim 64,
// with 168 of them, some went to scratch memory (96 single tokens 91 us instead
// of 85).
__device__ __forceinline__ void hide(int& x) { asm volatile("" : "+v"(x)); }

// A segment's work as one workgroup sees it (all uniform).
struct Work {
    int kv, kv_end;      // first position of the segment's key tile 0; positions from kv_end on are zeros
    int tok0, n_tok;     // first token row (packed), tokens of the row tile
    int rows;            // n_tok * group
    int seq;             // -1: the prefix, rows of any sequence
    int row0, base;      // of the sequence
    int kvh;
    int j0, j1;          // key tiles
    int dst;             // 0: out; 1: a slot; 2: whole rows
    const int32_t* table;
    float* slot;
    float* slot_stats;
};

template <typename T, int HD>
struct Kernel {
    typedef Elem<T> E;
    typedef typename E::v8 v8;
    typedef typename E::v4 v4;
    typedef typename E::v2 v2;
    typedef Tile<HD> L;
    // Two stages of the ring, and the workgroups of a CU that registers (and,
    // at head_dim 128, LDS) leave room for.  (More stages at head_dim 64 made
    // no difference: 3 instead of 2, batches of single tokens within 1%.)
    static constexpr int PER_CU = HD == 128 ? 2 : 3;
    static constexpr int RING = 2 * L::BYTES;
    // An offset stays while the largest weight is at most 2^kSlack above its start
    static constexpr float kSlack = 7.f;

    // What a row's scores x (before their scaling) are turned into weights
    // with: 2^(x scale2 + off), off near -max x scale2.  That product is
    // rounded, by 2^-4 below 2^20, but by whole units from 2^24 on, and the
    // largest weight would be that far from where it belongs, up to infinite
    // or zero.  From 2^20 on ("far") the weights are 2^((x - ref) scale2 +
    // kOffset) with the largest score itself as ref: x - ref is exact near it.
    // A far row looks at its level for every score: what rows need that are
    // not is then one comparison.
    struct Level {
        float lim = -__builtin_inff();  // nothing to do while no score is above this
        float off = -0.f;               // far: ref; -0 while all scores are -infinity (masked or not: their
                                        //   weights are zero with any offset, and no other level has this one)
        __device__ bool far() const { return lim == -__builtin_inff() && !minus_zero(off); }
        // For scores above lim, mx the largest: to the level that it asks for.
        // Returns what sums so far are to be multiplied by.  (Constants pass
        // through asm: held in registers for this path, which is rarely taken,
        // they cost more elsewhere.)
        __device__ float move(float mx, float scale2) {
            float k = E::kOffset, slack = kSlack;
            asm volatile("" : "+v"(k), "+v"(slack), "+v"(scale2));
            const bool was = far(), none = minus_zero(off);
            if (!(mx > (was ? off : lim))) return 1.f;
            const float t = mx * scale2, ref = was ? off : 0.f, from = was ? k : off;
            const bool f = fabsf(t) >= 1048576.f && mx < __builtin_inff();
            const float to = f ? k : k - t;
            lim = f ? -__builtin_inff() : __builtin_fmaf(slack, __builtin_amdgcn_rcpf(scale2), mx);
            off = f ? mx : to;
            return none ? 1.f : shrink(__builtin_fmaf(ref - (f ? mx : 0.f), scale2, -from) + to);
        }
        // A partial result's two numbers, with l for the sum of its weights.
        __device__ f32x2 stats(bool sees, float l) const {
            const bool none = minus_zero(off);
            return f32x2{none ? __builtin_inff() : off, none ? (sees ? l : -0.f) : far() ? -l : l};
        }
    };

    // ---- loads: wave w takes rows 16 w .. 16 w + 15 of K and V
    struct Loader {
        unsigned row, kp, vp;  // byte offset of this lane's first row, its pieces of K and V there
        unsigned lds;
        __device__ void init(const PagedAttendArgs& a, unsigned lds_off, int wave, int lane) {
            lds = lds_off + wave * 16 * L::ROW;
            const int r0 = lane / L::PIECES, p = lane % L::PIECES;
            row = r0 * a.c.pos_stride;
            kp = (p ^ L::swizzle_k(r0)) * 16;
            vp = (p ^ L::swizzle_v(r0)) * 16;
        }
        // (instruction i: rows i * RPI further on, whose K swizzle differs in
        // one bit or two, whose V swizzle is the same)
        __device__ __forceinline__ unsigned k_at(const PagedAttendArgs& a, int i) const {
            return (kp ^ (L::swizzle_k(i * L::RPI) * 16)) + (row + i * L::RPI * a.c.pos_stride);
        }
        __device__ __forceinline__ unsigned v_at(const PagedAttendArgs& a, int i) const {
            return vp + (row + i * L::RPI * a.c.pos_stride);
        }
        // Where the next 64 groups of 16 positions are, one a lane: offset
        // into K and V, bytes from there on that may be read (0: none).  From
        // these a step takes its own with three lane reads; found one by one,
        // by scalar loads and products, they took longer than its first
        // matrix products, and the loads were waited for with every LDS read.
        struct Groups {
            unsigned lo, hi, bytes;
        };
        // `stride` positions apart, from position `at` of the segment on.
        static __device__ __forceinline__ void locate(Groups& g, const PagedAttendArgs& a, const Work& s, int at,
                                                      int stride, int lane) {
            const int pos = s.kv + at + lane * stride;
            g = {0u, 0u, 0u};
            if (pos < s.kv_end) {
                const unsigned x = (unsigned)pos >> 4, i = a.page_magic ? __umulhi(x, a.page_magic) : x;
                const int page = gptr(s.table)[i];
                if (page >= 0 && page < a.c.n_pages) {
                    const unsigned long long o = (unsigned long long)page * (unsigned long long)a.c.page_stride +
                                                 (unsigned long long)(pos - (int)i * a.c.page_size) * (unsigned)a.c.pos_stride +
                                                 (unsigned long long)s.kvh * (unsigned)a.c.head_stride;
                    g.lo = (unsigned)o;
                    g.hi = (unsigned)(o >> 32);
                    g.bytes = (unsigned)(min(s.kv_end - pos, 16) - 1) * a.c.pos_stride + L::ROW;
                }
            }
            asm volatile("" : "+v"(g.lo), "+v"(g.hi), "+v"(g.bytes));  // (waited for here)
        }
        // A load of 2 * NI instructions, K first, to be issued one by one.
        struct Pending {
            u32x4 kr, vr;
            unsigned to;
        };
        __device__ __forceinline__ Pending prepare(const PagedAttendArgs& a, const Groups& g, int i, int stage) const {
            const unsigned long long o = (unsigned)__builtin_amdgcn_readlane(g.lo, i) |
                                         (unsigned long long)(unsigned)__builtin_amdgcn_readlane(g.hi, i) << 32;
            const unsigned bytes = (unsigned)__builtin_amdgcn_readlane(g.bytes, i);
            const unsigned long long kb = (unsigned long long)a.c.k + o, vb = (unsigned long long)a.c.v + o;
            return {{(unsigned)kb, (unsigned)(kb >> 32) & 0xFFFFu, bytes, 0x00020000u},
                    {(unsigned)vb, (unsigned)(vb >> 32) & 0xFFFFu, bytes, 0x00020000u},
                    lds + stage * L::BYTES};
        }
        template <bool kOnce>
        __device__ __forceinline__ void piece(const PagedAttendArgs& a, const Pending& p, int i) const {
            if (i < L::NI)
                load_to_lds<kOnce>(p.kr, k_at(a, i), p.to + i * 1024);
            else
                load_to_lds<kOnce>(p.vr, v_at(a, i - L::NI), p.to + L::V + (i - L::NI) * 1024);
        }
        template <bool kOnce>
        __device__ __forceinline__ void issue(const PagedAttendArgs& a, const Groups& g, int at, int stage) const {
            const Pending p = prepare(a, g, at, stage);
#pragma unroll
            for (int i = 0; i < 2 * L::NI; ++i) piece<kOnce>(a, p, i);
        }
    };

    // Positions (from the segment's first one on) that packed token row t of a segment sees.
    static __device__ int limit_of(const Work& s, int t, const Seqs& sq) {
        int base = s.base, r0 = s.row0;
        if (s.seq < 0) {
            int lo = 0, hi = sq.n;  // row0[lo] <= t < row0[hi]
            if (sq.row0[0] > t || sq.row0[hi] <= t) return 0;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (sq.row0[mid] <= t)
                    lo = mid;
                else
                    hi = mid;
            }
            base = sq.base[lo];
            r0 = sq.row0[lo];
        }
        return min(max(base + t - r0 + 1, 0), s.kv_end) - s.kv;
    }

    // Pointers of one row's partial sums.
    static __device__ float* sums_of(const PagedAttendArgs& a, const Work& s, int r, int t, int h) {
        return s.dst == 1 ? s.slot + (long long)r * HD
                          : a.whole + ((long long)(s.seq < 0 ? a.b.n_rows : 0) + t) * a.nh * HD + (long long)h * HD;
    }
    static __device__ float* stats_of(const PagedAttendArgs& a, const Work& s, int r, int t, int h) {
        return s.dst == 1 ? s.slot_stats + 2 * r
                          : a.whole_stats + (((long long)(s.seq < 0 ? a.b.n_rows : 0) + t) * a.nh + h) * 2;
    }

    // ---- up to 128 rows: wave w takes rows 32 w .. 32 w + 31 against the 64
    // keys of a tile.  S^T = K Q^T, so a lane's scores are all of query row
    // lane % 32: its statistics need no exchange but one with lane ^ 32, and S^T
    // in the accumulator layout is, up to the order of the keys, the operand of
    // O^T = V^T P^T.  That order is the same for V's operand: transposing
    // reads of four keys each.
    static __device__ __forceinline__ void rows128(const PagedAttendArgs& a, const Work& s, const Loader& ld,
                                                   TER_LDS char* ring, const Seqs& sq, int* shared, int& tick,
                                                   int w, int lane) {
        hide(lane);
        int* const lows = shared;                 // [kWaves]
        int* const flag = shared + kWaves;        // [2] the tick at which a tile of a stage held odd values
        const int half = lane >> 5, col = lane & 31;
        const int r = 32 * w + col, tok = r / a.group, t = s.tok0 + tok;
        const int h = s.kvh * a.group + (r - tok * a.group);
        const bool live = r < s.rows;
        const int lim = live ? limit_of(s, t, sq) : 0;
        v8 q[HD / 16];
        {
            const char* p = a.q + (live ? (long long)t * a.q_stride + (long long)h * L::ROW : 0) + half * 16;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) q[c] = *gptr(reinterpret_cast<const v8*>(p + c * 32));
        }
        // What every row sees, and what none of this wave's sees more than.
        // (On the prefix: all of it, or as if some row saw nothing.)
        int lo, hi;
        if (s.seq >= 0) {
            lo = min(max(s.base + s.tok0 - s.row0 + 1, 0), s.kv_end) - s.kv;
            hi = 32 * w < s.rows ? min(max(s.base + s.tok0 + (min(32 * w + 32, s.rows) - 1) / a.group - s.row0 + 1, 0),
                                       s.kv_end) - s.kv
                                 : 0;
        } else {
            const bool some = __ballot(live && lim < s.kv_end) != 0;
            if (lane == 0) lows[w] = some;  // (one lane: stores of several lanes to one place have no order)
            __syncthreads();
            lo = __builtin_amdgcn_readfirstlane(lows[0] | lows[1] | lows[2] | lows[3]) ? 0 : s.kv_end;
            hi = 32 * w < s.rows ? s.kv_end : 0;
        }

        f32x16 o[HD / 32];
        float l;
        Level level;

        // LDS offsets: K pieces of row col (+ 32 by offset); V rows of the
        // lane's transposing read
        // (pieces further on by exclusive or: rows and stages are multiples of
        // 128 bytes)
        const int ka = col * L::ROW + ((half ^ L::swizzle_k(col)) * 16);
        const int vr = 4 * half + ((lane & 15) >> 2);
        const int va = L::V + vr * L::ROW + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ L::swizzle_v(vr)) * 16) +
                       8 * (lane & 1);
        const auto mine = [&](int j) { return j * kPagedKeys + 16 * w; };
        // one tile ahead of the one in work
        typename Loader::Groups groups;
        int put = 0, todo = s.j0;
        auto group = [&]() {
            const int i = (todo - s.j0) & 63;
            if (i == 0) Loader::locate(groups, a, s, mine(todo), kPagedKeys, lane);
            ++todo;
            return i;
        };
        auto fetch = [&]() {
            if (todo < s.j1) {
                ld.template issue<false>(a, groups, group(), put);
                put ^= 1;
            }
        };
        // The same in pieces, spread over a step: a wave that issues all of
        // them at once waits a quarter of the step for the address unit.
        // (Behind the last tile they load what nobody reads, into a stage that is free.)
        typename Loader::Pending next;
        auto prepare = [&]() {
            next = ld.prepare(a, groups, group(), put);
            put ^= 1;
        };
        int stage = 0, j = s.j0;
        auto arrive = [&]() {  // tile j is in LDS
            wait_loads<0>();
            barrier_only();
        };
        // The same for a tile that some row does not see whole.  Values there
        // may be infinite or NaN, and a zero weight times those is NaN: they
        // are added to the sums of the rows that see them and set to zero in
        // LDS.  Each wave looks at the rows that it loaded.
        auto arrive_masked = [&]() {
            wait_loads<0>();
            TER_LDS char* const vt = ring + stage * L::BYTES + L::V;
            TER_LDS u32x4* const own = (TER_LDS u32x4*)(vt + w * 16 * L::ROW + lane * 16);
            unsigned odd = 0;
#pragma unroll
            for (int i = 0; i < L::NI; ++i) {
                const u32x4 y = own[64 * i];
#pragma unroll
                for (int m = 0; m < 4; ++m) odd |= odd_halves<T>(y[m]);
            }
            ++tick;
            if (odd) flag[stage] = tick;
            wait_lds();
            barrier_only();
            if (__builtin_amdgcn_readfirstlane(flag[stage]) != tick) return;
            settle_all(o);
#pragma clang loop unroll(disable)
            for (int k = 0; k < kPagedKeys; ++k) {
                const bool sees = j * kPagedKeys + k < lim;
                const TER_LDS char* v = vt + k * L::ROW + 8 * half;
#pragma unroll
                for (int d = 0; d < HD / 32; ++d) {
                    // (elements 32 d .. 32 d + 31 of the row: four pieces in a row, swizzled or not)
                    const TER_LDS char* vd = v + ((4 * d) ^ L::swizzle_v(k)) * 16;
#pragma unroll
                    for (int i = 0; i < 16; i += 4) add_odd<T>(o[d], i, *(const TER_LDS u32x2*)(vd + 4 * i), sees);
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < L::NI; ++i) {
                u32x4 y = own[64 * i];
#pragma unroll
                for (int m = 0; m < 4; ++m) y[m] = without_odd<T>(y[m]);
                own[64 * i] = y;
            }
            __syncthreads();
        };
        // One tile, its two halves of 32 keys staggered: while the matrix
        // cores form the second half's scores the vector units turn the first
        // half's into weights, and so on with the value products.  (A wave
        // issues in order, so the two kinds have to alternate in its code:
        // the scheduling groups below.)
        auto step = [&](auto masked) {
            constexpr bool kMasked = decltype(masked)::value;
            const int kt = (int)(size_t)ring + stage * L::BYTES + ka, vt = (int)(size_t)ring + stage * L::BYTES + va;
            f32x16 x[2];
            v8 k[HD / 16], p[2][2], y[2][HD / 32];
            float al = 1.f, wo;
            auto read_k = [&](int b, int c) { k[c] = *((const TER_LDS v8*)(size_t)(unsigned)(kt ^ (32 * c)) + b * 2 * L::ROW); };
            auto scores = [&](int b, int c) { x[b] = E::mma32(k[c], q[c], x[b]); };
            auto read_v = [&](int c, int d) {
                const TER_LDS char* v = (const TER_LDS char*)(size_t)(unsigned)(vt ^ (64 * d)) + c * 16 * L::ROW;
                const v4 y0 = E::read_tr(v), y1 = E::read_tr(v + 8 * L::ROW);
                y[c & 1][d] = __builtin_shufflevector(y0, y1, 0, 1, 2, 3, 4, 5, 6, 7);
            };
            auto value = [&](int c, int d) {
                o[d] = E::mma32(y[c & 1][d], p[c >> 1][c & 1], o[d]);
            };
            // The offset for half b; al is what sums so far are to be multiplied by.
            auto decide = [&](int b) {
                settle(x[b]);
                if (kMasked) {
                    const int n = lim - j * kPagedKeys - 32 * b - 4 * half;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (8 * (i >> 2) + (i & 3) >= n) x[b][i] = -__builtin_inff();
                }
                float mx = x[b][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[b][i]);
                mx = fmaxf(mx, lane_xor32(mx));
                const bool look = __ballot(mx > level.lim) != 0;
                wo = level.off;
                if (look) {
                    al = level.move(mx, a.scale2);
                    wo = level.off;
                    if (__ballot(level.far())) {
                        const float ref = level.far() ? level.off : 0.f;
                        wo = level.far() ? E::kOffset : level.off;
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[b][i] -= ref;
                    }
                }
                return look;
            };
            auto rescale = [&]() {
                l *= al;
                settle_all(o);
#pragma unroll
                for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= al;
            };
            auto weight = [&](int b, int i) {  // elements i, i + 1
                const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][i], a.scale2, wo));
                const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][i + 1], a.scale2, wo));
                const v2 e = {(T)e0, (T)e1};
                p[b][i >> 3][i & 7] = e[0];
                p[b][i >> 3][(i & 7) + 1] = e[1];
                l = E::add(e, l);
            };

#pragma unroll
            for (int c = 0; c < HD / 16; ++c) read_k(0, c);
            __builtin_amdgcn_sched_barrier(0);
            prepare();
#pragma unroll
            for (int i = 0; i < 16; ++i) x[0][i] = x[1][i] = 0.f;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
                scores(0, c);
                read_k(1, c);
                if (c % 4 == 2) ld.template piece<false>(a, next, c / 4);  // NI / 2
                __builtin_amdgcn_sched_barrier(0);
            }
            if (decide(0)) rescale();
            __builtin_amdgcn_sched_barrier(0);
            // (in this order: two weights for each of eight places in the code)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i % (128 / HD) == 0) {
                    const int c = i / (128 / HD);
                    scores(1, c);
                    if (c % 2 == 0) ld.template piece<false>(a, next, L::NI / 2 + c / 2);  // NI
                    if (c >= HD / 32) read_v(0, c - HD / 32);
                }
                weight(0, 2 * i);
                __builtin_amdgcn_sched_barrier(0);
            }
            // (weights are formed here, not where they are used)
            asm volatile("" : "+v"(p[0][0]), "+v"(p[0][1]), "+v"(l));
            __builtin_amdgcn_sched_barrier(0);
            const bool grown = decide(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) read_v(1, d);
            const float sum = l;
            l = 0.f;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i % (128 / HD) == 0) {
                    const int c = i / 4, d = i / (128 / HD) % (HD / 32);
                    value(c, d);
                    read_v(2 + c, d);
                    if (i % (16 / L::NI) == 2) ld.template piece<false>(a, next, L::NI * 3 / 2 + i / (16 / L::NI));  // NI / 2
                }
                weight(1, 2 * i);
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("" : "+v"(p[1][0]), "+v"(p[1][1]), "+v"(l));
            __builtin_amdgcn_sched_barrier(0);
            const float more = l;
            l = sum;
            if (grown) rescale();
            l += more;
#pragma unroll
            for (int c = 2; c < 4; ++c)
#pragma unroll
                for (int d = 0; d < HD / 32; ++d) value(c, d);
        };
        // tiles that every row sees whole, then the others
        for (int full = min(s.j1, max(s.j0, lo / kPagedKeys));; full = s.j0) {
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
            l = 0.f;
            level = Level{};
            fetch();
            for (; j < full; ++j, stage ^= 1) {
                arrive();
                step(std::false_type{});
            }
            for (; j < s.j1; ++j, stage ^= 1) {
                arrive_masked();
                if (j * kPagedKeys < hi)
                    step(std::true_type{});
                else
                    fetch();  // no row of this wave sees it
            }
            wait_loads<0>();
            settle_all(o);
            if (full == s.j0) break;
            // Infinite or NaN: once more, with every tile's values looked at
            const bool odd = __ballot(live && !all_finite(o)) != 0;
            if (lane == 0) lows[w] = odd;
            __syncthreads();
            if (!__builtin_amdgcn_readfirstlane(lows[0] | lows[1] | lows[2] | lows[3])) break;
            put = stage = 0;
            j = todo = s.j0;
        }
        l += lane_xor32(l);
        if (!live) return;
        if (s.dst == 0) {
            const float inv = lim > 0 ? 1.f / l : 0.f;
            char* p = a.out + (long long)t * a.out_stride + (long long)h * L::ROW + half * 8;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const v4 y = {(T)(o[d][i] * inv), (T)(o[d][i + 1] * inv), (T)(o[d][i + 2] * inv),
                                  (T)(o[d][i + 3] * inv)};
                    *gptr(reinterpret_cast<v4*>(p + 64 * d + 4 * i)) = y;
                }
            return;
        }
        float* p = sums_of(a, s, r, t, h) + half * 4;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *gptr(reinterpret_cast<f32x4*>(p + 32 * d + 2 * i)) =
                    f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
        if (half == 0)
            *gptr(reinterpret_cast<f32x2*>(stats_of(a, s, r, t, h))) = level.stats(lim > s.j0 * kPagedKeys, l);
    }

    // ---- up to 16 rows, 16 keys at a time.  kSolo: by one wave.  Else wave w
    // takes keys 16 w .. 16 w + 15 of every tile; no wave waits for another
    // before their sums meet in LDS at the end.
    template <bool kSolo>
    static __device__ __forceinline__ void rows16(const PagedAttendArgs& a, const Work& s, const Loader& ld,
                                                  TER_LDS char* ring, const Seqs& sq, int w, int lane) {
        hide(lane);
        const int quad = lane >> 4, col = lane & 15;
        const int tok = col / a.group, t = s.tok0 + tok, h = s.kvh * a.group + (col - tok * a.group);
        const bool live = col < s.rows;
        const int lim = live ? limit_of(s, t, sq) : 0;
        const int first = s.j0 * kPagedKeys + (kSolo ? 0 : 16 * w), stride = kSolo ? 16 : kPagedKeys;
        const int n = kSolo ? max(1, (min(s.j1 * kPagedKeys, s.kv_end - s.kv) - first + 15) / 16) : s.j1 - s.j0;
        typename Loader::Groups groups;
        int put = 0, todo = 0;
        auto fetch = [&]() {
            if (todo < n) {
                if ((todo & 63) == 0) Loader::locate(groups, a, s, first + todo * stride, stride, lane);
                ld.template issue<true>(a, groups, todo & 63, put);
                ++todo;
                put ^= 1;
            }
        };
        fetch();
        fetch();
        v8 q[HD / 32];
        {
            const char* p = a.q + (live ? (long long)t * a.q_stride + (long long)h * L::ROW : 0) + quad * 16;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) q[c] = *gptr(reinterpret_cast<const v8*>(p + c * 64));
        }
        int lo = 0;  // what every row sees (on the prefix: all of it or nothing)
        if (s.seq >= 0)
            lo = min(max(s.base + s.tok0 - s.row0 + 1, 0), s.kv_end) - s.kv;
        else if (__ballot(live && lim < s.kv_end) == 0)
            lo = s.kv_end;
        f32x4 o[HD / 16];
        float l;
        Level level;
        const int kr = 16 * w + col, vr = 16 * w + 4 * quad + (col >> 2);
        int ka[HD / 32], va[HD / 16];
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) ka[c] = kr * L::ROW + (((4 * c + quad) ^ L::swizzle_k(kr)) * 16);
#pragma unroll
        for (int d = 0; d < HD / 16; ++d)
            va[d] = L::V + vr * L::ROW + (((2 * d + ((lane & 3) >> 1)) ^ L::swizzle_v(vr)) * 16) + 8 * (lane & 1);
        for (bool again = false;; again = true) {
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
            l = 0.f;
            level = Level{};
            // The queries, which the compiler waits for, have to be here before the
            // loop: inside it that wait would be one for all loads in flight.
            wait_loads<0>();
            int stage = 0;
            for (int i = 0; i < n; ++i, stage ^= 1) {
                // the next keys' loads may still be in flight
                if (i + 1 < n)
                    wait_loads<2 * L::NI>();
                else
                    wait_loads<0>();
                const int at = first + i * stride;
                TER_LDS char* tile = ring + stage * L::BYTES;
                if (at + 16 > lo) {  // (as in rows128, by each wave for its own keys)
                    TER_LDS u32x4* const mine = (TER_LDS u32x4*)(tile + L::V + w * 16 * L::ROW + lane * 16);
                    unsigned odd = 0;
#pragma unroll
                    for (int i = 0; i < L::NI; ++i) {
                        const u32x4 y = mine[64 * i];
#pragma unroll
                        for (int m = 0; m < 4; ++m) odd |= odd_halves<T>(y[m]);
                    }
                    if (__ballot(odd != 0)) {
                        settle_all(o);
#pragma clang loop unroll(disable)
                        for (int k = 0; k < 16; ++k) {
                            const TER_LDS char* v = tile + L::V + (16 * w + k) * L::ROW + (quad & 1) * 8;
#pragma unroll
                            for (int d = 0; d < HD / 16; ++d)
                                add_odd<T>(o[d], 0,
                                           *(const TER_LDS u32x2*)(v + ((2 * d + (quad >> 1)) ^ L::swizzle_v(16 * w + k)) * 16),
                                           at + k < lim);
                        }
#pragma unroll
                        for (int i = 0; i < L::NI; ++i) {
                            u32x4 y = mine[64 * i];
#pragma unroll
                            for (int m = 0; m < 4; ++m) y[m] = without_odd<T>(y[m]);
                            mine[64 * i] = y;
                        }
                        wait_lds();
                    }
                }
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                v8 k[HD / 32];
                v4 y[HD / 16];
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) k[c] = *(const TER_LDS v8*)(tile + ka[c]);
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) y[d] = E::read_tr(tile + va[d]);
                __builtin_amdgcn_sched_barrier(0);  // all reads in flight before the first product
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) x = E::mma16(k[c], q[c], x);
                settle(x);
                if (at + 16 > lo) {
                    const int see = lim - at - 4 * quad;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k >= see) x[k] = -__builtin_inff();
                }
                float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                mx = fmaxf(mx, lane_xor16(mx));
                mx = fmaxf(mx, lane_xor32(mx));
                float wo = level.off;
                if (__ballot(mx > level.lim)) {
                    const float al = level.move(mx, a.scale2);
                    l *= al;
                    settle_all(o);
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d) o[d] *= al;
                    wo = level.off;
                    if (__ballot(level.far())) {
                        const float ref = level.far() ? level.off : 0.f;
                        wo = level.far() ? E::kOffset : level.off;
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] -= ref;
                    }
                }
                v4 p, rest;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.scale2, wo));
                    l += e;
                    p[i] = (T)e;
                    rest[i] = (T)(e - (float)p[i]);
                }
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) o[d] = E::mma16k16(y[d], p, o[d]);
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) o[d] = E::mma16k16(y[d], rest, o[d]);
                wait_lds();  // these keys' reads are done: their place is free
                fetch();
            }
            settle_all(o);
            // Infinite or NaN: once more, with every key's values looked at
            if (again || !__ballot(live && !all_finite(o))) break;
            lo = -0x7FFFFFFF;
            put = todo = 0;
            fetch();
            fetch();
        }
        l += lane_xor16(l);
        l += lane_xor32(l);
        if (kSolo) {
            if (!live) return;
            if (s.dst == 0) {
                const float inv = lim > 0 ? 1.f / l : 0.f;
                char* p = a.out + (long long)t * a.out_stride + (long long)h * L::ROW + quad * 8;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) {
                    const v4 y = {(T)(o[d][0] * inv), (T)(o[d][1] * inv), (T)(o[d][2] * inv), (T)(o[d][3] * inv)};
                    *gptr(reinterpret_cast<v4*>(p + 32 * d)) = y;
                }
            } else {
                float* p = sums_of(a, s, col, t, h) + 4 * quad;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) *gptr(reinterpret_cast<f32x4*>(p + 16 * d)) = o[d];
                if (quad == 0)
                    *gptr(reinterpret_cast<f32x2*>(stats_of(a, s, col, t, h))) = level.stats(lim > first, l);
            }
            return;
        }
        // the waves' sums: [wave][row][HD], then [wave][row][2]
        __syncthreads();
        TER_LDS float* sums = (TER_LDS float*)ring;
        TER_LDS float* stats = sums + kWaves * 16 * HD;
        if (live) {
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
                *(TER_LDS f32x4*)(sums + (w * 16 + col) * HD + 16 * d + 4 * quad) = o[d];
            if (quad == 0) *(TER_LDS f32x2*)(stats + (w * 16 + col) * 2) = level.stats(lim > first, l);
        }
        __syncthreads();
        for (int i = w * 64 + lane; i < s.rows * (HD / 4); i += kThreads) {
            const int r = i / (HD / 4), e = (i - r * (HD / 4)) * 4;
            PartSum<T> sum;
#pragma unroll
            for (int k = 0; k < kWaves; ++k)
                sum.add(*(TER_LDS f32x4*)(sums + (k * 16 + r) * HD + e), *(TER_LDS f32x2*)(stats + (k * 16 + r) * 2), a.scale2);
            const int rt = s.tok0 + r / a.group, rh = s.kvh * a.group + r % a.group;
            if (s.dst == 0) {
                *gptr(reinterpret_cast<v4*>(a.out + (long long)rt * a.out_stride + (long long)rh * L::ROW + e * 2)) = sum.result();
            } else {
                *gptr(reinterpret_cast<f32x4*>(sums_of(a, s, r, rt, rh) + e)) = sum.y;
                if (e == 0) *gptr(reinterpret_cast<f32x2*>(stats_of(a, s, r, rt, rh))) = sum.stats();
            }
        }
    }
};

template <int kCtrl, int kRows>
__device__ __forceinline__ unsigned dpp_add(unsigned v) {
    return __builtin_elementwise_add_sat(
        v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xF, false));
}
// Inclusive prefix sum over the wave, saturating: within rows of 16 lanes, then
// the last lanes of the rows before.
__device__ __forceinline__ unsigned wave_prefix(unsigned v) {
    v = dpp_add<0x111, 0xF>(v);  // row_shr:1
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);  // row_bcast:15
    return dpp_add<0x143, 0xC>(v);  // row_bcast:31
}

// Fills sq; returns the units of the whole line.  They fit 31 bits if row0 does
// not decrease; a batch whose sequences overlap may have more: then none is done.
__device__ __forceinline__ int count_units(const PagedAttendArgs& a, const PagedLine& l, const Seqs& sq, int* tmp) {
    const int n = a.b.n_seq, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int each = (n + kThreads - 1) / kThreads, i0 = tid * each, i1 = min(n, i0 + each);
    unsigned sum = 0;
    for (int i = i0; i < i1; ++i) {
        const int r0 = gptr(a.b.row0)[i], r1 = gptr(a.b.row0)[i + 1];
        const PagedSeq s = paged_seq(r0, r1, gptr(a.b.kv_len)[i], a.b.n_rows, a.b.capacity);
        sq.row0[i] = s.r0;
        sq.base[i] = s.base;
        if (i == n - 1) sq.row0[n] = min(max(r1, 0), a.b.n_rows);
        sq.before[i] = (int)sum;
        sum = __builtin_elementwise_add_sat(sum, (unsigned)(paged_units(s, l.group, l.q, l.kv0) * a.nkv));
    }
    const unsigned inc = wave_prefix(sum);
    if (lane == 63) tmp[w] = (int)inc;
    __syncthreads();
    unsigned add = l.prefix_units + inc - sum, total = l.prefix_units;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        if (k < w) add += (unsigned)tmp[k];
        total = __builtin_elementwise_add_sat(total, (unsigned)tmp[k]);
    }
    if (total > 0x7FFFFFFFu) total = 0;
    for (int i = i0; i < i1; ++i) sq.before[i] += (int)add;
    if (tid == 0) sq.before[n] = (int)total;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane((int)total);
}

template <typename T, int HD>
__global__ __launch_bounds__(kThreads, (Kernel<T, HD>::PER_CU)) void paged_attend_kernel(PagedAttendArgs a) {
    typedef Kernel<T, HD> K;
    extern __shared__ __align__(1024) unsigned char lds[];
    int* tmp = reinterpret_cast<int*>(lds + K::RING);  // [kWaves + 2]
    const Seqs sq(tmp + kWaves + 2, a.b.n_seq);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TER_LDS char* ring = (TER_LDS char*)lds;

    PagedLine l = paged_line(a.group, a.tokens_log2, a.shared, a.b.n_rows, a.nkv);
    const int total = count_units(a, l, sq, tmp);
    if (a.shared && blockIdx.x == 0)
        for (int i = threadIdx.x; i <= a.b.n_seq; i += kThreads) gptr(a.before)[i] = sq.before[i];
    paged_cut(l, total, a.cuts_by);
    // neighbouring ranges on one XCD (blocks go round the 8 XCDs): they read the same keys
    // (blocks beyond the last range have the numbers behind it: each number once)
    const int chunk = (l.n_wg + 7) / 8, x = (int)(blockIdx.x % 8), y = (int)(blockIdx.x / 8);
    const int g = y < chunk ? x * chunk + y : 8 * chunk + x * (a.cuts_by.max_wg / 8 - chunk) + y - chunk;
    if (g >= l.n_wg) {
        if (threadIdx.x == 0) gptr(a.cuts)[8 * g] = 0;
        return;
    }

    PagedSeq q{};  // the sequence of the segment found last
    auto segment = [&](int u) {
        if (u < l.prefix_units) return paged_segment(l, u, a.nkv, 0, q, 0, 0);
        const int b = sq.find(u), b0 = sq.before[b], b1 = sq.before[b + 1];
        q = sq[b];
        return paged_segment(l, u, a.nkv, b, q, Seqs::uniform(b0), Seqs::uniform(b1));
    };
    typename K::Loader ld;
    ld.init(a, (unsigned)(size_t)ring, w, lane);
    int tick = 0;
    if (threadIdx.x < 2) tmp[kWaves + threadIdx.x] = 0;  // (a barrier comes before each segment)
    const int raw1 = paged_cut_at(l, g + 1);
    int u0 = paged_cut_at(l, g);
    PagedSegment sg = segment(u0);
    u0 = paged_snap(l, sg, u0);
    if (u0 == sg.start + sg.n && u0 < total) sg = segment(u0);
    int turn = -1;  // of a run of short segments: the wave whose turn it is
    for (int u = u0;;) {
        const int end = raw1 >= sg.start + sg.n ? sg.start + sg.n : paged_snap(l, sg, raw1);
        if (end <= u) {
            if (u == u0 && threadIdx.x == 0) gptr(a.cuts)[8 * g] = 0;
            break;
        }
        Work s;
        s.seq = sg.seq;
        s.kvh = sg.kvh;
        s.j0 = max(u - sg.start - kPagedLead, 0);
        s.j1 = sg.lead ? end - sg.start - kPagedLead : paged_key_tiles(q, 0, l.q, l.kv0);
        const bool whole = u == sg.start && end == sg.start + sg.n;
        if (sg.seq < 0) {
            s.tok0 = sg.tile << l.q;
            s.n_tok = min(a.b.n_rows - s.tok0, 1 << l.q);
            s.kv = 0;
            s.kv_end = a.shared;
            s.row0 = s.base = 0;
            s.table = a.b.pages;
        } else {
            const int i = sg.tile << l.q;
            s.tok0 = q.r0 + i;
            s.n_tok = min(q.n - i, 1 << l.q);
            s.kv = a.shared;
            s.kv_end = max(paged_limit(q, i + s.n_tok - 1, a.b.capacity), a.shared);
            s.row0 = q.r0;
            s.base = q.base;
            s.table = a.b.pages + (long long)sg.seq * a.b.pages_stride;
        }
        s.rows = s.n_tok * a.group;
        s.dst = !whole ? 1 : a.shared ? 2 : 0;
        const int slot = 2 * g + (u == sg.start ? 1 : 0);
        s.slot = a.slots + (long long)slot * a.slot_rows * HD;
        s.slot_stats = a.slot_stats + (long long)slot * a.slot_rows * 2;
        if (sg.lead == 0 && (u > u0 || raw1 > end)) {
            // short ones beside others: the waves take turns, each by itself
            if (turn < 0) __syncthreads();
            turn = (turn + 1) & (kWaves - 1);
            if (turn == w) K::template rows16<true>(a, s, ld, ring, sq, w, lane);
        } else {
            turn = -1;
            __syncthreads();  // the ring is free
            if (s.rows > kPagedFew)
                K::rows128(a, s, ld, ring, sq, tmp, tick, w, lane);
            else
                K::template rows16<false>(a, s, ld, ring, sq, w, lane);
        }
        if (u == u0 && threadIdx.x == 0) {  // what the joining kernel has to know of this cut
            const PagedParts p = paged_parts(l, sg.start, sg.n, sg.lead);
            *gptr(reinterpret_cast<i32x4*>(a.cuts + 8 * g)) = i32x4{u == sg.start ? 0 : s.rows, s.tok0, s.kvh, p.first};
            gptr(a.cuts)[8 * g + 4] = p.last;
        }
        u = end;
        if (u < sg.start + sg.n || u >= total) break;
        if (!paged_advance(l, sg, q, a.nkv)) sg = segment(u);
    }
}

// ---- joining.  A row takes HD / 4 threads, S groups of them every S-th partial
// result of the row.
template <typename T, int HD>
struct Join {
    static constexpr int TPR = HD / 4, GROUPS = kThreads / TPR;
    typedef typename Elem<T>::v4 v4;
    struct Lds {
        float sums[GROUPS][HD];
        f32x2 stats[GROUPS];
    };
    // Partial result i of n of a row: place(i, sums, stats).  All threads call
    // it; those of a row's first group return with the whole, `live` rows write it.
    template <class Place>
    static __device__ void row(Lds& lds, int S, int n, bool live, float scale2, Place place, char* out) {
        const int grp = threadIdx.x / TPR, e = (threadIdx.x % TPR) * 4, sub = grp & (S - 1);
        PartSum<T> t;
        if (live) {
            constexpr int U = 4;  // partial results in flight
            for (int i0 = sub; i0 < n; i0 += U * S) {
                f32x4 v[U];
                f32x2 st[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i0 + u * S >= n) break;
                    const float *ps, *pt;
                    place(i0 + u * S, ps, pt);
                    v[u] = *gptr(reinterpret_cast<const f32x4*>(ps + e));
                    st[u] = *gptr(reinterpret_cast<const f32x2*>(pt));
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i0 + u * S < n) t.add(v[u], st[u], scale2);
            }
        }
        if (S > 1) {
            __syncthreads();
            *reinterpret_cast<f32x4*>(&lds.sums[grp][e]) = t.y;
            if (e == 0) lds.stats[grp] = t.stats();
            __syncthreads();
            if (sub == 0)
                for (int k = 1; k < S; ++k)
                    t.add(*reinterpret_cast<const f32x4*>(&lds.sums[grp + k][e]), lds.stats[grp + k], scale2);
        }
        if (live && sub == 0) *gptr(reinterpret_cast<v4*>(out + e * 2)) = t.result();
    }
};

// Without a shared prefix: the rows of each segment that was cut, spread over
// the workgroups of its cuts (a.cuts, written by the ranges that begin there).
template <typename T, int HD>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedAttendArgs a) {
    typedef Join<T, HD> J;
    __shared__ typename J::Lds lds;
    const ConstInts cut{a.cuts + 8 * blockIdx.x};
    const int rows = cut[0], g = blockIdx.x;
    if (rows == 0) return;
    const int tok0 = cut[1], kvh = cut[2], first = cut[3], n = cut[4] - first + 1;
    int S = 1;
    while (S < J::GROUPS && 4 * S < n) S *= 2;
    const int per = J::GROUPS / S, grp = threadIdx.x / J::TPR;
    const int worker = (g - first - 1) * gridDim.y + blockIdx.y, workers = (n - 1) * gridDim.y;
    for (int r0 = worker * per; r0 < rows; r0 += workers * per) {
        const int r = r0 + grp / S, tok = r / a.group, t = tok0 + tok, h = kvh * a.group + r - tok * a.group;
        J::row(
            lds, S, n, r < rows, a.scale2,
            [&](int i, const float*& sums, const float*& stats) {
                const long long at = (long long)(2 * (first + i) + (i == 0 ? 1 : 0)) * a.slot_rows + r;
                sums = a.slots + at * HD;
                stats = a.slot_stats + at * 2;
            },
            a.out + (long long)t * a.out_stride + (long long)h * HD * 2);
    }
}

// With a shared prefix: each row's own positions and the prefix, either of
// which may have been cut.  A workgroup is one token row of one KV head.
template <typename T, int HD>
__global__ __launch_bounds__(kThreads) void paged_join_shared_kernel(PagedAttendArgs a) {
    typedef Join<T, HD> J;
    __shared__ typename J::Lds lds;
    const int t = blockIdx.x, kvh = blockIdx.y, q = a.tokens_log2;
    const int b = paged_seq_of_row(a.b.row0, a.b.n_seq, t);
    if (b < 0) return;
    const ConstInts rows{a.b.row0}, lens{a.b.kv_len}, before{a.before};
    const PagedSeq s = paged_seq(rows[b], rows[b + 1], lens[b], a.b.n_rows, a.b.capacity);
    PagedLine l = paged_line(a.group, q, a.shared, a.b.n_rows, a.nkv);
    const int total = before[a.b.n_seq];
    if (t - s.r0 >= s.n || total == 0) return;  // (row0 decreases somewhere)
    paged_cut(l, total, a.cuts_by);
    const int tile = (t - s.r0) >> q, b0 = before[b], each = (before[b + 1] - b0) / a.nkv;
    const PagedParts own = paged_parts(l, b0 + kvh * each + paged_length_before(s, tile, q, l.kv0),
                                       paged_length(s, tile, a.group, q, l.kv0),
                                       paged_solid(s, a.group, q, l.kv0) ? 0 : kPagedLead);
    const PagedParts pre = paged_parts(l, (kvh * l.prefix_rows + (t >> q)) * l.prefix_length, l.prefix_length, kPagedLead);
    const int n_own = own.last - own.first + 1, n_pre = pre.last - pre.first + 1;
    const int own_row = ((t - s.r0) & ((1 << q) - 1)) * a.group, pre_row = (t & ((1 << q) - 1)) * a.group;
    int S = J::GROUPS;
    while (S > 1 && (J::GROUPS / S < a.group || 2 * S > n_own + n_pre)) S /= 2;
    const int per = J::GROUPS / S, grp = threadIdx.x / J::TPR;
    for (int i0 = 0; i0 < a.group; i0 += per) {
        const int i = i0 + grp / S, h = kvh * a.group + i;
        J::row(
            lds, S, n_own + n_pre, i < a.group, a.scale2,
            [&](int k, const float*& sums, const float*& stats) {
                const bool is_pre = k >= n_own;
                const PagedParts& p = is_pre ? pre : own;
                if (p.first == p.last) {
                    const long long at = ((long long)(is_pre ? a.b.n_rows : 0) + t) * a.nh + h;
                    sums = a.whole + at * HD;
                    stats = a.whole_stats + at * 2;
                } else {
                    const long long at = (long long)paged_slot(p, p.first + k - (is_pre ? n_own : 0)) * a.slot_rows +
                                         (is_pre ? pre_row : own_row) + i;
                    sums = a.slots + at * HD;
                    stats = a.slot_stats + at * 2;
                }
            },
            a.out + (long long)t * a.out_stride + (long long)h * HD * 2);
    }
}

template <typename T, int HD>
hipError_t launch(const PagedAttendArgs& a, hipStream_t st) {
    static LdsLimit limit;
    const int lds = Kernel<T, HD>::RING + (3 * a.b.n_seq + 2 + kWaves + 2) * 4;
    const void* fn = reinterpret_cast<const void*>(&paged_attend_kernel<T, HD>);
    hipError_t e = limit.allow(Kernel<T, HD>::RING + (3 * TER_HIP_PAGED_SEQ_MAX + 2 + kWaves + 2) * 4, {fn});
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((paged_attend_kernel<T, HD>), dim3(a.cuts_by.max_wg), dim3(kThreads), lds, st, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (!a.shared && a.cuts_by.uncut * kPagedKeys > a.b.capacity + a.b.n_rows) return hipSuccess;  // nothing is cut
    if (a.shared)
        hipLaunchKernelGGL((paged_join_shared_kernel<T, HD>), dim3(a.b.n_rows, a.nkv), dim3(kThreads), 0, st, a);
    else
        hipLaunchKernelGGL((paged_join_kernel<T, HD>), dim3(a.cuts_by.max_wg, 4), dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace

PagedAttendLayout paged_attend_layout(int device, int nh, int nkv, int hd, int n_seq, int n_rows, int capacity,
                                      int shared) {
    PagedAttendLayout p{};
    const int cus = device_cu_count(device);
    if (cus <= 0) return p;
    const int group = nh / nkv;
    p.tokens_log2 = paged_tokens_log2(group);
    const int64_t tiles = ((int64_t)n_rows >> p.tokens_log2) + n_seq;
    // no more ranges than there can be work for
    const int64_t units = nkv * (tiles * (kPagedLead + 1 + min((int64_t)capacity + n_rows, (int64_t)1 << 30) / kPagedKeys) +
                                 (shared ? tiles * (kPagedLead + 1 + shared / kPagedKeys) : 0));
    PagedCuts& c = p.cuts_by;
    c.resident = (hd == 128 ? Kernel<_Float16, 128>::PER_CU : Kernel<_Float16, 64>::PER_CU) * cus;
    // Rows that keep the matrix cores busy, one at a time: prompts of a batch
    // 124 us with equal ranges, 118 so, prompts among single tokens 79 and 75.
    // Single tokens alone share the memory evenly: 87 us with equal ranges, 90
    // so.  (With a prefix the joining kernel, in which each row looks for its
    // ranges, loses more than this gains: 37 and 39 us.)
    c.rounds = c.resident / cus;
    c.round = cus / 8;
    c.skew = cus % 8 == 0 && !shared && (int64_t)n_rows * group > kPagedFew * n_seq ? (hd == 128 ? 3 : 2) : 0;
    c.min_per = 2;
    c.target = 96;
    // Short tables: with nothing cut there is nothing to join, one launch less
    // (with a prefix there always is: four tokens behind 448 positions 15.8 us
    // uncut, 13.6 cut).
    c.uncut = !shared && capacity + n_rows <= 512 ? 9 : 1;
    // (as paged_cut has it for the most units there can be: each range needs
    // two places in the workspace, 96 single tokens 52 MB so instead of 208
    // with four times the resident ones)
    c.max_wg = (int)min(max((int64_t)c.resident, min((int64_t)4 * c.resident, units / c.target)),
                        (units + c.min_per - 1) / c.min_per);
    c.max_wg = (c.max_wg + 7) / 8 * 8;
    p.slot_rows = min(kPagedRows, (int)min((long long)n_rows * group, (long long)(1 << p.tokens_log2) * group));
    auto take = [&](size_t n) {
        const size_t at = p.bytes;
        p.bytes += (n + 255) / 256 * 256;
        return at;
    };
    const size_t slots = 2 * (size_t)c.max_wg * p.slot_rows, whole = shared ? 2 * (size_t)n_rows * nh : 0;
    p.cuts = take((size_t)c.max_wg * 32);
    p.before = take(shared ? (size_t)(n_seq + 1) * 4 : 0);
    p.slot_stats = take(slots * 2 * 4);
    p.whole_stats = take(whole * 2 * 4);
    p.slots = take(slots * hd * 4);
    p.whole = take(whole * hd * 4);
    return p;
}

hipError_t launch_paged_attend(const PagedAttendArgs& a, int hd, bool bf16, hipStream_t st) {
    if (hd == 128) return bf16 ? launch<__bf16, 128>(a, st) : launch<_Float16, 128>(a, st);
    return bf16 ? launch<__bf16, 64>(a, st) : launch<_Float16, 64>(a, st);
}

}  // namespace terhip

// sample.hip -- a token for each row of logits: temperature, top-k, top-p,
// min-p and a given random number.
//
// Every cut and the draw itself are places in one order: falling logits, of
// equal ones the lower index first.  A place is found by its measure, the
// number of elements up to it (top-k) or the sum of their weights (top-p, the
// draw), as the first element at which the running measure exceeds a target.
// Weights are integers (see Weights), so sums do not depend on the order in
// which a wave, an atomic or a workgroup adds them.
//
// A row is read three times: its extent, a histogram, the elements of the bins
// that matter; then a few elements are left.  Measured, extent + histogram + list
// + end: 1 x 128256 fp16, top_k 50, top_p 0.95: 3.4 + 4.2 + 6.4 + 6.0 us, dependent
// trips to memory and through LDS; 64 rows bf16 of mixed settings 6.3 + 12.0 +
// 12.8 + 15.0; 256 rows fp16, top_p 0.92: 12.5 (5.2 TB/s) + 29.3 + 22.2 + 13.5, the
// histogram by its 26 vector instructions an element (a weight in binary64 among
// them) and the list by its own 12, not by the 65 MB read.
//
// A row whose places lie among more than 8192 elements of one bin (equal logits,
// as zeros in 16 bits) or that has an infinite logit is searched by one
// workgroup, and the call waits for it: 64 x 128256 fp16, top_k 50, top_p 0.95, 31 us
// become 2770 with one row of zeros, of atomics that meet in one place, and 770
// with one infinity; of 32000 tokens 28, 715 and 215.
#include "common.h"
#include "sample.h"

namespace terhip {
namespace {

typedef unsigned long long u64;

template <int TYPE>
struct Logit {
    typedef uint16_t T;
    static __device__ float raw(T v) {
        return TYPE == TER_HIP_T_F16 ? half_bits_to_float(v) : __builtin_bit_cast(float, (unsigned)v << 16);
    }
};
template <>
struct Logit<TER_HIP_T_F32> {
    typedef float T;
    static __device__ float raw(T v) { return v; }
};

// NaN as -infinity, +infinity as the largest number, -0 as 0.
__device__ __forceinline__ float cleaned(float x) {
    return __builtin_fminf(__builtin_fmaxf(x, -__builtin_inff()), 3.402823466e38f) + 0.0f;
}

// Bits in the order of the values.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __builtin_bit_cast(unsigned, x);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

constexpr double kOne = 17592186044416.0;  // 2^44: the weight of the largest logit

// w(x) = 2^(t / 256), t = (x - m) 256 log2(e) / T, as a multiple of 2^-44.
// With n = rint(t), r = t - n (|r| <= 1/2): 2^((n & 255) / 256) from a table,
// 2^(r / 256) by its Taylor polynomial of degree 3 (the next term is below
// (ln 2 / 512)^4 / 24 = 2^-42.7), 2^(n >> 8) by the exponent.  t is rounded
// twice, relative 2^-52 of at most 2^13.5: 2^-47 of the result.
struct Weights {
    const double* table;  // 2^(44 + j / 256), in LDS
    double m, c;

    __device__ __forceinline__ double scaled(float x) const {
        // (from -12032, 2^-47, on all the same; also of -infinity, and of NaN, -infinity times 0)
        return of(__builtin_fmax(((double)x - m) * c, -12032.0));
    }
    __device__ __forceinline__ double of(double t) const {
        const double tn = t + 6755399441055744.0;  // 1.5 * 2^52: rounds to an integer, in the low bits
        const int n = (int)__builtin_bit_cast(u64, tn);
        const double r = t - (tn - 6755399441055744.0);
        constexpr double a = 0.0027076061740622863;  // ln 2 / 256
        double p = __builtin_fma(r, a * a * a / 6, a * a / 2);
        p = __builtin_fma(r, p, a);
        p = __builtin_fma(r, p, 1.0);
        // (the table's number times 2^(n >> 8): into its exponent)
        const u64 e = __builtin_bit_cast(u64, table[n & 255]) + ((u64)(unsigned)((n & ~255) << 12) << 32);
        return __builtin_bit_cast(double, e) * p;
    }
    // (below 2^52 the low bits of a number added to 2^52 are its nearest integer)
    static __device__ __forceinline__ u64 whole(double v) {
        return __builtin_bit_cast(u64, v + 4503599627370496.0) - 0x4330000000000000ull;
    }
    __device__ __forceinline__ u64 operator()(float x) const { return whole(scaled(x)); }
    // the same for logits less than 32 T below the largest; anything for others
    __device__ __forceinline__ u64 quick(float x) const { return whole(of(((double)x - m) * c)); }
};

__device__ __forceinline__ Weights weights_of(const double* table, float m, double T) {
    return Weights{table, (double)m, 369.32993046757463 / T};  // 256 log2(e) / T
}

// The settings of a row.
struct Settings {
    double T;
    int k;       // elements kept by top-k (V: all)
    float p;     // >= 1: off
    u64 least;   // weights kept by min-p (0: all)
    double u;
};

__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int row) {
    const float t = a.p.temperature_dev ? gptr(a.p.temperature_dev)[row] : a.p.temperature;
    const int k = a.p.top_k_dev ? gptr(a.p.top_k_dev)[row] : a.p.top_k;
    const float p = a.p.top_p_dev ? gptr(a.p.top_p_dev)[row] : a.p.top_p;
    const float q = a.p.min_p_dev ? gptr(a.p.min_p_dev)[row] : a.p.min_p;
    const float u = gptr(a.u)[row];
    Settings s;
    // (not below 2^-120: the bins of one below 2^-121 are past binary32)
    s.T = t > 0.f ? (double)__builtin_fmaxf(t, 0x1p-120f) : 0.0;
    s.k = k > 0 && k < a.V ? k : a.V;
    s.p = p < 1.f ? p : 1.f;  // (NaN: 1)
    s.least = q > 0.f ? (u64)__builtin_ceil((double)__builtin_fminf(q, 1.f) * kOne) : 0;
    s.u = (double)__builtin_fminf(__builtin_fmaxf(u, 0.f), 0.99999994f);
    return s;
}

template <int NT>
struct Shared {
    static constexpr int kWaves = NT / 64;
    u64 mass[256];
    unsigned count[256];
    u64 red[kWaves];
    unsigned part[kWaves];
    // what a search found
    u64 before_mass;
    unsigned before_count, prefix;
};

__device__ __forceinline__ u64 wave_sum(u64 v) {
    for (int s = 1; s < 64; s <<= 1) v += (u64)__shfl_xor((long long)v, s);
    return v;
}

// A row by its elements, one workgroup.
template <int TYPE, int kThreads>
struct Row {
    static constexpr int kWaves = kThreads / 64;
    typedef typename Logit<TYPE>::T T;
    typedef Shared<kThreads> Sh;
    const TER_GLOBAL T* x;
    int V;
    __device__ float operator[](int i) const { return cleaned(Logit<TYPE>::raw(x[i])); }

    __device__ unsigned largest(Sh& sh) const {
        unsigned k = 0;
        for (int i = threadIdx.x; i < V; i += kThreads) {
            const unsigned e = key_of((*this)[i]);
            k = e > k ? e : k;
        }
        for (int s = 1; s < 64; s <<= 1) {
            const unsigned o = (unsigned)__shfl_xor((int)k, s);
            k = o > k ? o : k;
        }
        if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = k;
        __syncthreads();
        for (int i = 0; i < kWaves; ++i) k = sh.part[i] > k ? sh.part[i] : k;
        __syncthreads();
        return k;
    }

    // Sum of the weights that are `least` or more.
    __device__ u64 mass(Sh& sh, const Weights& w, u64 least) const {
        u64 s = 0;
        for (int i = threadIdx.x; i < V; i += kThreads) {
            const u64 e = w((*this)[i]);
            s += e >= least ? e : 0;
        }
        s = wave_sum(s);
        if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = s;
        __syncthreads();
        s = 0;
        for (int i = 0; i < kWaves; ++i) s += sh.red[i];
        __syncthreads();
        return s;
    }

    // Index of element `rank` (from 0, by index) of those with key `key`.
    __device__ int tie(Sh& sh, unsigned key, unsigned rank) const {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const int per = ((V + kWaves - 1) / kWaves + 63) / 64 * 64, from = wave * per;
        const int to = from + per < V ? from + per : V;
        unsigned n = 0;
        for (int i = from; i < to; i += 64)
            n += __builtin_popcountll(__ballot(i + lane < to && key_of((*this)[i + lane]) == key));
        if (lane == 0) sh.part[wave] = n;
        __syncthreads();
        unsigned before = 0;
        for (int i = 0; i < wave; ++i) before += sh.part[i];
        if (rank >= before && rank < before + n) {  // (one wave)
            unsigned left = rank - before;
            for (int i = from; i < to; i += 64) {
                u64 b = __ballot(i + lane < to && key_of((*this)[i + lane]) == key);
                const unsigned c = __builtin_popcountll(b);
                if (left < c) {
                    for (; left; --left) b &= b - 1;
                    if (lane == 0) sh.prefix = (unsigned)(i + __builtin_ctzll(b));
                    break;
                }
                left -= c;
            }
        }
        __syncthreads();
        return (int)sh.prefix;
    }

    struct Place {
        unsigned key;      // of the element
        u64 before;        // weights of all larger elements
        unsigned n_before; // their number
    };

    // The value of the first element at which the running measure (the weights,
    // or the number where by_count) exceeds target, which the whole exceeds:
    // byte by byte of the key, each by a histogram of the elements that agree
    // so far.
    __device__ Place find(Sh& sh, const Weights& w, bool by_count, u64 target) const {
        Place at = {0, 0, 0};
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = threadIdx.x; i < 256; i += kThreads) {
                sh.mass[i] = 0;
                sh.count[i] = 0;
            }
            __syncthreads();
            const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
            for (int i = threadIdx.x; i < V; i += kThreads) {
                const float e = (*this)[i];
                const unsigned key = key_of(e);
                if ((key & mask) != at.key) continue;
                const unsigned b = key >> shift & 255;
                atomicAdd(&sh.count[b], 1u);
                atomicAdd(&sh.mass[b], w(e));
            }
            __syncthreads();
            if (threadIdx.x < 64) {
                // four bins a lane, from the largest
                const int lane = threadIdx.x;
                u64 mass = 0;
                unsigned count = 0;
                for (int i = 0; i < 4; ++i) {
                    mass += sh.mass[255 - 4 * lane - i];
                    count += sh.count[255 - 4 * lane - i];
                }
                u64 m = mass;
                unsigned c = count;
                for (int s = 1; s < 64; s <<= 1) {
                    const u64 om = (u64)__shfl_up((long long)m, s);
                    const unsigned oc = (unsigned)__shfl_up((int)c, s);
                    if (lane >= s) {
                        m += om;
                        c += oc;
                    }
                }
                const u64 got = by_count ? at.n_before + c : at.before + m;
                const u64 ends = __ballot(got > target);
                if (ends && lane == __builtin_ctzll(ends)) {
                    m = at.before + m - mass;
                    c = at.n_before + c - count;
                    int b = 255 - 4 * lane;
                    for (int i = 0; i < 3; ++i, --b) {
                        const u64 nm = m + sh.mass[b];
                        const unsigned nc = c + sh.count[b];
                        if ((by_count ? (u64)nc : nm) > target) break;
                        m = nm;
                        c = nc;
                    }
                    sh.before_mass = m;
                    sh.before_count = c;
                    sh.prefix = at.key | (unsigned)b << shift;
                }
            }
            __syncthreads();
            at = {sh.prefix, sh.before_mass, sh.before_count};
            __syncthreads();
        }
        return at;
    }
};

// One row by one workgroup: a search through the row's values for each cut and
// for the draw, four passes each.  Right for every row; the general path.
template <int TYPE, int NT>
__device__ __forceinline__ void sample_row(const SampleArgs& a, int row, const double* table, Shared<NT>& sh) {
    Row<TYPE, NT> x{gptr(reinterpret_cast<const typename Logit<TYPE>::T*>(a.logits + (long long)row * a.stride)), a.V};
    const unsigned top = x.largest(sh);
    const Settings s = settings_of(a, row);
    if (top == key_of(-__builtin_inff()) || s.T == 0.0) {
        const int i = top == key_of(-__builtin_inff()) ? -1 : x.tie(sh, top, 0);
        if (threadIdx.x == 0) {
            gptr(a.token)[row] = i;
            if (a.prob) gptr(a.prob)[row] = i < 0 ? 0.f : 1.f;
        }
        return;
    }
    const Weights w = weights_of(table, value_of(top), s.T);
    u64 sum = x.mass(sh, w, 0);
    if (s.k < a.V) {
        const auto at = x.find(sh, w, true, (u64)(s.k - 1));
        sum = at.before + ((unsigned)s.k - at.n_before) * w(value_of(at.key));
    }
    if (s.p < 1.f) {
        // elements with less than p * sum before them: up to the first at which the sum reaches it
        const double want = __builtin_ceil((double)s.p * (double)sum);
        const u64 target = want > 1.0 ? (u64)want - 1 : 0;
        const auto at = x.find(sh, w, false, target);
        const u64 e = w(value_of(at.key));
        const u64 kept = at.before + ((target - at.before) / e + 1) * e;
        sum = kept < sum ? kept : sum;
    }
    if (s.least) {
        const u64 kept = x.mass(sh, w, s.least);
        sum = kept < sum ? kept : sum;
    }
    const u64 target = (u64)(s.u * (double)sum);
    const auto at = x.find(sh, w, false, target);
    const float v = value_of(at.key);
    const int i = x.tie(sh, at.key, (unsigned)((target - at.before) / w(v)));
    if (threadIdx.x == 0) {
        gptr(a.token)[row] = i;
        if (a.prob) gptr(a.prob)[row] = (float)(w.scaled(v) / (double)sum);
    }
}

// ---- the usual path: bins of bins ----
//
// The row is cut into bins of falling logits: bin floor(y), y = (m - x) /
// range * (kBins - 2), in binary32, where range is the smallest of 31.5 T and
// the row's own.  Its steps are monotonic, so bins stand in the order of the
// logits and one holds all elements between two values.  The last bin, kBins -
// 1, takes what has no weight (31.5 T and more below m) and is not counted.  A
// histogram of numbers or of weights over the bins finds the bin of each cut
// and of the draw.  A cut moves what later ones start from, so a later place
// is known to a bin or two only: all of them are listed.  The same again over
// the listed elements, a bin cut into up to 256, leaves a few elements, which
// one wave compares with each other, or many equal ones.
constexpr int kCountK = 1024; // up to this top_k everything kept is listed, and weights are computed for the list alone
constexpr int kFew = 64;      // elements compared by one wave
constexpr int kValues = 64;   // different values among more elements than that, by their bins
constexpr int kOneByOne = 8;  // or one after another
constexpr int kSecond = 4096; // elements of the second list (a power of two)

struct Bins {
    float mh, cb;  // m / 2; bins for half a logit
    __device__ __forceinline__ float operator()(float x) const {
        return __builtin_fmaf(x, -0.5f, mh) * cb;  // (halves do not overflow; NaN of NaN, +infinity of -infinity)
    }
};
constexpr float kLast = (float)(kBins - 1);
constexpr int kSpare = 64;

// m, low: the largest logit and the smallest that is a number.
__device__ __forceinline__ Bins bins_of(float m, float low, double T) {
    const double range = __builtin_fmin(31.5 * T, ((double)m - (double)low) * 1.001);
    return Bins{0.5f * m, (float)__builtin_fmin(2.0 * (kBins - 2) / range, 3e38)};
}

// What a row's histogram counts.
enum Mode { kCount = 1, kMass = 2, kBoth = 3 };
__device__ __forceinline__ int mode_of(const Settings& s, int V) {
    return s.k <= kCountK && s.k < V ? kCount : s.k < V ? kBoth : kMass;
}

// A workgroup's LDS: for the extent of its logits, for a histogram, for the list
// too, and to the end.
template <int NT>
struct LdsScan {
    static constexpr int kThreads = NT, kWaves = NT / 64;
    u64 wave_mass[kWaves];
    unsigned wave_count[kWaves];
};

template <int NT>
struct LdsBins : LdsScan<NT> {
    double table[256];
    u64 mass[kBins + kSpare];
    unsigned count[kBins + kSpare];
    // places of a level: bin, sums at its start and end
    int at[8];
    u64 from[8], to[8];
    u64 least_mass;       // sum of the weights that min-p keeps
    int n;
};

template <int NT, int LIST>
struct LdsList : LdsBins<NT> {
    unsigned index[LIST];
};

template <int NT>
struct Lds : LdsList<NT, kList> {
    u64 list[kList];
    union {
        u64 second[kSecond];
        Shared<NT> general;
    };
    unsigned values[kValues], numbers[kValues];
};

// f(x, i), x an array of consecutive elements from i on, of all elements [i0,
// i1) of a row by the workgroup's threads, 16 bytes a load, four loads in flight.
template <int TYPE, int kThreads, typename F>
__device__ __forceinline__ void each(const typename Logit<TYPE>::T* row, int i0, int i1, F f) {
    typedef typename Logit<TYPE>::T T;
    typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
    constexpr int VE = 16 / (int)sizeof(T), U = 4;
    const int t = threadIdx.x;
    const TER_GLOBAL T* p = gptr(row) + i0;
    const int n = i1 - i0;
    int head = (int)((0 - reinterpret_cast<uintptr_t>(row + i0)) & 15) / (int)sizeof(T);
    head = head < n ? head : n;
    const int nv = (n - head) / VE, tail = head + nv * VE;
    // (the elements outside of whole vectors: at most 2 VE - 2, one a thread)
    const int odd = t < head ? t : t - head < n - tail ? tail + t - head : -1;
    if (odd >= 0) {
        const float x[1] = {Logit<TYPE>::raw(p[odd])};
        f(x, i0 + odd);
    }
    const TER_GLOBAL u32x4* v = reinterpret_cast<const TER_GLOBAL u32x4*>(p + head);
    for (int a = t; a < nv; a += U * kThreads) {
        u32x4 r[U];
#pragma unroll
        for (int q = 0; q < U; ++q) r[q] = v[a + q * kThreads < nv ? a + q * kThreads : nv - 1];
#pragma unroll
        for (int q = 0; q < U; ++q) {
            if (a + q * kThreads >= nv) break;
            float x[VE];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned w = r[q][e];
                if constexpr (TYPE == TER_HIP_T_F32) {
                    x[e] = __builtin_bit_cast(float, w);
                } else {
                    x[2 * e] = Logit<TYPE>::raw((uint16_t)w);
                    x[2 * e + 1] = Logit<TYPE>::raw((uint16_t)(w >> 16));
                }
            }
            f(x, i0 + head + (a + q * kThreads) * VE);
        }
    }
}

template <typename A>
constexpr int length_of(const A& x) { return (int)(sizeof(x) / sizeof(x[0])); }

// The largest logit of a row or slice, and the smallest that is a number.
struct Extent {
    float high, low;
    __device__ void join(float h, float l) {
        high = __builtin_fmaxf(high, h);
        low = __builtin_fminf(low, l);
    }
};

template <int TYPE, int NT>
__device__ Extent extent_of(const typename Logit<TYPE>::T* row, int i0, int i1, LdsScan<NT>& sh) {
    Extent x{-__builtin_inff(), __builtin_inff()};
    each<TYPE, NT>(row, i0, i1, [&](const auto& v, int) {
#pragma unroll
        for (int e = 0; e < length_of(v); ++e) x.join(v[e], v[e] == -__builtin_inff() ? x.low : v[e]);
    });
    for (int s = 1; s < 64; s <<= 1) x.join(__shfl_xor(x.high, s), __shfl_xor(x.low, s));
    if ((threadIdx.x & 63) == 0) {
        sh.wave_count[threadIdx.x >> 6] = __builtin_bit_cast(unsigned, x.high);
        sh.wave_mass[threadIdx.x >> 6] = __builtin_bit_cast(unsigned, x.low);
    }
    __syncthreads();
    for (int i = 0; i < NT / 64; ++i)
        x.join(__builtin_bit_cast(float, sh.wave_count[i]), __builtin_bit_cast(float, (unsigned)sh.wave_mass[i]));
    __syncthreads();
    return x;
}

// Index of the first element equal to m (V: none).
template <int TYPE, int NT>
__device__ int first_of(const typename Logit<TYPE>::T* row, int V, float m, LdsScan<NT>& sh) {
    int at = V;
    each<TYPE, NT>(row, 0, V, [&](const auto& x, int i) {
        for (int e = 0; e < length_of(x); ++e) at = cleaned(x[e]) == m && i + e < at ? i + e : at;
    });
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_xor(at, s);
        at = o < at ? o : at;
    }
    if ((threadIdx.x & 63) == 0) sh.wave_count[threadIdx.x >> 6] = (unsigned)at;
    __syncthreads();
    for (int i = 0; i < NT / 64; ++i) at = (int)sh.wave_count[i] < at ? (int)sh.wave_count[i] : at;
    __syncthreads();
    return at;
}

template <int NT>
__device__ __forceinline__ void clear_bins(LdsBins<NT>& sh) {
#pragma unroll 1
    for (int i = threadIdx.x; i < kBins; i += NT) {
        sh.mass[i] = 0;
        sh.count[i] = 0;
    }
    if (threadIdx.x == 0) sh.least_mass = 0;
    __syncthreads();
}

// Elements [i0, i1) into the histogram in LDS.  Those of the last bin go to one
// of kSpare more by their lane, which nobody reads, so that many do not meet in
// one place; their weights may be anything.  No branches: the weights of a
// load's elements are computed side by side.
template <int TYPE, int NT>
__device__ void fill_bins(const typename Logit<TYPE>::T* row, int i0, int i1, int mode, u64 least, const Bins& y,
                          const Weights& w, LdsBins<NT>& sh) {
    const float last = kLast + (float)(threadIdx.x & (kSpare - 1));
    if (mode == kCount) {
        each<TYPE, NT>(row, i0, i1, [&](const auto& x, int) {
#pragma unroll
            for (int e = 0; e < length_of(x); ++e) atomicAdd(&sh.count[(int)__builtin_fminf(y(x[e]), last)], 1u);
        });
    } else {
        u64 kept = 0;
        const bool sums = least != 0, counts = mode != kMass;
        each<TYPE, NT>(row, i0, i1, [&](const auto& x, int) {
            constexpr int N = sizeof(x) / sizeof(x[0]);
            u64 m[N];
            int b[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                b[e] = (int)__builtin_fminf(y(x[e]), last);
                m[e] = w.quick(x[e]);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) atomicAdd(&sh.mass[b[e]], m[e]);
            if (sums) {
#pragma unroll
                for (int e = 0; e < N; ++e) kept += b[e] < kBins - 1 && m[e] >= least ? m[e] : 0;
            }
            if (counts) {
#pragma unroll
                for (int e = 0; e < N; ++e) atomicAdd(&sh.count[b[e]], 1u);
            }
        });
        if (sums) {
            kept = wave_sum(kept);
            if ((threadIdx.x & 63) == 0) atomicAdd(&sh.least_mass, kept);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sh.mass[kBins - 1] = 0;
        sh.count[kBins - 1] = 0;
    }
    __syncthreads();
}

// m and n plus those of the lane that a DPP control names (0 where there is none).
template <int CTRL, int ROWS>
__device__ __forceinline__ void wave_scan_step(u64& m, unsigned& n) {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)m, CTRL, ROWS, 0xF, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(m >> 32), CTRL, ROWS, 0xF, false);
    m += (u64)hi << 32 | lo;
    n += (unsigned)__builtin_amdgcn_update_dpp(0, (int)n, CTRL, ROWS, 0xF, false);
}

// Exclusive running sums over a workgroup's threads; the whole in *all.
template <int NT>
__device__ __forceinline__ void block_scan(u64& m, unsigned& n, u64* all, LdsScan<NT>& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // within the wave by DPP: rows of 16 lanes, then the rows' last lanes
    u64 im = m;
    unsigned in = n;
    wave_scan_step<0x111, 0xF>(im, in);  // row_shr:1
    wave_scan_step<0x112, 0xF>(im, in);
    wave_scan_step<0x114, 0xF>(im, in);
    wave_scan_step<0x118, 0xF>(im, in);
    wave_scan_step<0x142, 0xA>(im, in);  // row_bcast:15
    wave_scan_step<0x143, 0xC>(im, in);  // row_bcast:31
    if (lane == 63) {
        sh.wave_mass[wave] = im;
        sh.wave_count[wave] = in;
    }
    __syncthreads();
    u64 bm = 0, sum = 0;
    unsigned bn = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        const u64 e = sh.wave_mass[i];
        const unsigned c = sh.wave_count[i];
        bm += i < wave ? e : 0;
        bn += i < wave ? c : 0;
        sum += e;
    }
    m = bm + im - m;
    n = bn + in - n;
    *all = sum;
    __syncthreads();
}

__device__ __forceinline__ u64 p_target(float p, u64 sum) {
    const double want = __builtin_ceil((double)p * (double)sum);
    return want > 1.0 ? (u64)want - 1 : 0;
}

constexpr int kNone = 1 << 20;

// The bins of a level that hold the places, up to three runs of them in their
// order, and the sums in front of each run.
struct Runs {
    int lo[3], hi[3];  // kNone: no run
    u64 mass[3];
    unsigned count[3];
    u64 total;         // sum of all weights (not before the list in mode kCount)
    u64 least_mass;
};

__device__ __forceinline__ void swap_runs(Runs& r, int i, int j) {
    if (r.lo[j] >= r.lo[i]) return;
    const int l = r.lo[i], h = r.hi[i];
    r.lo[i] = r.lo[j];
    r.hi[i] = r.hi[j];
    r.lo[j] = l;
    r.hi[j] = h;
}

// One level: the histogram in LDS becomes its running sums, those of each run
// of `before` (from bins 0, start1 and start2 on; null: one run of all) from the
// sums in front of it, and the places are found in it.  Listing of all up
// to the last element of the top_k where there are no weights (weighted =
// false).
template <int NT>
__device__ __forceinline__ Runs level_of(const Settings& s, int V, bool weighted, const Runs* before, int start1, int start2,
                                         LdsBins<NT>& sh) {
    constexpr int PER = kBins / NT;  // bins of a thread
    const int b0 = threadIdx.x * PER;
    u64 m[PER], e[PER], ms = 0;
    unsigned n[PER], c[PER], ns = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        m[i] = ms;
        n[i] = ns;
        ms += e[i] = sh.mass[b0 + i];
        ns += c[i] = sh.count[b0 + i];
    }
    Runs r;
    block_scan(ms, ns, &r.total, sh);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        sh.mass[b0 + i] = m[i] += ms;
        sh.count[b0 + i] = n[i] += ns;
    }
    if (threadIdx.x < 8) sh.at[threadIdx.x] = kNone;
    __syncthreads();
    if (before) {
        const int f1 = start1 < kBins ? start1 : 0, f2 = start2 < kBins ? start2 : 0;
        const u64 m0 = before->mass[0], m1 = before->mass[1] - sh.mass[f1], m2 = before->mass[2] - sh.mass[f2];
        const unsigned n0 = before->count[0], n1 = before->count[1] - sh.count[f1], n2 = before->count[2] - sh.count[f2];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int b = b0 + i;
            sh.mass[b] = m[i] += b >= start2 ? m2 : b >= start1 ? m1 : m0;
            sh.count[b] = n[i] += b >= start2 ? n2 : b >= start1 ? n1 : n0;
        }
        if (before->total) r.total = before->total;
    }
    r.least_mass = before && before->total ? before->least_mass : sh.least_mass;
    // the bin in which the running sum exceeds a target
    auto cross = [&](u64 target, int slot) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (m[i] <= target && target - m[i] < e[i]) {
                sh.at[slot] = b0 + i;
                sh.from[slot] = m[i];
                sh.to[slot] = m[i] + e[i];
            }
    };
    if (s.k < V) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (n[i] <= (unsigned)(s.k - 1) && (unsigned)(s.k - 1) - n[i] < c[i]) {
                sh.at[0] = b0 + i;
                sh.from[0] = m[i];
                sh.to[0] = m[i] + e[i];
            }
        __syncthreads();
    }
    const int bk = sh.at[0];  // (kNone: no top_k, or its last element has no weight)
#pragma unroll
    for (int i = 0; i < 3; ++i) r.lo[i] = r.hi[i] = kNone;
    if (!weighted) {
        r.lo[0] = 0;
        r.hi[0] = bk != kNone ? bk : kBins - 2;
        r.total = 0;
    } else {
        u64 lo = r.total, hi = r.total;  // the sum of what is kept, so far
        if (bk != kNone) {
            r.lo[0] = r.hi[0] = bk;
            lo = sh.from[0];
            hi = sh.to[0];
        }
        if (s.p < 1.f) {
            cross(p_target(s.p, lo), 1);
            cross(p_target(s.p, hi), 2);
            __syncthreads();
            r.lo[1] = sh.at[1];
            r.hi[1] = sh.at[2];
            const u64 a = sh.from[1], b = sh.to[2];
            lo = a < lo ? a : lo;
            hi = b < hi ? b : hi;
        }
        if (s.least) {
            lo = r.least_mass < lo ? r.least_mass : lo;
            hi = r.least_mass < hi ? r.least_mass : hi;
        }
        cross((u64)(s.u * (double)lo), 3);
        cross((u64)(s.u * (double)hi), 4);
        __syncthreads();
        r.lo[2] = sh.at[3];
        r.hi[2] = sh.at[4];
        // in their order, those that touch as one
        swap_runs(r, 0, 1);
        swap_runs(r, 1, 2);
        swap_runs(r, 0, 1);
        if (r.lo[2] != kNone && r.lo[2] <= r.hi[1] + 1) {
            r.hi[1] = r.hi[2] > r.hi[1] ? r.hi[2] : r.hi[1];
            r.lo[2] = r.hi[2] = kNone;
        }
        if (r.lo[1] != kNone && r.lo[1] <= r.hi[0] + 1) {
            r.hi[0] = r.hi[1] > r.hi[0] ? r.hi[1] : r.hi[0];
            r.lo[1] = r.lo[2];
            r.hi[1] = r.hi[2];
            r.lo[2] = r.hi[2] = kNone;
            if (r.lo[1] != kNone && r.lo[1] <= r.hi[0] + 1) {
                r.hi[0] = r.hi[1] > r.hi[0] ? r.hi[1] : r.hi[0];
                r.lo[1] = r.hi[1] = kNone;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int f = r.lo[i] < kBins ? r.lo[i] : 0;
        r.mass[i] = sh.mass[f];
        r.count[i] = sh.count[f];
    }
    __syncthreads();
    return r;
}

__device__ __forceinline__ u64 entry_of(float x, int i) { return (u64)~key_of(cleaned(x)) << 32 | (unsigned)i; }
__device__ __forceinline__ float entry_value(u64 l) { return value_of(~(unsigned)(l >> 32)); }

// Lists the elements of runs r among [i0, i1) by their indices: sh.n of them,
// those past LIST left out.
template <int TYPE, int NR, int NT, int LIST>
__device__ __forceinline__ void list_runs(const typename Logit<TYPE>::T* x, int i0, int i1, const Bins& y, const Runs& r,
                                          LdsList<NT, LIST>& sh) {
    float lo[NR], hi[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        lo[i] = (float)r.lo[i];
        hi[i] = (float)(r.hi[i] + 1);
    }
    each<TYPE, NT>(x, i0, i1, [&](const auto& v, int i) {
        constexpr int N = sizeof(v) / sizeof(v[0]);
        unsigned in = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float b = y(v[e]);
            bool one = false;
#pragma unroll
            for (int k = 0; k < NR; ++k) one |= (b >= lo[k]) & (b < hi[k]);
            in |= one ? 1u << e : 0;
        }
        if (in) {
            int at = atomicAdd(&sh.n, __builtin_popcount(in));
            for (; in; in &= in - 1, ++at)
                if (at < LIST) sh.index[at] = (unsigned)(i + __builtin_ctz(in));
        }
    });
}

template <int TYPE, int NT, int LIST>
__device__ void fill_list(const typename Logit<TYPE>::T* x, int i0, int i1, const Bins& y, const Runs& r,
                          LdsList<NT, LIST>& sh) {
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    if (r.lo[1] == kNone)
        list_runs<TYPE, 1>(x, i0, i1, y, r, sh);
    else if (r.lo[2] == kNone)
        list_runs<TYPE, 2>(x, i0, i1, y, r, sh);
    else
        list_runs<TYPE, 3>(x, i0, i1, y, r, sh);
    __syncthreads();
}

// a / b, where it is below 2^20 (in binary64, off by one at most, and put right).
__device__ __forceinline__ unsigned ratio(u64 a, u64 b) {
    unsigned q = (unsigned)((double)a / (double)b);
    q -= q * b > a;
    q += (q + 1) * b <= a;
    return q;
}

// One element of a group that is small or of few values: its sums in front.
struct Spot {
    u64 before, mass;       // sum of the weights in front of it; its own (of all equal ones)
    unsigned rank, number;  // elements in front of it; equal ones
};

// The value of lane i, the same for the wave.
__device__ __forceinline__ u64 lane_of(u64 v, int i) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), i) << 32 |
           (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, i);
}

// The places among the spots that a wave's lanes hold (`here`: this lane has
// one), each kept sum exact: the sum of all kept, and where u lies.
__device__ __forceinline__ u64 kept_of(const Settings& s, int V, const Spot& z, u64 weight, bool here, const Runs& r,
                                       u64* target) {
    auto pick = [&](bool mine, u64 v) -> u64 {
        const u64 b = __ballot(mine);
        if (!b) return 0;
        return lane_of(v, __builtin_ctzll(b));
    };
    u64 sum = r.total;
    if (s.k < V) {
        const unsigned k = (unsigned)(s.k - 1);
        const u64 got = pick(here && z.rank <= k && k - z.rank < z.number, z.before + (k - z.rank + 1) * weight);
        sum = got ? got : sum;  // (none: the top_k's last element has no weight)
    }
    u64 kept = sum;
    if (s.p < 1.f) {
        const u64 t = p_target(s.p, sum);
        const bool mine = here && z.before <= t && t - z.before < z.mass;
        const u64 got = pick(mine, z.before + (mine ? ratio(t - z.before, weight) + 1 : 0) * weight);
        if (!got) return 0;
        kept = got < kept ? got : kept;
    }
    if (s.least && r.least_mass < kept) kept = r.least_mass;
    *target = (u64)(s.u * (double)kept);
    return kept;
}

// k <= kFew elements, lane i of the first wave with l; b: its bin, whose sums in
// front are z's.
__device__ __forceinline__ bool finish_lanes(const SampleArgs& a, int row, const Settings& s, const Weights& w,
                                             const Runs& q, int k, u64 l, float x, u64 e, int b, Spot z) {
    const bool here = (int)(threadIdx.x & 63) < k;
    // (lanes from k on hold the largest entry: behind all.  Eight at a time: one
    // wave works here, and one by one each waits for the last.)
    for (int i8 = 0; i8 < k; i8 += 8)
#pragma unroll
        for (int i = i8; i < i8 + 8; ++i) {
            const u64 ol = lane_of(l, i), oe = lane_of(e, i);
            const bool ahead = __builtin_amdgcn_readlane(b, i) == b && ol < l;
            z.before += ahead ? oe : 0;
            z.rank += ahead;
        }
    u64 target = 0;
    const u64 sum = kept_of(s, a.V, z, e, here, q, &target);
    const bool mine = sum && here && z.before <= target && target - z.before < e;
    if (mine) {
        gptr(a.token)[row] = (int32_t)(unsigned)l;
        if (a.prob) gptr(a.prob)[row] = (float)(w.scaled(x) / (double)sum);
    }
    return __ballot(mine) != 0;
}

// The second list, if it has few elements.
template <int NT, typename B>
__device__ __forceinline__ bool finish_few(const SampleArgs& a, int row, const Settings& s, const B& bin, const Weights& w,
                                           const Runs& q, int k, Lds<NT>& sh) {
    if (threadIdx.x < 64) {
        const bool here = (int)threadIdx.x < k;
        const u64 l = here ? sh.second[threadIdx.x] : ~0ull;
        const float x = entry_value(l);
        const int b = here ? bin(x) : -1;
        const bool found = finish_lanes(a, row, s, w, q, k, l, x, here ? w(x) : 0, b,
                                        Spot{here ? sh.mass[b] : 0, here ? w(x) : 0, here ? sh.count[b] : 0, 1});
        if (threadIdx.x == 0) sh.at[7] = found;
    }
    __syncthreads();
    return sh.at[7] != 0;
}

// The first list, if it has few elements: its runs are the bins.
template <int NT>
__device__ __forceinline__ bool finish_short(const SampleArgs& a, int row, const Settings& s, const Bins& y, const Weights& w,
                                             const Runs& r, int n, Lds<NT>& sh) {
    if (threadIdx.x < 64) {
        const bool here = (int)threadIdx.x < n;
        const u64 l = here ? sh.list[threadIdx.x] : ~0ull;
        const float x = entry_value(l);
        const u64 e = here ? w(x) : 0;
        const int f = (int)y(x);
        const int b = here ? (f >= r.lo[1]) + (f >= r.lo[2]) : -1;
        Runs q = r;
        if (r.total == 0) {
            q.total = wave_sum(e);
            q.least_mass = wave_sum(e >= s.least ? e : 0);
        }
        Spot z{r.mass[0], e, r.count[0], 1};
        const u64 m1 = r.mass[1] - z.before, m2 = r.mass[2] - z.before - m1;
        const unsigned c1 = r.count[1] - z.rank, c2 = r.count[2] - z.rank - c1;
        z.before += (b >= 1 ? m1 : 0) + (b >= 2 ? m2 : 0);
        z.rank += (b >= 1 ? c1 : 0) + (b >= 2 ? c2 : 0);
        const bool found = finish_lanes(a, row, s, w, q, n, l, x, e, b, z);
        if (threadIdx.x == 0) sh.at[7] = found;
    }
    __syncthreads();
    return sh.at[7] != 0;
}

// The slot of a bin of the runs: those of the first, then of the others.
__device__ __forceinline__ int slot_of(const Runs& q, int b) {
    const int n0 = q.hi[0] - q.lo[0] + 1, n1 = q.lo[1] != kNone ? q.hi[1] - q.lo[1] + 1 : 0;
    int i = b - q.lo[0];
    i += b >= q.lo[1] ? q.lo[0] + n0 - q.lo[1] : 0;
    i += b >= q.lo[2] ? q.lo[1] + n1 - q.lo[2] : 0;
    return i;
}

// The different values among the k elements of the second list, falling, and
// their numbers; how many, 0 where they are more than kValues or not found here.
// Equal logits, as 16 bits have many, stand in a bin by themselves: the bins'
// values, if the runs have few bins; else the largest value left, one by one.
template <int NT, typename B>
__device__ __forceinline__ int values_of(const B& bin, const Runs& q, int k, Lds<NT>& sh) {
    const int lane = threadIdx.x & 63;
    const int last = q.lo[2] != kNone ? q.hi[2] : q.lo[1] != kNone ? q.hi[1] : q.hi[0];
    const int bins = slot_of(q, last) + 1;
    if (threadIdx.x < kValues) sh.numbers[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.at[5] = 0;
    if (bins <= kValues) {
        for (int i = threadIdx.x; i < k; i += NT)
            sh.values[slot_of(q, bin(entry_value(sh.second[i])))] = (unsigned)(sh.second[i] >> 32);  // (any one's)
        __syncthreads();
        for (int i = threadIdx.x; i < k; i += NT) {
            const int slot = slot_of(q, bin(entry_value(sh.second[i])));
            if ((unsigned)(sh.second[i] >> 32) != sh.values[slot]) sh.at[5] = 1;
            atomicAdd(&sh.numbers[slot], 1u);
        }
        __syncthreads();
        return sh.at[5] ? 0 : bins;
    }
    if (threadIdx.x < kValues) sh.values[threadIdx.x] = ~0u;
    __syncthreads();
    unsigned after = 0;  // (inverted keys rise as logits fall; 0 inverted is a NaN's)
    for (int nv = 0; nv <= kOneByOne; ++nv) {
        unsigned v = ~0u;
        for (int i = threadIdx.x; i < k; i += NT) {
            const unsigned e = (unsigned)(sh.second[i] >> 32);
            v = e > after && e < v ? e : v;
        }
        for (int d = 1; d < 64; d <<= 1) {
            const unsigned o = (unsigned)__shfl_xor((int)v, d);
            v = o < v ? o : v;
        }
        if (lane == 0 && v != ~0u) atomicMin(&sh.values[nv], v);
        __syncthreads();
        after = sh.values[nv];
        if (after == ~0u) return nv;
        unsigned c = 0;
        for (int i = threadIdx.x; i - lane < k; i += NT)
            c += __builtin_popcountll(__ballot(i < k && (unsigned)(sh.second[i] >> 32) == after));
        if (lane == 0 && c) atomicAdd(&sh.numbers[nv], c);
    }
    return 0;
}

// Elements of nv different values: those as spots, then the token among equal
// ones by its index.
template <int NT, typename B>
__device__ __forceinline__ bool finish_values(const SampleArgs& a, int row, const Settings& s, const B& bin, const Weights& w,
                                              const Runs& q, int k, int nv, Lds<NT>& sh) {
    __syncthreads();
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        const unsigned c = lane < nv ? sh.numbers[lane] : 0;
        const bool here = c != 0;
        const unsigned key = here ? sh.values[lane] : 0x7FFFFFFFu;
        const float x = value_of(~key);
        const u64 e = here ? w(x) : 0;
        const int b = here ? bin(x) : -1;
        Spot z{here ? sh.mass[b] : 0, e * c, here ? sh.count[b] : 0, c};
        for (int i = 0; i < nv; ++i) {  // (values that share a bin)
            const u64 oe = lane_of(z.mass, i);
            const unsigned oc = (unsigned)__builtin_amdgcn_readlane((int)c, i);
            const bool ahead = __builtin_amdgcn_readlane(b, i) == b && i < lane;
            z.before += ahead ? oe : 0;
            z.rank += ahead ? oc : 0;
        }
        u64 target = 0;
        const u64 sum = kept_of(s, a.V, z, e, here, q, &target);
        const bool mine = sum && here && z.before <= target && target - z.before < z.mass;
        if (mine) {
            sh.at[5] = (int)ratio(target - z.before, e);
            sh.at[6] = (int)key;
            if (a.prob) gptr(a.prob)[row] = (float)(w.scaled(x) / (double)sum);
        }
        const bool found = __ballot(mine) != 0;
        if (lane == 0) sh.at[7] = found;
    }
    __syncthreads();
    if (!sh.at[7]) return false;
    const unsigned rank = (unsigned)sh.at[5], key = (unsigned)sh.at[6];
    // of the equal ones the one with `rank` lower indices: by the index's upper bits, then among those that share them
    static_assert(TER_HIP_SAMPLE_V_MAX <= kBins << 8, "");
    clear_bins(sh);
    for (int i = threadIdx.x; i < k; i += NT)
        if ((unsigned)(sh.second[i] >> 32) == key) atomicAdd(&sh.count[(unsigned)sh.second[i] >> 8], 1u);
    __syncthreads();
    constexpr int PER = kBins / NT;
    const int b0 = threadIdx.x * PER;
    u64 none = 0, all;
    unsigned n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += sh.count[b0 + i];
    block_scan(none, n, &all, sh);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const unsigned c = sh.count[b0 + i];
        if (n <= rank && rank - n < c) {
            sh.at[0] = b0 + i;
            sh.at[1] = (int)(rank - n);
        }
        n += c;
    }
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    const int bucket = sh.at[0];
    for (int i = threadIdx.x; i < k; i += NT)
        if ((unsigned)(sh.second[i] >> 32) == key && (int)((unsigned)sh.second[i] >> 8) == bucket)
            sh.mass[atomicAdd(&sh.n, 1)] = (unsigned)sh.second[i];  // (256 at most)
    __syncthreads();
    if ((int)threadIdx.x < sh.n) {
        const u64 me = sh.mass[threadIdx.x];
        int lower = 0;
        for (int i = 0; i < sh.n; ++i) lower += sh.mass[i] < me;
        if (lower == sh.at[1]) gptr(a.token)[row] = (int32_t)me;
    }
    return true;
}

// Any elements: sorted.
template <int NT, typename B>
__device__ __forceinline__ bool finish_sorted(const SampleArgs& a, int row, const Settings& s, const B& bin, const Weights& w,
                                              const Runs& q, int k, Lds<NT>& sh) {
    int size = 128;
    while (size < k) size *= 2;
    for (int i = k + threadIdx.x; i < size; i += NT) sh.second[i] = ~0ull;
    __syncthreads();
    for (int m = 2; m <= size; m *= 2)
        for (int j = m / 2; j > 0; j /= 2) {
            for (int i = threadIdx.x; i < size / 2; i += NT) {
                const int f = (i & -j) * 2 + (i & (j - 1)), g = f + j;
                const u64 x = sh.second[f], y = sh.second[g];
                if ((x > y) == ((f & m) == 0)) {
                    sh.second[f] = y;
                    sh.second[g] = x;
                }
            }
            __syncthreads();
        }
    // Sums in front of each element: those of its bin, and of the bin's elements
    // before it.  The bin's first takes the list's sum there off the bin's.
    const int per = (k + NT - 1) / NT, i0 = threadIdx.x * per, i1 = i0 + per < k ? i0 + per : k;
    u64 sum = 0, all;
    unsigned none = 0;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) sum += w(entry_value(sh.second[i]));
    block_scan(sum, none, &all, sh);
    u64 p = sum;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        const float x = entry_value(sh.second[i]);
        const int b = bin(x);
        if (i == 0 || bin(entry_value(sh.second[i - 1])) != b) {
            sh.mass[b] -= p;
            sh.count[b] -= (unsigned)i;
        }
        p += w(x);
    }
    if (threadIdx.x < 8) {
        sh.at[threadIdx.x] = 0;
        sh.to[threadIdx.x] = 0;
    }
    __syncthreads();
    // the first element whose running sum is above target: that sum, and the element
    auto place = [&](u64 target, int slot) {
        u64 r = sum;
#pragma unroll 1
        for (int i = i0; i < i1; ++i) {
            const float x = entry_value(sh.second[i]);
            const u64 e = w(x), before = sh.mass[bin(x)] + r;
            if (before <= target && target - before < e) {
                sh.to[slot] = before + e;
                sh.at[slot] = i + 1;
            }
            r += e;
        }
        __syncthreads();
        return sh.to[slot];
    };
    u64 top = q.total;
    if (s.k < a.V) {
        u64 r = sum;
#pragma unroll 1
        for (int i = i0; i < i1; ++i) {
            const float x = entry_value(sh.second[i]);
            const int b = bin(x);
            r += w(x);
            if (sh.count[b] + (unsigned)i == (unsigned)(s.k - 1)) sh.to[0] = sh.mass[b] + r;
        }
        __syncthreads();
        if (sh.to[0]) top = sh.to[0];
    }
    u64 kept = top;
    if (s.p < 1.f) {
        const u64 got = place(p_target(s.p, top), 1);
        if (!got) return false;
        kept = got < kept ? got : kept;
    }
    if (s.least && q.least_mass < kept) kept = q.least_mass;
    place((u64)(s.u * (double)kept), 2);
    if (!sh.at[2]) return false;
    if (threadIdx.x == 0) {
        const u64 l = sh.second[sh.at[2] - 1];
        gptr(a.token)[row] = (int32_t)(unsigned)l;
        if (a.prob) gptr(a.prob)[row] = (float)(w.scaled(entry_value(l)) / (double)kept);
    }
    return true;
}

// The token from the n elements in the list, which are all of runs r; false
// where its place is not found (too many elements close together).
template <int NT>
__device__ __forceinline__ bool finish_row(const SampleArgs& a, int row, const Settings& s, const Bins& y, const Weights& w,
                                           const Runs& r, int n, Lds<NT>& sh) {
    if (n <= kFew) return finish_short(a, row, s, y, w, r, n, sh);
    // the runs' bins, each cut into 2^shift (no choice between variables: the
    // compiler makes it an array in LDS, addressed by the dispatch packet, which is in host memory: 10 us)
    const int len0 = r.hi[0] - r.lo[0] + 1, len1 = r.lo[1] != kNone ? r.hi[1] - r.lo[1] + 1 : 0;
    const int len2 = r.lo[2] != kNone ? r.hi[2] - r.lo[2] + 1 : 0;
    int shift = 8;
    while (((len0 + len1 + len2) << shift) > kBins) --shift;
    const int start1 = r.lo[1] != kNone ? len0 << shift : kNone;
    const int start2 = r.lo[2] != kNone ? (len0 + len1) << shift : kNone;
    const int lo1 = r.lo[1], lo2 = r.lo[2];
    const int off0 = -r.lo[0] * (1 << shift), off1 = (len0 - lo1) * (1 << shift) - off0;
    const int off2 = (len0 + len1 - lo2) * (1 << shift) - off1 - off0;
    auto bin = [=](float x) {
        const int f = (int)(y(x) * 256.f), b = f >> 8;  // (exact; below 0 by a rounding: the first)
        int i = (f >> (8 - shift)) + off0;
        i += b >= lo1 ? off1 : 0;
        i += b >= lo2 ? off2 : 0;
        return i < 0 ? 0 : i < kBins ? i : kBins - 1;
    };
    clear_bins(sh);
    u64 kept = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += NT) {
        const float x = entry_value(sh.list[i]);
        const u64 e = w(x);
        const int b = bin(x);
        atomicAdd(&sh.mass[b], e);
        atomicAdd(&sh.count[b], 1u);
        kept += e >= s.least ? e : 0;
    }
    if (r.total == 0 && s.least) {
        kept = wave_sum(kept);
        if ((threadIdx.x & 63) == 0) atomicAdd(&sh.least_mass, kept);
    }
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    const Runs q = level_of(s, a.V, true, &r, start1, start2, sh);
    // the elements of its runs
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += NT) {
        const u64 e = sh.list[i];
        const int b = bin(entry_value(e));
        if ((b >= q.lo[0] && b <= q.hi[0]) || (b >= q.lo[1] && b <= q.hi[1]) || (b >= q.lo[2] && b <= q.hi[2])) {
            const int at = atomicAdd(&sh.n, 1);
            if (at < kSecond) sh.second[at] = e;
        }
    }
    __syncthreads();
    const int k = sh.n;
    if (k <= kFew) return finish_few(a, row, s, bin, w, q, k, sh);
    if (k > kSecond) return false;
    const int nv = values_of(bin, q, k, sh);
    return nv ? finish_values(a, row, s, bin, w, q, k, nv, sh) : finish_sorted(a, row, s, bin, w, q, k, sh);
}

// 2^44 times 2^(j / 256).
__device__ __forceinline__ void fill_table(double* table) {
    if (threadIdx.x < 256) table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 256) + 44.0);
    __syncthreads();
}

template <int TYPE>
__device__ __forceinline__ const typename Logit<TYPE>::T* row_of(const SampleArgs& a, int row) {
    return reinterpret_cast<const typename Logit<TYPE>::T*>(a.logits + (long long)row * a.stride);
}

// Rows that need no sums: of nothing to draw, and at temperature 0.
__device__ __forceinline__ bool no_sums(const Extent& x, const Settings& s) {
    return x.high == -__builtin_inff() || s.T == 0.0;
}
// Rows with an infinite logit go the general path.
__device__ __forceinline__ bool infinite(const Extent& x) { return x.high == __builtin_inff(); }

template <int TYPE, int NT>
__device__ __forceinline__ void settle(const SampleArgs& a, int row, const Extent& x, LdsScan<NT>& sh) {
    const bool none = x.high == -__builtin_inff();
    const int i = none ? -1 : first_of<TYPE>(row_of<TYPE>(a, row), a.V, cleaned(x.high), sh);
    if (threadIdx.x == 0) {
        gptr(a.token)[row] = i;
        if (a.prob) gptr(a.prob)[row] = none ? 0.f : 1.f;
    }
}

constexpr int kRowThreads = 1024, kSliceThreads = 512;
constexpr int kSliceList = 4096;

// One workgroup a row, start to end.
template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_rows_kernel(SampleArgs a) {
    __shared__ Lds<kRowThreads> sh;
    const int row = blockIdx.x;
    const auto* x = row_of<TYPE>(a, row);
    const Settings s = settings_of(a, row);
    fill_table(sh.table);
    const Extent ext = extent_of<TYPE>(x, 0, a.V, sh);
    if (no_sums(ext, s)) {
        settle<TYPE>(a, row, ext, sh);
        return;
    }
    if (!infinite(ext)) {
        const Bins y = bins_of(ext.high, ext.low, s.T);
        const Weights w = weights_of(sh.table, cleaned(ext.high), s.T);
        const int mode = mode_of(s, a.V);
        clear_bins(sh);
        fill_bins<TYPE>(x, 0, a.V, mode, s.least, y, w, sh);
        const Runs r = level_of(s, a.V, mode != kCount, nullptr, kNone, kNone, sh);
        fill_list<TYPE>(x, 0, a.V, y, r, sh);
        const int n = sh.n;
        if (n <= kList) {
            for (int i = threadIdx.x; i < n; i += kRowThreads)
                sh.list[i] = entry_of(Logit<TYPE>::raw(gptr(x)[sh.index[i]]), (int)sh.index[i]);
            __syncthreads();
            if (finish_row(a, row, s, y, w, r, n, sh)) return;
        }
        __syncthreads();
    }
    sample_row<TYPE>(a, row, sh.table, sh.general);
}

// ---- few rows: slices of a row by many workgroups, four launches ----

__device__ __forceinline__ void slice_of(const SampleArgs& a, int& row, int& g, int& i0, int& i1) {
    row = blockIdx.x / a.slices;
    g = blockIdx.x - row * a.slices;
    const int per = ((a.V + a.slices - 1) / a.slices + 7) / 8 * 8;
    i0 = g * per < a.V ? g * per : a.V;
    i1 = i0 + per < a.V ? i0 + per : a.V;
}

__device__ __forceinline__ Extent row_extent(const SampleArgs& a, const SampleRow* z) {
    Extent x{-__builtin_inff(), __builtin_inff()};
    const int i = threadIdx.x & 63;
    if (i < a.slices) x = Extent{gptr(z->slice_high)[i], gptr(z->slice_low)[i]};
    for (int s = 1; s < 64; s <<= 1) x.join(__shfl_xor(x.high, s), __shfl_xor(x.low, s));
    return x;
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void sample_max_kernel(SampleArgs a) {
    constexpr int NT = kSliceThreads;
    __shared__ LdsScan<NT> sh;
    int row, g, i0, i1;
    slice_of(a, row, g, i0, i1);
    SampleRow* z = a.ws + row;
    // the row's sums, cleared for the next launch
    for (int i = g * NT + threadIdx.x; i < kBins; i += a.slices * NT) {
        gptr(z->mass)[i] = 0;
        gptr(z->count)[i] = 0;
    }
    const Extent x = extent_of<TYPE>(row_of<TYPE>(a, row), i0, i1, sh);
    if (threadIdx.x == 0) {
        gptr(z->slice_high)[g] = x.high;
        gptr(z->slice_low)[g] = x.low;
        if (g == 0) {
            *gptr(&z->n) = 0;
            *gptr(&z->least_mass) = 0;
        }
    }
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void sample_bins_kernel(SampleArgs a) {
    constexpr int NT = kSliceThreads;
    __shared__ LdsBins<NT> sh;
    int row, g, i0, i1;
    slice_of(a, row, g, i0, i1);
    SampleRow* z = a.ws + row;
    const Extent x = row_extent(a, z);
    const Settings s = settings_of(a, row);
    if (no_sums(x, s) || infinite(x)) return;
    const int mode = mode_of(s, a.V);
    if (mode != kCount) fill_table(sh.table);
    clear_bins(sh);
    fill_bins<TYPE>(row_of<TYPE>(a, row), i0, i1, mode, s.least, bins_of(x.high, x.low, s.T),
                    weights_of(sh.table, x.high, s.T), sh);
    for (int i = threadIdx.x; i < kBins; i += NT) {
        if (mode != kCount && sh.mass[i]) atomicAdd(&z->mass[i], sh.mass[i]);
        if (mode != kMass && sh.count[i]) atomicAdd(&z->count[i], sh.count[i]);
    }
    if (threadIdx.x == 0 && sh.least_mass) atomicAdd(&z->least_mass, sh.least_mass);
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void sample_list_kernel(SampleArgs a) {
    constexpr int NT = kSliceThreads;
    __shared__ LdsList<NT, kSliceList> sh;
    int row, g, i0, i1;
    slice_of(a, row, g, i0, i1);
    SampleRow* z = a.ws + row;
    const Extent x = row_extent(a, z);
    const Settings s = settings_of(a, row);
    if (no_sums(x, s) || infinite(x)) return;
    {
        constexpr int PER = kBins / NT;
        u64 m[PER];
        unsigned c[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            m[i] = gptr(z->mass)[threadIdx.x + i * NT];
            c[i] = gptr(z->count)[threadIdx.x + i * NT];
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            sh.mass[threadIdx.x + i * NT] = m[i];
            sh.count[threadIdx.x + i * NT] = c[i];
        }
    }
    if (threadIdx.x == 0) sh.least_mass = *gptr(&z->least_mass);
    __syncthreads();
    const Runs r = level_of(s, a.V, mode_of(s, a.V) != kCount, nullptr, kNone, kNone, sh);
    if (g == 0 && threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            z->lo[i] = r.lo[i];
            z->hi[i] = r.hi[i];
            z->run_mass[i] = r.mass[i];
            z->run_count[i] = r.count[i];
        }
        z->total = r.total;
    }
    fill_list<TYPE>(row_of<TYPE>(a, row), i0, i1, bins_of(x.high, x.low, s.T), r, sh);
    const int n = sh.n;
    // (more than the slice's list holds: none of the row's list is used)
    if (threadIdx.x == 0) sh.at[0] = n ? (int)atomicAdd(&z->n, (unsigned)(n <= kSliceList ? n : kList + 1)) : 0;
    __syncthreads();
    const int at = sh.at[0];
    for (int i = threadIdx.x; i < n && i < kSliceList && at + i < kList; i += NT)
        gptr(z->list)[at + i] = entry_of(Logit<TYPE>::raw(gptr(row_of<TYPE>(a, row))[sh.index[i]]), (int)sh.index[i]);
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void sample_finish_kernel(SampleArgs a) {
    constexpr int NT = kSliceThreads;
    __shared__ Lds<NT> sh;
    const int row = blockIdx.x;
    const SampleRow* z = a.ws + row;
    const Extent x = row_extent(a, z);
    const Settings s = settings_of(a, row);
    const int n = (int)*gptr(&z->n);
    Runs r;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        r.lo[i] = gptr(z->lo)[i];
        r.hi[i] = gptr(z->hi)[i];
        r.mass[i] = gptr(z->run_mass)[i];
        r.count[i] = gptr(z->run_count)[i];
    }
    r.total = *gptr(&z->total);
    r.least_mass = *gptr(&z->least_mass);
    if (no_sums(x, s)) {
        settle<TYPE>(a, row, x, sh);
        return;
    }
    fill_table(sh.table);
    if (!infinite(x) && n <= kList) {
        for (int i = threadIdx.x; i < n; i += NT) sh.list[i] = gptr(z->list)[i];
        __syncthreads();
        if (finish_row(a, row, s, bins_of(x.high, x.low, s.T), weights_of(sh.table, x.high, s.T), r, n, sh)) return;
        __syncthreads();
    }
    sample_row<TYPE>(a, row, sh.table, sh.general);
}

// ---- calls that take the largest logit of every row, whatever else: temperature
// 0 or top_k 1 on the host.  No workgroup needs what another found, so a row's
// slices and one wave that joins them are two launches, the logits read once:
// 300 x 128256 27.3 us and 43.4 with temperatures of 0 on the device, 64 rows
// 10.6 and 27.6 of kernels, 3 rows 5.9 and 33. ----

// The least entry of a workgroup's threads, to the first wave.
template <int NT>
__device__ __forceinline__ u64 least_entry(u64 l, u64* red) {
    auto wave = [](u64 v) {
        for (int s = 1; s < 64; s <<= 1) {
            const u64 o = (u64)__shfl_xor((long long)v, s);
            v = o < v ? o : v;
        }
        return v;
    };
    l = wave(l);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = l;
    __syncthreads();
    return wave(threadIdx.x < NT / 64 ? red[threadIdx.x] : ~0ull);
}

__device__ __forceinline__ void settle_entry(const SampleArgs& a, int row, u64 l) {
    const bool none = (unsigned)(l >> 32) == ~key_of(-__builtin_inff());
    gptr(a.token)[row] = none ? -1 : (int32_t)(unsigned)l;
    if (a.prob) gptr(a.prob)[row] = none ? 0.f : 1.f;
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void sample_largest_kernel(SampleArgs a) {
    constexpr int NT = kSliceThreads;
    __shared__ u64 red[NT / 64];
    int row, g, i0, i1;
    slice_of(a, row, g, i0, i1);
    float best = -__builtin_inff();
    int at = i0;
    each<TYPE, NT>(row_of<TYPE>(a, row), i0, i1, [&](const auto& v, int i) {
#pragma unroll
        for (int e = 0; e < length_of(v); ++e) {
            const float x = cleaned(v[e]);
            const bool more = x > best || (x == best && i + e < at);
            best = more ? x : best;
            at = more ? i + e : at;
        }
    });
    const u64 l = least_entry<NT>(entry_of(best, at), red);
    if (threadIdx.x != 0) return;
    if (a.slices == 1)
        settle_entry(a, row, l);
    else
        gptr(a.ws[row].list)[g] = l;
}

__global__ __launch_bounds__(64) void sample_largest_join_kernel(SampleArgs a) {
    __shared__ u64 red[1];
    const int i = threadIdx.x;
    const u64 l = least_entry<64>(i < a.slices ? gptr(a.ws[blockIdx.x].list)[i] : ~0ull, red);
    if (i == 0) settle_entry(a, blockIdx.x, l);
}

template <int TYPE>
hipError_t launch_largest(const SampleArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(sample_largest_kernel<TYPE>, dim3(a.rows * a.slices), dim3(kSliceThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.slices == 1) return e;
    hipLaunchKernelGGL(sample_largest_join_kernel, dim3(a.rows), dim3(64), 0, st, a);
    return hipGetLastError();
}

template <int TYPE>
hipError_t launch(const SampleArgs& a, hipStream_t st) {
    const bool cold = !a.p.temperature_dev && a.p.temperature == 0.f, one = !a.p.top_k_dev && a.p.top_k == 1;
    if (cold || one) return launch_largest<TYPE>(a, st);
    const dim3 rows(a.rows), block(kSliceThreads);
    if (a.slices == 1) {
        hipLaunchKernelGGL(sample_rows_kernel<TYPE>, rows, dim3(kRowThreads), 0, st, a);
        return hipGetLastError();
    }
    const dim3 grid(a.rows * a.slices);
    hipLaunchKernelGGL(sample_max_kernel<TYPE>, grid, block, 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(sample_bins_kernel<TYPE>, grid, block, 0, st, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(sample_list_kernel<TYPE>, grid, block, 0, st, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(sample_finish_kernel<TYPE>, rows, block, 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, int type, hipStream_t st) {
    if (type == TER_HIP_T_F16) return launch<TER_HIP_T_F16>(a, st);
    if (type == TER_HIP_T_BF16) return launch<TER_HIP_T_BF16>(a, st);
    return launch<TER_HIP_T_F32>(a, st);
}

}  // namespace terhip

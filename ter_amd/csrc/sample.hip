// sample.hip -- a token for each row of logits: temperature, top-k, top-p,
// min-p and a given random number.
//
// Every cut and the draw itself are places in one order: falling logits, of
// equal ones the lower index first.  A place is found by its measure, the
// number of elements up to it (top-k) or the sum of their weights (top-p, the
// draw), as the first element at which the running measure exceeds a target.
// Weights are integers (see Weights), so sums do not depend on the order in
// which a wave, an atomic or a workgroup adds them.
#include "common.h"
#include "sample.h"

namespace terhip {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;

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
    const double* table;  // 2^(j / 256), in LDS
    double m, c;

    __device__ __forceinline__ double scaled(float x) const {
        double t = ((double)x - m) * c;
        t = __builtin_fmax(t, -12032.0);  // 2^-47; also of -infinity, and of NaN (-infinity times 0)
        const double tn = t + 6755399441055744.0;  // 1.5 * 2^52: rounds to an integer, in the low bits
        const int n = (int)__builtin_bit_cast(u64, tn);
        const double r = t - (tn - 6755399441055744.0);
        constexpr double a = 0.0027076061740622863;  // ln 2 / 256
        double p = __builtin_fma(r, a * a * a / 6, a * a / 2);
        p = __builtin_fma(r, p, a);
        p = __builtin_fma(r, p, 1.0);
        return __builtin_ldexp(table[n & 255] * p, 44 + (n >> 8));
    }
    __device__ __forceinline__ u64 operator()(float x) const {
        // (below 2^52 the low bits of a number added to 2^52 are its nearest integer)
        return __builtin_bit_cast(u64, scaled(x) + 4503599627370496.0) - 0x4330000000000000ull;
    }
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
    s.T = t > 0.f ? (double)t : 0.0;
    s.k = k > 0 && k < a.V ? k : a.V;
    s.p = p < 1.f ? p : 1.f;  // (NaN: 1)
    s.least = q > 0.f ? (u64)__builtin_ceil((double)__builtin_fminf(q, 1.f) * kOne) : 0;
    s.u = (double)__builtin_fminf(__builtin_fmaxf(u, 0.f), 0.99999994f);
    return s;
}

struct Shared {
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
template <int TYPE>
struct Row {
    typedef typename Logit<TYPE>::T T;
    const TER_GLOBAL T* x;
    int V;
    __device__ float operator[](int i) const { return cleaned(Logit<TYPE>::raw(x[i])); }

    __device__ unsigned largest(Shared& sh) const {
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
    __device__ u64 mass(Shared& sh, const Weights& w, u64 least) const {
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
    __device__ int tie(Shared& sh, unsigned key, unsigned rank) const {
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
    __device__ Place find(Shared& sh, const Weights& w, bool by_count, u64 target) const {
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
// for the draw.  Right for every row; the general path.
template <int TYPE>
__device__ void sample_row(const SampleArgs& a, int row, const double* table, Shared& sh) {
    Row<TYPE> x{gptr(reinterpret_cast<const typename Logit<TYPE>::T*>(a.logits + (long long)row * a.stride)), a.V};
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


// ---- the usual path: two levels ----
//
// The row is cut into bins of falling weight: bin b of logit x is
// floor((m - x) / T * (kBins - 1) / 31.5), clipped to kBins - 1, in binary32.
// Its steps are monotonic, so bins stand in the order of the logits and one
// holds all elements between two values; from 31.5 on weights are 0, so the
// last bin has none (and is not counted up).  A histogram of numbers or of
// weights over the bins finds the bin of each cut and of the draw; the elements
// of those bins, few, are then listed, sorted, and the places found exactly.
// A cut moves what later ones start from, so before the list is there a later
// place is known to a bin or two only: all of them are listed.
constexpr int kCountK = 1024; // up to this top_k everything kept is listed, and weights are computed for the list alone

struct Bins {
    float mh, cb;  // m / 2; bins for half a logit
    __device__ __forceinline__ int operator()(float x) const {
        // (halves do not overflow; NaN and -infinity: the last; +infinity: the first)
        return (int)(unsigned)__builtin_fminf(__builtin_fmaf(x, -0.5f, mh) * cb, (float)(kBins - 1));
    }
};

__device__ __forceinline__ Bins bins_of(float m, double T) {
    return Bins{0.5f * m, (float)__builtin_fmin(2.0 * (kBins - 1) / 31.5 / T, 3e38)};
}

// What a row's histogram counts.
enum Mode { kCount = 1, kMass = 2, kBoth = 3 };
__device__ __forceinline__ int mode_of(const Settings& s, int V) {
    return s.k <= kCountK && s.k < V ? kCount : s.k < V ? kBoth : kMass;
}

struct Lds {
    double table[256];
    union {
        struct {
            u64 mass[kBins];
            unsigned count[kBins];
            u64 list[kList];
        };
        Shared general;
    };
    u64 wave_mass[kWaves];
    unsigned wave_count[kWaves];
    u64 place[8];
    int cross[8];
    int n;
};

// f(x) or f(x, i) of elements [i0, i1) of a row by `nt` threads, 16 bytes a
// load, four loads in flight.
template <int TYPE, typename F>
__device__ __forceinline__ void each(const typename Logit<TYPE>::T* row, int i0, int i1, int t, int nt, F f) {
    typedef typename Logit<TYPE>::T T;
    typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
    constexpr int VE = 16 / (int)sizeof(T), U = 4;
    const TER_GLOBAL T* p = gptr(row) + i0;
    const int n = i1 - i0;
    int head = (int)((0 - reinterpret_cast<uintptr_t>(row + i0)) & 15) / (int)sizeof(T);
    head = head < n ? head : n;
    const int nv = (n - head) / VE, tail = head + nv * VE;
    if (t < head) f(Logit<TYPE>::raw(p[t]), i0 + t);
    if (t < n - tail) f(Logit<TYPE>::raw(p[tail + t]), i0 + tail + t);
    const TER_GLOBAL u32x4* v = reinterpret_cast<const TER_GLOBAL u32x4*>(p + head);
    for (int a = t; a < nv; a += U * nt) {
        u32x4 r[U];
#pragma unroll
        for (int q = 0; q < U; ++q) r[q] = v[a + q * nt < nv ? a + q * nt : nv - 1];
#pragma unroll
        for (int q = 0; q < U; ++q) {
            if (a + q * nt >= nv) break;
            const int i = i0 + head + (a + q * nt) * VE;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned w = r[q][e];
                if constexpr (TYPE == TER_HIP_T_F32) {
                    f(__builtin_bit_cast(float, w), i + e);
                } else {
                    f(Logit<TYPE>::raw((uint16_t)w), i + 2 * e);
                    f(Logit<TYPE>::raw((uint16_t)(w >> 16)), i + 2 * e + 1);
                }
            }
        }
    }
}

// The largest logit of [i0, i1), to every thread of the workgroup.
template <int TYPE>
__device__ float largest_of(const typename Logit<TYPE>::T* row, int i0, int i1, Lds& sh) {
    float m = -__builtin_inff();
    each<TYPE>(row, i0, i1, threadIdx.x, kThreads, [&](float x, int) { m = __builtin_fmaxf(m, x); });
    for (int s = 1; s < 64; s <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, s));
    if ((threadIdx.x & 63) == 0) sh.wave_count[threadIdx.x >> 6] = __builtin_bit_cast(unsigned, m);
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) m = __builtin_fmaxf(m, __builtin_bit_cast(float, sh.wave_count[i]));
    __syncthreads();
    return cleaned(m);
}

// Index of the first element equal to m (V: none).
template <int TYPE>
__device__ int first_of(const typename Logit<TYPE>::T* row, int V, float m, Lds& sh) {
    int at = V;
    each<TYPE>(row, 0, V, threadIdx.x, kThreads, [&](float x, int i) { at = cleaned(x) == m && i < at ? i : at; });
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_xor(at, s);
        at = o < at ? o : at;
    }
    if ((threadIdx.x & 63) == 0) sh.wave_count[threadIdx.x >> 6] = (unsigned)at;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) at = (int)sh.wave_count[i] < at ? (int)sh.wave_count[i] : at;
    __syncthreads();
    return at;
}

__device__ __forceinline__ void clear_bins(Lds& sh) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        sh.mass[i] = 0;
        sh.count[i] = 0;
    }
}

// Elements [i0, i1) into the histogram in LDS.
template <int TYPE>
__device__ void fill_bins(const typename Logit<TYPE>::T* row, int i0, int i1, int mode, const Bins& bin,
                          const Weights& w, Lds& sh) {
    if (mode == kCount) {
        each<TYPE>(row, i0, i1, threadIdx.x, kThreads, [&](float x, int) {
            const int b = bin(x);
            if (b < kBins - 1) atomicAdd(&sh.count[b], 1u);
        });
    } else if (mode == kMass) {
        each<TYPE>(row, i0, i1, threadIdx.x, kThreads, [&](float x, int) {
            const int b = bin(x);
            if (b < kBins - 1) atomicAdd(&sh.mass[b], w(x));
        });
    } else {
        each<TYPE>(row, i0, i1, threadIdx.x, kThreads, [&](float x, int) {
            const int b = bin(x);
            if (b < kBins - 1) {
                atomicAdd(&sh.count[b], 1u);
                atomicAdd(&sh.mass[b], w(x));
            }
        });
    }
}

// Exclusive running sums over a workgroup's threads of m and n; the whole in *tm.
__device__ void block_scan(u64& m, unsigned& n, u64* tm, Lds& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 im = m;
    unsigned in = n;
    for (int s = 1; s < 64; s <<= 1) {
        const u64 om = (u64)__shfl_up((long long)im, s);
        const unsigned on = (unsigned)__shfl_up((int)in, s);
        if (lane >= s) {
            im += om;
            in += on;
        }
    }
    if (lane == 63) {
        sh.wave_mass[wave] = im;
        sh.wave_count[wave] = in;
    }
    __syncthreads();
    u64 bm = 0, all = 0;
    unsigned bn = 0;
    for (int i = 0; i < kWaves; ++i) {
        const u64 e = sh.wave_mass[i];
        bm += i < wave ? e : 0;
        bn += i < wave ? sh.wave_count[i] : 0;
        all += e;
    }
    m = bm + im - m;
    n = bn + in - n;
    *tm = all;
    __syncthreads();
}

// The bins to list, from the histogram in LDS, which becomes its running sums.
struct Ranges {
    int lo[4], hi[4];  // (lo > hi: none)
    int bk;            // bin of the last element of the top_k (kBins - 1: weightless, or no top_k)
    u64 total;         // sum of all weights (not of mode kCount)
    u64 least_before;  // sum of the weights before bin lo[2]
    __device__ __forceinline__ bool has(int b) const {
        bool r = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) r = r || (b >= lo[i] && b <= hi[i]);
        return r;
    }
};

__device__ __forceinline__ u64 p_target(float p, u64 sum) {
    const double want = __builtin_ceil((double)p * (double)sum);
    return want > 1.0 ? (u64)want - 1 : 0;
}

__device__ Ranges ranges_of(const Settings& s, int V, int mode, Lds& sh) {
    constexpr int PER = kBins / kThreads;  // bins of a thread
    const int b0 = threadIdx.x * PER;
    u64 m[PER], ms = 0;
    unsigned n[PER], ns = 0;
    for (int i = 0; i < PER; ++i) {
        m[i] = ms;
        n[i] = ns;
        ms += sh.mass[b0 + i];
        ns += sh.count[b0 + i];
    }
    const u64 thread_mass = ms;
    const unsigned thread_count = ns;
    Ranges r;
    block_scan(ms, ns, &r.total, sh);
    for (int i = 0; i < PER; ++i) {
        sh.mass[b0 + i] = m[i] += ms;
        sh.count[b0 + i] = n[i] += ns;
    }
    const u64 mass_end = ms + thread_mass;
    const unsigned count_end = ns + thread_count;
    // the bin in which a running sum exceeds a target
    auto cross = [&](u64 target, int slot) {
        for (int i = 0; i < PER; ++i)
            if (m[i] <= target && target < (i + 1 < PER ? m[i + 1] : mass_end)) sh.cross[slot] = b0 + i;
    };
    if (threadIdx.x == 0)
        for (int i = 0; i < 8; ++i) sh.cross[i] = kBins - 1;
    __syncthreads();
    if (s.k < V)
        for (int i = 0; i < PER; ++i)
            if (n[i] <= (unsigned)(s.k - 1) && (unsigned)(s.k - 1) < (i + 1 < PER ? n[i + 1] : count_end))
                sh.cross[0] = b0 + i;
    __syncthreads();
    r.bk = sh.cross[0];
    for (int i = 0; i < 4; ++i) {
        r.lo[i] = 1;
        r.hi[i] = 0;
    }
    r.least_before = 0;
    if (mode == kCount) {
        r.lo[0] = 0;
        r.hi[0] = r.bk < kBins - 1 ? r.bk : kBins - 2;
        __syncthreads();
        return r;
    }
    u64 lo = r.total, hi = r.total;  // the sum of what is kept, so far
    if (r.bk < kBins - 1) {
        lo = sh.mass[r.bk];
        hi = sh.mass[r.bk + 1];
        r.lo[0] = r.hi[0] = r.bk;
    }
    if (s.p < 1.f) {
        cross(p_target(s.p, lo), 1);
        cross(p_target(s.p, hi), 2);
        __syncthreads();
        const int bl = sh.cross[1], bh = sh.cross[2];  // (both below the last: their targets are below the total)
        r.lo[1] = bl;
        r.hi[1] = bh;
        const u64 a = sh.mass[bl], b = sh.mass[bh + 1];
        lo = a < lo ? a : lo;
        hi = b < hi ? b : hi;
    }
    if (s.least) {
        // where weights fall below `least` (2^-44 or more: bin 1983 at most): the bin of that logit, give or take
        // the rounding of its place
        const int c = (int)(-log((double)s.least / kOne) * ((kBins - 1) / 31.5));
        r.lo[2] = c > 0 ? c - 1 : 0;
        r.hi[2] = c + 1;
        const u64 a = r.least_before = sh.mass[r.lo[2]], b = sh.mass[r.hi[2] + 1];
        lo = a < lo ? a : lo;
        hi = b < hi ? b : hi;
    }
    cross((u64)(s.u * (double)lo), 3);
    cross((u64)(s.u * (double)hi), 4);
    __syncthreads();
    r.lo[3] = sh.cross[3];
    r.hi[3] = sh.cross[4];
    __syncthreads();
    return r;
}

// The list's n elements (key and index, inverted key first), padded to a power
// of two, into their order.
__device__ void sort_list(u64* list, int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int i = threadIdx.x; i < size / 2; i += kThreads) {
                const int a = (i & -j) * 2 + (i & (j - 1)), b = a + j;
                const u64 x = list[a], y = list[b];
                if ((x > y) == ((a & k) == 0)) {
                    list[a] = y;
                    list[b] = x;
                }
            }
            __syncthreads();
        }
}

__device__ __forceinline__ u64 entry_of(float x, int i) { return (u64)~key_of(cleaned(x)) << 32 | (unsigned)i; }

// The token from the listed elements of ranges r, whose running sums are in
// LDS; false where a place is not among them.
__device__ bool finish_row(const SampleArgs& a, int row, const Settings& s, int mode, const Bins& bin, const Weights& w,
                           const Ranges& r, int n, Lds& sh) {
    constexpr int PER = kList / kThreads;
    sort_list(sh.list, n);
    const int per = (n + kThreads - 1) / kThreads, i0 = threadIdx.x * per;
    const int n0 = n - i0 < per ? n - i0 : per;  // elements of this thread (below 0: none)
    auto value = [&](int i) { return value_of(~(unsigned)(sh.list[i0 + i] >> 32)); };
    u64 e[PER], before = 0;
    unsigned none = 0;
    for (int i = 0; i < PER; ++i) {
        e[i] = i < n0 ? w(value(i)) : 0;
        before += e[i];
    }
    u64 all;
    block_scan(before, none, &all, sh);
    // running sums over the whole row: of the bin's start, and of its elements so far
    if (mode != kCount) {
        u64 p = before;
        for (int i = 0; i < PER; ++i) {
            if (i >= n0) break;
            const int b = bin(value(i));
            if (i0 + i == 0 || bin(value(i - 1)) != b) {
                sh.mass[b] -= p;
                sh.count[b] -= (unsigned)(i0 + i);
            }
            p += e[i];
        }
    }
    if (threadIdx.x < 8) sh.place[threadIdx.x] = 0;
    __syncthreads();
    u64 at[PER];
    unsigned rank[PER];
    for (int i = 0; i < PER; ++i) {
        at[i] = before;
        rank[i] = (unsigned)(i0 + i);
        if (mode != kCount && i < n0) {
            const int b = bin(value(i));
            at[i] += sh.mass[b];
            rank[i] += sh.count[b];
        }
        before += e[i];
    }
    // places are written as their running sum, which is above 0
    u64 sum = mode == kCount ? all : r.total;
    if (r.bk < kBins - 1) {
        for (int i = 0; i < PER; ++i)
            if (i < n0 && rank[i] == (unsigned)(s.k - 1)) sh.place[0] = at[i] + e[i];
        __syncthreads();
        sum = sh.place[0];
    }
    u64 kept = sum;
    if (s.p < 1.f) {
        const u64 target = p_target(s.p, sum);
        for (int i = 0; i < PER; ++i)
            if (i < n0 && at[i] <= target && target < at[i] + e[i]) sh.place[1] = at[i] + e[i];
        __syncthreads();
        kept = sh.place[1] < kept ? sh.place[1] : kept;
    }
    if (s.least) {
        u64 most = threadIdx.x == 0 ? r.least_before : 0;
        for (int i = 0; i < PER; ++i)
            if (i < n0 && e[i] >= s.least) most = at[i] + e[i] > most ? at[i] + e[i] : most;
        if (most) atomicMax(&sh.place[2], most);
        __syncthreads();
        kept = sh.place[2] < kept ? sh.place[2] : kept;
    }
    const u64 target = (u64)(s.u * (double)kept);
    for (int i = 0; i < PER; ++i)
        if (i < n0 && at[i] <= target && target < at[i] + e[i]) {
            const u64 l = sh.list[i0 + i];
            gptr(a.token)[row] = (int32_t)(unsigned)l;
            if (a.prob) gptr(a.prob)[row] = (float)(w.scaled(value(i)) / (double)kept);
            sh.place[3] = 1;
        }
    __syncthreads();
    return kept != 0 && sh.place[3] != 0;
}

__device__ __forceinline__ void fill_table(double* table) {
    if (threadIdx.x < 256) table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 256));
    __syncthreads();
}

// Rows that need no sums: of nothing to draw, and at temperature 0.
template <int TYPE>
__device__ __forceinline__ bool settled(const SampleArgs& a, int row, const typename Logit<TYPE>::T* x, float m, double T,
                                        Lds& sh) {
    const bool none = m == -__builtin_inff();
    if (!none && T > 0.0) return false;
    const int i = none ? -1 : first_of<TYPE>(x, a.V, m, sh);
    if (threadIdx.x == 0) {
        gptr(a.token)[row] = i;
        if (a.prob) gptr(a.prob)[row] = none ? 0.f : 1.f;
    }
    return true;
}

template <int TYPE>
__device__ __forceinline__ const typename Logit<TYPE>::T* row_of(const SampleArgs& a, int row) {
    return reinterpret_cast<const typename Logit<TYPE>::T*>(a.logits + (long long)row * a.stride);
}

// Lists the elements of r among [i0, i1): sh.n of them, those past kList left out.
template <int TYPE>
__device__ void fill_list(const typename Logit<TYPE>::T* x, int i0, int i1, const Bins& bin, const Ranges& r, Lds& sh) {
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    each<TYPE>(x, i0, i1, threadIdx.x, kThreads, [&](float v, int i) {
        if (!r.has(bin(v))) return;
        const int at = atomicAdd(&sh.n, 1);
        if (at < kList) sh.list[at] = entry_of(v, i);
    });
    __syncthreads();
}

// One workgroup a row, start to end.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs a) {
    __shared__ Lds sh;
    const int row = blockIdx.x;
    const auto* x = row_of<TYPE>(a, row);
    fill_table(sh.table);
    const float m = largest_of<TYPE>(x, 0, a.V, sh);
    const Settings s = settings_of(a, row);
    if (settled<TYPE>(a, row, x, m, s.T, sh)) return;
    const Bins bin = bins_of(m, s.T);
    const Weights w = weights_of(sh.table, m, s.T);
    const int mode = mode_of(s, a.V);
    clear_bins(sh);
    __syncthreads();
    fill_bins<TYPE>(x, 0, a.V, mode, bin, w, sh);
    __syncthreads();
    const Ranges r = ranges_of(s, a.V, mode, sh);
    fill_list<TYPE>(x, 0, a.V, bin, r, sh);
    const int n = sh.n;
    if (n <= kList && finish_row(a, row, s, mode, bin, w, r, n, sh)) return;
    __syncthreads();
    sample_row<TYPE>(a, row, sh.table, sh.general);
}

// ---- few rows: slices of a row by many workgroups, four launches ----

__device__ __forceinline__ void slice_of(const SampleArgs& a, int& row, int& i0, int& i1) {
    row = blockIdx.x / a.slices;
    const int g = blockIdx.x - row * a.slices;
    const int per = ((a.V + a.slices - 1) / a.slices + 7) / 8 * 8;
    i0 = g * per < a.V ? g * per : a.V;
    i1 = i0 + per < a.V ? i0 + per : a.V;
}

__device__ __forceinline__ SampleRow* ws_of(const SampleArgs& a, int row) { return a.ws + row; }

__device__ __forceinline__ float row_max(const SampleArgs& a, const SampleRow* z) {
    float m = -__builtin_inff();
    for (int i = 0; i < a.slices; ++i) m = __builtin_fmaxf(m, gptr(z->slice_max)[i]);
    return m;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(SampleArgs a) {
    __shared__ Lds sh;
    int row, i0, i1;
    slice_of(a, row, i0, i1);
    const int g = blockIdx.x - row * a.slices;
    SampleRow* z = ws_of(a, row);
    // the row's sums, cleared for the next launch
    for (int i = g * kThreads + threadIdx.x; i < kBins; i += a.slices * kThreads) {
        gptr(z->mass)[i] = 0;
        gptr(z->count)[i] = 0;
    }
    const float m = largest_of<TYPE>(row_of<TYPE>(a, row), i0, i1, sh);
    if (threadIdx.x == 0) {
        gptr(z->slice_max)[g] = m;
        if (g == 0) *gptr(&z->n) = 0;
    }
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleArgs a) {
    __shared__ Lds sh;
    int row, i0, i1;
    slice_of(a, row, i0, i1);
    SampleRow* z = ws_of(a, row);
    const float m = row_max(a, z);
    const Settings s = settings_of(a, row);
    if (m == -__builtin_inff() || s.T == 0.0) return;
    const int mode = mode_of(s, a.V);
    if (mode != kCount) fill_table(sh.table);
    clear_bins(sh);
    __syncthreads();
    fill_bins<TYPE>(row_of<TYPE>(a, row), i0, i1, mode, bins_of(m, s.T), weights_of(sh.table, m, s.T), sh);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        if (mode != kCount && sh.mass[i]) atomicAdd(&z->mass[i], sh.mass[i]);
        if (mode != kMass && sh.count[i]) atomicAdd(&z->count[i], sh.count[i]);
    }
}

__device__ __forceinline__ void load_bins(const SampleRow* z, Lds& sh) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        sh.mass[i] = gptr(z->mass)[i];
        sh.count[i] = gptr(z->count)[i];
    }
    __syncthreads();
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_list_kernel(SampleArgs a) {
    __shared__ Lds sh;
    int row, i0, i1;
    slice_of(a, row, i0, i1);
    SampleRow* z = ws_of(a, row);
    const float m = row_max(a, z);
    const Settings s = settings_of(a, row);
    if (m == -__builtin_inff() || s.T == 0.0) return;
    load_bins(z, sh);
    const Ranges r = ranges_of(s, a.V, mode_of(s, a.V), sh);
    fill_list<TYPE>(row_of<TYPE>(a, row), i0, i1, bins_of(m, s.T), r, sh);
    const int n = sh.n;
    if (threadIdx.x == 0) sh.cross[0] = n ? (int)atomicAdd(&z->n, (unsigned)n) : 0;  // (V at most in all)
    __syncthreads();
    const int at = sh.cross[0];
    for (int i = threadIdx.x; i < n && i < kList && at + i < kList; i += kThreads) gptr(z->list)[at + i] = sh.list[i];
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleArgs a) {
    __shared__ Lds sh;
    const int row = blockIdx.x;
    const SampleRow* z = ws_of(a, row);
    const float m = row_max(a, z);
    const Settings s = settings_of(a, row);
    if (settled<TYPE>(a, row, row_of<TYPE>(a, row), m, s.T, sh)) return;
    const int mode = mode_of(s, a.V);
    fill_table(sh.table);
    load_bins(z, sh);
    const Ranges r = ranges_of(s, a.V, mode, sh);
    const int n = (int)*gptr(&z->n);
    if (n <= kList) {
        for (int i = threadIdx.x; i < n; i += kThreads) sh.list[i] = gptr(z->list)[i];
        __syncthreads();
        if (finish_row(a, row, s, mode, bins_of(m, s.T), weights_of(sh.table, m, s.T), r, n, sh)) return;
    }
    __syncthreads();
    sample_row<TYPE>(a, row, sh.table, sh.general);
}

template <int TYPE>
hipError_t launch(const SampleArgs& a, hipStream_t st) {
    const dim3 rows(a.rows), block(kThreads);
    if (a.slices <= 1) {
        hipLaunchKernelGGL(sample_rows_kernel<TYPE>, rows, block, 0, st, a);
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

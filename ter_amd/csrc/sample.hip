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
    double table[256];
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
__device__ void sample_row(const SampleArgs& a, int row, Shared& sh) {
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
    const Weights w{sh.table, (double)value_of(top), 369.32993046757463 / s.T};  // 256 log2(e) / T
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

__device__ __forceinline__ void fill_table(Shared& sh) {
    if (threadIdx.x < 256) sh.table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 256));
    __syncthreads();
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs a) {
    __shared__ Shared sh;
    fill_table(sh);
    sample_row<TYPE>(a, blockIdx.x, sh);
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, int type, hipStream_t st) {
    const dim3 grid(a.rows);
    if (type == TER_HIP_T_F16)
        hipLaunchKernelGGL(sample_rows_kernel<TER_HIP_T_F16>, grid, dim3(kThreads), 0, st, a);
    else if (type == TER_HIP_T_BF16)
        hipLaunchKernelGGL(sample_rows_kernel<TER_HIP_T_BF16>, grid, dim3(kThreads), 0, st, a);
    else
        hipLaunchKernelGGL(sample_rows_kernel<TER_HIP_T_F32>, grid, dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace terhip

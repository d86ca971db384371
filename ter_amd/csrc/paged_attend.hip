// paged_attend.hip -- causal attention of the new rows of a batch of sequences
// over a paged cache.  The simple form: one wave per row and query head, 64
// positions at a time (lane = position for the scores, lane = output elements
// for the sums), with the running maximum and sum of a softmax in one pass.
#include "common.h"
#include "paged.h"

namespace terhip {
namespace {

template <typename T, int HD>
__global__ __launch_bounds__(64) void paged_attend_kernel(PagedAttendArgs a) {
    constexpr int D = HD / 64;
    const int t = blockIdx.x, h = blockIdx.y, g = h / a.group, lane = threadIdx.x;
    const int b = paged_seq_of_row(a.b.row0, a.b.n_seq, t);
    if (b < 0) return;
    const int r0 = max(a.b.row0[b], 0), r1 = min(a.b.row0[b + 1], a.b.n_rows);
    const long long pos = (long long)max(a.b.kv_len[b], 0) - (r1 - r0) + (t - r0);
    const int lim = (int)min(max(pos + 1, 0ll), (long long)a.b.capacity);
    const int32_t* table = a.b.pages + (long long)b * a.b.pages_stride;
    const T* q = reinterpret_cast<const T*>(a.q + (long long)t * a.q_stride) + h * HD;
    float m = -__builtin_inff(), l = 0.f, o[D];
    for (int j = 0; j < D; ++j) o[j] = 0.f;
    for (int s0 = 0; s0 < lim; s0 += 64) {
        const int s = s0 + lane, n = min(64, lim - s0);
        long long at = -1;
        float score = -__builtin_inff();
        if (s < lim) {
            const int slot = s / a.c.page_size, page = table[slot];
            float dot = 0.f;
            if (page >= 0 && page < a.c.n_pages) {
                at = page * a.c.page_stride + (long long)(s - slot * a.c.page_size) * a.c.pos_stride +
                     (long long)g * a.c.head_stride;
                const T* k = reinterpret_cast<const T*>(a.c.k + at);
                for (int d = 0; d < HD; ++d) dot = __builtin_fmaf((float)q[d], (float)k[d], dot);
            }
            score = dot * a.scale;
        }
        float mx = score;
        for (int w = 32; w; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
        const float mn = fmaxf(m, mx), ref = mn == -__builtin_inff() ? 0.f : mn;
        const float al = __expf(m - ref), p = s < lim ? __expf(score - ref) : 0.f;
        l *= al;
        for (int j = 0; j < D; ++j) o[j] *= al;
        float sum = p;
        for (int w = 32; w; w >>= 1) sum += __shfl_xor(sum, w);
        l += sum;
        m = mn;
        for (int i = 0; i < n; ++i) {
            const float pi = __shfl(p, i);
            const long long ai = __shfl(at, i);
            if (ai < 0) continue;
            const T* v = reinterpret_cast<const T*>(a.c.v + ai);
            for (int j = 0; j < D; ++j) o[j] = __builtin_fmaf(pi, (float)v[lane * D + j], o[j]);
        }
    }
    T* out = reinterpret_cast<T*>(a.out + (long long)t * a.out_stride) + h * HD + lane * D;
    for (int j = 0; j < D; ++j) out[j] = (T)(lim > 0 ? o[j] / l : 0.f);
}

}  // namespace

hipError_t launch_paged_attend(const PagedAttendArgs& a, int hd, bool bf16, hipStream_t st) {
    const dim3 grid(a.b.n_rows, a.nh), block(64);
    if (hd == 128) {
        if (bf16)
            hipLaunchKernelGGL((paged_attend_kernel<__bf16, 128>), grid, block, 0, st, a);
        else
            hipLaunchKernelGGL((paged_attend_kernel<_Float16, 128>), grid, block, 0, st, a);
    } else {
        if (bf16)
            hipLaunchKernelGGL((paged_attend_kernel<__bf16, 64>), grid, block, 0, st, a);
        else
            hipLaunchKernelGGL((paged_attend_kernel<_Float16, 64>), grid, block, 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace terhip

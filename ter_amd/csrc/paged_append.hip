// paged_append.hip -- new keys and values of a batch of sequences into their
// cache pages, the position rotation of queries and keys applied on the way.
//
// For a row at position p and pair k of a head, angle a = p * theta^(-2k/d):
//   (x0, x1) -> (x0 cos a - x1 sin a, x0 sin a + x1 cos a),
// one fused multiply-add over the other product in binary32 each, rounded once
// to the element type.  cos and sin come from a table of the context: the
// angle of a far position needs more than binary32 (at position 10^5 its
// rounding alone is 4e-3 rad), so the table is made from angles in double.
//
// Bound by memory: every element is read and written once (30 heads of 128
// in a BitNet row: 15 KB), and a row's table entries (512 B) once.  A
// workgroup is one row, so its sequence, position and page are found once, by
// wave-uniform code, while its q, k and v loads are already in flight; a thread takes
// the two 16-byte pieces that hold eight whole pairs.  Measured: 8,760 rows of
// prompts (20 + 5 + 5 heads of 128, 135 MB) 24.7 us, 5.4 TB/s (a large copy
// reaches 4.85); 192 single tokens 3.7 us and one 2.7 us, the chain of
// boundary, length, page and store.
#include "common.h"
#include "paged.h"

namespace terhip {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Freqs {
    double f[64];
};

__global__ void paged_rope_table_kernel(float* tab, int half, int max_pos, Freqs fr) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)max_pos * half) return;
    const int p = (int)(i / half), k = (int)(i - (long long)p * half);
    double s, c;
    sincos((double)p * fr.f[k], &s, &c);
    gptr(tab)[2 * i] = (float)c;
    gptr(tab)[2 * i + 1] = (float)s;
}

template <typename T, int HD, bool kNeox>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    constexpr int P = HD / 16;  // threads (of two pieces) a head
    const int t = blockIdx.x;
    const int nq = a.q ? a.nh : 0;
    const int n = (nq + 2 * a.nkv) * P;
    int b = -2;
    long long pos = 0;
    char *kd = nullptr, *vd = nullptr;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        // (threads past the last item load it too, so that every lane takes
        // part in the search below, and store nothing)
        const int i = min(i0 + (int)threadIdx.x, n - 1), hh = i / P, c = i - hh * P;
        const bool is_q = hh < nq, is_k = !is_q && hh < nq + a.nkv;
        const int h = is_q ? hh : is_k ? hh - nq : hh - nq - a.nkv;
        // bytes of the thread's two pieces within the head
        const int o0 = kNeox ? 16 * c : 32 * c, o1 = kNeox ? 16 * c + HD : 32 * c + 16;
        const char* src = (is_q   ? a.q + (long long)t * a.q_stride
                           : is_k ? a.k + (long long)t * a.k_stride
                                  : a.v + (long long)t * a.v_stride) +
                          (long long)h * HD * 2;
        u32x4 x0 = *gptr(reinterpret_cast<const u32x4*>(src + o0));
        u32x4 x1 = *gptr(reinterpret_cast<const u32x4*>(src + o1));
        if (i0 == 0) {
            b = paged_seq_of_row(a.b.row0, a.b.n_seq, t);
            if (b < 0) return;  // a row of no sequence
            const int r0 = max(a.b.row0[b], 0), r1 = min(a.b.row0[b + 1], a.b.n_rows);
            pos = (long long)max(a.b.kv_len[b], 0) - (r1 - r0) + (t - r0);
            if (pos < 0 || pos >= a.max_pos) return;
            if (pos < a.b.capacity) {
                const int slot = (int)pos / a.c.page_size;
                const int page = a.b.pages[(long long)b * a.b.pages_stride + slot];
                if (page >= 0 && page < a.c.n_pages) {
                    const long long o = page * a.c.page_stride +
                                        (long long)((int)pos - slot * a.c.page_size) * a.c.pos_stride;
                    kd = a.c.k + o;
                    vd = a.c.v + o;
                }
            }
        }
        if (is_q || is_k) {
            const TER_GLOBAL f32x4* tab = gptr(reinterpret_cast<const f32x4*>(a.rope + pos * HD + 16 * c));
            const f32x4 t0 = tab[0], t1 = tab[1], t2 = tab[2], t3 = tab[3];
            const float cs[16] = {t0[0], t0[1], t0[2], t0[3], t1[0], t1[1], t1[2], t1[3],
                                  t2[0], t2[1], t2[2], t2[3], t3[0], t3[1], t3[2], t3[3]};
            vec8 y0 = __builtin_bit_cast(vec8, x0), y1 = __builtin_bit_cast(vec8, x1);
            T e[16];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = y0[k], e[8 + k] = y1[k];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                // pair k of the eight: (k of the first piece, k of the second),
                // or two elements in a row
                T& e0 = e[kNeox ? k : 2 * k];
                T& e1 = e[kNeox ? 8 + k : 2 * k + 1];
                const float v0 = (float)e0, v1 = (float)e1, co = cs[2 * k], si = cs[2 * k + 1];
                e0 = (T)__builtin_fmaf(v0, co, -(v1 * si));
                e1 = (T)__builtin_fmaf(v0, si, v1 * co);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) y0[k] = e[k], y1[k] = e[8 + k];
            x0 = __builtin_bit_cast(u32x4, y0);
            x1 = __builtin_bit_cast(u32x4, y1);
        }
        if (i0 + (int)threadIdx.x >= n || (!is_q && !kd)) continue;
        char* dst = is_q ? a.q_out + (long long)t * a.qo_stride + (long long)h * HD * 2
                         : (is_k ? kd : vd) + (long long)h * a.c.head_stride;
        // (nothing here reads them again: the rows of prompts 24.7 us so, 30.8
        // with stores that stay in the L2, which are written back at the end)
        __builtin_nontemporal_store(x0, gptr(reinterpret_cast<u32x4*>(dst + o0)));
        __builtin_nontemporal_store(x1, gptr(reinterpret_cast<u32x4*>(dst + o1)));
    }
}

template <typename T, int HD>
void launch(const PagedAppendArgs& a, bool neox, hipStream_t st) {
    const int n = ((a.q ? a.nh : 0) + 2 * a.nkv) * (HD / 16);
    const dim3 grid(a.b.n_rows), block(n < 256 ? (n + 63) / 64 * 64 : 256);
    if (neox)
        hipLaunchKernelGGL((paged_append_kernel<T, HD, true>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((paged_append_kernel<T, HD, false>), grid, block, 0, st, a);
}

}  // namespace

hipError_t launch_paged_rope_table(float* tab, int hd, int max_pos, double theta, hipStream_t st) {
    Freqs fr;
    for (int k = 0; k < 64; ++k) fr.f[k] = k < hd / 2 ? __builtin_pow(theta, -2.0 * k / hd) : 0.0;
    const long long n = (long long)max_pos * (hd / 2);
    hipLaunchKernelGGL(paged_rope_table_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, tab, hd / 2,
                       max_pos, fr);
    return hipGetLastError();
}

hipError_t launch_paged_append(const PagedAppendArgs& a, int hd, bool neox, bool bf16, hipStream_t st) {
    if (hd == 128)
        bf16 ? launch<__bf16, 128>(a, neox, st) : launch<_Float16, 128>(a, neox, st);
    else
        bf16 ? launch<__bf16, 64>(a, neox, st) : launch<_Float16, 64>(a, neox, st);
    return hipGetLastError();
}

}  // namespace terhip

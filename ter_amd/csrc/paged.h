// paged.h -- shared definitions of the paged-cache operators (include/ter_hip_paged.h):
// what their kernels are launched with.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_plan.h"
#include "ter_hip_paged.h"

namespace terhip {

struct PagedBatch {
    const int32_t* row0;    // [n_seq + 1]
    const int32_t* kv_len;  // [n_seq]
    const int32_t* pages;   // [n_seq][pages_stride]
    long long pages_stride;
    int n_seq, n_rows;
    int capacity;           // positions of a table row: max_pages * page_size, at most POS_MAX
};

struct PagedCache {
    char* k;
    char* v;
    long long page_stride;  // bytes
    int pos_stride, head_stride;
    int n_pages, page_size;
};

struct PagedAppendArgs {
    PagedBatch b;
    PagedCache c;
    const char* q;  // null: keys and values only
    const char* k;
    const char* v;
    char* q_out;
    long long q_stride, k_stride, v_stride, qo_stride;  // bytes
    const float* rope;                                  // [max_pos][hd/2][2] (cos, sin)
    int nh, nkv, max_pos;
};

struct PagedAttendArgs {
    PagedBatch b;
    PagedCache c;
    const char* q;
    char* out;
    long long q_stride, out_stride;  // bytes
    float scale2;                    // scale * log2(e)
    int nh, nkv, group, tokens_log2;
    int shared;                      // a multiple of 16
    unsigned page_magic;             // ceil(2^32 / (page_size / 16)); 0 for pages of 16
    PagedCuts cuts_by;
    // the workspace (paged_attend_layout)
    int* cuts;                       // [max_wg][8] where a range begins inside a segment: rows of the row tile
                                     //   (0: it does not), first token row, KV head, first and last range of it
    int* before;                     // shared: [n_seq + 1] units before each sequence
    float* slots;                    // [2 max_wg][slot_rows][hd], then [2 max_wg][slot_rows][2]
    float* slot_stats;
    int slot_rows;
    float* whole;                    // shared: [2: own positions, prefix][n_rows nh][hd], then [..][2]
    float* whole_stats;
};

// How a call is cut, and where its parts lie in the workspace (offsets in
// bytes; the rows of `whole` are there with a shared prefix only).
struct PagedAttendLayout {
    int tokens_log2, slot_rows;
    PagedCuts cuts_by;
    size_t cuts, before, slots, slot_stats, whole, whole_stats, bytes;
};
// (bytes 0: the device cannot be asked for its CUs)
PagedAttendLayout paged_attend_layout(int device, int nh, int nkv, int hd, int n_seq, int n_rows, int capacity,
                                      int shared);

hipError_t launch_paged_rope_table(float* tab, int hd, int max_pos, double theta, hipStream_t st);
hipError_t launch_paged_append(const PagedAppendArgs& a, int hd, bool neox, bool bf16, hipStream_t st);
hipError_t launch_paged_attend(const PagedAttendArgs& a, int hd, bool bf16, hipStream_t st);

#if defined(__HIPCC__)
// The sequence of row t (row0[b] <= t < row0[b + 1]), or -1; the same in every
// lane.  The wave looks at 64 boundaries at once: two rounds of loads for up
// to 4096 sequences.  Every index is within [0, n_seq] whatever row0 holds.
__device__ __forceinline__ int paged_seq_of_row(const int32_t* row0, int n_seq, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    if (n_seq > 64) {
        const int step = (n_seq + 63) / 64;
        const int i = min((lane + 1) * step, n_seq);
        const int c = __builtin_popcountll(__ballot(row0[i] <= t && (lane + 1) * step < n_seq));
        lo = c * step;
        const int j = min(lo + lane + 1, n_seq);
        lo += __builtin_popcountll(__ballot(lane < step && lo + lane < n_seq && row0[j] <= t));
    } else {
        lo = __builtin_popcountll(__ballot(lane < n_seq && row0[min(lane + 1, n_seq)] <= t));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    return lo < n_seq && row0[lo] <= t ? lo : -1;
}
#endif

}  // namespace terhip

/*
 * ter_hip_paged.h -- attention for batches of sequences over a paged cache on
 * MI355X (gfx950): the C-ABI of the operators that serve prompts and many
 * sequences at once, beside the one-sequence decode attention of ter_hip.h
 * (ter_hip_attn_decode, ter_hip_rope; the same status codes and conventions:
 * device pointers, a HIP stream as void*, arguments checked on the host, no
 * aborts).  No counterpart in the reference, whose forward decodes one
 * sequence over a contiguous cache (cuda/ter_cuda_forward_bitnet.cu:848-913).
 *
 * A batch is n_seq sequences.  The rows (tokens) of a call are packed: those
 * of sequence b are rows row0[b] .. row0[b+1] - 1 of q, k, v and out, and
 * they are the last ones of its kv_len[b] positions: row row0[b] + i is at
 * position kv_len[b] - (row0[b+1] - row0[b]) + i.  A prompt is a sequence
 * whose rows are all its positions, a decode step has one row a sequence, and
 * both may stand in one batch.  Position p of sequence b lies in page
 * pages[b][p / page_size], slot p % page_size.
 *
 * Lengths and tables are read on the device, when the launch runs: a captured
 * graph serves batches whose lengths grow.  So the host cannot refuse what
 * they hold; the kernels bound every access by them:
 *   - row0 entries are clamped to [0, n_rows]; rows in no sequence are left as
 *     they were;
 *   - positions from max_pages * page_size on do not exist: append writes
 *     nothing there, attend sees none;
 *   - a page id outside [0, n_pages) is no page: append writes nothing there,
 *     attend reads zeros as its keys and values;
 *   - rows at positions below 0 (kv_len[b] less than the rows given): append
 *     leaves them, attend writes zeros.
 * row0 must not decrease (where it does, results of the rows concerned are
 * undefined; accesses stay in bounds).  Two rows of one call must not have the same page
 * and slot (append); pages may be shared between sequences for reading.
 */
#ifndef TER_HIP_PAGED_H
#define TER_HIP_PAGED_H

#include "ter_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TER_HIP_PAGED_F16  0
#define TER_HIP_PAGED_BF16 1

#define TER_HIP_PAGED_SEQ_MAX 1024       /* sequences per call                */
#define TER_HIP_PAGED_ROWS_MAX (1 << 17) /* rows per call                     */
#define TER_HIP_PAGED_POS_MAX (1 << 20)  /* positions per sequence            */

/* One layer's pages.  Element (page, slot, head, d) of k (v) is at
 * k + page * page_stride + slot * pos_stride + head * head_stride + d: any
 * order of slots and heads, and k and v interleaved in one allocation, are
 * fine. */
typedef struct ter_hip_paged_cache {
    void*   k;           /* device fp16 / bf16, 16-byte aligned              */
    void*   v;
    int64_t page_stride; /* elements; multiples of 8                         */
    int64_t pos_stride;
    int64_t head_stride;
    int32_t n_pages;
    int32_t page_size;   /* a multiple of 16, at most 65536                  */
} ter_hip_paged_cache_t;

typedef struct ter_hip_paged_batch {
    const int32_t* row0;         /* device [n_seq + 1]                       */
    const int32_t* kv_len;       /* device [n_seq]: positions, new rows included */
    const int32_t* pages;        /* device [n_seq][pages_stride]             */
    int64_t        pages_stride; /* >= max_pages                             */
    int32_t        max_pages;    /* columns of pages that may be read        */
    int32_t        n_seq;
} ter_hip_paged_batch_t;

typedef struct ter_hip_paged ter_hip_paged_t;

/* Context for one model shape: n_heads query heads (a multiple of n_kv_heads,
 * at most 128 per KV head; query head h reads KV head h * n_kv_heads /
 * n_heads), head_dim 64 or 128, element type TER_HIP_PAGED_*, RoPE base theta
 * and pairing TER_HIP_ROPE_* for positions below max_pos.  Belongs to the
 * device that is current at creation; calls on another one are refused
 * (TER_HIP_ERR_HIP).  Holds the RoPE table only (max_pos * head_dim fp32:
 * angles pos * theta^(-2k/head_dim) in double, cos and sin rounded once):
 * nothing in it changes between calls, so calls on different streams may use
 * one context at the same time. */
int ter_hip_paged_create(ter_hip_paged_t** ctx, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                         int32_t max_pos, float theta, int32_t rope_type, int32_t dtype);
void ter_hip_paged_destroy(ter_hip_paged_t* ctx);

/* Rotates the new queries and keys to their positions and writes keys and
 * values to their pages, one launch.  q [n_rows][n_heads][head_dim], k and v
 * [n_rows][n_kv_heads][head_dim], each row contiguous, rows *_stride elements
 * apart (parts of one fused projection output are fine), 16-byte aligned with
 * strides that are multiples of 8.  q_out receives the rotated queries; it may
 * be q.  q and q_out both NULL: keys and values only.  Rows at positions from
 * max_pos on are left alone. */
int ter_hip_paged_append(const ter_hip_paged_t* ctx, const ter_hip_paged_batch_t* batch,
                         const ter_hip_paged_cache_t* cache, int32_t n_rows, const void* q, int64_t q_stride,
                         const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* q_out,
                         int64_t q_out_stride, void* stream);

/* Causal attention of the rows over the pages (their own positions included:
 * append first): out[r][h] = sum_{s <= p(r)} softmax_s(scale * q[r][h] . K[s])
 * V[s].  q holds rotated queries, laid out as for append; out likewise.  scale
 * > 0, or 0 for 1 / sqrt(head_dim).  Scores q . K may have any size that
 * binary32 holds, and their products with scale any at all.
 *
 * Rounding: scores, the softmax and all sums are binary32, the result is
 * rounded once.  On its way into the product with V a weight is rounded to two
 * elements of the cache's type (22 bits of fp16, 16 of bf16) where a KV head's
 * query heads times the sequence's rows in a tile are 16 or fewer, as those of
 * single tokens are, and to one element (11 or 8 bits) where they are more: of
 * prompts, and of all sequences' rows together on a shared prefix.  In fp16
 * weights below 2^-33 of a row's largest are zero.  Where a row sees infinite
 * values or NaN its result has them, whatever their weights.
 *
 * shared: the first `shared` positions of every sequence are the same pages
 * (row 0 of the table is read for them); rounded down to a multiple of 16.
 * Results are those of shared = 0 up to rounding: those positions are
 * multiplied once with the rows of all sequences instead of once for each.
 *
 * ws: ws_bytes >= ter_hip_paged_attend_ws(...) bytes of device memory,
 * 16-byte aligned, of any contents, used by this call until it ends: calls
 * that may overlap in time (other streams, other captured graphs) need one
 * each. */
size_t ter_hip_paged_attend_ws(const ter_hip_paged_t* ctx, const ter_hip_paged_batch_t* batch,
                               const ter_hip_paged_cache_t* cache, int32_t n_rows, int32_t shared);
int ter_hip_paged_attend(const ter_hip_paged_t* ctx, const ter_hip_paged_batch_t* batch,
                         const ter_hip_paged_cache_t* cache, int32_t n_rows, const void* q, int64_t q_stride,
                         void* out, int64_t out_stride, int32_t shared, float scale, void* ws, size_t ws_bytes,
                         void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TER_HIP_PAGED_H */

// paged_abi.hip -- the extern "C" boundary of the paged-cache operators
// (include/ter_hip_paged.h): every argument the host can see is checked before
// any device work, and nothing throws or aborts.
#include <hip/hip_runtime.h>

#include <cmath>
#include <new>

#include "common.h"
#include "paged.h"

using namespace terhip;

struct ter_hip_paged {
    int nh = 0, nkv = 0, hd = 0, max_pos = 0, device = 0;
    bool neox = true, bf16 = false;
    float* rope = nullptr;  // [max_pos][hd/2][2]
};

namespace {

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Rows of `width` elements, `stride` elements apart.
int check_rows(const char* what, const void* p, int64_t stride, int64_t width) {
    if (!p) return fail(TER_HIP_ERR_NULL, "null %s", what);
    if (!aligned(p, 16) || stride % 8) return fail(TER_HIP_ERR_ALIGN, "%s rows must be 16-byte aligned", what);
    if (stride < width || stride > (1ll << 40))
        return fail(TER_HIP_ERR_SHAPE, "%s row stride %lld (rows of %lld)", what, (long long)stride, (long long)width);
    return TER_HIP_OK;
}

int check_device(const ter_hip_paged_t* ctx) {
    int dev = -1;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_fail(e, "current device");
    if (dev != ctx->device)
        return fail(TER_HIP_ERR_HIP, "the context belongs to device %d, device %d is current", ctx->device, dev);
    return TER_HIP_OK;
}

// The batch and the cache as the kernels take them.
int check_batch(const ter_hip_paged_t* ctx, const ter_hip_paged_batch_t* b, const ter_hip_paged_cache_t* c, int n_rows,
                PagedBatch* pb, PagedCache* pc) {
    if (!ctx || !b || !c) return fail(TER_HIP_ERR_NULL, "null context, batch or cache");
    if (b->n_seq < 0 || b->n_seq > TER_HIP_PAGED_SEQ_MAX || n_rows < 0 || n_rows > TER_HIP_PAGED_ROWS_MAX)
        return fail(TER_HIP_ERR_SHAPE, "n_seq=%d n_rows=%d", b->n_seq, n_rows);
    if (c->page_size < 16 || c->page_size > 65536 || c->page_size % 16 || c->n_pages < 1)
        return fail(TER_HIP_ERR_SHAPE, "page_size=%d (a multiple of 16 to 65536) n_pages=%d", c->page_size, c->n_pages);
    if (b->max_pages < 0 || b->pages_stride < b->max_pages || b->pages_stride > (1ll << 40))
        return fail(TER_HIP_ERR_SHAPE, "max_pages=%d pages_stride=%lld", b->max_pages, (long long)b->pages_stride);
    if (!b->row0 || (b->n_seq > 0 && (!b->kv_len || (b->max_pages > 0 && !b->pages))) || !c->k || !c->v)
        return fail(TER_HIP_ERR_NULL, "null table or cache pointer");
    if (!aligned(b->row0, 4) || !aligned(b->kv_len, 4) || !aligned(b->pages, 4) || !aligned(c->k, 16) ||
        !aligned(c->v, 16) || c->page_stride % 8 || c->pos_stride % 8 || c->head_stride % 8)
        return fail(TER_HIP_ERR_ALIGN, "cache pointers and strides must be 16-byte aligned");
    // a page within 2^31 bytes, heads and slots within a page
    const int64_t last = (int64_t)(c->page_size - 1) * c->pos_stride + (int64_t)(ctx->nkv - 1) * c->head_stride + ctx->hd;
    if (c->pos_stride < ctx->hd || c->head_stride < ctx->hd || c->pos_stride > (1 << 28) || c->head_stride > (1 << 28) ||
        last * 2 > 0x7FFFFFFFll || c->page_stride < ctx->hd || c->page_stride > (1ll << 40))
        return fail(TER_HIP_ERR_SHAPE, "cache strides %lld, %lld, %lld", (long long)c->page_stride,
                    (long long)c->pos_stride, (long long)c->head_stride);
    const int64_t cap = (int64_t)b->max_pages * c->page_size;
    if (cap > TER_HIP_PAGED_POS_MAX + 65535)
        return fail(TER_HIP_ERR_SHAPE, "%d pages of %d positions in a sequence", b->max_pages, c->page_size);
    pb->row0 = b->row0;
    pb->kv_len = b->kv_len;
    pb->pages = b->pages;
    pb->pages_stride = b->pages_stride;
    pb->n_seq = b->n_seq;
    pb->n_rows = n_rows;
    pb->capacity = (int)cap;
    pc->k = static_cast<char*>(c->k);
    pc->v = static_cast<char*>(c->v);
    pc->page_stride = c->page_stride * 2;
    pc->pos_stride = (int)c->pos_stride * 2;
    pc->head_stride = (int)c->head_stride * 2;
    pc->n_pages = c->n_pages;
    pc->page_size = c->page_size;
    return TER_HIP_OK;
}

}  // namespace

extern "C" {

int ter_hip_paged_create(ter_hip_paged_t** out, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_pos,
                         float theta, int32_t rope_type, int32_t dtype) {
    if (!out) return fail(TER_HIP_ERR_NULL, "null context pointer");
    *out = nullptr;
    if (n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads || n_heads / n_kv_heads > 128 || n_heads > 65535 ||
        (head_dim != 64 && head_dim != 128) || max_pos < 1 || max_pos > TER_HIP_PAGED_POS_MAX)
        return fail(TER_HIP_ERR_SHAPE, "paged attention shape nh=%d nkv=%d hd=%d max_pos=%d unsupported", n_heads,
                    n_kv_heads, head_dim, max_pos);
    if (rope_type != TER_HIP_ROPE_NORM && rope_type != TER_HIP_ROPE_NEOX)
        return fail(TER_HIP_ERR_PAYLOAD, "unknown RoPE type %d", rope_type);
    if (dtype != TER_HIP_PAGED_F16 && dtype != TER_HIP_PAGED_BF16)
        return fail(TER_HIP_ERR_PAYLOAD, "unknown element type %d", dtype);
    if (!(theta > 0.f) || std::isinf(theta)) return fail(TER_HIP_ERR_SHAPE, "RoPE theta must be > 0 and finite");
    ter_hip_paged* c = new (std::nothrow) ter_hip_paged();
    if (!c) return fail(TER_HIP_ERR_ALLOC, "paged attention context");
    c->nh = n_heads;
    c->nkv = n_kv_heads;
    c->hd = head_dim;
    c->max_pos = max_pos;
    c->neox = rope_type == TER_HIP_ROPE_NEOX;
    c->bf16 = dtype == TER_HIP_PAGED_BF16;
    hipError_t e = hipGetDevice(&c->device);
    if (e == hipSuccess) e = hipMalloc(&c->rope, (size_t)max_pos * head_dim * sizeof(float));
    if (e == hipSuccess) e = launch_paged_rope_table(c->rope, head_dim, max_pos, (double)theta, nullptr);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
    if (e != hipSuccess) {
        ter_hip_paged_destroy(c);
        return hip_fail(e, "paged attention context");
    }
    *out = c;
    return TER_HIP_OK;
}

void ter_hip_paged_destroy(ter_hip_paged_t* c) {
    if (!c) return;
    (void)hipFree(c->rope);
    delete c;
}

int ter_hip_paged_append(const ter_hip_paged_t* ctx, const ter_hip_paged_batch_t* batch,
                         const ter_hip_paged_cache_t* cache, int32_t n_rows, const void* q, int64_t q_stride,
                         const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* q_out,
                         int64_t q_out_stride, void* stream) {
    PagedAppendArgs a{};
    int rc = check_batch(ctx, batch, cache, n_rows, &a.b, &a.c);
    if (rc) return rc;
    if (n_rows == 0 || batch->n_seq == 0) return TER_HIP_OK;
    if ((q == nullptr) != (q_out == nullptr)) return fail(TER_HIP_ERR_NULL, "q and q_out go together");
    if (q && (rc = check_rows("q", q, q_stride, (int64_t)ctx->nh * ctx->hd))) return rc;
    if (q && (rc = check_rows("q_out", q_out, q_out_stride, (int64_t)ctx->nh * ctx->hd))) return rc;
    if ((rc = check_rows("k", k, k_stride, (int64_t)ctx->nkv * ctx->hd))) return rc;
    if ((rc = check_rows("v", v, v_stride, (int64_t)ctx->nkv * ctx->hd))) return rc;
    if ((rc = check_device(ctx))) return rc;
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k);
    a.v = static_cast<const char*>(v);
    a.q_out = static_cast<char*>(q_out);
    a.q_stride = q_stride * 2;
    a.k_stride = k_stride * 2;
    a.v_stride = v_stride * 2;
    a.qo_stride = q_out_stride * 2;
    a.rope = ctx->rope;
    a.nh = ctx->nh;
    a.nkv = ctx->nkv;
    a.max_pos = ctx->max_pos;
    const hipError_t e = launch_paged_append(a, ctx->hd, ctx->neox, ctx->bf16, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "paged append launch");
    return TER_HIP_OK;
}

size_t ter_hip_paged_attend_ws(const ter_hip_paged_t* ctx, const ter_hip_paged_batch_t* batch,
                               const ter_hip_paged_cache_t* cache, int32_t n_rows, int32_t shared) {
    PagedBatch b;
    PagedCache c;
    if (check_batch(ctx, batch, cache, n_rows, &b, &c) || n_rows == 0 || b.n_seq == 0 || shared < 0) return 0;
    return paged_attend_layout(ctx->device, ctx->nh, ctx->nkv, ctx->hd, b.n_seq, n_rows, b.capacity, shared / 16 * 16)
        .bytes;
}

int ter_hip_paged_attend(const ter_hip_paged_t* ctx, const ter_hip_paged_batch_t* batch,
                         const ter_hip_paged_cache_t* cache, int32_t n_rows, const void* q, int64_t q_stride,
                         void* out, int64_t out_stride, int32_t shared, float scale, void* ws, size_t ws_bytes,
                         void* stream) {
    PagedAttendArgs a{};
    int rc = check_batch(ctx, batch, cache, n_rows, &a.b, &a.c);
    if (rc) return rc;
    if (shared < 0 || shared > a.b.capacity)
        return fail(TER_HIP_ERR_SHAPE, "shared=%d of %d positions", shared, a.b.capacity);
    if (!(scale >= 0.f) || scale > 1e38f) return fail(TER_HIP_ERR_SHAPE, "scale must be > 0 and finite, or 0");
    if (n_rows == 0 || batch->n_seq == 0) return TER_HIP_OK;
    if ((rc = check_rows("q", q, q_stride, (int64_t)ctx->nh * ctx->hd))) return rc;
    if ((rc = check_rows("out", out, out_stride, (int64_t)ctx->nh * ctx->hd))) return rc;
    shared = shared / 16 * 16;
    const PagedAttendLayout p =
        paged_attend_layout(ctx->device, ctx->nh, ctx->nkv, ctx->hd, batch->n_seq, n_rows, a.b.capacity, shared);
    if (p.bytes == 0) return fail(TER_HIP_ERR_HIP, "cannot query CU count");
    // units are counted in 31 bits (a sequence's rows may lie behind its whole table)
    const int64_t tiles = ((int64_t)n_rows >> p.tokens_log2) + batch->n_seq;
    if (tiles * ctx->nkv * (((int64_t)a.b.capacity + n_rows) / 64 + 10 + shared / 64) > 0x7FFFFFFFll)
        return fail(TER_HIP_ERR_SHAPE, "%d rows over %d positions are too many for one call", n_rows, a.b.capacity);
    if (!ws) return fail(TER_HIP_ERR_NULL, "null workspace");
    if (ws_bytes < p.bytes) return fail(TER_HIP_ERR_SHAPE, "workspace of %zu bytes, %zu needed", ws_bytes, p.bytes);
    if (!aligned(ws, 16)) return fail(TER_HIP_ERR_ALIGN, "workspace misaligned");
    if ((rc = check_device(ctx))) return rc;
    a.q = static_cast<const char*>(q);
    a.out = static_cast<char*>(out);
    a.q_stride = q_stride * 2;
    a.out_stride = out_stride * 2;
    a.scale2 = (float)((scale > 0.f ? (double)scale : 1.0 / std::sqrt((double)ctx->hd)) * 1.4426950408889634);
    a.nh = ctx->nh;
    a.nkv = ctx->nkv;
    a.group = ctx->nh / ctx->nkv;
    a.tokens_log2 = p.tokens_log2;
    a.shared = shared;
    const unsigned d = (unsigned)a.c.page_size / 16;  // x / d = x * magic >> 32 for x < 2^17, d <= 4096
    a.page_magic = d == 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d);
    a.cuts_by = p.cuts_by;
    a.slot_rows = p.slot_rows;
    char* w = static_cast<char*>(ws);
    a.cuts = reinterpret_cast<int*>(w + p.cuts);
    a.before = reinterpret_cast<int*>(w + p.before);
    a.slots = reinterpret_cast<float*>(w + p.slots);
    a.slot_stats = reinterpret_cast<float*>(w + p.slot_stats);
    a.whole = reinterpret_cast<float*>(w + p.whole);
    a.whole_stats = reinterpret_cast<float*>(w + p.whole_stats);
    const hipError_t e = launch_paged_attend(a, ctx->hd, ctx->bf16, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "paged attention launch");
    return TER_HIP_OK;
}

}  // extern "C"

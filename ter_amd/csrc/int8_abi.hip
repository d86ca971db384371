// int8_abi.hip -- the extern "C" boundary of the 8-bit products
// (include/ter_hip_int8.h): every argument the host can see is checked before
// any device work, and nothing throws or aborts.
#include <hip/hip_runtime.h>

#include "common.h"
#include "int8.h"

using namespace terhip;

namespace {

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

bool shape_ok(int K, int N) { return K >= 1 && K <= TER_HIP_INT8_K_MAX && N >= 1 && N <= TER_HIP_INT8_N_MAX; }

int check_w8(const ter_hip_w8_t* w) {
    if (!w || !w->data || !w->scale) return fail(TER_HIP_ERR_NULL, "null weight handle or buffer");
    if (!shape_ok(w->K, w->N)) return fail(TER_HIP_ERR_SHAPE, "8-bit weight shape K=%d N=%d out of range", w->K, w->N);
    if (w->bytes < ter_hip_w8_bytes(w->K, w->N)) return fail(TER_HIP_ERR_SHAPE, "8-bit weight buffer too small");
    if (!aligned(w->data, 256) || !aligned(w->scale, 16)) return fail(TER_HIP_ERR_ALIGN, "8-bit weight buffer misaligned");
    return TER_HIP_OK;
}

int elem_bytes(int type) {
    switch (type) {
        case TER_HIP_T_F16:
        case TER_HIP_T_BF16: return 2;
        case TER_HIP_T_F32:
        case TER_HIP_T_I32: return 4;
        case TER_HIP_T_I8: return 1;
        default: return 0;
    }
}

// A matrix of rows, `width` elements each, `stride` apart.
int check_rows(const char* what, const void* p, int type, int64_t stride, int64_t width) {
    if (!p) return fail(TER_HIP_ERR_NULL, "null %s", what);
    if (!aligned(p, (size_t)elem_bytes(type))) return fail(TER_HIP_ERR_ALIGN, "%s misaligned", what);
    if (stride < width || stride > (1ll << 36))
        return fail(TER_HIP_ERR_SHAPE, "%s row stride %lld (rows of %lld)", what, (long long)stride, (long long)width);
    return TER_HIP_OK;
}

int check_x(const ter_hip_w8_t* w, const ter_hip_rows_t* x) {
    if (!x) return fail(TER_HIP_ERR_NULL, "null rows");
    if (x->type < TER_HIP_T_F16 || x->type > TER_HIP_T_I8) return fail(TER_HIP_ERR_PAYLOAD, "unknown row type %d", x->type);
    if (x->n < 0 || x->n > TER_HIP_INT8_M_MAX || (long long)x->n * w->N > TER_HIP_INT8_Y_MAX)
        return fail(TER_HIP_ERR_SHAPE, "%d rows by %d channels", x->n, w->N);
    if (x->n == 0) return TER_HIP_OK;
    return check_rows("rows", x->data, x->type, x->stride, w->K);
}

// Whether the kernels read the rows where they are (256 of them within 32-bit
// offsets).
bool in_place(const ter_hip_w8_t* w, const ter_hip_rows_t* x) {
    return x->type == TER_HIP_T_I8 && w->K % 16 == 0 && aligned(x->data, 16) &&
           ((x->stride % 16 == 0 && x->stride <= 1 << 22) || x->n == 1);
}

// Whether the product's kernel quantizes the rows itself.
bool quant_within(const ter_hip_w8_t* w, const ter_hip_rows_t* x) {
    return x->type != TER_HIP_T_I8 && i8_quant_within(x->n, i8_units(w->K));
}

size_t row_bytes(const ter_hip_w8_t* w) { return (size_t)i8_units(w->K) * kI8Unit; }

// Of the workspace: the rows in 8 bits, and their scales.
size_t rows_bytes_of(const ter_hip_w8_t* w, const ter_hip_rows_t* x) {
    if (x->n == 0 || in_place(w, x) || quant_within(w, x)) return 0;
    return (size_t)x->n * (row_bytes(w) + 4);
}

int parts_of(const ter_hip_w8_t* w, const ter_hip_rows_t* x) {
    return i8_in_tiles(x->n, w->N) ? i8_parts(x->n, w->N, i8_units(w->K)) : 1;
}

// Behind them the sums of parts of K.
size_t sums_at(const ter_hip_w8_t* w, const ter_hip_rows_t* x) { return (rows_bytes_of(w, x) + 15) / 16 * 16; }

size_t ws_bytes_of(const ter_hip_w8_t* w, const ter_hip_rows_t* x) {
    const int parts = parts_of(w, x);
    if (parts == 1) return rows_bytes_of(w, x);
    return sums_at(w, x) + (size_t)parts * x->n * i8_sums_stride(w->N) * 4;
}

}  // namespace

extern "C" {

size_t ter_hip_w8_bytes(int32_t K, int32_t N) {
    if (!shape_ok(K, N)) return 0;
    return i8_tile_bytes(K, N) + (size_t)i8_pairs(N) * 32 * sizeof(float);
}

int ter_hip_w8_init(ter_hip_w8_t* w, void* buf, size_t buf_bytes, int32_t K, int32_t N) {
    if (!w || !buf) return fail(TER_HIP_ERR_NULL, "null weight handle or buffer");
    if (!shape_ok(K, N)) return fail(TER_HIP_ERR_SHAPE, "8-bit weight shape K=%d N=%d out of range", K, N);
    if (buf_bytes < ter_hip_w8_bytes(K, N))
        return fail(TER_HIP_ERR_SHAPE, "buffer of %zu bytes, %zu needed", buf_bytes, ter_hip_w8_bytes(K, N));
    if (!aligned(buf, 256)) return fail(TER_HIP_ERR_ALIGN, "8-bit weight buffer must be 256-byte aligned");
    w->data = buf;
    w->scale = reinterpret_cast<float*>(static_cast<char*>(buf) + i8_tile_bytes(K, N));
    w->bytes = buf_bytes;
    w->K = K;
    w->N = N;
    return TER_HIP_OK;
}

int ter_hip_w8_pack(const ter_hip_w8_t* w, const int8_t* q, int64_t q_stride, const float* scale, void* stream) {
    int rc = check_w8(w);
    if (rc) return rc;
    if ((rc = check_rows("integers", q, TER_HIP_T_I8, q_stride, w->K))) return rc;
    if (!scale) return fail(TER_HIP_ERR_NULL, "null scales");
    if (!aligned(scale, 4)) return fail(TER_HIP_ERR_ALIGN, "scales misaligned");
    const hipError_t e = launch_w8_pack(q, q_stride, scale, static_cast<uint8_t*>(w->data), w->scale, w->K, w->N,
                                        static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "8-bit weight pack launch");
    return TER_HIP_OK;
}

int ter_hip_w8_quantize(const ter_hip_w8_t* w, const void* src, int32_t type, int64_t src_stride, void* stream) {
    int rc = check_w8(w);
    if (rc) return rc;
    if (type < TER_HIP_T_F16 || type > TER_HIP_T_F32) return fail(TER_HIP_ERR_PAYLOAD, "unknown weight type %d", type);
    if ((rc = check_rows("weights", src, type, src_stride, w->K))) return rc;
    const hipError_t e = launch_w8_quantize(src, type, src_stride, static_cast<uint8_t*>(w->data), w->scale, w->K, w->N,
                                            static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "8-bit weight quantize launch");
    return TER_HIP_OK;
}

int ter_hip_w8_unpack(const ter_hip_w8_t* w, int8_t* q, float* scale, void* stream) {
    const int rc = check_w8(w);
    if (rc) return rc;
    if (!aligned(scale, 4)) return fail(TER_HIP_ERR_ALIGN, "scales misaligned");
    if (!q && !scale) return TER_HIP_OK;
    const hipError_t e = launch_w8_unpack(static_cast<const uint8_t*>(w->data), w->scale, q, scale, w->K, w->N,
                                          static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "8-bit weight unpack launch");
    return TER_HIP_OK;
}

size_t ter_hip_w8_mm_ws(const ter_hip_w8_t* w, const ter_hip_rows_t* x) {
    if (check_w8(w) || check_x(w, x)) return 0;
    return ws_bytes_of(w, x);
}

int ter_hip_w8_mm(const ter_hip_w8_t* w, const ter_hip_rows_t* x, void* y, int64_t y_stride, int32_t y_type, void* ws,
                  size_t ws_bytes, void* stream) {
    int rc = check_w8(w);
    if (rc) return rc;
    if ((rc = check_x(w, x))) return rc;
    if (y_type < TER_HIP_T_F16 || y_type > TER_HIP_T_I32 || y_type == TER_HIP_T_I8)
        return fail(TER_HIP_ERR_PAYLOAD, "unknown result type %d", y_type);
    if (y_type == TER_HIP_T_I32 && x->type != TER_HIP_T_I8)
        return fail(TER_HIP_ERR_PAYLOAD, "bare sums need integer rows");
    if (x->n == 0) return TER_HIP_OK;
    if ((rc = check_rows("results", y, y_type, y_stride, w->N))) return rc;
    if (x->type == TER_HIP_T_I8 && y_type != TER_HIP_T_I32) {
        if (!x->scale) return fail(TER_HIP_ERR_NULL, "integer rows need their scales");
        if (!aligned(x->scale, 4)) return fail(TER_HIP_ERR_ALIGN, "row scales misaligned");
    }
    const size_t need = ws_bytes_of(w, x);
    if (need) {
        if (!ws) return fail(TER_HIP_ERR_NULL, "null workspace");
        if (ws_bytes < need) return fail(TER_HIP_ERR_SHAPE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
        if (!aligned(ws, 16)) return fail(TER_HIP_ERR_ALIGN, "workspace misaligned");
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    Int8MmArgs a{};
    a.w = static_cast<const uint8_t*>(w->data);
    a.ws = w->scale;
    a.y = static_cast<char*>(y);
    a.ldy = y_stride;
    a.M = x->n;
    a.N = w->N;
    a.Ku = i8_units(w->K);
    a.y_type = y_type;
    a.x_type = TER_HIP_T_I8;
    a.parts = parts_of(w, x);
    if (a.parts > 1) a.sums = reinterpret_cast<int*>(static_cast<char*>(ws) + sums_at(w, x));
    if (quant_within(w, x)) {
        a.x = static_cast<const int8_t*>(x->data);
        a.ldx = x->stride;
        a.Kx = w->K;
        a.x_type = x->type;
        a.vec = aligned(x->data, 16) && (x->n == 1 || x->stride * elem_bytes(x->type) % 16 == 0);
    } else if (in_place(w, x)) {
        a.x = static_cast<const int8_t*>(x->data);
        a.xs = x->scale;
        a.ldx = x->n == 1 ? w->K : x->stride;
        a.Kx = w->K;
    } else {
        int8_t* q = static_cast<int8_t*>(ws);
        const size_t ldq = row_bytes(w);
        float* s = reinterpret_cast<float*>(q + (size_t)x->n * ldq);
        const hipError_t e = launch_rows8(x->data, x->type, x->stride, x->n, w->K, q, (long long)ldq, s, st);
        if (e != hipSuccess) return hip_fail(e, "row quantization launch");
        a.x = q;
        a.xs = x->type == TER_HIP_T_I8 ? x->scale : s;
        a.ldx = (long long)ldq;
        a.Kx = (int)ldq;
    }
    const hipError_t e = launch_int8_mm(a, st);
    if (e != hipSuccess) return hip_fail(e, "8-bit product launch");
    return TER_HIP_OK;
}

}  // extern "C"

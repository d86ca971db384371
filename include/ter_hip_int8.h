/*
 * ter_hip_int8.h -- matrix products in 8-bit integers with a scale for each
 * token and each channel on MI355X (gfx950): the C-ABI of the weights that
 * are not ternary, beside the packed trits of ter_hip.h (ter_hip_gemv,
 * ter_hip_gemm; the same status codes and conventions: device pointers, a HIP
 * stream as void*, arguments checked on the host, no aborts).  No counterpart
 * in the reference, whose lm_head is fp16 for one row
 * (cuda/ter_cuda_forward_bitnet.cu:388-429).
 *
 *   y[m][n] = (sum_k x[m][k] w[n][k]) * (x_scale[m] * w_scale[n])
 *
 * The sum is exact (int32: K is at most TER_HIP_INT8_K_MAX, so 128 * 128 * K
 * stays below 2^31); it is converted to binary32, multiplied by the binary32
 * product of the scales, and rounded once more where y is fp16 or bf16.  A
 * value beyond the type's range becomes an infinity.
 *
 * Rows that are not integers are quantized within the call, each by its own
 * largest magnitude, in binary32 as ter_hip_quant_int8 does:
 *   s = 127 / (max_k |x[m][k]| + 1e-9f), q = rint(x * s), x_scale = 1 / s.
 * A row that holds an infinity or NaN has x_scale NaN: its results are NaN,
 * those of other rows are not touched by it.
 */
#ifndef TER_HIP_INT8_H
#define TER_HIP_INT8_H

#include "ter_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TER_HIP_INT8_K_MAX 131071
#define TER_HIP_INT8_N_MAX (1 << 23)
#define TER_HIP_INT8_M_MAX (1 << 23)
#define TER_HIP_INT8_Y_MAX (1ll << 36) /* results of one call: n * N */

/* Element types of rows and results. */
#define TER_HIP_T_F16  0
#define TER_HIP_T_BF16 1
#define TER_HIP_T_F32  2
#define TER_HIP_T_I8   3  /* rows only    */
#define TER_HIP_T_I32  4  /* results only */

/* A K x N weight (N channels of K values) on the device, in the layout that
 * the kernels stream: a caller-owned buffer of ter_hip_w8_bytes(K, N) bytes,
 * 256-byte aligned. */
typedef struct ter_hip_w8 {
    void*   data;
    float*  scale;   /* device [N], within the buffer */
    size_t  bytes;
    int32_t K, N;
} ter_hip_w8_t;

/* Bytes of the buffer; 0 for a K or N out of range. */
size_t ter_hip_w8_bytes(int32_t K, int32_t N);
int ter_hip_w8_init(ter_hip_w8_t* w, void* buf, size_t buf_bytes, int32_t K, int32_t N);

/* Fills the weight: from integers q [N][K] (rows q_stride >= K apart) and
 * their scales [N]; or from w [N][K] of type TER_HIP_T_F16, _BF16 or _F32,
 * each channel quantized by the steps above.  Any alignment of an element. */
int ter_hip_w8_pack(const ter_hip_w8_t* w, const int8_t* q, int64_t q_stride, const float* scale, void* stream);
int ter_hip_w8_quantize(const ter_hip_w8_t* w, const void* src, int32_t type, int64_t src_stride, void* stream);
/* The integers [N][K] (contiguous) and scales [N] back; either may be NULL. */
int ter_hip_w8_unpack(const ter_hip_w8_t* w, int8_t* q, float* scale, void* stream);

/* Rows of a call: n rows of K elements, stride elements apart (>= K, any
 * alignment of an element).  Integer rows at 16-byte aligned addresses with K
 * a multiple of 16 are read where they are, others are laid out first.
 * scale: device [n], for TER_HIP_T_I8 only, where results are not integers. */
typedef struct ter_hip_rows {
    const void*  data;
    const float* scale;
    int64_t      stride;
    int32_t      type;   /* TER_HIP_T_* */
    int32_t      n;
} ter_hip_rows_t;

/* y [n][N] (rows y_stride >= N elements apart) of type y_type: TER_HIP_T_I32
 * gives the bare sums and needs integer rows.  y may not overlap an input.
 * ws: ws_bytes >= ter_hip_w8_mm_ws(...) bytes of device memory (0: none
 * needed), 16-byte aligned, of any contents, used by this call until it ends:
 * calls that may overlap in time (other streams, other captured graphs) need
 * one each.  The size depends on K, N, the rows' type, number, stride and
 * 16-byte alignment.  n = 0 launches nothing.  Capturable. */
size_t ter_hip_w8_mm_ws(const ter_hip_w8_t* w, const ter_hip_rows_t* x);
int ter_hip_w8_mm(const ter_hip_w8_t* w, const ter_hip_rows_t* x, void* y, int64_t y_stride, int32_t y_type, void* ws,
                  size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TER_HIP_INT8_H */

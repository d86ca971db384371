/*
 * ter_hip_sample.h -- tokens drawn from the logits of a batch on MI355X
 * (gfx950): temperature, top-k, top-p and min-p with random numbers that the
 * caller gives, beside the argmax of one row in ter_hip.h
 * (ter_hip_argmax_f16; the same status codes and conventions: device pointers,
 * a HIP stream as void*, arguments checked on the host, no aborts).  No
 * counterpart in the reference's GPU code, which takes the largest logit
 * (cuda/ter_cuda_forward_bitnet.cu:454-495).
 *
 * For one row of logits l, in the order of falling l (of equal ones the lower
 * index first):
 *   w = exp((l - max l) / temperature)
 *   of all, the first top_k;
 *   of those, the ones whose predecessors' w sum to less than top_p times the
 *   sum over the top_k (the first always);
 *   of those, the ones with w >= min_p (the first always);
 * and the token is the first of the kept, in the same order, at which the
 * running sum of w exceeds u times the sum over all kept.
 *
 * Weights are computed in binary64 (relative error below 2^-42) and summed as
 * integers, multiples of 2^-44 of the largest: sums are exact in any order, so
 * a row gives the same token in every batch and launch, and one whose weight
 * is below 2^-45 of the largest is never drawn.
 *
 *   - temperature 0 (or, read on the device, not above 0) takes the largest
 *     logit, whatever top_k, top_p, min_p and u; one above 0 and below 2^-120
 *     counts as 2^-120;
 *   - top_k 0 (or below, or V and more) keeps all; so do top_p 1 (and, on the
 *     device, more or NaN) and min_p 0 (below or NaN; above 1 counts as 1);
 *   - u is in [0, 1); on the device others count as the nearest in it, NaN as 0;
 *   - logits that are -infinity or NaN are never drawn; +infinity counts as the
 *     largest finite binary32; a row with nothing to draw gives token -1, prob 0.
 *
 * Thousands of logits next to each other where a cut or the draw falls (a row of
 * zeros), and infinite ones, are slow: milliseconds for a row of 128256, and the
 * call takes as long.  Rows that only fill up a batch are best given temperature
 * 0 on the device, or logits of -infinity, which are settled at once.
 */
#ifndef TER_HIP_SAMPLE_H
#define TER_HIP_SAMPLE_H

#include "ter_hip.h"
#include "ter_hip_int8.h" /* element types */

#ifdef __cplusplus
extern "C" {
#endif

#define TER_HIP_SAMPLE_V_MAX    (1 << 19)
#define TER_HIP_SAMPLE_ROWS_MAX (1 << 20)

/* Settings of a call: a device array with one value a row, or NULL and one
 * value for all rows (checked on the host: temperature finite and >= 0, top_k
 * >= 0, top_p and min_p in [0, 1]). */
typedef struct ter_hip_sample_params {
    const float*   temperature_dev;  /* [rows] or NULL */
    const int32_t* top_k_dev;
    const float*   top_p_dev;
    const float*   min_p_dev;
    float          temperature;
    int32_t        top_k;
    float          top_p;
    float          min_p;
} ter_hip_sample_params_t;

/* Draws token[r] for each of `rows` rows of V logits of type TER_HIP_T_F16,
 * _BF16 or _F32 (ter_hip_int8.h), rows stride >= V elements apart, with u[r].
 * prob (or NULL) receives the probability with which the token was drawn, its
 * w over the sum of the kept.  Settings, u and logits are read on the device
 * when the launch runs.  ws: ws_bytes >= ter_hip_sample_ws(rows, V) bytes of
 * device memory (0: none needed), 16-byte aligned, of any contents, used by
 * this call until it ends: calls that may overlap in time need one each. */
size_t ter_hip_sample_ws(int32_t rows, int32_t V);
int ter_hip_sample(const void* logits, int32_t type, int64_t stride, int32_t rows, int32_t V, const float* u,
                   const ter_hip_sample_params_t* params, int32_t* token, float* prob, void* ws, size_t ws_bytes,
                   void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TER_HIP_SAMPLE_H */

// sample_abi.hip -- the extern "C" boundary of the sampling operator
// (include/ter_hip_sample.h): every argument the host can see is checked
// before any device work, and nothing throws or aborts.
#include <hip/hip_runtime.h>

#include "common.h"
#include "sample.h"

using namespace terhip;

namespace {

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

bool shape_ok(int rows, int V) {
    return rows >= 0 && rows <= TER_HIP_SAMPLE_ROWS_MAX && V >= 1 && V <= TER_HIP_SAMPLE_V_MAX;
}

}  // namespace

extern "C" {

size_t ter_hip_sample_ws(int32_t rows, int32_t V) {
    if (!shape_ok(rows, V) || sample_slices(rows, V) <= 1) return 0;
    return (size_t)rows * sizeof(SampleRow);
}

int ter_hip_sample(const void* logits, int32_t type, int64_t stride, int32_t rows, int32_t V, const float* u,
                   const ter_hip_sample_params_t* params, int32_t* token, float* prob, void* ws, size_t ws_bytes,
                   void* stream) {
    if (!params) return fail(TER_HIP_ERR_NULL, "null settings");
    if (type < TER_HIP_T_F16 || type > TER_HIP_T_F32) return fail(TER_HIP_ERR_PAYLOAD, "unknown logit type %d", type);
    if (!shape_ok(rows, V)) return fail(TER_HIP_ERR_SHAPE, "%d rows of %d logits", rows, V);
    const ter_hip_sample_params_t& p = *params;
    if (!p.temperature_dev && !(p.temperature >= 0.f && p.temperature <= 3.402823466e38f))
        return fail(TER_HIP_ERR_SHAPE, "temperature must be finite and >= 0");
    if (!p.top_k_dev && p.top_k < 0) return fail(TER_HIP_ERR_SHAPE, "top_k must be >= 0");
    if (!p.top_p_dev && !(p.top_p >= 0.f && p.top_p <= 1.f)) return fail(TER_HIP_ERR_SHAPE, "top_p must be in [0, 1]");
    if (!p.min_p_dev && !(p.min_p >= 0.f && p.min_p <= 1.f)) return fail(TER_HIP_ERR_SHAPE, "min_p must be in [0, 1]");
    if (rows == 0) return TER_HIP_OK;
    if (!logits || !u || !token) return fail(TER_HIP_ERR_NULL, "null logits, random numbers or tokens");
    const size_t el = type == TER_HIP_T_F32 ? 4 : 2;
    if (stride < V || stride > (1ll << 36)) return fail(TER_HIP_ERR_SHAPE, "row stride %lld (rows of %d)", (long long)stride, V);
    if (!aligned(logits, el) || !aligned(u, 4) || !aligned(token, 4) || !aligned(prob, 4) ||
        !aligned(p.temperature_dev, 4) || !aligned(p.top_k_dev, 4) || !aligned(p.top_p_dev, 4) || !aligned(p.min_p_dev, 4))
        return fail(TER_HIP_ERR_ALIGN, "logits, settings or results misaligned");
    const size_t need = ter_hip_sample_ws(rows, V);
    if (need) {
        if (!ws) return fail(TER_HIP_ERR_NULL, "null workspace");
        if (ws_bytes < need) return fail(TER_HIP_ERR_SHAPE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
        if (!aligned(ws, 16)) return fail(TER_HIP_ERR_ALIGN, "workspace misaligned");
    }
    SampleArgs a{};
    a.logits = static_cast<const char*>(logits);
    a.stride = stride * (int64_t)el;
    a.rows = rows;
    a.V = V;
    a.u = u;
    a.p = p;
    a.token = token;
    a.prob = prob;
    a.ws = static_cast<SampleRow*>(ws);
    a.slices = sample_slices(rows, V);
    const hipError_t e = launch_sample(a, type, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "sampling launch");
    return TER_HIP_OK;
}

}  // extern "C"

// sample.h -- shared definitions of the sampling operator (include/ter_hip_sample.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ter_hip_sample.h"

namespace terhip {

struct SampleArgs {
    const char* logits;
    long long stride;  // bytes
    int rows, V;
    const float* u;
    ter_hip_sample_params_t p;
    int32_t* token;
    float* prob;  // or null
};

hipError_t launch_sample(const SampleArgs& a, int type, hipStream_t st);

}  // namespace terhip

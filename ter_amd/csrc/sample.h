// sample.h -- shared definitions of the sampling operator (include/ter_hip_sample.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ter_hip_sample.h"

namespace terhip {

constexpr int kBins = 2048;   // of a row's histogram (sample.hip)
constexpr int kList = 8192;   // elements listed at most: else the general path
constexpr int kSlices = 64;   // workgroups of a row at most

// Workspace of a row that several workgroups work on.
struct SampleRow {
    unsigned long long mass[kBins];
    unsigned long long list[kList];
    unsigned count[kBins];
    unsigned long long run_mass[3], total, least_mass;
    unsigned run_count[3];
    int lo[3], hi[3];
    unsigned n;  // elements listed (more than kList: not all are)
    float slice_high[kSlices], slice_low[kSlices];
    unsigned pad[4];
};
static_assert(sizeof(SampleRow) % 16 == 0, "");

// Workgroups of a row: 1 where rows alone fill the GPU (a call needs no
// workspace then).
inline int sample_slices(int rows, int V) {
    const int want = (V + 4095) / 4096, fit = 512 / (rows > 0 ? rows : 1);
    int n = want < fit ? want : fit;
    n = n < kSlices ? n : kSlices;
    return n > 1 ? n : 1;
}

struct SampleArgs {
    const char* logits;
    long long stride;  // bytes
    int rows, V;
    const float* u;
    ter_hip_sample_params_t p;
    int32_t* token;
    float* prob;  // or null
    SampleRow* ws;
    int slices;
};

hipError_t launch_sample(const SampleArgs& a, int type, hipStream_t st);

}  // namespace terhip

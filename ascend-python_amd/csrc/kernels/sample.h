// Arguments of the sampling kernels (validated by the C ABI).
#pragma once

#include "common.h"

namespace qk {

struct SampleArgs {
    const void* x;  // [rows][vocab] logits
    int dtype;
    int64_t rows, vocab, row_stride;
    const float* uniform;      // [rows], as the others; these may be nullptr:
    const float* temperature;  // 1
    const int32_t* top_k;      // all
    const float* top_p;        // 1
    const float* min_p;        // 0
    int32_t* tokens;
    float* logprobs;
};
size_t sample_workspace(int64_t rows, int64_t vocab, int dtype);
hipError_t launch_sample(const SampleArgs& a, void* workspace, hipStream_t stream);

}  // namespace qk

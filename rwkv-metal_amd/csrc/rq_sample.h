// rq_sample.h -- the sampler's arguments, shared by its kernel and the entry point.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/rwkvq_rwkv7.h"

namespace rq {

constexpr int64_t kSampleMaxVocab = 1 << 20;

struct SampleArgs {
    const void* logits;
    int dt;
    int64_t rows, vocab;
    const float* u;
    // one for each row, or NULL and one for all
    const float* temperature;
    const int64_t* top_k;
    const float* top_p;
    const float* min_p;
    float temperature_all;
    int64_t top_k_all;
    float top_p_all, min_p_all;
    int64_t* token;
    float* logprob;  // or NULL
};

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream);

}  // namespace rq

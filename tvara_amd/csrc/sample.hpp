// The next token of each row of logits, drawn by given random numbers
// (tvara_sample_plan_*).
#pragma once

#include <cstddef>
#include <cstdint>

#include "buffers.hpp"

namespace tvara_amd {

constexpr int kSampleChunks = 1024;  // most chunks of a row

struct SampleArgs {
    const float* logits;  // [rows] rows of vocab, stride apart
    size_t stride;
    int rows, vocab;
    int chunk, chunks;  // logits of a chunk (a multiple of 256), chunks of a row
    const float* uniforms;     // [rows]
    const float* temperature;  // [rows] or null: 1
    const int32_t* top_k;      // [rows] or null: all
    const float* top_p;        // [rows] or null: 1
    const float* min_p;        // [rows] or null: 0
    uint32_t* tokens;          // [rows]
    float* probability;        // [rows] or null
    float* chunk_max;          // [rows][chunks]
    double* chunk_mass;        // [rows][chunks]: sum of exp((x - maximum) / temperature)
    int* err;                  // [0]: logits without a token, [1]: parameters
};

// sample.hip
void launch_sample(const SampleArgs& a, hipStream_t s);

struct SamplePlan {
    int rows = 0, vocab = 0, chunk = 0, chunks = 0, device = 0;
    DeviceBuffer space;
    PinnedBuffer flag;
    hipStream_t last = nullptr;

    void build(size_t rows, size_t vocab);
    void launch(size_t n, const float* logits, size_t stride, const float* uniforms, const float* temperature,
                const int32_t* top_k, const float* top_p, const float* min_p, uint32_t* tokens, float* probability,
                hipStream_t s);
    void check();
};

}  // namespace tvara_amd

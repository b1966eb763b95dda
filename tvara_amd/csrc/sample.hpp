// The next token of each row of logits, drawn by given random numbers
// (tvara_sample_plan_*).
#pragma once

#include <cstddef>
#include <cstdint>

#include "buffers.hpp"

namespace tvara_amd {

constexpr int kSampleChunks = 1024;  // most chunks of a row
constexpr int kSampleGroup = 4;      // chunks whose mass is one number
constexpr int kSampleGroups = kSampleChunks / kSampleGroup;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 4096;    // candidates of a row's list

struct SampleCandidate {
    uint32_t key, index;  // of the logit's order; in the row
};

// What the launches tell each other of a row.
struct SampleRow {
    int done;         // its token is written
    int size, swept;  // candidates, and those in the borders' bins
    int last;         // the last bin of a candidate
    float top;        // the largest logit
    unsigned long long total;           // the row's mass (not with top-k)
    unsigned long long above, between;  // masses before top-p's bins, and from them to top-k's
};

struct SampleArgs {
    const float* logits;  // [rows] rows of vocab, stride apart
    size_t stride;
    int rows, vocab;
    int chunk, chunks;  // logits of a chunk (a multiple of 256), chunks of a row
    double one;         // units of mass to the largest weight, a power of two
    const float* uniforms;     // [rows]
    const float* temperature;  // [rows] or null: 1
    const int32_t* top_k;      // [rows] or null: all
    const float* top_p;        // [rows] or null: 1
    const float* min_p;        // [rows] or null: 0
    uint32_t* tokens;          // [rows]
    float* probability;        // [rows] or null
    float* chunk_max;     // [rows][chunks]
    double* group_mass;   // [rows][kSampleGroups]: sum of exp((x - their maximum) / temperature)
    unsigned long long* chunk_mass;  // [rows][chunks]: what is kept of a chunk whole
    unsigned long long* bin_mass;    // [rows][kSampleBins], null where the list holds a vocabulary
    uint32_t* bin_count;             // [rows][kSampleBins]
    SampleCandidate* list;           // [rows][room]
    int room;
    SampleRow* rows_state;  // [rows]
    int* err;                  // [0]: logits without a token, [1]: parameters
};

// sample.hip
void launch_sample(const SampleArgs& a, hipStream_t s);

struct SamplePlan {
    int rows = 0, vocab = 0, chunk = 0, chunks = 0, room = 0, device = 0;
    double one = 0;
    DeviceBuffer space;
    PinnedBuffer flag;
    hipStream_t last = nullptr;
    size_t bytes = 0;

    void carve(char* base, SampleArgs* a);
    void build(size_t rows, size_t vocab);
    void launch(size_t n, const float* logits, size_t stride, const float* uniforms, const float* temperature,
                const int32_t* top_k, const float* top_p, const float* min_p, uint32_t* tokens, float* probability,
                hipStream_t s);
    void check();
};

}  // namespace tvara_amd

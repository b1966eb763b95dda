// Attention over the paged cache whose scores are capped or biased by distance,
// each row within a range of keys of its own (tvara_score_plan_*).
#pragma once

#include <cstddef>
#include <cstdint>
#include <vector>

#include "kv_cache.hpp"
#include "tree.hpp"

namespace tvara_amd {

// A batch as the kernels read it.  Row r of the packed rows sees keys
// ranges[r].x .. ranges[r].y - 1 (x >= y: none, and its output is zeros); an
// attention row is a (row, query head) pair.
struct ScoreArgs {
    const char* pool;
    BlockLayout lay;
    int layer, heads, group;
    const int32_t* tables;
    // three entries a workgroup (ScorePlan::build): x: table offset, y: tokens of the
    // sequence, z: rows of the block, w: the first of them; x: query head, y: query heads,
    // z: first step, w: end; x: run, y: runs, z: the first row's partial, w: its position
    const int4* work;
    const int2* ranges;
    const int2* runs;  // [rows]: first partial, runs (one run: written to out)
    int rows;
    const float* q;  // [rows][heads][head_dim]
    float* out;
    float* part_acc;  // [partials][heads][head_dim]
    float* part_ml;   // [partials][heads][2]: maximum (log2 units), normaliser
    float qscale;     // of a product: to log2 units, or (cap) to the argument of tanh
    float cap;        // in log2 units; 0: none
    const float* slopes;  // [heads], in log2 units; null: none
    int* err;
};

// score.hip
void launch_score_rows(const ScoreArgs& a, int items, hipStream_t s);
void launch_score_merge(const ScoreArgs& a, hipStream_t s);
// score_tiles.hip (the layouts of tree_tiles_supported): blocks of up to 16
// attention rows, or of up to kScoreMany
constexpr int kScoreFew = 16, kScoreMany = 256;
// Steps of a wave whose parts are added up in a row in f32.  Behind a large one each may be
// lost, up to half an ulp, while the normaliser keeps them all: 64 are 3.8e-6 of a column at
// the very worst, 128 7.6e-6, 4,096 2.4e-4.  Runs of few rows end there, of which four waves
// share the steps, and join with what is rounded away; many rows' sums go to memory (2 x
// 2,048 rows after 14,336, 32 heads on 8 of 128: 3,810 us, and 3,740 in one chain of 512).
constexpr int kScoreChain = 64, kScoreManyChain = 128;
int score_step(const BlockLayout& lay, int block);   // keys of a step
int score_units(const BlockLayout& lay, int block);  // workgroups of a CU
void launch_score_tiles(const ScoreArgs& a, int block, int workgroups, hipStream_t s);

struct ScorePlan {
    DeviceCache* cache = nullptr;
    uint64_t epoch = 0;
    size_t rows = 0, slots = 0;
    float qscale = 0.f, cap = 0.f;
    bool tiles = false, biased = false;
    int heads = 0, group = 0;
    int few = 0, many = 0, items = 0;  // workgroups of each kernel
    PlanRegion region;
    size_t tables_at = 0, ranges_at = 0, runs_at = 0, slopes_at = 0, few_at = 0, many_at = 0, acc_at = 0, ml_at = 0;

    void build(DeviceCache* c, const uint64_t* sequences, size_t n, size_t heads, size_t context, const size_t* start,
               const size_t* rows, const size_t* first, const size_t* end, float scale, float cap, const float* slopes,
               bool parts);  // whether long chunks' products may be of fp16 parts (score_tiles.hip)
    void launch(int layer, const float* q, float* out, hipStream_t s);
    void check();
};

}  // namespace tvara_amd

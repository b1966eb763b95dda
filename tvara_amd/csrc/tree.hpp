// One step of speculative decoding with trees of drafted tokens over the
// paged cache: attention of the trees, greedy acceptance, slot maps with block
// tables, and the write of the accepted rows.
#pragma once

#include <cstddef>
#include <cstdint>
#include <memory>
#include <vector>

#include "kv_cache.hpp"

namespace tvara_amd {

// most nodes of one tree (its ancestor masks are 32 words a node)
constexpr size_t kMaxTreeNodes = 1024;
// most floats from one node's keys to the next one's: a tile's 32 rows lie within
// the 32 bits of a buffer's offsets
constexpr size_t kMaxRowStride = size_t(1) << 23;

// A batch of trees as the kernels read it.  Node rows are packed, one tree
// after the other; an attention row is a (node, query head) pair.
struct TreeArgs {
    const char* pool;
    BlockLayout lay;
    int layer, heads, group;
    const int32_t* tables;
    const int4* trees;     // x: table offset, y: cached tokens seen, z: nodes, w: first node row
    const uint32_t* mask;  // [node rows][words]: bit k of word s: the node sees node 32s + k of its tree
    int words;
    bool alone;            // tiles: an entry of work for each wave, not each workgroup
    const int4* work;      // see the kernels
    int split_tokens;      // row kernel: cached tokens of a run
    const int2* runs;      // per node row: first partial, runs (one run: written to out)
    int rows;
    const float* q;        // [node rows][heads][head_dim]
    const float* keys;     // [node rows] rows of kv_width floats, row_stride apart
    const float* values;
    size_t row_stride;
    float* out;            // [node rows][heads][head_dim]
    float* part_acc;       // [partials][heads][head_dim]
    float* part_ml;        // [partials][heads][2]: maximum (log2 units), normaliser
    bool check;            // a merged result that is not finite sets *err
    float qscale;          // log2(e) / sqrt(head_dim)
    int* err;
};

// greedy acceptance (launch_tree_accept)
struct AcceptArgs {
    const int4* trees;       // as TreeArgs
    const int32_t* parents;  // [node rows], within the tree; -1: a root
    int count, rows;
    const uint32_t* tokens;  // [node rows]
    const uint32_t* first;   // [trees]: the token a root has to be
    const float* logits;     // [node rows], logits_stride apart
    size_t vocab, logits_stride;
    int splits;              // parts of a row's vocabulary
    size_t part;             // logits of a part
    uint64_t* best;          // [node rows][splits]
    int* done;               // [trees]: parts done in this launch, zero between launches (null: a launch of its own walks)
    const int32_t* tree_of;  // [node rows]
    bool every_tree_has_nodes;
    int32_t* path;           // [trees][path_stride]: accepted node rows, -1 behind
    size_t path_stride;
    int32_t* accepted;       // [trees]
    uint32_t* next;          // [trees]
    int* err;
};

// slot maps and block tables (launch_slot_map)
struct SlotArgs {
    const int32_t* ids;      // the sequences' block ids; a set sign bit: shared
    const int2* seqs;        // x: first id, y: blocks
    int count, tpb;
    const int32_t* starts;   // [count]
    const int32_t* counts;   // [count]
    size_t stride, capacity;
    int32_t* offsets;        // [count + 1] or null
    int32_t* positions;      // [capacity] or null
    int64_t* slots;          // [capacity] or null
    int32_t* tables;         // [count][width] or null
    size_t width;
    int* err;
};

struct WriteArgs {
    char* pool;
    BlockLayout lay;
    int64_t slot_count;      // slots of the pool
    const int64_t* slots;    // [n], -1: nothing to write
    const int32_t* rows;     // [n] or null: row t
    size_t n, row_count;
    const float* keys;       // element (row, layer, column) at row * row_stride + layer * layer_stride + column
    const float* values;
    size_t row_stride, layer_stride;
    int* err;
};

// tree.hip
void launch_tree_rows(const TreeArgs& a, int items, hipStream_t s);
void launch_tree_merge(const TreeArgs& a, int most_runs, hipStream_t s);
// tree_tiles.hip: head_dim 64 and 128.  Work has three entries a workgroup (TreeArgs::
// alone: a wave): the tree (as trees); KV head, first row, first step, end; run, runs, the
// tree's first partial.
bool tree_tiles_supported(const BlockLayout& lay);
constexpr int kTreeStep = 32;  // keys of a step
constexpr int kTreeWaves = 4;  // of a workgroup
struct TreeTileShape {
    int rows;   // of a workgroup
    int units;  // workgroups that share a CU
    int least;  // steps of a run
    int alone_from, alone_to;  // workgroups a CU from which, steps of one to which waves work alone
};
// of 16 rows, or for f32x3 32 or 128 too
TreeTileShape tree_tile_shape(const BlockLayout& lay, int rows, bool x3);
void launch_tree_tiles(const TreeArgs& a, int rows, int workgroups, bool x3, hipStream_t s);
// tree_accept.hip: chooses part, splits and whether done stays; rows * splits is at
// most rows + kAcceptParts
constexpr size_t kAcceptParts = 4096;
void tree_accept_parts(AcceptArgs& a);
void launch_tree_accept(const AcceptArgs& a, hipStream_t s);
// slots.hip
void launch_slot_map(const SlotArgs& a, hipStream_t s);
void launch_slot_write(const WriteArgs& a, hipStream_t s);

// The device memory of a plan: sections of one region, the first of them
// uploaded in one copy on the cache's stream.  Plans that stayed on the null
// stream give their buffers to the cache's pool for its next plans, as decode
// plans do (PlanPool).
class PlanRegion {
public:
    PlanRegion() = default;
    ~PlanRegion();
    PlanRegion(const PlanRegion&) = delete;
    PlanRegion& operator=(const PlanRegion&) = delete;

    // sections of the uploaded part, then (data null) of the rest
    struct Section {
        const void* data;
        size_t bytes;
        size_t at = 0;
    };
    void place(DeviceCache& c, std::vector<Section>& sections);
    char* device() const { return static_cast<char*>(buf_->region.ptr); }
    // the kernels' error words, in pinned host memory
    int* flags() const { return static_cast<int*>(buf_->flag.ptr); }
    static constexpr int kFlags = 2;
    void launched(hipStream_t s);
    // waits for the last launch's stream; the words that were set (bit i: word
    // i), which are cleared
    int check();

private:
    std::unique_ptr<PlanPool::Set> buf_;
    std::shared_ptr<PlanPool> home_;
    bool null_stream_ = true;
    hipStream_t last_ = nullptr;
};

// the nodes' depths, a root's 1; refuses a parent that does not come before its node
// and depths above `room`
void tree_depths(const int32_t* parents, size_t nodes, size_t room, std::vector<size_t>& depth);

// Trees of drafted tokens over cached sequences (tvara_tree_plan_*).
struct TreePlan {
    DeviceCache* cache = nullptr;
    uint64_t epoch = 0;
    int heads = 0, group = 0, precision = 0, words = 1, items = 0, split_tokens = 0;
    TreeTileShape tiles{};  // rows 0: the row kernel
    bool alone = false;     // an entry of work for each wave of the tiles
    int most_runs = 1;
    size_t count = 0, rows = 0, slots = 0;
    PlanRegion region;
    size_t tables_at = 0, trees_at = 0, mask_at = 0, work_at = 0, runs_at = 0, parents_at = 0, acc_at = 0, ml_at = 0,
           best_at = 0, done_at = 0, tree_of_at = 0;
    bool every_tree_has_nodes = true;

    void build(DeviceCache* c, const uint64_t* sequences, size_t n, size_t heads, size_t context,
               const size_t* visible, const size_t* nodes, const int32_t* parents, int precision);
    TreeTileShape tile_shape(const std::vector<int4>& trees) const;
    // the workgroups of the kernel, and each node row's first partial and runs
    void row_work(const std::vector<int4>& trees, std::vector<int4>& work, std::vector<int2>& runs);
    void tile_work(const std::vector<int4>& trees, std::vector<int4>& work, std::vector<int2>& runs);
    void launch(int layer, const float* q, const float* keys, const float* values, size_t row_stride, float* out,
                hipStream_t s);
    void accept(const uint32_t* tokens, const uint32_t* first, const float* logits, size_t vocab, size_t logits_stride,
                int32_t* path, size_t path_stride, int32_t* accepted, uint32_t* next, hipStream_t s);
    void check();
};

// Slots and block tables of listed sequences (tvara_slot_plan_*).
struct SlotPlan {
    DeviceCache* cache = nullptr;
    uint64_t epoch = 0;
    size_t count = 0, seqs_at = 0;
    PlanRegion region;

    void build(DeviceCache* c, const uint64_t* sequences, size_t n);
    void map(const int32_t* starts, const int32_t* counts, size_t stride, size_t capacity, int32_t* offsets,
             int32_t* positions, int64_t* slots, int32_t* tables, size_t width, hipStream_t s);
    void write(const int64_t* slots, const int32_t* rows, size_t n, const float* keys, const float* values,
               size_t row_count, size_t row_stride, size_t layer_stride, hipStream_t s);
    void check();
};

}  // namespace tvara_amd

// Plans of speculative decoding with token trees (tree.hpp): what the host
// checks and lays out; the kernels are in tree.hip, tree_accept.hip and slots.hip.
#include "tree.hpp"

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <limits>
#include <map>

namespace tvara_amd {

namespace {
constexpr size_t kIntMax = static_cast<size_t>(std::numeric_limits<int32_t>::max());
// of a launch: 2^32 threads, here in workgroups of up to 256
constexpr size_t kMaxThreads = std::numeric_limits<uint32_t>::max(), kMaxWorkgroups = kMaxThreads / 256;

// steps from which on a run is a long one, and those that its start and merge are worth
constexpr size_t kLongRun = 64, kRunStart = 5;

size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
}  // namespace

// ------------------------------------------------------------ the region

PlanRegion::~PlanRegion() {
    if (buf_ && home_ && null_stream_) home_->give(std::move(buf_));
}

void PlanRegion::place(DeviceCache& c, std::vector<Section>& sections) {
    c.flush();  // (as AttnPlan::compute)
    size_t total = 0, copied = 0;
    for (Section& s : sections) {
        s.at = total;
        total = round_up(total + std::max<size_t>(s.bytes, 1), 256);
        if (s.data) copied = total;
    }
    hipStream_t s = c.stream();
    null_stream_ = s == nullptr;
    home_ = c.plan_pool();
    buf_ = s ? std::make_unique<PlanPool::Set>() : home_->take(total);
    try {
        buf_->region.ensure(total);
    } catch (const std::runtime_error&) {  // no memory, unless closed plans hold some
        (void)hipGetLastError();
        home_->clear();
        buf_->region.ensure(total);
    }
    if (copied) {
        char* host = static_cast<char*>(buf_->staging.acquire(copied));
        std::memset(host, 0, copied);
        for (const Section& x : sections)
            if (x.data && x.bytes) std::memcpy(host + x.at, x.data, x.bytes);
        TVARA_HIP(hipMemcpyAsync(device(), host, copied, hipMemcpyHostToDevice, s));
        buf_->staging.release(s);
    }
    auto* f = static_cast<volatile int*>(buf_->flag.acquire(kFlags * sizeof(int)));
    for (int i = 0; i < kFlags; ++i) f[i] = 0;
    last_ = s;
}

void PlanRegion::launched(hipStream_t s) {
    null_stream_ &= s == nullptr;
    last_ = s;
}

int PlanRegion::check() {
    TVARA_HIP(hipStreamSynchronize(last_));
    auto* f = static_cast<volatile int*>(buf_->flag.ptr);
    int set = 0;
    for (int i = 0; i < kFlags; ++i) {
        if (f[i]) set |= 1 << i;
        f[i] = 0;
    }
    return set;
}

// -------------------------------------------------------------- the trees

void tree_depths(const int32_t* parents, size_t nodes, size_t room, std::vector<size_t>& depth) {
    depth.resize(nodes);
    for (size_t j = 0; j < nodes; ++j) {
        const int32_t p = parents[j];
        if (p < -1 || p >= static_cast<int32_t>(j)) throw std::invalid_argument("invalid token tree");
        depth[j] = p < 0 ? 1 : depth[p] + 1;
        if (depth[j] > room) throw std::invalid_argument("token tree exceeds the context");
    }
}

void TreePlan::build(DeviceCache* c, const uint64_t* sequences, size_t n, size_t h, size_t context,
                     const size_t* visible, const size_t* nodes, const int32_t* parents, int prec) {
    cache = c;
    const Geometry& g = c->geometry();
    c->check_device();
    if (!n || !sequences || !nodes) throw std::invalid_argument("empty tree plan");
    if (prec != 0 && prec != 2) throw std::invalid_argument("tree attention is f32 or f32x3");
    if (h > 65535) throw std::invalid_argument("invalid fused attention shape");  // (a grid's second dimension)
    heads = static_cast<int>(h);
    group = static_cast<int>(h / g.kv_heads);
    precision = prec;
    count = n;
    rows = 0;
    size_t most = 0;
    for (size_t i = 0; i < n; ++i) {
        if (nodes[i] > kMaxTreeNodes) throw std::invalid_argument("a token tree has at most 1,024 nodes");
        rows += nodes[i];
        most = std::max(most, nodes[i]);
        // (the merge has a thread for two columns, acceptance a workgroup a row and more)
        if (rows > kMaxWorkgroups - kAcceptParts || rows > std::min(kIntMax, kMaxThreads / g.head_dim) / h)
            throw std::invalid_argument("attention batch too large");
    }
    if (rows && !parents) throw std::invalid_argument("invalid token tree");
    words = static_cast<int>(std::max<size_t>(1, (most + 31) / 32));

    std::vector<int4> trees(n);
    std::vector<uint32_t> mask(rows * words, 0);
    std::vector<int32_t> tab;
    std::map<uint64_t, int32_t> offset;
    std::vector<size_t> depth;
    size_t row0 = 0;
    for (size_t i = 0; i < n; ++i) {
        const Table& t = c->sequence(sequences[i]);
        const size_t seen = visible ? std::min(visible[i], t.length) : t.length;
        if (seen > kIntMax - kMaxTreeNodes) throw std::invalid_argument("sequence too long for the device kernels");
        if (seen > context) throw std::invalid_argument("invalid fused attention shape");
        tree_depths(parents + row0, nodes[i], context - seen, depth);
        for (size_t j = 0; j < nodes[i]; ++j) {
            const int32_t p = parents[row0 + j];
            uint32_t* m = &mask[(row0 + j) * words];
            if (p >= 0) std::copy_n(&mask[(row0 + p) * words], words, m);
            m[j / 32] |= 1u << (j % 32);
        }
        if (!offset.count(sequences[i])) {
            offset[sequences[i]] = static_cast<int32_t>(tab.size());
            for (const Handle& b : t.blocks) tab.push_back(static_cast<int32_t>(b.id));
            if (tab.size() > kIntMax) throw std::invalid_argument("attention batch too large");
        }
        trees[i] = make_int4(offset[sequences[i]], static_cast<int>(seen), static_cast<int>(nodes[i]), static_cast<int>(row0));
        row0 += nodes[i];
    }
    epoch = c->epoch();

    std::vector<int4> work;
    std::vector<int2> runs(rows);
    slots = 0;
    tiles = tree_tiles_supported(c->layout()) ? tile_shape(trees) : TreeTileShape{};
    if (tiles.rows)
        tile_work(trees, work, runs);
    else
        row_work(trees, work, runs);
    if (slots > kIntMax / h || work.size() > 3 * kMaxWorkgroups) throw std::invalid_argument("attention batch too large");
    items = static_cast<int>(tiles.rows ? work.size() / (alone ? 3 * kTreeWaves : 3) : work.size());
    most_runs = 1;
    for (const int2& r : runs) most_runs = std::max(most_runs, r.y);

    // acceptance's: each row's tree, and counters that start at zero
    std::vector<int32_t> tree_of(rows), zeros(n, 0);
    every_tree_has_nodes = true;
    for (size_t i = 0; i < n; ++i) {
        std::fill_n(tree_of.begin() + trees[i].w, trees[i].z, static_cast<int32_t>(i));
        every_tree_has_nodes &= trees[i].z > 0;
    }

    std::vector<PlanRegion::Section> s = {
        {tab.data(), tab.size() * sizeof(int32_t)},   {trees.data(), n * sizeof(int4)},
        {mask.data(), mask.size() * sizeof(uint32_t)}, {work.data(), work.size() * sizeof(int4)},
        {runs.data(), runs.size() * sizeof(int2)},     {parents, rows * sizeof(int32_t)},
        {tree_of.data(), rows * sizeof(int32_t)},      {zeros.data(), n * sizeof(int)},
        {nullptr, slots * h * g.head_dim * sizeof(float)}, {nullptr, slots * h * 2 * sizeof(float)},
        {nullptr, (rows + kAcceptParts) * sizeof(uint64_t)},
    };
    region.place(*c, s);
    size_t* at[] = {&tables_at, &trees_at, &mask_at, &work_at, &runs_at, &parents_at, &tree_of_at, &done_at, &acc_at, &ml_at, &best_at};
    for (size_t i = 0; i < s.size(); ++i) *at[i] = s[i].at;
}

// Runs of cached tokens, so that a long context fills the chip: about four waves
// a SIMD, 64 tokens or more each; the last run takes the tree's own.
void TreePlan::row_work(const std::vector<int4>& trees, std::vector<int4>& work, std::vector<int2>& runs) {
    size_t total = 0;
    for (const int4& t : trees) total += static_cast<size_t>(t.y) * t.z;
    const size_t target = std::max<size_t>(1, static_cast<size_t>(cache->compute_units()) * 16 / heads);
    const size_t split = std::min(round_up(std::max<size_t>(total / target, 64), 64), kIntMax / 2);
    split_tokens = static_cast<int>(split);
    for (size_t i = 0; i < trees.size(); ++i) {
        const int4& t = trees[i];
        const int parts = static_cast<int>(std::max<size_t>(1, (static_cast<size_t>(t.y) + split - 1) / split));
        for (int j = 0; j < t.z; ++j) {
            runs[t.w + j] = make_int2(static_cast<int>(slots), parts);
            if (parts > 1) slots += parts;
            for (int p = 0; p < parts; ++p) work.push_back(make_int4(static_cast<int>(i), j, p, parts));
        }
    }
}

namespace {
int cached_steps(const int4& t) { return (t.y + kTreeStep - 1) / kTreeStep; }
// steps over the tree's own nodes of the row block from row r0
int own_steps(const int4& t, int r0, int rows, int group) {
    return (std::min(t.z * group, r0 + rows) - 1) / group / kTreeStep + 1;
}
}  // namespace

// Rows of a workgroup.  f32: 16 (MI355X, 16 contexts of 2048, 32 heads on 8, head_dim 64,
// 64 rows a KV head 16: 54.8 us  32: 64.5; head_dim 128, 32 rows 58.7 and 65.6).  f32x3
// can share a key's two parts among 32 rows in registers or 128 in LDS.  Many rows need
// that, but as long as the work is short, the fewest rows are best for which the chip
// holds all workgroups at once (eight trees of 16 nodes after 250 tokens 16: 11.8  32: 17.4
// 128: 20.1; 60 such 90.3, 67.4, 42.5), and then blocks that fill it.  Else by the
// most rows of a tree (16 contexts of 2048, 16 rows 16: 51.6  32: 55.3; 64 rows 32: 58.7
// 128: 72.5; 80 rows 32: 113  128: 79).  Over 404 shapes (1 to 60 trees of 4 to 28
// nodes after 30 to 16,000 tokens, both widths and formats) this is 0.6% from the
// best of the three on average, 45% at worst; by rows alone it would be 11%.  16 uneven
// contexts (200 to 2,000 tokens) fill the chip with blocks of 16 in one run each, which
// end with the longest: 27.3 us, 23.0 in blocks of 32.
// TVARA_TREE_ROWS (16, 32 or 128) chooses for f32x3 instead.
TreeTileShape TreePlan::tile_shape(const std::vector<int4>& trees) const {
    constexpr size_t kShort = 40;  // steps of a place for a workgroup
    const bool x3 = precision == 2;
    if (!x3) return tree_tile_shape(cache->layout(), 16, x3);
    int most = 0;
    for (const int4& t : trees) most = std::max(most, t.z * group);
    const char* choice = std::getenv("TVARA_TREE_ROWS");
    for (const int high : {16, 32, 128})
        if (choice && std::atoi(choice) == high) return tree_tile_shape(cache->layout(), high, x3);
    bool crowded = false;  // few steps, and not in one round
    for (const int high : {16, 32, 128}) {
        const TreeTileShape shape = tree_tile_shape(cache->layout(), high, x3);
        const size_t units = static_cast<size_t>(cache->compute_units()) * shape.units;
        size_t workgroups = 0, steps = 0;
        int longest = 0;
        for (const int4& t : trees) {
            if (!t.z) continue;
            const int blocks = (t.z * group - 1) / high + 1, each = cached_steps(t) + own_steps(t, t.z * group - 1, high, group);
            workgroups += static_cast<size_t>(blocks) * cache->layout().kv_heads;
            steps += static_cast<size_t>(blocks) * cache->layout().kv_heads * each;
            longest = std::max(longest, each);
        }
        // (where a run a tree fills the chip, the longest may not end much later than the rest)
        const bool even = longest <= 8 || 2 * workgroups <= units || 2 * longest * workgroups <= 3 * steps;
        // (in blocks of 128, 32 rows leave half of the waves without any)
        const size_t most_steps = high == 128 && most <= 32 ? kShort / 4 : kShort;
        if (workgroups <= units && steps <= most_steps * units && even && (high < 128 || (most > 16 && 2 * workgroups >= units)))
            return shape;
        crowded |= high == 32 && workgroups > units && longest < kTreeWaves;
    }
    return tree_tile_shape(cache->layout(), most <= 16 ? 16 : most <= 64 && !crowded ? 32 : 128, x3);
}

// Runs of steps of the tiles, as many as give every CU its workgroups.  Ids go to the
// XCDs round-robin: the row blocks of one run, which read the same keys, go to one
// XCD, whose L2 then has them, and the XCDs' lists are filled by the fewest steps so
// far, each ordered from the longest run to the shortest.
void TreePlan::tile_work(const std::vector<int4>& trees, std::vector<int4>& work, std::vector<int2>& runs) {
    const int kv_heads = cache->layout().kv_heads, xcds = std::max(1, cache->xcds()), high = tiles.rows;
    auto steps_of = [&](const int4& t) {  // of its last row block, which has the most
        return cached_steps(t) + own_steps(t, t.z * group - 1, high, group);
    };
    size_t total = 0;
    for (const int4& t : trees)
        for (int r0 = 0; r0 < t.z * group; r0 += high)
            total += static_cast<size_t>(kv_heads) * (cached_steps(t) + own_steps(t, r0, high, group));
    // Steps of a run: an even share, or up to twice that if the chip then holds all
    // workgroups at once.  Where the share is long, the length with the least rounds of
    // workgroups * their mean steps: a second round for a few of them costs a share
    // (MI355X, f32, head_dim 128: six trees of 23 nodes after 6,263 tokens in 288
    // workgroups for 256 places 240 us, cut so 179); short ones would pay more for the
    // launch of a merge (62 trees of 7 nodes after 191: 20.2 us, cut so 26.9).
    const size_t units = static_cast<size_t>(cache->compute_units()) * tiles.units, least = tiles.least;
    const size_t even = std::max(least, (total + units - 1) / units);
    const bool lengthy = even >= kLongRun;
    size_t per = even, best = std::numeric_limits<size_t>::max();
    for (size_t p = lengthy ? even / 6 : even; p <= 2 * even; p += (p + 15) / 16) {
        size_t workgroups = 0, longest = 0;
        for (const int4& t : trees) {
            if (!t.z) continue;
            const size_t steps = steps_of(t), parts = (steps + p - 1) / p;
            workgroups += parts * ((t.z * group - 1) / high + 1) * kv_heads;
            longest = std::max(longest, (steps + parts - 1) / parts);
        }
        if (!lengthy) {
            if (workgroups > units) continue;
            per = p;
            break;
        }
        const size_t rounds = (workgroups + units - 1) / units;
        const size_t end = std::max((longest + kRunStart) * units, rounds * (total * units / workgroups + kRunStart * units));
        if (end < best) {
            best = end;
            per = p;
        }
    }
    size_t workgroups = 0, most_steps = 0;
    for (const int4& t : trees) {
        if (!t.z) continue;
        workgroups += (steps_of(t) + per - 1) / per * ((t.z * group - 1) / high + 1) * kv_heads;
        most_steps = std::max(most_steps, std::min<size_t>(per, steps_of(t)));
    }
    alone = workgroups / cache->compute_units() >= static_cast<size_t>(tiles.alone_from) &&
           most_steps <= static_cast<size_t>(tiles.alone_to);
    struct Group {  // the row blocks of a run
        int tree, head, run, runs, slot, step, end;
    };
    std::vector<Group> groups;
    for (size_t i = 0; i < trees.size(); ++i) {
        const int4& t = trees[i];
        if (!t.z) continue;
        const int steps = steps_of(t);
        const int parts = static_cast<int>((steps + per - 1) / per), len = (steps + parts - 1) / parts;
        for (int p = 0; p < parts; ++p)
            for (int h = 0; h < kv_heads; ++h)
                groups.push_back({static_cast<int>(i), h, p, parts, static_cast<int>(slots), p * len, std::min((p + 1) * len, steps)});
        for (int j = 0; j < t.z; ++j) runs[t.w + j] = make_int2(static_cast<int>(slots + static_cast<size_t>(j) * parts), parts);
        if (parts > 1) slots += static_cast<size_t>(t.z) * parts;
        if (slots > kIntMax / heads) throw std::invalid_argument("attention batch too large");
    }
    std::stable_sort(groups.begin(), groups.end(), [](const Group& x, const Group& y) { return x.end - x.step > y.end - y.step; });
    std::vector<std::vector<int4>> lists(xcds);
    std::vector<size_t> load(xcds, 0);
    for (const Group& x : groups) {
        const int4& t = trees[x.tree];
        const size_t to = std::min_element(load.begin(), load.end()) - load.begin();
        for (int r0 = 0; r0 < t.z * group; r0 += high) {
            const int all = cached_steps(t) + own_steps(t, r0, high, group);
            const int step = std::min(x.step, all), end = std::min(x.end, all);
            lists[to].insert(lists[to].end(), {t, make_int4(x.head, r0, step, end), make_int4(x.run, x.runs, x.slot, 0)});
            load[to] += end - step + 1;
        }
    }
    // an XCD's list becomes that of every xcds-th workgroup
    const size_t chunk = alone ? 3 * kTreeWaves : 3;
    size_t longest = 0;
    for (const auto& l : lists) longest = std::max(longest, round_up(l.size(), chunk));
    work.assign(longest * xcds, make_int4(0, 0, 0, 0));  // (padding has no nodes)
    for (int x = 0; x < xcds; ++x)
        for (size_t k = 0; k < lists[x].size(); ++k) work[chunk * (k / chunk * xcds + x) + k % chunk] = lists[x][k];
}

void TreePlan::launch(int layer, const float* q, const float* keys, const float* values, size_t row_stride, float* out,
                      hipStream_t s) {
    if (cache->epoch() != epoch) throw std::invalid_argument("tree plan is stale: the cache changed");
    const Geometry& g = cache->geometry();
    if (layer < 0 || static_cast<size_t>(layer) >= g.layers) throw std::invalid_argument("invalid fused attention shape");
    if (!row_stride) row_stride = g.kv_width();
    if (row_stride < g.kv_width()) throw std::invalid_argument("token rows overlap");
    if (row_stride > kMaxRowStride) throw std::invalid_argument("token rows too far apart");
    if (!rows) return;
    cache->check_device();
    cache->enter(s);
    char* d = region.device();
    TreeArgs a{};
    a.pool = cache->pool();
    a.lay = cache->layout();
    a.layer = layer;
    a.heads = heads;
    a.group = group;
    a.tables = reinterpret_cast<const int32_t*>(d + tables_at);
    a.trees = reinterpret_cast<const int4*>(d + trees_at);
    a.mask = reinterpret_cast<const uint32_t*>(d + mask_at);
    a.words = words;
    a.work = reinterpret_cast<const int4*>(d + work_at);
    a.alone = alone;
    a.split_tokens = split_tokens;
    a.runs = reinterpret_cast<const int2*>(d + runs_at);
    a.rows = static_cast<int>(rows);
    a.q = q;
    a.keys = keys;
    a.values = values;
    a.row_stride = row_stride;
    a.out = out;
    a.part_acc = reinterpret_cast<float*>(d + acc_at);
    a.part_ml = reinterpret_cast<float*>(d + ml_at);
    a.qscale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(g.head_dim)));
    a.check = tiles.rows && precision == 2;
    a.err = region.flags();
    if (tiles.rows)
        launch_tree_tiles(a, tiles.rows, items, precision == 2, s);
    else
        launch_tree_rows(a, items, s);
    if (slots) launch_tree_merge(a, most_runs, s);
    cache->leave(s);
    region.launched(s);
}

void TreePlan::accept(const uint32_t* tokens, const uint32_t* first, const float* logits, size_t vocab,
                      size_t logits_stride, int32_t* path, size_t path_stride, int32_t* accepted, uint32_t* next,
                      hipStream_t s) {
    if (!vocab || vocab > kIntMax) throw std::invalid_argument("invalid vocabulary");
    if (!logits_stride) logits_stride = vocab;
    if (logits_stride < vocab) throw std::invalid_argument("logit rows overlap");
    cache->check_device();
    AcceptArgs a{};
    char* d = region.device();
    a.trees = reinterpret_cast<const int4*>(d + trees_at);
    a.parents = reinterpret_cast<const int32_t*>(d + parents_at);
    a.count = static_cast<int>(count);
    a.rows = static_cast<int>(rows);
    a.tokens = tokens;
    a.first = first;
    a.logits = logits;
    a.vocab = vocab;
    a.logits_stride = logits_stride;
    a.done = reinterpret_cast<int*>(d + done_at);
    a.tree_of = reinterpret_cast<const int32_t*>(d + tree_of_at);
    a.every_tree_has_nodes = every_tree_has_nodes;
    tree_accept_parts(a);
    a.best = reinterpret_cast<uint64_t*>(d + best_at);
    a.path = path;
    a.path_stride = path_stride;
    a.accepted = accepted;
    a.next = next;
    a.err = region.flags() + 1;
    cache->enter(s);  // (the plan's upload)
    launch_tree_accept(a, s);
    cache->leave(s);
    region.launched(s);
}

void TreePlan::check() {
    const int set = region.check();
    if (set & 1) throw std::invalid_argument("invalid online attention input");
    if (set & 2) throw std::invalid_argument("invalid logits or path of a token tree");
}

// -------------------------------------------------------------- the slots

void SlotPlan::build(DeviceCache* c, const uint64_t* sequences, size_t n) {
    cache = c;
    c->check_device();
    if (!n || !sequences) throw std::invalid_argument("empty slot plan");
    if (n > 65535) throw std::invalid_argument("a slot plan has at most 65,535 sequences");
    count = n;
    std::vector<int32_t> ids;
    std::vector<int2> seqs(n);
    for (size_t i = 0; i < n; ++i) {
        const Table& t = c->sequence(sequences[i]);
        if (ids.size() + t.blocks.size() > kIntMax) throw std::invalid_argument("slot plan too large");
        seqs[i] = make_int2(static_cast<int>(ids.size()), static_cast<int>(t.blocks.size()));
        // a block that others hold too is not this sequence's to write
        for (const Handle& b : t.blocks) {
            const uint32_t shared = c->references(b) > 1 ? 0x80000000u : 0u;
            ids.push_back(static_cast<int32_t>(static_cast<uint32_t>(b.id) | shared));
        }
    }
    epoch = c->epoch();
    std::vector<PlanRegion::Section> s = {{ids.data(), ids.size() * sizeof(int32_t)}, {seqs.data(), n * sizeof(int2)}};
    region.place(*c, s);
    seqs_at = s[1].at;
}

void SlotPlan::map(const int32_t* starts, const int32_t* counts, size_t stride, size_t capacity, int32_t* offsets,
                   int32_t* positions, int64_t* slots, int32_t* tables, size_t width, hipStream_t s) {
    if (cache->epoch() != epoch) throw std::invalid_argument("slot plan is stale: the cache changed");
    if (capacity > kIntMax || stride > kIntMax || width > kIntMax || (tables && width > kIntMax / count))
        throw std::invalid_argument("slot map too large");
    if (stride && capacity < stride * count) throw std::invalid_argument("slot map smaller than its sequences");
    cache->check_device();
    cache->enter(s);
    SlotArgs a{};
    a.ids = reinterpret_cast<const int32_t*>(region.device());
    a.seqs = reinterpret_cast<const int2*>(region.device() + seqs_at);
    a.count = static_cast<int>(count);
    a.tpb = cache->layout().tpb;
    a.starts = starts;
    a.counts = counts;
    a.stride = stride;
    a.capacity = capacity;
    a.offsets = offsets;
    a.positions = positions;
    a.slots = slots;
    a.tables = tables;
    a.width = width;
    a.err = region.flags();
    launch_slot_map(a, s);
    cache->leave(s);
    region.launched(s);
}

void SlotPlan::write(const int64_t* slots, const int32_t* rows, size_t n, const float* keys, const float* values,
                     size_t row_count, size_t row_stride, size_t layer_stride, hipStream_t s) {
    if (cache->epoch() != epoch) throw std::invalid_argument("slot plan is stale: the cache changed");
    const Geometry& g = cache->geometry();
    // (a thread has up to four floats of a row, and 32 bits for their place in a block)
    if (n > kMaxWorkgroups || row_count > kIntMax || 2 * g.layers * g.kv_width() > size_t(65535) * 256 ||
        2 * g.layers * g.kv_width() * g.tokens_per_block > kMaxThreads)
        throw std::invalid_argument("KV write too large");
    if (row_stride < g.kv_width() || (g.layers > 1 && layer_stride < g.kv_width()))
        throw std::invalid_argument("token rows overlap");
    if (cache->format() == kQ8 && (row_stride % 4 || (g.layers > 1 && layer_stride % 4)))
        throw std::invalid_argument("device buffers must be 16-byte aligned");
    if (!n) return;
    cache->check_device();
    cache->enter(s);
    WriteArgs a{};
    a.pool = cache->pool();
    a.lay = cache->layout();
    a.slot_count = static_cast<int64_t>(g.max_blocks * g.tokens_per_block);
    a.slots = slots;
    a.rows = rows;
    a.n = n;
    a.row_count = row_count;
    a.keys = keys;
    a.values = values;
    a.row_stride = row_stride;
    a.layer_stride = layer_stride;
    a.err = region.flags() + 1;
    launch_slot_write(a, s);
    cache->leave(s);
    region.launched(s);
}

// whether `count` rows of floats this far apart may pass the end of the address space
static bool wraps(size_t count, size_t stride) { return count && stride > (size_t(1) << 59) / count; }

void SlotPlan::rotate(RotateArgs a, hipStream_t s) {
    if (cache->epoch() != epoch) throw std::invalid_argument("slot plan is stale: the cache changed");
    const Geometry& g = cache->geometry();
    if (a.layer < 0 || static_cast<size_t>(a.layer) >= g.layers || a.heads < 1 || a.heads % static_cast<int>(g.kv_heads) ||
        a.heads + 2 * g.kv_heads > 65535 || g.head_dim % 2 || g.head_dim > 512 || a.rotary < 0 || a.rotary % 2 ||
        static_cast<size_t>(a.rotary) > g.head_dim)
        throw std::invalid_argument("invalid rotation shape");
    if (!(a.eps >= 0) || !std::isfinite(a.eps)) throw std::invalid_argument("invalid norm epsilon");
    const size_t hidden = a.heads * g.head_dim;
    if (!a.q_stride) a.q_stride = hidden;
    if (!a.kv_stride) a.kv_stride = g.kv_width();
    if (a.q_stride < hidden || a.kv_stride < g.kv_width() || wraps(a.n, a.q_stride) || wraps(a.n, a.kv_stride))
        throw std::invalid_argument("token rows overlap");
    // (rows of other strides would be written while others are read)
    if ((a.q_out && a.q_out == a.q && a.q_stride != hidden) || (a.k_out && a.k_out == a.keys && a.kv_stride != g.kv_width()))
        throw std::invalid_argument("token rows overlap");
    if (a.n > kMaxWorkgroups || 2 * g.layers * g.kv_width() * g.tokens_per_block > kMaxThreads)
        throw std::invalid_argument("KV write too large");
    if (!a.n) return;
    cache->check_device();
    cache->enter(s);
    a.pool = cache->pool();
    a.lay = cache->layout();
    a.slot_count = static_cast<int64_t>(g.max_blocks * g.tokens_per_block);
    a.err = region.flags() + 2;
    launch_rotate(a, s);
    cache->leave(s);
    region.launched(s);
}

void SlotPlan::read(ReadArgs a, hipStream_t s) {
    if (cache->epoch() != epoch) throw std::invalid_argument("slot plan is stale: the cache changed");
    const Geometry& g = cache->geometry();
    if (a.layer < 0 || a.layers < 0 || static_cast<size_t>(a.layer) > g.layers || static_cast<size_t>(a.layers) > g.layers - a.layer)
        throw std::invalid_argument("layers outside the cache");
    if (a.row_stride < g.kv_width() || (a.layers > 1 && a.layer_stride < g.kv_width()))
        throw std::invalid_argument("token rows overlap");
    // one row's layers before the next row, or one layer's rows before the next layer, all
    // of them without a turn round the address space
    const size_t layers = std::max(a.layers, 1), rows = std::max<size_t>(a.n, 1);
    if (wraps(rows, a.row_stride) || wraps(layers, a.layer_stride) ||
        (rows > 1 && layers > 1 && a.row_stride < (layers - 1) * a.layer_stride + g.kv_width() &&
         a.layer_stride < (rows - 1) * a.row_stride + g.kv_width()))
        throw std::invalid_argument("token rows overlap");
    if (a.n > kMaxWorkgroups || 2 * g.layers * g.kv_width() > size_t(65535) * 256 ||
        2 * g.layers * g.kv_width() * g.tokens_per_block > kMaxThreads)
        throw std::invalid_argument("KV read too large");
    if (cache->format() == kQ8 && (a.row_stride % 4 || (a.layers > 1 && a.layer_stride % 4)))
        throw std::invalid_argument("device buffers must be 16-byte aligned");
    if (!a.n || !a.layers) return;
    cache->check_device();
    cache->enter(s);
    a.pool = cache->pool();
    a.lay = cache->layout();
    a.slot_count = static_cast<int64_t>(g.max_blocks * g.tokens_per_block);
    a.err = region.flags() + 2;
    launch_slot_read(a, s);
    cache->leave(s);
    region.launched(s);
}

void SlotPlan::check() {
    const int set = region.check();
    if (set & 1) throw std::invalid_argument("slot map outside the sequences' own blocks");
    if (set & 2) throw std::invalid_argument("KV write outside the pool or the rows");
    if (set & 4) throw std::invalid_argument("slot outside the pool");
}

}  // namespace tvara_amd

// Plans of scored attention (score.hpp): what the host checks and lays out.
#include "score.hpp"

#include <algorithm>
#include <cmath>
#include <limits>
#include <map>

namespace tvara_amd {

namespace {

constexpr size_t kIntMax = static_cast<size_t>(std::numeric_limits<int32_t>::max());
// of a launch: 2^32 threads, here in workgroups of up to 512
constexpr size_t kMaxThreads = std::numeric_limits<uint32_t>::max(), kMaxWorkgroups = kMaxThreads / 512;
// keys of a run of the row kernel, at least
constexpr size_t kRowRun = 64;
// caps that are none
constexpr float kNoCap = 18446744073709551616.f;  // 2^64
// the largest bias of a score, in log2 units, with room for the score in f32
constexpr float kMaxBias = 8.5e37f;
// rounds of workgroups that runs are cut for; what a run of few and of many rows costs
// beside its steps, in steps (many: six prompts of 3 to 700 rows behind up to 2,500 keys, 32
// heads of 64: 134 us at 2, whose runs are shorter and want merging, 130 at 8 and at 24)
constexpr size_t kRounds = 4, kRunCost[2] = {12, 8};

// A block of rows of a sequence that read the same keys: they share its runs.
struct Block {
    int seq, row, rows;  // the first of the packed rows, how many
    int position;        // of the first
    int step, end;
    int runs, slot;
};

}  // namespace

void ScorePlan::build(DeviceCache* c, const uint64_t* sequences, size_t n, size_t h, size_t context, const size_t* start,
                      const size_t* counts, const size_t* first, const size_t* end, float scale, float limit,
                      const float* slopes, bool parts_too) {
    cache = c;
    const Geometry& g = c->geometry();
    c->check_device();
    if (!n || !sequences || !start || !counts) throw std::invalid_argument("empty score plan");
    if (h > 65535) throw std::invalid_argument("invalid fused attention shape");  // (a grid's second dimension)
    if (!scale) scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(g.head_dim)));
    constexpr double kLog2e = 1.4426950408889634;
    // (of scores up to 2^52 such a cap changes nothing that f32 holds, and scale / cap would
    // leave the numbers that operands in parts hold: fp16's and bf16's)
    if (limit >= kNoCap && std::isfinite(static_cast<float>(limit * kLog2e))) limit = 0;
    qscale = static_cast<float>(limit ? static_cast<double>(scale) / limit : scale * kLog2e);
    cap = static_cast<float>(limit * kLog2e);
    if (!(scale > 0) || !(limit >= 0) || !std::isfinite(qscale) || !(qscale > 0) || !std::isfinite(cap))
        throw std::invalid_argument("invalid score scale or cap");
    biased = slopes != nullptr;
    std::vector<float> bias(biased ? h : 0);
    for (size_t i = 0; i < bias.size(); ++i) {
        bias[i] = static_cast<float>(slopes[i] * kLog2e);
        if (!std::isfinite(bias[i])) throw std::invalid_argument("invalid score slope");
    }
    heads = static_cast<int>(h);
    group = static_cast<int>(h / g.kv_heads);
    rows = 0;
    for (size_t i = 0; i < n; ++i) {
        // (the merge has 256 threads a row in its grid's first dimension)
        if (counts[i] > kIntMax || (rows += counts[i]) > std::min(kIntMax, kMaxThreads / g.head_dim) / h || rows > kMaxThreads / 256)
            throw std::invalid_argument("attention batch too large");
    }

    const BlockLayout& lay = c->layout();
    tiles = tree_tiles_supported(lay);
    if (!tiles && g.head_dim > 512) throw std::invalid_argument("head_dim above 512 is not supported");
    // a position's query heads of one KV head that a block takes: all, or an even part
    const int parts = (group + kScoreFew - 1) / kScoreFew, per_block = (group + parts - 1) / parts;
    std::vector<int2> ranges(rows), runs(rows, make_int2(0, 1));
    std::vector<int32_t> tab;
    std::map<uint64_t, int32_t> offset;
    std::vector<int4> seqs(n);
    std::vector<Block> blocks[2];  // of few rows (or the row kernel's), of many
    const int step[2] = {tiles ? score_step(lay, kScoreFew) : 1, tiles ? score_step(lay, kScoreMany) : 1};
    size_t row0 = 0, longest = 0;
    for (size_t i = 0; i < n; ++i) {
        const Table& t = c->sequence(sequences[i]);
        if (t.length > kIntMax / 2) throw std::invalid_argument("sequence too long for the device kernels");
        if (t.length > context || start[i] > t.length || counts[i] > t.length - start[i])
            throw std::invalid_argument("invalid fused attention shape");
        longest = std::max(longest, t.length);
        if (!offset.count(sequences[i])) {
            offset[sequences[i]] = static_cast<int32_t>(tab.size());
            for (const Handle& b : t.blocks) tab.push_back(static_cast<int32_t>(b.id));
            if (tab.size() > kIntMax) throw std::invalid_argument("attention batch too large");
        }
        for (size_t j = 0; j < counts[i]; ++j) {
            const size_t lo = first ? first[row0 + j] : 0, hi = end ? end[row0 + j] : start[i] + j + 1;
            if (hi > t.length) throw std::invalid_argument("visible keys behind the sequence's end");
            ranges[row0 + j] = lo < hi ? make_int2(static_cast<int>(lo), static_cast<int>(hi)) : make_int2(0, 0);
        }
        seqs[i] = make_int4(offset[sequences[i]], static_cast<int>(t.length), static_cast<int>(counts[i]), static_cast<int>(row0));
        // Blocks of many rows, whose products are of fp16 parts, are for plans that allow
        // these.  They share a key's parts among them and pay for padding and
        // splitting with few: eight contexts of 2,000, 32 heads on 8, attention rows a KV
        // head, few against many (f32, us): head_dim 64 96 rows 51 and 57, 128 69 and 61;
        // head_dim 128 64 rows 58 and 82, 96 90 and 85; (Q8_0) 64 128 rows 52 and 61, 256 78
        // and 63; 128 128 rows 79 and 90, 256 123 and 93.
        const int kind = tiles && parts_too && counts[i] * per_block > (lay.format == kQ8 ? 160 : 96) ? 1 : 0;
        const size_t high = tiles ? (kind ? kScoreMany : kScoreFew) / per_block : 1;
        for (size_t j = 0; j < counts[i]; j += high) {
            Block b{static_cast<int>(i), static_cast<int>(row0 + j), static_cast<int>(std::min(high, counts[i] - j)),
                    static_cast<int>(start[i] + j), std::numeric_limits<int>::max(), 0, 1, 0};
            for (int r = b.row; r < b.row + b.rows; ++r)
                if (ranges[r].x < ranges[r].y) {
                    b.step = std::min(b.step, ranges[r].x / step[kind]);
                    b.end = std::max(b.end, (ranges[r].y + step[kind] - 1) / step[kind]);
                }
            if (b.end == 0) b.step = 0;  // no keys: zeros are written
            blocks[kind].push_back(b);
        }
        row0 += counts[i];
    }
    epoch = c->epoch();
    // (a bias that is infinite would take a key that a row sees from it, or be all that it has)
    for (const float b : bias)
        if (std::fabs(b) * static_cast<float>(longest) > kMaxBias) throw std::invalid_argument("invalid score slope");

    // Runs of steps, as many as give every CU its workgroups.
    slots = 0;
    const int kv_heads = lay.kv_heads, xcds = std::max(1, c->xcds());
    std::vector<int4> work[2];
    for (int kind = 0; kind < 2; ++kind) {
        const int block = kind ? kScoreMany : kScoreFew;
        const size_t slices = tiles ? static_cast<size_t>(kv_heads) * parts : h;
        size_t total = 0, units = static_cast<size_t>(c->compute_units()) * 16, least = kRowRun;
        if (tiles) {
            units = static_cast<size_t>(c->compute_units()) * score_units(lay, block);
            least = 4;
        }
        size_t longest_block = 0;
        for (const Block& b : blocks[kind]) {
            total += static_cast<size_t>(b.end - b.step) * slices;
            longest_block = std::max(longest_block, static_cast<size_t>(b.end - b.step));
        }
        // Runs of the same length that the chip takes in as few whole rounds as possible: in
        // one, two, … rounds the shortest that leave no workgroup for another, and of those the
        // least time. (Cut by the average alone, the ragged lengths leave a few workgroups
        // behind, for as long as all the others took.)
        size_t per = std::max(least, (total + units - 1) / units), time = std::numeric_limits<size_t>::max();
        auto cuts = [&](size_t length) {
            size_t count = 0;
            for (const Block& b : blocks[kind]) count += std::max<size_t>(1, (b.end - b.step + length - 1) / length) * slices;
            return count;
        };
        bool at_once = false;
        for (size_t rounds = 1; tiles && rounds <= kRounds; ++rounds) {
            size_t low = std::max(least, (total + rounds * units - 1) / (rounds * units)), high = std::max(low, longest_block);
            if (cuts(high) > rounds * units) continue;
            while (low < high) {
                const size_t mid = low + (high - low) / 2;
                if (cuts(mid) <= rounds * units)
                    high = mid;
                else
                    low = mid + 1;
            }
            if (rounds * (low + kRunCost[kind]) < time) {
                time = rounds * (low + kRunCost[kind]);
                per = low;
                at_once = rounds == 1;
            }
        }
        if (tiles && !kind && per > 4 * kScoreChain) {
            per = 4 * kScoreChain;
            at_once = false;
        }
        std::vector<int4> list;
        std::vector<size_t> load;
        for (Block& b : blocks[kind]) {
            const size_t steps = b.end - b.step;
            const int cut = static_cast<int>(std::max<size_t>(1, (steps + per - 1) / per));
            const int len = static_cast<int>((steps + cut - 1) / cut);
            b.runs = std::max(1, len ? static_cast<int>((steps + len - 1) / len) : 1);
            b.slot = static_cast<int>(slots);
            if (b.runs > 1) {
                for (int j = 0; j < b.rows; ++j) runs[b.row + j] = make_int2(static_cast<int>(slots) + j * b.runs, b.runs);
                slots += static_cast<size_t>(b.rows) * b.runs;
                if (slots > kIntMax / h) throw std::invalid_argument("attention batch too large");
            }
            if (work[0].size() + list.size() > 3 * kMaxWorkgroups) throw std::invalid_argument("attention batch too large");
            if (!tiles)
                for (int r = 0; r < b.runs; ++r) {
                    work[0].push_back(make_int4(seqs[b.seq].x, seqs[b.seq].y, 1, b.row));
                    work[0].push_back(make_int4(0, 0, b.step + r * len, std::min(b.step + (r + 1) * len, b.end)));
                    work[0].push_back(make_int4(r, b.runs, b.slot, b.position));
                }
        }
        if (!tiles) continue;
        // Workgroups that read the same keys one after the other, cut into the XCDs' equal
        // shares (workgroup ids go to the XCDs round-robin), each from the longest down: shares
        // of the work, or of the workgroups where all of them run at once.
        size_t sum = 0;
        for (size_t at = 0; at < blocks[kind].size();) {
            size_t to = at;
            int most = 1;
            while (to < blocks[kind].size() && blocks[kind][to].seq == blocks[kind][at].seq) most = std::max(most, blocks[kind][to++].runs);
            for (int kh = 0; kh < kv_heads; ++kh)
                for (int p = 0; p < parts; ++p)
                    for (int r = 0; r < most; ++r)
                        for (size_t k = at; k < to; ++k) {
                            const Block& b = blocks[kind][k];
                            if (r >= b.runs) continue;
                            const int len = (b.end - b.step + b.runs - 1) / b.runs, h0 = p * per_block;
                            const int s0 = b.step + r * len, s1 = std::min(s0 + len, b.end);
                            list.push_back(make_int4(seqs[b.seq].x, seqs[b.seq].y, b.rows, b.row));
                            list.push_back(make_int4(kh * group + h0, std::min(per_block, group - h0), s0, s1));
                            list.push_back(make_int4(r, b.runs, b.slot, b.position));
                            load.push_back(s1 - s0 + kRunCost[kind]);
                            sum += at_once ? 1 : load.back();
                            if (load.size() > kMaxWorkgroups / 2) throw std::invalid_argument("attention batch too large");
                        }
            at = to;
        }
        std::vector<std::vector<size_t>> lists(xcds);
        size_t done = 0, longest = 0;
        for (size_t k = 0; k < load.size(); ++k) {
            lists[std::min<size_t>(xcds - 1, done * xcds / std::max<size_t>(sum, 1))].push_back(k);
            done += at_once ? 1 : load[k];
        }
        for (auto& l : lists) {
            std::stable_sort(l.begin(), l.end(), [&](size_t x, size_t y) { return load[x] > load[y]; });
            longest = std::max(longest, l.size());
        }
        work[kind].assign(3 * longest * xcds, make_int4(0, 0, 0, 0));  // (padding has no rows)
        for (int x = 0; x < xcds; ++x)
            for (size_t k = 0; k < lists[x].size(); ++k)
                std::copy_n(&list[3 * lists[x][k]], 3, &work[kind][3 * (k * xcds + x)]);
        if (work[kind].size() > 3 * kMaxWorkgroups) throw std::invalid_argument("attention batch too large");
    }
    few = tiles ? static_cast<int>(work[0].size() / 3) : 0;
    many = static_cast<int>(work[1].size() / 3);
    items = tiles ? 0 : static_cast<int>(work[0].size() / 3);

    std::vector<PlanRegion::Section> s = {
        {tab.data(), tab.size() * sizeof(int32_t)},  {ranges.data(), rows * sizeof(int2)},
        {runs.data(), rows * sizeof(int2)},          {bias.data(), bias.size() * sizeof(float)},
        {work[0].data(), work[0].size() * sizeof(int4)}, {work[1].data(), work[1].size() * sizeof(int4)},
        {nullptr, slots * h * g.head_dim * sizeof(float)}, {nullptr, slots * h * 2 * sizeof(float)},
    };
    region.place(*c, s);
    size_t* at[] = {&tables_at, &ranges_at, &runs_at, &slopes_at, &few_at, &many_at, &acc_at, &ml_at};
    for (size_t i = 0; i < s.size(); ++i) *at[i] = s[i].at;
}

void ScorePlan::launch(int layer, const float* q, float* out, hipStream_t s) {
    if (cache->epoch() != epoch) throw std::invalid_argument("score plan is stale: the cache changed");
    if (layer < 0 || static_cast<size_t>(layer) >= cache->geometry().layers)
        throw std::invalid_argument("invalid fused attention shape");
    if (!rows) return;
    cache->check_device();
    cache->enter(s);
    char* d = region.device();
    ScoreArgs a{};
    a.pool = cache->pool();
    a.lay = cache->layout();
    a.layer = layer;
    a.heads = heads;
    a.group = group;
    a.tables = reinterpret_cast<const int32_t*>(d + tables_at);
    a.ranges = reinterpret_cast<const int2*>(d + ranges_at);
    a.runs = reinterpret_cast<const int2*>(d + runs_at);
    a.rows = static_cast<int>(rows);
    a.q = q;
    a.out = out;
    a.part_acc = reinterpret_cast<float*>(d + acc_at);
    a.part_ml = reinterpret_cast<float*>(d + ml_at);
    a.qscale = qscale;
    a.cap = cap;
    a.slopes = biased ? reinterpret_cast<const float*>(d + slopes_at) : nullptr;
    a.err = region.flags();
    a.work = reinterpret_cast<const int4*>(d + few_at);
    if (items) launch_score_rows(a, items, s);
    if (few) launch_score_tiles(a, kScoreFew, few, s);
    a.work = reinterpret_cast<const int4*>(d + many_at);
    if (many) launch_score_tiles(a, kScoreMany, many, s);
    if (slots) launch_score_merge(a, s);
    cache->leave(s);
    region.launched(s);
}

void ScorePlan::check() {
    if (region.check()) throw std::invalid_argument("invalid online attention input");
}

}  // namespace tvara_amd

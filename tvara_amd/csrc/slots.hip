// Slot maps and block tables from a batch's lengths, and the write of K/V rows
// through them.  Token j of sequence i has position start_i + j and slot
// block * tokens_per_block + position % tokens_per_block, where block is the
// id of block position / tokens_per_block of the sequence.
#include <algorithm>

#include "common.hpp"
#include "q8.hpp"
#include "tree.hpp"

namespace tvara_amd {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ long long block_sum(long long v, long long* part) {
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    long long sum = 0;
    for (int w = 0; w < kThreads / 64; ++w) sum += part[w];
    return sum;
}

// grid.x: sequence, the last: what lies behind the sequences; grid.y: a share of
// its tokens and of its table.  Bound: the chain of dependent loads (the counts
// before, the ids), so a thread has about one token and one table entry, and what
// does not depend on the sum is requested before it.  MI355X: 4.3 us for one sequence's
// five tokens, 5.6 us for 256 sequences with 88,619 (positions, slots and tables).
__global__ __launch_bounds__(kThreads) void slot_map_kernel(const SlotArgs a) {
    __shared__ long long part[kThreads / 64];
    const int i = blockIdx.x, tid = threadIdx.x;
    const int32_t* __restrict__ ids = a.ids;
    const size_t step = static_cast<size_t>(gridDim.y) * kThreads, t0 = static_cast<size_t>(blockIdx.y) * kThreads + tid;
    const bool behind = i == a.count;
    const int2 seq = behind ? make_int2(0, 0) : a.seqs[i];
    const int start = behind ? 0 : a.starts[i], count = behind ? 0 : a.counts[i];
    if (a.tables && !behind)
        for (size_t b = t0; b < a.width; b += step)
            a.tables[i * a.width + b] = b < static_cast<size_t>(seq.y) ? ids[seq.x + b] & 0x7fffffff : -1;
    // tokens of the sequences before this one
    long long before = 0;
    for (int k = tid; k < i; k += kThreads) before += max(a.counts[k], 0);
    before = block_sum(before, part);
    if (blockIdx.y == 0 && tid == 0 && a.offsets) a.offsets[i] = static_cast<int32_t>(min(before, 0x7fffffffll));
    auto fill = [&](size_t from, size_t to) {
        for (size_t t = from + t0; t < to; t += step) {
            if (a.positions) a.positions[t] = -1;
            if (a.slots) a.slots[t] = -1;
        }
    };
    if (behind) {
        fill(min(a.stride ? a.stride * a.count : static_cast<size_t>(before), a.capacity), a.capacity);
        return;
    }
    const size_t first = a.stride ? a.stride * i : static_cast<size_t>(before);
    const size_t room = first < a.capacity ? a.capacity - first : 0;
    const size_t n = min(static_cast<size_t>(max(count, 0)), a.stride ? a.stride : room);
    bool bad = count < 0 || n < static_cast<size_t>(max(count, 0));
    for (size_t j = t0; j < n; j += step) {
        const unsigned pos = static_cast<unsigned>(start) + static_cast<unsigned>(j);  // (negative ones wrap past every block)
        const unsigned b = pos / static_cast<unsigned>(a.tpb);
        const int id = b < static_cast<unsigned>(seq.y) ? ids[seq.x + b] : -1;
        bad |= id < 0;  // outside the sequence's blocks, or a shared one
        if (a.positions) a.positions[first + j] = static_cast<int32_t>(pos);
        if (a.slots) a.slots[first + j] = id < 0 ? -1 : static_cast<int64_t>(id) * a.tpb + (pos - b * a.tpb);
    }
    if (bad) *a.err = 1;
    if (a.stride) fill(first + n, first + a.stride);
}

// whether token t is written, and from which row into which block and slot
__device__ __forceinline__ bool placed(const WriteArgs& a, size_t t, size_t& row, int64_t& block, int& slot) {
    const int64_t to = a.slots[t];
    if (to < 0) return false;
    const int64_t r = a.rows ? a.rows[t] : static_cast<int64_t>(t);
    if (to >= a.slot_count || r < 0 || static_cast<size_t>(r) >= a.row_count) {
        *a.err = 1;
        return false;
    }
    row = static_cast<size_t>(r);
    block = to / a.lay.tpb;
    slot = static_cast<int>(to - block * a.lay.tpb);
    return true;
}

// grid.x: token, grid.y: a share of its rows of every (layer, kind).  Four floats a
// thread and turn, the turns' loads requested together; stores that nothing in the
// launch reads back pass the caches.  Bound: HBM.  MI355X, 229 rows of 16 layers of
// 2 x 512 floats: 6.9 us, 4.4 TB/s read and written.
constexpr int kTurns = 4, kTurnsQ8 = 1;

template <int kVec>
__global__ __launch_bounds__(kThreads) void slot_write_f32_kernel(const WriteArgs a) {
    typedef float vec __attribute__((ext_vector_type(kVec)));
    size_t row;
    int64_t block;
    int slot;
    if (!placed(a, blockIdx.x, row, block, slot)) return;
    const unsigned w = a.lay.kv_width / kVec, units = 2 * a.lay.layers * w;
    const unsigned u0 = blockIdx.y * (kTurns * kThreads) + threadIdx.x;
    char* base = a.pool + block * a.lay.stride;
    vec x[kTurns];
    unsigned to[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
        const unsigned u = min(u0 + k * kThreads, units - 1), r = u / w, c = u - r * w;  // r: layer * 2 + kind
        const float* src = ((r & 1) ? a.values : a.keys) + row * a.row_stride + (r >> 1) * a.layer_stride;
        x[k] = reinterpret_cast<const vec*>(src)[c];
        to[k] = (r * a.lay.tpb + slot) * w + c;
    }
#pragma unroll
    for (int k = 0; k < kTurns; ++k)
        if (u0 + k * kThreads < units) __builtin_nontemporal_store(x[k], reinterpret_cast<vec*>(base) + to[k]);
}

// The encoder of appends (q8_encode_element), four elements a lane: eight lanes
// share a group's maximum and scale.  Bound at these sizes: the chain slot, row,
// maximum, store (100 rows of 8 layers of 2 x 1024 floats, 8.3 MB: 6.8 us).
__global__ __launch_bounds__(kThreads) void slot_write_q8_kernel(const WriteArgs a) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    size_t row;
    int64_t block;
    int slot;
    if (!placed(a, blockIdx.x, row, block, slot)) return;
    const unsigned w = a.lay.kv_width / 4, units = 2 * a.lay.layers * w;  // (a multiple of 8 lanes)
    const unsigned u0 = blockIdx.y * (kTurnsQ8 * kThreads) + threadIdx.x;
    char* base = a.pool + block * a.lay.stride;
    f32x4 x[kTurnsQ8];
#pragma unroll
    for (int k = 0; k < kTurnsQ8; ++k) {
        const unsigned u = min(u0 + k * kThreads, units - 1), r = u / w, c = u - r * w;
        const float* src = ((r & 1) ? a.values : a.keys) + row * a.row_stride + (r >> 1) * a.layer_stride;
        x[k] = *reinterpret_cast<const f32x4*>(src + 4 * c);
    }
#pragma unroll
    for (int k = 0; k < kTurnsQ8; ++k) {
        const unsigned u = min(u0 + k * kThreads, units - 1), r = u / w, c = u - r * w;
        float amax = fmaxf(fmaxf(fabsf(x[k][0]), fabsf(x[k][1])), fmaxf(fabsf(x[k][2]), fabsf(x[k][3])));
        for (int m = 4; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 8));
        uint16_t d;
        int8_t q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q8_encode_element(x[k][e], amax, &d, &q[e]);
        if (u0 + k * kThreads >= units) continue;
        char* sec = base + static_cast<size_t>(r) * a.lay.section;
        const uint32_t four = static_cast<uint8_t>(q[0]) | static_cast<uint8_t>(q[1]) << 8 | static_cast<uint8_t>(q[2]) << 16 |
                              static_cast<uint32_t>(static_cast<uint8_t>(q[3])) << 24;
        *reinterpret_cast<uint32_t*>(sec + q8_byte_offset(a.lay, slot, 4 * c)) = four;
        if (c % 8 == 0) *reinterpret_cast<uint16_t*>(sec + q8_scale_offset(a.lay, slot, c / 8)) = d;
    }
}

}  // namespace

void launch_slot_map(const SlotArgs& a, hipStream_t s) {
    const size_t each = std::max(a.capacity, a.width * a.count) / a.count;
    const unsigned shares = static_cast<unsigned>(std::clamp<size_t>((each + kThreads / 2 - 1) / (kThreads / 2), 1, 64));
    launch("slot_map", slot_map_kernel, dim3(a.count + 1, shares), dim3(kThreads), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

void launch_slot_write(const WriteArgs& a, hipStream_t s) {
    const bool wide = a.lay.format == kQ8 || (a.lay.kv_width % 4 == 0 && a.row_stride % 4 == 0 && a.layer_stride % 4 == 0);
    const size_t units = static_cast<size_t>(2) * a.lay.layers * a.lay.kv_width / (wide ? 4 : 1);
    const size_t share = static_cast<size_t>(a.lay.format == kQ8 ? kTurnsQ8 : kTurns) * kThreads;
    const dim3 grid(static_cast<unsigned>(a.n), static_cast<unsigned>((units + share - 1) / share));
    launch("slot_write",
           a.lay.format == kQ8 ? slot_write_q8_kernel : wide ? slot_write_f32_kernel<4> : slot_write_f32_kernel<1>, grid,
           dim3(kThreads), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

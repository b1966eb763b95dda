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

// grid.x: sequence, the last: what lies behind the sequences; grid.y: a share
// of its tokens and of its table.
__global__ __launch_bounds__(kThreads) void slot_map_kernel(const SlotArgs a) {
    __shared__ long long part[kThreads / 64];
    const int i = blockIdx.x, tid = threadIdx.x;
    // tokens of the sequences before this one
    long long before = 0;
    for (int k = tid; k < i; k += kThreads) before += max(a.counts[k], 0);
    before = block_sum(before, part);
    const size_t step = static_cast<size_t>(gridDim.y) * kThreads, t0 = static_cast<size_t>(blockIdx.y) * kThreads + tid;
    if (blockIdx.y == 0 && tid == 0 && a.offsets) a.offsets[i] = static_cast<int32_t>(min(before, 0x7fffffffll));
    auto fill = [&](size_t from, size_t to) {
        for (size_t t = from + t0; t < to; t += step) {
            if (a.positions) a.positions[t] = -1;
            if (a.slots) a.slots[t] = -1;
        }
    };
    if (i == a.count) {
        fill(min(a.stride ? a.stride * a.count : static_cast<size_t>(before), a.capacity), a.capacity);
        return;
    }
    const int2 seq = a.seqs[i];
    const int start = a.starts[i], count = a.counts[i];
    const size_t first = a.stride ? a.stride * i : static_cast<size_t>(before);
    const size_t room = first < a.capacity ? a.capacity - first : 0;
    const size_t n = min(static_cast<size_t>(max(count, 0)), a.stride ? a.stride : room);
    bool bad = count < 0 || n < static_cast<size_t>(max(count, 0));
    for (size_t j = t0; j < n; j += step) {
        const long long pos = static_cast<long long>(start) + static_cast<long long>(j);
        const long long b = pos / a.tpb;
        const int id = pos >= 0 && b < seq.y ? a.ids[seq.x + b] : -1;
        bad |= id < 0;  // outside the sequence's blocks, or a shared one
        if (a.positions) a.positions[first + j] = static_cast<int32_t>(pos);
        if (a.slots) a.slots[first + j] = id < 0 ? -1 : static_cast<int64_t>(id) * a.tpb + pos % a.tpb;
    }
    if (bad) *a.err = 1;
    if (a.stride) fill(first + n, first + a.stride);
    if (a.tables)
        for (size_t b = t0; b < a.width; b += step)
            a.tables[i * a.width + b] = b < static_cast<size_t>(seq.y) ? a.ids[seq.x + b] & 0x7fffffff : -1;
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

// grid.x: token, grid.y: layer * 2 + kind
__global__ __launch_bounds__(kThreads) void slot_write_f32_kernel(const WriteArgs a) {
    size_t row;
    int64_t block;
    int slot;
    if (!placed(a, blockIdx.x, row, block, slot)) return;
    const int layer = blockIdx.y >> 1, w = a.lay.kv_width;
    const float* src = ((blockIdx.y & 1) ? a.values : a.keys) + row * a.row_stride + layer * a.layer_stride;
    float* dst = reinterpret_cast<float*>(a.pool + block * a.lay.stride) +
                 (static_cast<size_t>(blockIdx.y) * a.lay.tpb + slot) * w;
    for (int c = threadIdx.x; c < w; c += kThreads) dst[c] = src[c];
}

__global__ __launch_bounds__(kThreads) void slot_write_q8_kernel(const WriteArgs a) {
    size_t row;
    int64_t block;
    int slot;
    if (!placed(a, blockIdx.x, row, block, slot)) return;
    const int layer = blockIdx.y >> 1, l32 = threadIdx.x & 31;
    const float* src = ((blockIdx.y & 1) ? a.values : a.keys) + row * a.row_stride + layer * a.layer_stride;
    char* sec = a.pool + block * a.lay.stride + static_cast<size_t>(blockIdx.y) * a.lay.section;
    for (int g = threadIdx.x >> 5; g < a.lay.kv_width / 32; g += kThreads / 32) {
        const float x = src[g * 32 + l32];
        float amax = fabsf(x);
        for (int m = 16; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 32));
        uint16_t d;
        int8_t q;
        q8_encode_element(x, amax, &d, &q);
        reinterpret_cast<int8_t*>(sec)[q8_byte_offset(a.lay, slot, g * 32 + l32)] = q;
        if (l32 == 0) *reinterpret_cast<uint16_t*>(sec + q8_scale_offset(a.lay, slot, g)) = d;
    }
}

}  // namespace

void launch_slot_map(const SlotArgs& a, hipStream_t s) {
    const size_t each = std::max(a.capacity, a.width * a.count) / a.count;
    const unsigned shares = static_cast<unsigned>(std::clamp<size_t>(each / (4 * kThreads), 1, 64));
    launch("slot_map", slot_map_kernel, dim3(a.count + 1, shares), dim3(kThreads), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

void launch_slot_write(const WriteArgs& a, hipStream_t s) {
    launch("slot_write", a.lay.format == kF32 ? slot_write_f32_kernel : slot_write_q8_kernel,
           dim3(static_cast<unsigned>(a.n), a.lay.layers * 2), dim3(kThreads), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

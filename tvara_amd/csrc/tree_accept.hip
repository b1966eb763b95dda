// Greedy acceptance of token trees: which drafted nodes the model's own greedy
// choices confirm.  Per tree, e = first; while a child of the current node (a
// root at the start) has token e, the lowest such child is accepted and
// e = argmax(its logits), the lowest index on ties; next = e at the end.
#include <algorithm>

#include "common.hpp"
#include "tree.hpp"

namespace tvara_amd {
namespace {

// A logit's place in the order, above its index's complement: the maximum of
// these is the lowest index of the largest logit.  NaN is below every number.
__device__ __forceinline__ uint64_t ranked(float x, uint32_t index) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == 0.f ? 0.f : x);  // (-0 ties with 0)
    const uint32_t order = x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return static_cast<uint64_t>(order) << 32 | ~index;
}

// a workgroup per (row, part of its vocabulary): the part's best
__global__ __launch_bounds__(256) void tree_argmax_kernel(const AcceptArgs a) {
    __shared__ uint64_t part[4];
    const size_t row = blockIdx.x;
    const size_t per = (a.vocab + a.splits - 1) / a.splits, lo = blockIdx.y * per;
    const size_t hi = min(lo + per, a.vocab);
    const float* x = a.logits + row * a.logits_stride;
    uint64_t best = 0;
    bool bad = false;
    for (size_t i = lo + threadIdx.x; i < hi; i += 256) {
        const float v = x[i];
        bad |= v != v;
        best = max(best, ranked(v, static_cast<uint32_t>(i)));
    }
    if (bad) *a.err = 1;
    for (int m = 32; m >= 1; m >>= 1) best = max(best, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(best), m)));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0) a.best[row * a.splits + blockIdx.y] = max(max(part[0], part[1]), max(part[2], part[3]));
}

// a wave per tree walks it: 64 nodes are looked at together
__global__ __launch_bounds__(64) void tree_walk_kernel(const AcceptArgs a) {
    const int lane = threadIdx.x, tree = blockIdx.x;
    const int4 t = a.trees[tree];
    uint32_t want = a.first[tree];
    int at = -1, count = 0;
    int32_t* path = a.path + static_cast<size_t>(tree) * a.path_stride;
    for (;;) {
        int found = -1;
        for (int base = max(at, 0); base < t.z; base += 64) {  // children follow their parents
            const int j = base + lane;
            const bool hit = j < t.z && a.parents[t.w + j] == at && a.tokens[t.w + j] == want;
            const uint64_t hits = __ballot(hit);
            if (hits) {
                found = base + __builtin_ctzll(hits);
                break;
            }
        }
        if (found < 0) break;
        if (static_cast<size_t>(count) >= a.path_stride) {  // no room for it
            if (lane == 0) *a.err = 1;
            break;
        }
        const size_t row = static_cast<size_t>(t.w) + found;
        if (lane == 0) path[count] = static_cast<int32_t>(row);
        ++count;
        at = found;
        uint64_t best = 0;
        for (int s = lane; s < a.splits; s += 64) best = max(best, a.best[row * a.splits + s]);
        for (int m = 32; m >= 1; m >>= 1) best = max(best, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(best), m)));
        want = ~static_cast<uint32_t>(best);
    }
    for (size_t i = static_cast<size_t>(count) + lane; i < a.path_stride; i += 64) path[i] = -1;
    if (lane == 0) {
        a.accepted[tree] = count;
        a.next[tree] = want;
    }
}

}  // namespace

// about kAcceptParts workgroups, of 2,048 logits or more each
int tree_accept_splits(size_t rows, size_t vocab) {
    if (!rows) return 1;
    const size_t most = std::max<size_t>(1, vocab / 2048);
    return static_cast<int>(std::min(most, std::max<size_t>(1, kAcceptParts / rows)));
}

void launch_tree_accept(const AcceptArgs& a, hipStream_t s) {
    if (a.rows)
        launch("tree_argmax", tree_argmax_kernel, dim3(a.rows, a.splits), dim3(256), 0, s, a);
    launch("tree_walk", tree_walk_kernel, dim3(a.count), dim3(64), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

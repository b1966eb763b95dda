// Greedy acceptance of token trees: which drafted nodes the model's own greedy
// choices confirm.  Per tree, e = first; while a child of the current node (a
// root at the start) has token e, the lowest such child is accepted and
// e = argmax(its logits), the lowest index on ties; next = e at the end.
//
// Which rows are needed is known only on the way, so every row's argmax is taken,
// in parts of a workgroup each, and a workgroup then walks a tree.  Bound: one read
// of the logits.  A launch of few parts ends with the walk in the last workgroup of
// a tree (one launch); larger ones take a second launch, since the last arriver's
// release writes its XCD's L2 back, one workgroup after the other.  MI355X, 32 trees
// (503 nodes) over 128,256 tokens: 45.4 us, 5.7 TB/s, of which the walk is 4.6.
#include <algorithm>

#include "common.hpp"
#include "tree.hpp"

namespace tvara_amd {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr size_t kFusedParts = 128;

// A logit's place in the order, above its index's complement: the maximum of
// these is the lowest index of the largest logit.
__device__ __forceinline__ uint64_t ranked(float x, uint32_t index) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == 0.f ? 0.f : x);  // (-0 ties with 0)
    const uint32_t order = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return static_cast<uint64_t>(order) << 32 | ~index;
}

__device__ __forceinline__ uint64_t wave_max(uint64_t v, int width) {
    for (int m = width / 2; m >= 1; m >>= 1) v = max(v, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(v), m)));
    return v;
}

// A tree walked by the workgroup: its nodes' parents, tokens and choices come
// into LDS at once, then the first wave looks at 64 nodes together.
__device__ __forceinline__ void walk(const AcceptArgs& a, int tree) {
    __shared__ int32_t parent[kMaxTreeNodes];
    __shared__ uint32_t token[kMaxTreeNodes], choice[kMaxTreeNodes];
    __shared__ int length;
    const int tid = threadIdx.x, lane = tid & 63;
    const int4 t = a.trees[tree];
    uint32_t want = a.first[tree];
    for (int j = tid; j < t.z; j += kThreads) {
        parent[j] = a.parents[t.w + j];
        token[j] = a.tokens[t.w + j];
    }
    for (int j = tid / 16; j < t.z; j += kThreads / 16) {  // 16 lanes a node
        const uint64_t* parts = a.best + (static_cast<size_t>(t.w) + j) * a.splits;
        uint64_t best = 0;
        for (int s = tid & 15; s < a.splits; s += 16)
            best = max(best, __hip_atomic_load(parts + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        best = wave_max(best, 16);
        // (a row of NaN has no choice: its lowest index)
        if ((tid & 15) == 0) choice[j] = best ? ~static_cast<uint32_t>(best) : 0u;
    }
    __syncthreads();
    int32_t* path = a.path + static_cast<size_t>(tree) * a.path_stride;
    if (tid < 64) {
        int at = -1, count = 0;
        for (;;) {
            int found = -1;
            for (int base = at + 1; base < t.z; base += 64) {  // children follow their parents
                const int j = base + lane;
                const uint64_t hits = __ballot(j < t.z && parent[min(j, t.z - 1)] == at && token[min(j, t.z - 1)] == want);
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
            if (lane == 0) path[count] = t.w + found;
            ++count;
            at = found;
            want = choice[found];
        }
        if (lane == 0) {
            length = count;
            a.accepted[tree] = count;
            a.next[tree] = want;
        }
    }
    __syncthreads();
    for (size_t i = static_cast<size_t>(length) + tid; i < a.path_stride; i += kThreads) path[i] = -1;
}

// The best of a part of a row.  A thread keeps the first of its largest values: it
// goes up through its indexes, so a later one has to be larger.  Eight 16-byte loads
// of a thread are in flight.
template <bool kWide>
__global__ __launch_bounds__(kThreads) void tree_argmax_kernel(const AcceptArgs a) {
    __shared__ uint64_t part[kThreads / 64];
    __shared__ bool last;
    const int tid = threadIdx.x;
    const size_t row = blockIdx.x / static_cast<unsigned>(a.splits), split = blockIdx.x % static_cast<unsigned>(a.splits);
    const uint32_t lo = static_cast<uint32_t>(split * a.part), hi = static_cast<uint32_t>(min(a.vocab, (split + 1) * a.part));
    const float* x = a.logits + row * a.logits_stride;
    float top = -INFINITY, seen = 0.f;
    uint32_t where = 0xffffffffu;
    auto take = [&](float v, uint32_t i) {
        const bool more = v > top || (where == 0xffffffffu && v == v);
        top = more ? v : top;
        where = more ? i : where;
        seen = v != v ? v : seen;
    };
    uint32_t i = lo;
    if constexpr (kWide) {  // (lo and the row start on 16 bytes)
        constexpr int U = 8;
        for (; i + U * kThreads * 4 <= hi; i += U * kThreads * 4) {
            f32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(x + i + 4 * (u * kThreads + tid)));
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) take(v[u][e], i + 4 * (u * kThreads + tid) + e);
        }
        for (; i + kThreads * 4 <= hi; i += kThreads * 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(x + i + 4 * tid);
#pragma unroll
            for (int e = 0; e < 4; ++e) take(v[e], i + 4 * tid + e);
        }
    }
    for (i += tid; i < hi; i += kThreads) take(x[i], i);
    if (seen != seen) *a.err = 1;
    uint64_t best = where == 0xffffffffu ? 0 : ranked(top, where);
    best = wave_max(best, 64);
    if ((tid & 63) == 0) part[tid >> 6] = best;
    __syncthreads();
    if (tid == 0)
        __hip_atomic_store(a.best + blockIdx.x, max(max(part[0], part[1]), max(part[2], part[3])), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    if (!a.done) return;
    const int tree = a.tree_of[row];
    if (tid == 0) {
        const int all = a.trees[tree].z * a.splits;
        const int before = __hip_atomic_fetch_add(a.done + tree, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        last = before == all - 1;
        if (last) __hip_atomic_store(a.done + tree, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (last) walk(a, tree);
}

__global__ __launch_bounds__(kThreads) void tree_walk_kernel(const AcceptArgs a) { walk(a, blockIdx.x); }

}  // namespace

// About kAcceptParts parts in all, of 1,024 logits or more and a multiple of them;
// of at most kFusedParts where they are 32 KiB each at most (MI355X, one tree of
// eight over 32,000: two launches 8.25 us, one in few parts 7.34).
void tree_accept_parts(AcceptArgs& a) {
    const size_t rows = std::max(a.rows, 1), all = rows * a.vocab;
    auto part = [&](size_t parts) { return std::max<size_t>(1, (all / parts + 1023) / 1024) * 1024; };
    a.part = part(kAcceptParts);
    if (!a.every_tree_has_nodes || rows * ((a.vocab + part(kFusedParts / 2) - 1) / part(kFusedParts / 2)) > kFusedParts ||
        part(kFusedParts / 2) > 8192)
        a.done = nullptr;
    else
        a.part = part(kFusedParts / 2);
    a.splits = static_cast<int>((a.vocab + a.part - 1) / a.part);
}

void launch_tree_accept(const AcceptArgs& a, hipStream_t s) {
    if (a.rows)
        launch("tree_argmax", a.logits_stride % 4 ? tree_argmax_kernel<false> : tree_argmax_kernel<true>,
               dim3(static_cast<unsigned>(a.rows) * static_cast<unsigned>(a.splits)), dim3(kThreads), 0, s, a);
    if (!a.done) launch("tree_walk", tree_walk_kernel, dim3(a.count), dim3(kThreads), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

// Attention of token trees over the paged cache: row r of a tree attends to
// the sequence's cached tokens, the nodes above it and itself,
//   o = sum_k p_k v_k,  p = softmax_k(q . k / sqrt(d)),
// with the nodes' K/V in rows of their own, outside the cache (they join it only
// when they are accepted).
#include <algorithm>

#include "common.hpp"
#include "device_util.hpp"
#include "q8.hpp"
#include "tree.hpp"

namespace tvara_amd {
namespace {

constexpr int kMaxDim = 512;
// Groups of a row's runs where the rows alone leave CUs idle.  MI355X, one context of
// 32,400 tokens with 5 nodes (10 workgroups, 64 runs): the whole call 32.1 us without
// and 22.1 with; 86 nodes of 32 heads of 128 (344 workgroups, 16 runs): 8.5 and 9.0.
constexpr int kMergeGroups = 8;
constexpr size_t kMergeFew = 256;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// element `column` of a cached K (kind 0) or V row
__device__ __forceinline__ float cached_element(const TreeArgs& a, int block, int kind, int slot, int column) {
    const char* base = a.pool + static_cast<size_t>(block) * a.lay.stride;
    const size_t sec = static_cast<size_t>(a.layer) * 2 + kind;
    if (a.lay.format == kF32)
        return reinterpret_cast<const float*>(base)[(sec * a.lay.tpb + slot) * a.lay.kv_width + column];
    const char* s = base + sec * a.lay.section;
    const int8_t q = reinterpret_cast<const int8_t*>(s)[q8_byte_offset(a.lay, slot, column)];
    return half_bits_to_float(*reinterpret_cast<const uint16_t*>(s + q8_scale_offset(a.lay, slot, column / 32))) *
           static_cast<float>(q);
}

// Any head_dim and block size, f32 arithmetic: a wave per (run of a node's
// cached tokens, query head); lanes are keys for the scores and columns for the
// output.  A work item is x: tree, y: node, z: run, w: runs; the last run takes
// the tree's nodes.  For the layouts that the matrix cores' tiles do not take; bound
// by loads of single elements, every row for itself.
__global__ __launch_bounds__(64) void tree_rows_kernel(const TreeArgs a) {
    __shared__ float qs[kMaxDim];
    const int lane = threadIdx.x, h = blockIdx.y, kh = h / a.group;
    const int D = a.lay.head_dim, tpb = a.lay.tpb;
    const int4 it = a.work[blockIdx.x], tree = a.trees[it.x];
    const size_t row = static_cast<size_t>(tree.w) + it.y;
    const int k0 = it.z * a.split_tokens, k1 = it.z + 1 == it.w ? tree.y : k0 + a.split_tokens;
    const int cached = k1 - k0, keys = cached + (it.z + 1 == it.w ? it.y + 1 : 0);
    const int32_t* tab = a.tables + tree.x;
    const uint32_t* mask = a.mask + row * a.words;
    const float* qr = a.q + (row * a.heads + h) * D;
    for (int d = lane; d < D; d += 64) qs[d] = qr[d] * a.qscale;
    __syncthreads();
    auto node_row = [&](const float* rows, int node) {
        return rows + (static_cast<size_t>(tree.w) + node) * a.row_stride + static_cast<size_t>(kh) * D;
    };
    auto seen = [&](int j) {
        if (j >= keys) return false;
        const int node = j - cached;
        return node < 0 || (mask[node >> 5] >> (node & 31) & 1);
    };
    // A batch of 64 keys is added up by itself and then joins the rest, the normaliser
    // with what its additions have rounded away (one key 21 above 32,768 of N(0,1): 1.7e-5
    // of every output key by key, 1e-6 so; the same time).
    float m = -INFINITY, l = 0.f, rounded = 0.f, acc[kMaxDim / 64];
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) acc[i] = 0.f;
    bool bad = false;
    for (int base = 0; base < keys; base += 64) {
        const int j = base + lane;
        const bool ok = seen(j);
        float s = -INFINITY;
        if (ok) {
            s = 0.f;
            if (j < cached) {
                const int p = k0 + j, block = tab[p / tpb], slot = p % tpb;
                for (int d = 0; d < D; ++d) s = fmaf(qs[d], cached_element(a, block, 0, slot, kh * D + d), s);
            } else {
                const float* k = node_row(a.keys, j - cached);
                for (int d = 0; d < D; ++d) s = fmaf(qs[d], k[d], s);
            }
            bad |= !__builtin_isfinite(s);
        }
        float mx = s;
        for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        const float mnew = fmaxf(m, mx);
        if (mnew == -INFINITY) continue;  // no key seen yet
        const float alpha = fast_exp2(m - mnew), pj = ok ? fast_exp2(s - mnew) : 0.f;
        float ps = pj;
        for (int o = 32; o >= 1; o >>= 1) ps += __shfl_xor(ps, o);
        const float y = ps - rounded * alpha, before = l * alpha;
        l = before + y;
        rounded = (l - before) - y;
        m = mnew;
        float part[kMaxDim / 64];
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i) part[i] = 0.f;
        uint64_t left = __ballot(ok);  // values of keys that are not seen are not read
        while (left) {
            const int jj = __builtin_ctzll(left);
            left &= left - 1;
            const float w = __shfl(pj, jj);
            const int p = k0 + base + jj;
            const float* v = base + jj < cached ? nullptr : node_row(a.values, base + jj - cached);
            const int block = v ? 0 : tab[p / tpb], slot = p % tpb;
#pragma unroll
            for (int i = 0; i < kMaxDim / 64; ++i) {
                const int d = i * 64 + lane;
                if (d < D) part[i] = fmaf(w, v ? v[d] : cached_element(a, block, 1, slot, kh * D + d), part[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i) acc[i] = fmaf(acc[i], alpha, part[i]);
    }
    if (__any(bad) && lane == 0) *a.err = 1;
    const bool whole = it.w == 1;
    const size_t at = whole ? row * a.heads + h : (static_cast<size_t>(a.runs[row].x) + it.z) * a.heads + h;
    float* o = (whole ? a.out : a.part_acc) + at * D;
    const float inv = whole ? l : 1.f;
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) {
        const int d = i * 64 + lane;
        if (d < D) o[d] = acc[i] / inv;
    }
    if (!whole && lane == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(m, l);
}

// A row's runs combined: a thread per four columns (two where head_dim is no
// multiple of four) and per `groups` runs, the loads of four of its runs in flight;
// the groups meet in LDS, in order.  Bound: the memory behind the L2s, which the
// partials come from (86 nodes of 32 heads of 128, 16 runs: 8.5 us, 2.8 TB/s; 512
// nodes, 4 runs: 9.1 us, 4.6 TB/s).
template <int kVec, bool kGroups>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeArgs a, int groups) {
    typedef float vec __attribute__((ext_vector_type(kVec)));
    __shared__ float2 stats[kGroups ? 256 : 1];
    __shared__ vec sums[kGroups ? 256 : 1];
    const int D = a.lay.head_dim, parts = D / kVec, unit = parts * groups, each = 256 / unit;
    const int tid = threadIdx.x, mine = tid / unit, group = tid % unit / parts;
    const size_t at = static_cast<size_t>(blockIdx.x) * each + mine;
    const bool in = mine < each && at < static_cast<size_t>(a.rows) * a.heads;
    const int2 runs = in ? a.runs[at / a.heads] : make_int2(0, 1);
    const int c = kVec * (tid % parts), h = static_cast<int>(at % a.heads);
    constexpr int kTogether = 4;
    float m = -INFINITY, l = 0.f;
    vec sum = 0.f;
    auto add = [&](float2 ml, vec x) __attribute__((always_inline)) {
        if (ml.x == -INFINITY) return;
        const float mn = fmaxf(m, ml.x), wm = fast_exp2(m - mn), wr = fast_exp2(ml.x - mn);
        l = l * wm + ml.y * wr;
        sum = sum * wm + x * wr;
        m = mn;
    };
    if (runs.y > 1)
        for (int r0 = group; r0 < runs.y; r0 += kTogether * groups) {
            float2 ml[kTogether];
            vec x[kTogether];
#pragma unroll
            for (int r = 0; r < kTogether; ++r) {
                const size_t p = (static_cast<size_t>(runs.x) + min(r0 + r * groups, runs.y - 1)) * a.heads + h;
                ml[r] = *reinterpret_cast<const float2*>(a.part_ml + 2 * p);
                x[r] = *reinterpret_cast<const vec*>(a.part_acc + p * D + c);
            }
#pragma unroll
            for (int r = 0; r < kTogether; ++r)
                if (r0 + r * groups < runs.y) add(ml[r], x[r]);
        }
    if constexpr (kGroups) {
        stats[tid] = make_float2(m, l);
        sums[tid] = sum;
        __syncthreads();
        if (group || !in) return;
        for (int g = 1; g < groups; ++g) add(stats[tid + g * parts], sums[tid + g * parts]);
    }
    if (runs.y == 1) return;  // (written by the attention itself, or no row)
    const vec o = sum / l;
    bool finite = true;
#pragma unroll
    for (int e = 0; e < kVec; ++e) finite &= __builtin_isfinite(o[e]);
    if (a.check && !finite) *a.err = 1;
    *reinterpret_cast<vec*>(a.out + at * D + c) = o;
}

}  // namespace

void launch_tree_rows(const TreeArgs& a, int items, hipStream_t s) {
    if (a.lay.head_dim > kMaxDim) throw std::invalid_argument("head_dim above 512 is not supported");
    launch("tree_attention", tree_rows_kernel, dim3(items, a.heads), dim3(64), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

void launch_tree_merge(const TreeArgs& a, int most_runs, hipStream_t s) {
    const int vec = a.lay.head_dim % 4 ? 2 : 4, parts = a.lay.head_dim / vec;
    auto workgroups = [&](int groups) {
        const size_t each = 256 / (parts * groups);
        return (static_cast<size_t>(a.rows) * a.heads + each - 1) / each;
    };
    const int groups = workgroups(1) < kMergeFew ? std::max(1, std::min({(most_runs + 3) / 4, 256 / parts, kMergeGroups})) : 1;
    const size_t blocks = workgroups(groups);
    auto go = [&](auto kernel) {
        launch("tree_attention_merge", kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a, groups);
    };
    if (vec == 4)
        groups > 1 ? go(tree_merge_kernel<4, true>) : go(tree_merge_kernel<4, false>);
    else
        groups > 1 ? go(tree_merge_kernel<2, true>) : go(tree_merge_kernel<2, false>);
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

// Scored attention over the paged cache: row r of position p and query head h has
//   s_k = scale q . k,  s_k = cap tanh(s_k / cap) if there is a cap,
//   s_k -= slope_h |p - k|,  o = sum_k softmax(s)_k v_k  over first_r <= k < end_r,
// zeros where it sees no key.  Here: the kernel of any layout, and the merge of
// rows whose keys were cut into runs; the matrix cores' tiles are in score_tiles.hip.
#include <algorithm>

#include "score_util.hpp"

namespace tvara_amd {
namespace {

constexpr int kMaxDim = 512;

// Any head_dim and block size, f32 arithmetic: a wave per (run of a row's keys, query
// head); lanes are keys for the scores, which read their rows four columns at a time where
// rows are aligned, and kColumns columns each for the output.  For the layouts that the
// tiles do not take; bound by its loads, every row and head for itself: eight contexts of
// 2,000, 32 heads on 8 of 80 51 us (201 by single elements, a value at a time), 16 on 4 of 256 57
// (217), and 100 rows of each of two contexts of 1,000 496 (2,749).
template <int kColumns, bool kQ8>
__global__ __launch_bounds__(64) void score_rows_kernel(const ScoreArgs a) {
    constexpr int kTogether = kColumns < 4 ? 8 : 16 / kColumns;
    __shared__ __attribute__((aligned(16))) float qs[kMaxDim];
    const int lane = threadIdx.x, h = blockIdx.y, kh = h / a.group;
    const int D = a.lay.head_dim, tpb = a.lay.tpb, groups = D / 32;
    const bool aligned = kQ8 || D % 4 == 0;  // (Q8_0: rows of whole groups, heads at multiples of 16 bytes)
    const int4* w = a.work + 3 * static_cast<size_t>(blockIdx.x);
    const int4 seq = w[0], part = w[1], run = w[2];
    const int32_t* tab = a.tables + seq.x;
    const size_t row = seq.w;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    for (int d = lane; d < D; d += 64) qs[d] = a.q[(row * a.heads + h) * D + d] * a.qscale;
    __syncthreads();
    // a KV head's keys of the layer in a block, its values behind them, the bytes of a slot;
    // of Q8_0 the scales lie behind a block's bytes
    const size_t section = kQ8 ? a.lay.section : static_cast<size_t>(tpb) * a.lay.kv_width * 4;
    const size_t pitch = kQ8 ? D : 4 * static_cast<size_t>(a.lay.kv_width);
    const char* heads = a.pool + static_cast<size_t>(a.layer) * 2 * section + kh * (kQ8 ? a.lay.head_bytes : static_cast<size_t>(D) * 4);
    auto scale_of = [&](const char* head, int slot, int group) {
        return half_bits_to_float(*reinterpret_cast<const uint16_t*>(head + static_cast<size_t>(tpb) * D + (static_cast<size_t>(slot) * groups + group) * 2));
    };
    auto element = [&](const char* head, const char* at, int slot, int d) {
        if constexpr (kQ8) return scale_of(head, slot, d / 32) * static_cast<float>(reinterpret_cast<const int8_t*>(at)[d]);
        else return reinterpret_cast<const float*>(at)[d];
    };
    // A batch of 64 keys is added up by itself and then joins the rest, with what the
    // additions before have rounded away.
    float m = -INFINITY, l = 0.f, rounded = 0.f, acc[kColumns], rest[kColumns];
#pragma unroll
    for (int i = 0; i < kColumns; ++i) acc[i] = rest[i] = 0.f;
    bool bad = false;
    for (int base = part.z; base < part.w; base += 64) {
        const int key = base + lane;
        const bool ok = key < part.w;  // (a run lies within the row's range)
        float s = -INFINITY;
        int block = 0, slot = 0;
        if (ok) {
            s = 0.f;
            block = tab[key / tpb];
            slot = key % tpb;
            const char* head = heads + static_cast<size_t>(block) * a.lay.stride;
            const char* k = head + static_cast<size_t>(slot) * pitch;
            auto four = [&](int d) {
                if constexpr (kQ8) {
                    const char4 x = *reinterpret_cast<const char4*>(k + d);
                    const float scale = scale_of(head, slot, d / 32);
                    return f32x4{scale * static_cast<float>(x.x), scale * static_cast<float>(x.y), scale * static_cast<float>(x.z),
                                 scale * static_cast<float>(x.w)};
                } else {
                    return *reinterpret_cast<const f32x4*>(k + 4 * d);
                }
            };
            if (aligned) {
#pragma unroll 8
                for (int d = 0; d < D; d += 4) {
                    const f32x4 x = four(d), q = *reinterpret_cast<const f32x4*>(qs + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s = fmaf(q[e], x[e], s);
                }
            } else {
                for (int d = 0; d < D; ++d) s = fmaf(qs[d], element(head, k, slot, d), s);
            }
            bad |= !__builtin_isfinite(s);
            if (a.cap != 0.f) s = a.cap * any_tanh(s);
            if (a.slopes) s = fmaf(-slope, static_cast<float>(abs(run.w - key)), s);
        }
        float mx = s;
        for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        const float mnew = fmaxf(m, mx);
        if (mnew == -INFINITY) continue;
        const float alpha = fast_exp2(m - mnew), pj = ok ? fast_exp2(s - mnew) : 0.f;
        float ps = pj;
        for (int o = 32; o >= 1; o >>= 1) ps += __shfl_xor(ps, o);
        l *= alpha;
        rounded *= alpha;
        add_to(l, rounded, ps);
        m = mnew;
        float sum[kColumns];
#pragma unroll
        for (int i = 0; i < kColumns; ++i) sum[i] = 0.f;
        const int keys = min(64, part.w - base);
        for (int j = 0; j < keys; j += kTogether) {
            float x[kTogether][kColumns];
#pragma unroll
            for (int t = 0; t < kTogether; ++t) {
                const int from = min(j + t, keys - 1), of = __builtin_amdgcn_readlane(slot, from);
                const char* head = heads + static_cast<size_t>(__builtin_amdgcn_readlane(block, from)) * a.lay.stride + section;
#pragma unroll
                for (int i = 0; i < kColumns; ++i)  // (lanes behind the row write nothing)
                    x[t][i] = element(head, head + static_cast<size_t>(of) * pitch, of, min(i * 64 + lane, D - 1));
            }
#pragma unroll
            for (int t = 0; t < kTogether; ++t) {
                const float p = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, pj), min(j + t, keys - 1)));
                if (j + t < keys)
#pragma unroll
                    for (int i = 0; i < kColumns; ++i) sum[i] = fmaf(p, x[t][i], sum[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kColumns; ++i) {
            acc[i] *= alpha;
            rest[i] *= alpha;
            add_to(acc[i], rest[i], sum[i]);
        }
    }
    bad |= !__builtin_isfinite(l);  // (a score and its bias may be finite and their sum not)
    if (__any(bad) && lane == 0) *a.err = 1;
    const bool whole = run.y == 1;
    const size_t at = (whole ? row : static_cast<size_t>(run.z) + run.x) * a.heads + h;
    float* o = (whole ? a.out : a.part_acc) + at * D;
    const float div = whole && l != 0.f ? l : 1.f;
#pragma unroll
    for (int i = 0; i < kColumns; ++i) {
        const int d = i * 64 + lane;
        if (d < D) o[d] = acc[i] / div;
    }
    if (!whole && lane == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(m, l);
}

// (rows, heads) up to which four waves take one
constexpr size_t kMergeSpread = 8192;

// A row's runs combined: waves take runs in turn, lanes are columns, the maxima and sums of
// 64 runs in a wave's lanes at once.  The loads of four runs are in flight.  What the
// additions round away is kept (add_to): beside one run with all the weight the others'
// parts may each be less than half an ulp.  A workgroup takes a (row, head) with its four
// waves where the chip has waves to spare, or one with each (2,200 rows
// of 32 heads: 24 us, and 76 with four; a row of nine after 4,000 keys, with its attention,
// 13.5, and 10.4 with four).
template <int kColumns, int kWaves>
__global__ __launch_bounds__(256) void score_merge_kernel(const ScoreArgs a) {
    constexpr int kTogether = 4;
    __shared__ float2 stats[4];
    __shared__ float sums[4][64 * kColumns];
    const int lane = threadIdx.x & 63, in_group = threadIdx.x >> 6, wave = in_group % kWaves, D = a.lay.head_dim;
    const size_t row = blockIdx.x;
    const int h = kWaves == 4 ? blockIdx.y : 4 * blockIdx.y + in_group;
    const int2 runs = a.runs[row];
    if (runs.y == 1) return;  // (written by the attention itself)
    if (kWaves == 1 && h >= a.heads) return;
    float m = -INFINITY, l = 0.f, l_rest = 0.f, acc[kColumns], rest[kColumns];
#pragma unroll
    for (int i = 0; i < kColumns; ++i) acc[i] = rest[i] = 0.f;
    for (int r0 = 0; r0 < runs.y; r0 += 64 * kWaves) {  // run r0 + kWaves * lane + wave
        const int mine = r0 + kWaves * lane + wave, n = min(64, (runs.y - r0 - wave + kWaves - 1) / kWaves);
        float2 ml = make_float2(-INFINITY, 0.f);
        if (mine < runs.y) ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * ((static_cast<size_t>(runs.x) + mine) * a.heads + h));
        float mx = ml.x;
        for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        const float mnew = fmaxf(m, mx);
        if (mnew == -INFINITY) continue;
        const float alpha = fast_exp2(m - mnew), weight = fast_exp2(ml.x - mnew);
        float ls = ml.y * weight;
        for (int o = 32; o >= 1; o >>= 1) ls += __shfl_xor(ls, o);
        l *= alpha;
        l_rest *= alpha;
        add_to(l, l_rest, ls);
        m = mnew;
#pragma unroll
        for (int i = 0; i < kColumns; ++i) {
            acc[i] *= alpha;
            rest[i] *= alpha;
        }
        for (int r = 0; r < n; r += kTogether) {
            float x[kTogether][kColumns], w[kTogether];
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
                const int at = min(r + k, n - 1);
                w[k] = r + k < n ? __shfl(weight, at) : 0.f;
                const float* p = a.part_acc + ((static_cast<size_t>(runs.x) + r0 + kWaves * at + wave) * a.heads + h) * D;
#pragma unroll
                for (int i = 0; i < kColumns; ++i) x[k][i] = i * 64 + lane < D ? p[i * 64 + lane] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < kTogether; ++k)
                if (r + k < n)
#pragma unroll
                    for (int i = 0; i < kColumns; ++i) add_to(acc[i], rest[i], w[k] * x[k][i]);
        }
    }
    if constexpr (kWaves == 1) {
        const float div = l != 0.f ? l : 1.f;
#pragma unroll
        for (int i = 0; i < kColumns; ++i)
            if (i * 64 + lane < D) a.out[(row * a.heads + h) * D + i * 64 + lane] = acc[i] / div;
        return;
    }
    if (lane == 0) stats[wave] = make_float2(m, l);
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w].x);
    const float base = top == -INFINITY ? 0.f : top, scale = fast_exp2(m - base);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total = fmaf(fast_exp2(stats[w].x - base), stats[w].y, total);
#pragma unroll
    for (int i = 0; i < kColumns; ++i) sums[wave][i * 64 + lane] = acc[i] * scale;
    __syncthreads();
    const float div = total != 0.f ? total : 1.f;
    for (int d = threadIdx.x; d < D; d += 64 * kWaves) {
        float o = sums[0][d];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) o += sums[w][d];
        a.out[(row * a.heads + h) * D + d] = o / div;
    }
}

}  // namespace

void launch_score_rows(const ScoreArgs& a, int items, hipStream_t s) {
    if (a.lay.head_dim > kMaxDim) throw std::invalid_argument("head_dim above 512 is not supported");
    auto go = [&](auto kernel) { launch("score_attention", kernel, dim3(items, a.heads), dim3(64), 0, s, a); };
    const int columns = (a.lay.head_dim + 63) / 64;
    if (a.lay.format == kQ8)
        columns == 1   ? go(score_rows_kernel<1, true>)
        : columns == 2 ? go(score_rows_kernel<2, true>)
        : columns <= 4 ? go(score_rows_kernel<4, true>)
                       : go(score_rows_kernel<kMaxDim / 64, true>);
    else
        columns == 1   ? go(score_rows_kernel<1, false>)
        : columns == 2 ? go(score_rows_kernel<2, false>)
        : columns <= 4 ? go(score_rows_kernel<4, false>)
                       : go(score_rows_kernel<kMaxDim / 64, false>);
    TVARA_HIP(hipGetLastError());
}

void launch_score_merge(const ScoreArgs& a, hipStream_t s) {
    auto go = [&](auto kernel, int groups) {
        launch("score_attention_merge", kernel, dim3(static_cast<unsigned>(a.rows), static_cast<unsigned>(groups)), dim3(256), 0, s, a);
    };
    const int columns = (a.lay.head_dim + 63) / 64;
    if (static_cast<size_t>(a.rows) * a.heads > kMergeSpread) {
        const int groups = (a.heads + 3) / 4;
        columns == 1   ? go(score_merge_kernel<1, 1>, groups)
        : columns == 2 ? go(score_merge_kernel<2, 1>, groups)
                       : go(score_merge_kernel<kMaxDim / 64, 1>, groups);
    } else {
        columns == 1   ? go(score_merge_kernel<1, 4>, a.heads)
        : columns == 2 ? go(score_merge_kernel<2, 4>, a.heads)
                       : go(score_merge_kernel<kMaxDim / 64, 4>, a.heads);
    }
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

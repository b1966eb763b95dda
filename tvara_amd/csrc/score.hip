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
// head); lanes are keys for the scores and columns for the output.  For the layouts
// that the tiles do not take; bound by loads of single elements, every row for itself.
__global__ __launch_bounds__(64) void score_rows_kernel(const ScoreArgs a) {
    __shared__ float qs[kMaxDim];
    const int lane = threadIdx.x, h = blockIdx.y, kh = h / a.group;
    const int D = a.lay.head_dim, tpb = a.lay.tpb;
    const int4* w = a.work + 3 * static_cast<size_t>(blockIdx.x);
    const int4 seq = w[0], part = w[1], run = w[2];
    const int32_t* tab = a.tables + seq.x;
    const size_t row = seq.w;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    for (int d = lane; d < D; d += 64) qs[d] = a.q[(row * a.heads + h) * D + d] * a.qscale;
    __syncthreads();
    // A batch of 64 keys is added up by itself and then joins the rest, the normaliser
    // with what its additions have rounded away.
    float m = -INFINITY, l = 0.f, rounded = 0.f, acc[kMaxDim / 64];
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) acc[i] = 0.f;
    bool bad = false;
    for (int base = part.z; base < part.w; base += 64) {
        const int key = base + lane;
        const bool ok = key < part.w;  // (a run lies within the row's range)
        float s = -INFINITY;
        if (ok) {
            s = 0.f;
            const int block = tab[key / tpb], slot = key % tpb;
            for (int d = 0; d < D; ++d) s = fmaf(qs[d], score_element(a, block, 0, slot, kh * D + d), s);
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
        float sum[kMaxDim / 64];
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i) sum[i] = 0.f;
        const int keys = min(64, part.w - base);
        for (int j = 0; j < keys; ++j) {
            const float p = __shfl(pj, j);
            const int block = tab[(base + j) / tpb], slot = (base + j) % tpb;
#pragma unroll
            for (int i = 0; i < kMaxDim / 64; ++i) {
                const int d = i * 64 + lane;
                if (d < D) sum[i] = fmaf(p, score_element(a, block, 1, slot, kh * D + d), sum[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kMaxDim / 64; ++i) acc[i] = fmaf(acc[i], alpha, sum[i]);
    }
    if (__any(bad) && lane == 0) *a.err = 1;
    const bool whole = run.y == 1;
    const size_t at = (whole ? row : static_cast<size_t>(run.z) + run.x) * a.heads + h;
    float* o = (whole ? a.out : a.part_acc) + at * D;
    const float div = whole && l != 0.f ? l : 1.f;
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) {
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
    launch("score_attention", score_rows_kernel, dim3(items, a.heads), dim3(64), 0, s, a);
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

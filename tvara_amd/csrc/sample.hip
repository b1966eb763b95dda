// The next token of each row of logits x, by a given random number u:
//   w_i = exp((x_i - max x) / temperature)
//   top-k: the k largest x (the lowest index first among equals)
//   top-p: of those, from the largest down, as many as it takes to reach p of their mass
//   min-p: w_i >= min_p
// and then the first index up to which the kept mass exceeds u times all of it.
//
// Masses are whole numbers of 2^-44 of the largest weight in 64 bits, each weight from an
// exponential in f64: sums are then exact and the same in any order, so that neither the
// split of a row nor the order of atomics decides a token, and a border between two of
// 100,000 tokens is missed by 1e-9 of a token's mass.  (Weights below 2^-45 are zero.)
// From 2^20 logits on, whose sum may reach 2^64 of these, the unit is so much larger that
// it does not (SamplePlan::build).
//
// Four launches.
//  chunks: one read of the logits: of every 256 (a chunk) the maximum and, where the row
//    may keep every token, of every four chunks the mass.
//  gather: what the chunks' maxima and the mass say bounds the kept logits from below; the
//    logits above that go into a list while there is room, their counts and masses (in
//    f32) into bins by their distance to the maximum.  Rows without filters end here.
//  sweep: where the list was too short, the bins that hold the borders of top-k and top-p
//    go into the list, and the masses of what lies above are summed.
//  finish: the borders exactly, from the list, and the draw.
// Bound: the first by HBM and its f64 exponentials; the others by the steps of a
// workgroup, and, where rows are many and flat, by their instructions.  In us: a row of 32,000
// logits 4, 7, 2 and 8; 32 rows of 128,256 with parameters of all kinds 8, 16, 20 and 22; 256 rows
// of 128,256 with top-p (131 MB, 24 us to read) 45, 60, 92 and 24.
#include <algorithm>

#include "common.hpp"
#include "device_util.hpp"
#include "sample.hpp"

namespace tvara_amd {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;  // of all launches but the first
constexpr int kWaves = kThreads / 64;
constexpr int kBins = kSampleBins;
constexpr float kSpan = 32.f;  // of x / temperature that the bins cover: further down, weights are zero
constexpr int kList = kSampleList;
constexpr uint32_t kNone = 0xffffffffu;

// 2^a for a in [-1000, 0], 1e-14 of it: Taylor's series of 2^f, |f| <= 1/2, and a's whole
// part (the low word of a + 1.5 * 2^52) into the exponent
__device__ __forceinline__ double exp2_of(double a) {
    const double shifted = a + 6755399441055744.0, f = a - (shifted - 6755399441055744.0);
    double p = 4.44553827187081007394e-10;
    p = fma(p, f, 7.05491162080112087744e-09);
    p = fma(p, f, 1.01780860092396959520e-07);
    p = fma(p, f, 1.32154867901443052734e-06);
    p = fma(p, f, 1.52527338040598376946e-05);
    p = fma(p, f, 1.54035303933816060656e-04);
    p = fma(p, f, 1.33335581464284411157e-03);
    p = fma(p, f, 9.61812910762847687873e-03);
    p = fma(p, f, 5.55041086648215761801e-02);
    p = fma(p, f, 2.40226506959100694072e-01);
    p = fma(p, f, 6.93147180559945286227e-01);
    p = fma(p, f, 1.0);
    const u64 n = __builtin_bit_cast(u64, shifted);
    return __builtin_bit_cast(double, __builtin_bit_cast(u64, p) + (n << 52));
}

// exp((x - top) / temperature) of x <= top; c = log2(e) / temperature
__device__ __forceinline__ double weight_of(float x, float top, double c) {
    const double w = exp2_of(fmax((static_cast<double>(x) - static_cast<double>(top)) * c, -1000.0));
    return x == top ? 1.0 : w;
}

// in whole units, `one` to a weight of 1 (2^44 or less), rounded to nearest: the low bits of
// w * one + 2^52
__device__ __forceinline__ u64 units_of(double w, double one) {
    constexpr double kShift = 4503599627370496.0;
    return __builtin_bit_cast(u64, fma(w, one, kShift)) - __builtin_bit_cast(u64, kShift);
}

// the order of floats as that of numbers (-0 as 0)
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == 0.f ? 0.f : x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __builtin_bit_cast(float, (k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// maximum and sum over a wave's lanes, in all of them
template <int kControl>
__device__ __forceinline__ float moved(float v) {
    const int b = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, kControl, 0xf, 0xf, false));
}
template <int kControl>
__device__ __forceinline__ double moved(double v) {
    const u64 b = __builtin_bit_cast(u64, v);
    const int lo = static_cast<int>(b), hi = static_cast<int>(b >> 32);
    const uint32_t l = __builtin_amdgcn_update_dpp(lo, lo, kControl, 0xf, 0xf, false);
    const uint32_t h = __builtin_amdgcn_update_dpp(hi, hi, kControl, 0xf, 0xf, false);
    return __builtin_bit_cast(double, static_cast<u64>(h) << 32 | l);
}
constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;  // within 16 lanes
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, moved<kSwap1>(v));
    v = fmaxf(v, moved<kSwap2>(v));
    v = fmaxf(v, moved<kHalfMirror>(v));
    v = fmaxf(v, moved<kMirror>(v));
    return cross_row_max(v);
}
__device__ __forceinline__ double wave_sum(double v) {
    v += moved<kSwap1>(v);
    v += moved<kSwap2>(v);
    v += moved<kHalfMirror>(v);
    v += moved<kMirror>(v);
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// What a row asks for.
struct Asked {
    float temperature, min_p;
    double top_p;
    uint32_t top_k;  // vocab: all
    bool valid, greedy, by_k, by_p;
};
__device__ __forceinline__ Asked asked_of(const SampleArgs& a, int row) {
    Asked r;
    r.temperature = a.temperature ? a.temperature[row] : 1.f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f;
    r.min_p = a.min_p ? a.min_p[row] : 0.f;
    r.top_p = p;
    r.top_k = k <= 0 || k > a.vocab ? a.vocab : k;
    r.valid = r.temperature >= 0.f && r.temperature < INFINITY && k >= 0 && p >= 0.f && p <= 1.f && r.min_p >= 0.f && r.min_p <= 1.f;
    r.greedy = r.temperature == 0.f || r.top_k == 1 || p == 0.f;
    r.by_k = r.top_k < static_cast<uint32_t>(a.vocab);
    r.by_p = p < 1.f;
    return r;
}

// four logits from index i on (a multiple of 4), -inf behind the row and for NaN
template <bool kWide>
__device__ __forceinline__ f32x4 four_of(const float* x, int i, int vocab, bool& odd) {
    f32x4 v;
    if (kWide && i + 4 <= vocab) {
        v = *reinterpret_cast<const f32x4*>(x + i);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < vocab ? x[i + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (v[e] != v[e]) {
            odd = true;
            v[e] = -INFINITY;
        }
    return v;
}

// A wave kSampleGroup chunks, whose loads are in flight together (of chunks of 256).
// What the later launches count in starts from zero here.
template <bool kWide>
__global__ __launch_bounds__(256) void sample_chunks_kernel(const SampleArgs a) {
    constexpr int P = kSampleGroup;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.y, group = blockIdx.x * 4 + wave, c0 = group * P;
    const float* x = a.logits + row * a.stride;
    const Asked ask = asked_of(a, row);
    const bool mass = ask.valid && !ask.greedy && !ask.by_k;
    const double c = 1.4426950408889634 / static_cast<double>(ask.temperature);
    if (a.bin_mass)
        for (int i = blockIdx.x * 256 + threadIdx.x; i < kBins; i += gridDim.x * 256) {
            a.bin_mass[static_cast<size_t>(row) * kBins + i] = 0;
            a.bin_count[static_cast<size_t>(row) * kBins + i] = 0;
        }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.rows_state[row] = SampleRow{};
    if (c0 >= a.chunks) return;
    bool odd = false;
    float top = -INFINITY;
    double sum = 0;
    f32x4 v[P];
    const bool small = a.chunk == 256;
    if (small) {
#pragma unroll
        for (int k = 0; k < P; ++k) v[k] = four_of<kWide>(x, (c0 + k) * 256 + 4 * lane, a.vocab, odd);
    }
    for (int k = 0; k < P; ++k) {
        if (c0 + k >= a.chunks) break;
        float m = -INFINITY;
        if (small) {
            const f32x4 y = k == 0 ? v[0] : k == 1 ? v[1] : k == 2 ? v[2] : v[3];
            m = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
        } else {
            for (int i = (c0 + k) * a.chunk + 4 * lane; i < min((c0 + k + 1) * a.chunk, a.vocab); i += 256) {
                const f32x4 y = four_of<kWide>(x, i, a.vocab, odd);
                m = fmaxf(m, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
            }
        }
        m = wave_max(m);
        if (lane == 0) a.chunk_max[static_cast<size_t>(row) * a.chunks + c0 + k] = m;
        top = fmaxf(top, m);
    }
    if (__any(odd) && lane == 0) a.err[0] = 1;
    if (!mass || top == -INFINITY) return;
    if (small) {
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += weight_of(v[k][e], top, c);
    } else {
        for (int i = c0 * a.chunk + 4 * lane; i < min((c0 + P) * a.chunk, a.vocab); i += 256) {
            const f32x4 y = four_of<kWide>(x, i, a.vocab, odd);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += weight_of(y[e], top, c);
        }
    }
    sum = wave_sum(sum);
    if (lane == 0) a.group_mass[static_cast<size_t>(row) * kSampleGroups + group] = sum;
}

// ------------------------------------------------- workgroups of a row

struct Shared {
    float chunk_max[kSampleChunks];
    u64 chunk_mass[kSampleChunks];
    uint32_t chunk_ties[kSampleChunks];
    uint32_t count[kBins];
    u64 mass[kBins];
    SampleCandidate list[kList];
    float queue[kWaves][256];  // a wave's logits of a turn that are worth an exponential
    u64 wave_sums[kWaves];
    u64 told, left, rank;
    int found;
};

__device__ __forceinline__ u64 wave_scan(u64 v) {  // inclusive
    const int lane = threadIdx.x & 63;
    for (int o = 1; o < 64; o <<= 1) {
        const u64 below = __shfl_up(v, o);
        if (lane >= o) v += below;
    }
    return v;
}

// The inclusive sums of the workgroup's values, thread by thread.
__device__ __forceinline__ u64 block_scan(Shared& s, u64 v) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) s.wave_sums[wave] = v;
    __syncthreads();
    u64 before = 0;
    for (int w = 0; w < wave; ++w) before += s.wave_sums[w];
    return v + before;
}
__device__ __forceinline__ u64 block_sum(Shared& s, u64 v) {
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave_sums[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 sum = 0;
    for (int w = 0; w < kWaves; ++w) sum += s.wave_sums[w];
    return sum;
}

// The first of n places (two a thread) up to which the values' sum reaches `need` (1 or
// more), and the sum before it; n, and all of it, where they do not reach it.
template <class F>
__device__ __forceinline__ int find(Shared& s, int n, u64 need, F&& value, u64& before) {
    const int i = 2 * threadIdx.x;
    const u64 v0 = i < n ? value(i) : 0, v1 = i + 1 < n ? value(i + 1) : 0;
    const u64 upto = block_scan(s, v0 + v1), b0 = upto - v1 - v0, b1 = upto - v1;
    if (threadIdx.x == kThreads - 1 && upto < need) {
        s.found = n;
        s.told = upto;
    }
    if (b0 < need && b1 >= need) {
        s.found = i;
        s.told = b0;
    } else if (b1 < need && upto >= need) {
        s.found = i + 1;
        s.told = b1;
    }
    __syncthreads();
    before = s.told;
    const int at = s.found;
    __syncthreads();
    return at;
}

// A row as its workgroups see it.
struct Row {
    const float* x;
    int vocab, chunk, chunks;
    float top, scale;  // scale: bins for two units of a logit
    double c;          // log2(e) / temperature
    double min_p;
    double one;        // a mass of 1 (SampleArgs::one)

    __device__ __forceinline__ float distance(float v) const {
        return (v == top ? 0.f : 0.5f * top - 0.5f * v) * scale;  // (top - v may be beyond f32)
    }
    __device__ __forceinline__ int bin(float v) const {  // kBins: zero weight
        return static_cast<int>(fminf(distance(v), static_cast<float>(kBins)));
    }
    __device__ __forceinline__ double weight(float v) const { return weight_of(v, top, c); }
    __device__ __forceinline__ u64 units(float v) const { return units_of(weight(v), one); }
    __device__ __forceinline__ float share(float v, u64 sum) const {
        return static_cast<float>(weight(v) / (static_cast<double>(sum) / one));
    }
};

__device__ __forceinline__ Row row_of(const SampleArgs& a, int row, const Asked& ask, float top) {
    Row r;
    r.x = a.logits + row * a.stride;
    r.vocab = a.vocab;
    r.chunk = a.chunk;
    r.chunks = a.chunks;
    r.top = top;
    r.c = 1.4426950408889634 / static_cast<double>(ask.temperature);
    r.scale = fminf(2.f * kBins / kSpan / ask.temperature, 3e38f);
    r.min_p = ask.min_p;
    r.one = a.one;
    return r;
}

// f(four logits, the first's index, their chunk) for the row's chunks whose maximum's bin
// is at most `last`, a wave `own` of `waves` a chunk, the loads of four chunks in flight;
// none(chunk) for the others
template <bool kWide, class F, class G>
__device__ __forceinline__ void each_turn(const Shared& s, const Row& r, int last, int own, int waves, F&& f, G&& none) {
    constexpr int kTogether = 4;
    const int lane = threadIdx.x & 63;
    for (int k0 = own; k0 < r.chunks; k0 += waves * kTogether) {
        bool on[kTogether];
        f32x4 v[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            const int c = k0 + k * waves;
            on[k] = c < r.chunks && s.chunk_max[c] != -INFINITY && r.bin(s.chunk_max[c]) <= last;
            bool odd = false;
            if (on[k]) v[k] = four_of<kWide>(r.x, c * r.chunk + 4 * lane, r.vocab, odd);
        }
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            const int c = k0 + k * waves;
            if (!on[k]) {
                if (c < r.chunks) none(c);
                continue;
            }
            f(v[k], c * r.chunk + 4 * lane, c);
            for (int i = 256; i < r.chunk; i += 256) {  // (large vocabularies)
                bool odd = false;
                const int at = c * r.chunk + i + 4 * lane;
                f(four_of<kWide>(r.x, at, r.vocab, odd), at, c);
            }
        }
    }
}

// Where a lane's chosen ones of a turn (bit e: its e-th) go among the wave's; all: how many.
__device__ __forceinline__ int packed_place(uint32_t chosen, int& all) {
    int before = 0;
    all = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const u64 b = __ballot(chosen >> e & 1);
        before += __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(b >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(b), 0));
        all += __builtin_popcountll(b);
    }
    return before;
}

// f(x) for a wave's chosen logits of a turn, packed into its first lanes: of a row's many
// few are worth an exponential
template <class F>
__device__ __forceinline__ void each_packed(Shared& s, f32x4 v, uint32_t chosen, F&& f) {
    const int lane = threadIdx.x & 63;
    float* queue = s.queue[threadIdx.x >> 6];
    int all, at = packed_place(chosen, all);
    if (!all) return;
    asm volatile("" ::: "memory");  // (a wave's accesses to LDS stay in order)
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (chosen >> e & 1) queue[at++] = v[e];
    asm volatile("" ::: "memory");
    for (int i = lane; i < all; i += 64) f(queue[i]);
    asm volatile("" ::: "memory");
}

// A wave's chosen logits of a turn into the row's list while there is room; all are counted.
__device__ __forceinline__ void append(int* size, SampleCandidate* list, int room, f32x4 v, int index, uint32_t chosen) {
    int all, at = packed_place(chosen, all);
    if (!all) return;
    int base = 0;
    if ((threadIdx.x & 63) == 0) base = atomicAdd(size, all);
    at += __builtin_amdgcn_readfirstlane(base);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (chosen >> e & 1) {
            if (at < room) list[at] = {ordered(v[e]), static_cast<uint32_t>(index + e)};
            ++at;
        }
}

__device__ __forceinline__ void answer(const SampleArgs& a, int row, uint32_t token, float p) {
    a.tokens[row] = token;
    if (a.probability) a.probability[row] = p;
}

// The token of a stretch of the row that the random number falls on: the first in order of
// index up to which the kept mass exceeds `left`.  units(x, rank) is what x counts, where
// `rank` ties of the border come before it; tie(x) whether it is one of them.  A wave.
template <bool kWide, class F, class G>
__device__ __forceinline__ uint32_t pick(const Row& r, int from, int to, u64 left, u64 rank, F&& units, G&& tie, float& x) {
    const int lane = threadIdx.x & 63;
    uint32_t last = kNone;
    for (int i0 = from; i0 < min(to, r.vocab); i0 += 256) {
        bool odd = false;
        const int i = i0 + 4 * lane;
        const f32x4 v = four_of<kWide>(r.x, i, r.vocab, odd);
        uint32_t tied = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (v[e] != -INFINITY && tie(v[e])) tied |= 1u << e;
        const u64 tied_upto = wave_scan(__builtin_popcount(tied));
        u64 before = rank + tied_upto - __builtin_popcount(tied), w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = v[e] == -INFINITY ? 0 : units(v[e], before);
            before += tied >> e & 1;
        }
        rank += __shfl(tied_upto, 63);
        const u64 own = w[0] + w[1] + w[2] + w[3], upto = wave_scan(own);
        const u64 hit = __ballot(upto > left), any = __ballot(own != 0);
        const bool found = hit != 0;
        if (found || any) {  // the token, or the stretch's last kept one so far
            const int who = found ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
            u64 at = upto - own;
            int e = 0;
            if (found) {
                while (e < 3 && at + w[e] <= left) at += w[e++];
            } else {
                for (int k = 0; k < 4; ++k)
                    if (w[k]) e = k;
            }
            last = __shfl(static_cast<uint32_t>(i + e), who);
            x = __shfl(e == 0 ? v[0] : e == 1 ? v[1] : e == 2 ? v[2] : v[3], who);
        }
        if (found) return last;
        left -= __shfl(upto, 63);
    }
    return last;
}

// Candidates, rows that end here, and the bounds that the other launches go by.  grid.x:
// a share of the row's chunks.
template <bool kWide>
__global__ __launch_bounds__(kThreads) void sample_gather_kernel(const SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Asked ask = asked_of(a, row);
    const float u = a.uniforms[row];
    const bool first = blockIdx.x == 0;
    SampleRow* state = a.rows_state + row;
    if (!ask.valid || !(u >= 0.f && u < 1.f)) {
        if (first && tid == 0) {
            a.err[1] = 1;
            answer(a, row, kNone, 0.f);
            state->done = 1;
        }
        return;
    }
    const size_t at0 = static_cast<size_t>(row) * a.chunks;
    float mine = -INFINITY;
    if (tid < a.chunks) s.chunk_max[tid] = mine = a.chunk_max[at0 + tid];
    float top = wave_max(mine);
    if (lane == 0) s.wave_sums[wave] = __builtin_bit_cast(uint32_t, top);
    if (tid == 0) s.found = a.chunks;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, __builtin_bit_cast(float, static_cast<uint32_t>(s.wave_sums[w])));
    if (top == -INFINITY || ask.greedy) {
        if (!first) return;
        if (tid == 0) state->done = 1;
        if (top == -INFINITY) {  // nothing to draw
            if (tid == 0) {
                a.err[0] = 1;
                answer(a, row, kNone, 0.f);
            }
            return;
        }
        // the lowest index of the maximum, in the first chunk that has it
        if (mine == top) atomicMin(&s.found, tid);
        __syncthreads();
        if (tid >= 64) return;
        const float* x = a.logits + row * a.stride;
        for (int i = s.found * a.chunk; i < min((s.found + 1) * a.chunk, a.vocab); i += 64) {
            const u64 hit = __ballot(i + lane < a.vocab && x[min(i + lane, a.vocab - 1)] == top);
            if (!hit) continue;
            if (lane == 0) answer(a, row, static_cast<uint32_t>(i + __builtin_ctzll(hit)), 1.f);
            return;
        }
        return;
    }
    const Row r = row_of(a, row, ask, top);
    // the masses of four chunks each, and all of it (where top-k does not leave that open)
    const int groups = (a.chunks + kSampleGroup - 1) / kSampleGroup;
    u64 total = 0;
    if (!ask.by_k) {
        u64 units = 0;
        if (tid < groups) {
            float m = -INFINITY;
            for (int k = tid * kSampleGroup; k < min((tid + 1) * kSampleGroup, a.chunks); ++k) m = fmaxf(m, s.chunk_max[k]);
            if (m != -INFINITY)
                units = static_cast<u64>(__builtin_rint(a.group_mass[static_cast<size_t>(row) * kSampleGroups + tid] * r.weight(m) * a.one));
        }
        if (!ask.by_p && ask.min_p == 0.f) {  // every token: the draw
            if (!first) return;
            const u64 upto = block_scan(s, units), sum = block_sum(s, units);
            const u64 target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(sum));
            __syncthreads();
            if (upto - units <= target && upto > target) {
                s.found = tid;
                s.left = target - (upto - units);
            }
            __syncthreads();
            if (tid >= 64) return;
            const int from = s.found * kSampleGroup * a.chunk, to = from + kSampleGroup * a.chunk;
            float x = top;
            uint32_t token = pick<kWide>(r, from, to, s.left, 0, [&](float v, u64) { return r.units(v); }, [](float) { return false; }, x);
            if (token == kNone) {
                // (each alone rounds to nothing, together they did not: the largest of them)
                float m = -INFINITY;
                for (int k = s.found * kSampleGroup; k < min((s.found + 1) * kSampleGroup, a.chunks); ++k) m = fmaxf(m, s.chunk_max[k]);
                for (int i = from; i < min(to, a.vocab) && token == kNone; i += 64) {
                    const u64 hit = __ballot(i + lane < a.vocab && r.x[min(i + lane, a.vocab - 1)] == m);
                    if (hit) token = static_cast<uint32_t>(i + __builtin_ctzll(hit));
                }
                x = m;
            }
            if (lane == 0) {
                answer(a, row, token, r.share(x, sum));
                state->done = 1;
            }
            return;
        }
        total = block_sum(s, units);
    }
    const u64 need = ask.by_p && !ask.by_k ? max(static_cast<u64>(__builtin_ceil(ask.top_p * static_cast<double>(total))), u64(1)) : 0;

    // The last bin that can hold a kept logit.
    int last = kBins - 1;
    auto down_to = [&](double w) {  // the bin of a weight, or the one behind it
        last = min(last, static_cast<int>(fminf(-__log2f(static_cast<float>(w)) * 0.693147181f * (kBins / kSpan), 2.f * kBins)) + 1);
    };
    if (!ask.by_k && ask.min_p > 0.f) down_to(ask.min_p);
    // weights below (1 - p) of the mean weigh less than 1 - p together
    if (need) down_to(fmin((1.0 - ask.top_p) * static_cast<double>(total) / a.one / a.vocab, 1.0));
    for (int i = tid; i < kBins; i += kThreads) {
        s.mass[i] = 0;
        s.count[i] = 0;
    }
    // the chunks' maxima alone reach k, or p of the mass
    if (need || (ask.by_k && ask.top_k <= static_cast<uint32_t>(a.chunks))) {
        __syncthreads();
        if (mine != -INFINITY) {
            const int b = r.bin(mine);
            if (b < kBins) atomicAdd(&s.mass[b], ask.by_k ? u64(1) : r.units(mine));
        }
        __syncthreads();
        u64 before;
        last = min(last, find(s, kBins, ask.by_k ? ask.top_k : need, [&](int i) { return s.mass[i]; }, before));
        for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0;
    }
    __syncthreads();
    if (first && tid == 0) {
        state->top = top;
        state->last = last;
        state->total = total;
    }
    // masses here are of f32 exponentials, in units of 2^-31
    const bool bins = a.bin_mass != nullptr, counts = bins && ask.by_k, masses = bins && ask.by_p;
    SampleCandidate* list = a.list + static_cast<size_t>(row) * a.room;
    constexpr float kTurn = -1.44269504f * kSpan / kBins;
    each_turn<kWide>(
        s, r, last, blockIdx.x * kWaves + wave, gridDim.x * kWaves,
        [&](f32x4 v, int at, int) {
            uint32_t chosen = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = r.distance(v[e]);
                const int b = static_cast<int>(fminf(d, static_cast<float>(kBins)));
                if (v[e] == -INFINITY || b > last) continue;
                chosen |= 1u << e;
                if (counts) atomicAdd(&s.count[b], 1u);
                if (masses) atomicAdd(&s.mass[b], static_cast<u64>(static_cast<uint32_t>(fast_exp2(d * kTurn) * 2147483648.f)));
            }
            append(&state->size, list, a.room, v, at, chosen);
        },
        [](int) {});
    if (!bins) return;
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) {
        if (s.count[i]) atomicAdd(a.bin_count + static_cast<size_t>(row) * kBins + i, s.count[i]);
        if (s.mass[i]) atomicAdd(a.bin_mass + static_cast<size_t>(row) * kBins + i, s.mass[i]);
    }
}

// The bins that a row's borders lie in, from all counts and masses of its candidates:
// top-k's, and first to last of those that top-p's can be in, its masses being off by
// 2e-5 of themselves (the arguments of their exponentials) and a unit each.
struct Window {
    int k, p0, p1;  // k, p0: kBins where there is none
};
__device__ __forceinline__ Window window_of(const SampleArgs& a, Shared& s, int row, const Asked& ask, const SampleRow& state) {
    const u64* mass = a.bin_mass + static_cast<size_t>(row) * kBins;
    const uint32_t* count = a.bin_count + static_cast<size_t>(row) * kBins;
    Window w{kBins, kBins, -1};
    u64 before;
    if (ask.by_k && static_cast<u64>(state.size) > ask.top_k)
        w.k = find(s, kBins, ask.top_k, [&](int i) { return static_cast<u64>(count[i]); }, before);
    if (ask.by_p) {
        double lo = static_cast<double>(state.total) * (2147483648.0 / a.one), hi = lo;
        if (ask.by_k) {  // of what top-k keeps: up to its bin, or with all of that
            u64 up = 0;
            for (int i = threadIdx.x; i < kBins; i += kThreads)
                if (i < w.k) up += mass[i];
            lo = static_cast<double>(block_sum(s, up));
            hi = lo + (w.k < kBins ? static_cast<double>(mass[w.k]) : 0.0);
        }
        lo = fmax(ask.top_p * lo * (1 - 2e-5) - a.vocab, 1.0);
        hi = ask.top_p * hi * (1 + 2e-5) + a.vocab;
        w.p0 = find(s, kBins, static_cast<u64>(lo), [&](int i) { return mass[i]; }, before);
        w.p1 = min(find(s, kBins, static_cast<u64>(hi) + 1, [&](int i) { return mass[i]; }, before), kBins - 1);
        if (w.p0 > w.k) w.p0 = w.k;
        if (w.p1 > w.k) w.p1 = w.k;
    }
    return w;
}

// Rows whose candidates the list does not hold: the borders' bins into the list, the
// masses of what lies above them by chunks, and in all.
template <bool kWide>
__global__ __launch_bounds__(kThreads) void sample_sweep_kernel(const SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    SampleRow* state = a.rows_state + row;
    const SampleRow st = *state;
    if (st.done || st.size <= a.room) return;
    const Asked ask = asked_of(a, row);
    const Row r = row_of(a, row, ask, st.top);
    if (tid < a.chunks) s.chunk_max[tid] = a.chunk_max[static_cast<size_t>(row) * a.chunks + tid];
    const Window w = window_of(a, s, row, ask, st);
    __syncthreads();
    const int last = st.last, kept = min(min(w.p0, w.k), last + 1);  // bins before are kept whole
    SampleCandidate* list = a.list + static_cast<size_t>(row) * a.room;
    u64 *chunk_mass = a.chunk_mass + static_cast<size_t>(row) * a.chunks, above = 0, between = 0;
    each_turn<kWide>(
        s, r, last, blockIdx.x * kWaves + wave, gridDim.x * kWaves,
        [&](f32x4 v, int at, int chunk) {
            uint32_t before = 0, in = 0, rest = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int b = v[e] == -INFINITY ? kBins : r.bin(v[e]);
                if (b < kept)
                    before |= 1u << e;
                else if (b <= last && ((b >= w.p0 && b <= w.p1) || b == w.k))
                    in |= 1u << e;
                else if (ask.by_p && ask.by_k && b <= last && b < w.k)
                    rest |= 1u << e;  // (what top-k keeps behind top-p's bins)
            }
            append(&state->swept, list, a.room, v, at, in);
            u64 units = 0;
            each_packed(s, v, before, [&](float x) {
                const double y = r.weight(x);
                const u64 n = units_of(y, r.one);
                above += n;
                if (y >= r.min_p) units += n;
            });
            each_packed(s, v, rest, [&](float x) { between += r.units(x); });
            // (up to 256 times 2^44: exact in f64)
            const double sum = wave_sum(static_cast<double>(units));
            if (lane == 0) {
                const u64 n = static_cast<u64>(sum);
                chunk_mass[chunk] = at % a.chunk < 256 ? n : chunk_mass[chunk] + n;
            }
        },
        [&](int chunk) {
            if (lane == 0) chunk_mass[chunk] = 0;
        });
    above = block_sum(s, above);
    between = block_sum(s, between);
    if (tid == 0) {
        if (above) atomicAdd(&state->above, above);
        if (between) atomicAdd(&state->between, between);
    }
}

// The workgroup's values in descending order, one a thread (of the first n, a power of
// two from 64): Batcher's bitonic network, within waves by shuffles, by way of `space`
// where waves meet.
__device__ __forceinline__ u64 sort_down(u64 v, int n, u64* space) {
    const int t = threadIdx.x;
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j >= 1; j >>= 1) {
            u64 other;
            if (j >= 64) {
                __syncthreads();
                space[t] = v;
                __syncthreads();
                other = space[t ^ j];
            } else {
                other = __shfl_xor(v, j);
            }
            const bool first = (t & j) == 0, down = (t & k) == 0;
            v = first == down ? max(v, other) : min(v, other);
        }
    return v;
}

// sums of the first n threads' values (a wave's where n is 64: no barrier)
__device__ __forceinline__ u64 scan_of(Shared& s, u64 v, int n) { return n == 64 ? wave_scan(v) : block_scan(s, v); }
// thread `who`'s value, in every thread
__device__ __forceinline__ u64 from_thread(Shared& s, u64 v, int who, int n) {
    if (n == 64) return __shfl(v, who);
    __syncthreads();
    if (static_cast<int>(threadIdx.x) == who) s.told = v;
    __syncthreads();
    return s.told;
}

// Candidates of which a thread takes one: in order of their logits, top-k is a count and
// top-p a running mass; in order of their indexes, so is the draw.
__device__ __forceinline__ void draw_listed(const SampleArgs& a, int row, Shared& s, const SampleCandidate* list, const Row& r, const Asked& ask,
                                            int size, u64 total, float u) {
    const int t = threadIdx.x;
    int n = 64;
    while (n < size) n *= 2;
    if (n == 64 && t >= 64) return;
    const SampleCandidate mine = t < size ? list[t] : SampleCandidate{0, kNone};
    // (a larger key first, then a lower index)
    const u64 order = sort_down(static_cast<u64>(mine.key) << 32 | (kNone - mine.index), n, s.mass);
    const uint32_t key = static_cast<uint32_t>(order >> 32), index = kNone - static_cast<uint32_t>(order);
    const bool in = t < size && static_cast<uint32_t>(t) < ask.top_k;
    const double w = in ? r.weight(unordered(key)) : 0.0;
    const u64 units = in ? units_of(w, r.one) : 0;
    const u64 upto = scan_of(s, units, n);
    u64 need = 0;
    if (ask.by_p) {
        if (ask.by_k) total = from_thread(s, upto, n - 1, n);
        need = max(static_cast<u64>(__builtin_ceil(ask.top_p * static_cast<double>(total))), u64(1));
    }
    const bool kept = in && w >= r.min_p && (!need || upto - units < need);
    // by index, what is not kept behind; the place in the order of logits goes along
    const u64 by_index = sort_down(kept ? static_cast<u64>(kNone - index) << 32 | static_cast<uint32_t>(t) : 0, n, s.mass);
    const int place = static_cast<int>(by_index & 0xffffffffu);
    u64 own;
    uint32_t own_key;
    if (n == 64) {
        own = __shfl(units, place);
        own_key = __shfl(key, place);
    } else {
        __syncthreads();
        s.mass[t] = units;
        s.count[t] = key;
        __syncthreads();
        own = s.mass[place];
        own_key = s.count[place];
    }
    if (!by_index) own = 0;
    const u64 drawn = scan_of(s, own, n), sum = from_thread(s, drawn, n - 1, n);
    const u64 target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(sum));
    if (drawn > target && drawn - own <= target) answer(a, row, kNone - static_cast<uint32_t>(by_index >> 32), r.share(unordered(own_key), sum));
}

// What is kept: keys above `key`, and of those at it the first `ties` by index.
struct Border {
    uint32_t key;
    u64 ties;
    u64 mass;  // above the ties, of what was looked at
};

// The place at which `need` is reached from the largest down, by counts or masses, exactly:
// by 11, 11 and 10 bits of the keys.  each(f): f(key) for all that is looked at.
template <class Each>
__device__ __forceinline__ Border place(Shared& s, const Row& r, bool by_mass, u64 need, Each&& each) {
    uint32_t prefix = 0, mask = 0;
    u64 mass = 0;
    for (int shift = 21; shift >= 0; shift -= shift == 21 ? 11 : 10) {
        const int n = 1 << (shift ? 11 : 10);
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            s.count[i] = 0;
            s.mass[i] = 0;
        }
        __syncthreads();
        each([&](uint32_t key) {
            if ((key & mask) != prefix) return;
            const int at = n - 1 - static_cast<int>(key >> shift & (n - 1));
            if (!by_mass) atomicAdd(&s.count[at], 1u);
            const u64 w = r.units(unordered(key));
            if (w) atomicAdd(&s.mass[at], w);
        });
        __syncthreads();
        u64 before, other = 0;
        const int at = by_mass ? find(s, n, need, [&](int i) { return s.mass[i]; }, before)
                               : find(s, n, need, [&](int i) { return static_cast<u64>(s.count[i]); }, before);
        if (at == n) return {0, 0, mass + before};  // (not reached: all of it is kept, and no key is 0)
        if (by_mass) {
            mass += before;
        } else {
            for (int i = threadIdx.x; i < at; i += kThreads) other += s.mass[i];
            mass += block_sum(s, other);
        }
        need -= before;
        mask |= static_cast<uint32_t>(n - 1) << shift;
        prefix |= static_cast<uint32_t>(n - 1 - at) << shift;
    }
    const u64 each_one = r.units(unordered(prefix));
    return {prefix, by_mass ? (need + each_one - 1) / max(each_one, u64(1)) : need, mass};
}

// The borders and the draw.
template <bool kWide>
__global__ __launch_bounds__(kThreads) void sample_finish_kernel(const SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const SampleRow st = a.rows_state[row];
    if (st.done) return;
    const Asked ask = asked_of(a, row);
    const float u = a.uniforms[row];
    const Row r = row_of(a, row, ask, st.top);
    const SampleCandidate* given = a.list + static_cast<size_t>(row) * a.room;
    if (st.size <= kThreads) {
        draw_listed(a, row, s, given, r, ask, st.size, st.total, u);
        return;
    }
    const bool all = st.size <= a.room;  // the list has all candidates; else those in the borders' bins
    const int listed = all ? st.size : st.swept;
    const bool in_list = listed <= a.room;  // (else they come from memory again)
    if (tid < a.chunks) s.chunk_max[tid] = a.chunk_max[static_cast<size_t>(row) * a.chunks + tid];
    if (in_list)
        for (int i = tid; i < listed; i += kThreads) s.list[i] = given[i];
    Window w{kBins, kBins, -1};
    u64 count_before = 0;
    if (!all) {
        w = window_of(a, s, row, ask, st);
        if (w.k < kBins) {
            u64 n = 0;
            for (int i = tid; i < w.k; i += kThreads) n += a.bin_count[static_cast<size_t>(row) * kBins + i];
            count_before = block_sum(s, n);
        }
    }
    __syncthreads();
    // f(key, index) for what is in the bins lo to hi
    auto each = [&](int lo, int hi, auto&& f) {
        if (in_list) {
            for (int i = tid; i < listed; i += kThreads) {
                const SampleCandidate c = s.list[i];
                const int b = r.bin(unordered(c.key));
                if (b >= lo && b <= hi) f(c.key, static_cast<int>(c.index));
            }
        } else {
            each_turn<kWide>(
                s, r, st.last, wave, kWaves,
                [&](f32x4 v, int at, int) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int b = r.bin(v[e]);
                        if (v[e] != -INFINITY && b <= st.last && b >= lo && b <= hi) f(ordered(v[e]), at + e);
                    }
                },
                [](int) {});
        }
    };
    Border kept{0, 0, 0};  // (no key is 0: everything)
    const bool cut = ask.by_k && static_cast<u64>(st.size) > ask.top_k;
    if (cut)
        kept = place(s, r, false, ask.top_k - count_before,
                     [&](auto&& f) { each(all ? 0 : w.k, all ? kBins : w.k, [&](uint32_t key, int) { f(key); }); });
    if (ask.by_p) {
        u64 total = st.total;
        if (ask.by_k) {
            // what top-k keeps: above top-p's bins, in them, between them and its own, and
            // there what it keeps
            if (all && !cut) {
                u64 units = 0;
                each(0, kBins, [&](uint32_t key, int) { units += r.units(unordered(key)); });
                kept.mass = block_sum(s, units);
            }
            total = kept.mass + kept.ties * r.units(unordered(kept.key));
            if (!all) {
                u64 units = 0;
                each(w.p0, min(w.p1, w.k - 1), [&](uint32_t key, int) { units += r.units(unordered(key)); });
                total = (cut ? total : 0) + st.above + st.between + block_sum(s, units);
            }
        }
        const u64 need = max(static_cast<u64>(__builtin_ceil(ask.top_p * static_cast<double>(total))), u64(1));
        if (all || w.p0 <= w.p1) {
            const u64 above = all ? 0 : st.above;
            const Border p = need > above ? place(s, r, true, need - above,
                                                  [&](auto&& f) { each(all ? 0 : w.p0, all ? kBins : w.p1, [&](uint32_t key, int) { f(key); }); })
                                          : Border{0, 0, 0};
            // (top-k's border may lie before, or leave fewer of the same ties)
            if (p.key > kept.key || (p.key == kept.key && p.ties < kept.ties)) kept = p;
        }
    }
    // what is kept, by chunks
    __syncthreads();
    if (tid < a.chunks) {
        s.chunk_mass[tid] = all ? 0 : a.chunk_mass[static_cast<size_t>(row) * a.chunks + tid];
        s.chunk_ties[tid] = 0;
    }
    __syncthreads();
    const int from_bin = all ? 0 : min(min(w.p0, w.k), st.last + 1);
    each(from_bin, kBins, [&](uint32_t key, int i) {
        if (key < kept.key) return;
        const double y = r.weight(unordered(key));
        if (y < r.min_p) return;
        if (key == kept.key) {
            atomicAdd(&s.chunk_ties[i / a.chunk], 1u);
            return;
        }
        const u64 n = units_of(y, r.one);
        if (n) atomicAdd(&s.chunk_mass[i / a.chunk], n);
    });
    __syncthreads();
    // ties by index, then the chunk and the token that the random number falls on
    const u64 tie_units = kept.key ? r.units(unordered(kept.key)) : 0;
    const u64 ties = tid < a.chunks ? s.chunk_ties[tid] : 0, ties_before = block_scan(s, ties) - ties;
    u64 units = tid < a.chunks ? s.chunk_mass[tid] : 0;
    if (ties_before < kept.ties) units += min(ties, kept.ties - ties_before) * tie_units;
    const u64 upto = block_scan(s, units), sum = block_sum(s, units);
    const u64 target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(sum));
    __syncthreads();
    if (upto - units <= target && upto > target) {
        s.found = tid;
        s.left = target - (upto - units);
        s.rank = ties_before;
    }
    __syncthreads();
    if (tid >= 64) return;
    float x = st.top;
    auto tie = [&](float v) { return ordered(v) == kept.key && r.weight(v) >= r.min_p; };
    const uint32_t token = pick<kWide>(
        r, s.found * a.chunk, (s.found + 1) * a.chunk, s.left, s.rank,
        [&](float v, u64 rank) {
            const uint32_t key = ordered(v);
            const double y = r.weight(v);
            if (key < kept.key || y < r.min_p || r.bin(v) > st.last) return u64(0);
            return key > kept.key ? units_of(y, r.one) : rank < kept.ties ? tie_units : u64(0);
        },
        tie, x);
    if (lane == 0) answer(a, row, token, r.share(x, sum));
}

}  // namespace

void launch_sample(const SampleArgs& a, hipStream_t s) {
    const bool wide = a.stride % 4 == 0;
    const unsigned rows = static_cast<unsigned>(a.rows);
    const unsigned groups = static_cast<unsigned>((a.chunks + kSampleGroup - 1) / kSampleGroup);
    launch("sample_chunks", wide ? sample_chunks_kernel<true> : sample_chunks_kernel<false>, dim3((groups + 3) / 4, rows), dim3(256), 0, s, a);
    // as many workgroups a row as give every CU one, of a turn for each wave at the least
    // (128,256 logits, all launches, us, for 128, 256, 512 and 1,024 workgroups in all: 32 rows
    // of all kinds 82, 66, 66 and 74; 256 rows with top-p 216, 216, 229 and 264; a CU holds one
    // at a time, for its 90,272 bytes of LDS and 1,024 threads of 74 to 128 registers, so that
    // more than 256 wait for each other)
    const unsigned shares = std::clamp(256 / rows, 1u, (static_cast<unsigned>(a.chunks) + kWaves - 1) / kWaves);
    launch("sample_gather", wide ? sample_gather_kernel<true> : sample_gather_kernel<false>, dim3(shares, rows), dim3(kThreads), 0, s, a);
    if (a.bin_mass)
        launch("sample_sweep", wide ? sample_sweep_kernel<true> : sample_sweep_kernel<false>, dim3(shares, rows), dim3(kThreads), 0, s, a);
    launch("sample_finish", wide ? sample_finish_kernel<true> : sample_finish_kernel<false>, dim3(rows), dim3(kThreads), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

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
//
// Two launches.  The first reads the logits once: of every chunk of 256 its maximum and,
// where the row may keep every token, its mass.  The second, a workgroup a row, goes by
// the chunks that can hold a kept token: what the largest chunk maxima and the total mass
// say bounds the kept logits from below.  Bound: the first by HBM, the second, where
// many tokens are kept, by f64 exponentials and LDS atomics.
#include "common.hpp"
#include "sample.hpp"

namespace tvara_amd {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

constexpr int kThreads = 1024;  // of the second launch
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr float kSpan = 32.f;  // of x / temperature that the bins cover: further down, weights are zero
constexpr int kList = 4096;    // candidates that LDS holds
constexpr uint32_t kNone = 0xffffffffu;

// 2^a for a in [-1100, 0], 1e-14 of it: Taylor's series of e^(f ln 2), |f| <= 1/2
__device__ __forceinline__ double exp2_of(double a) {
    const double n = __builtin_rint(a), z = (a - n) * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = fma(p, z, 1.0 / 3628800.0);
    p = fma(p, z, 1.0 / 362880.0);
    p = fma(p, z, 1.0 / 40320.0);
    p = fma(p, z, 1.0 / 5040.0);
    p = fma(p, z, 1.0 / 720.0);
    p = fma(p, z, 1.0 / 120.0);
    p = fma(p, z, 1.0 / 24.0);
    p = fma(p, z, 1.0 / 6.0);
    p = fma(p, z, 0.5);
    p = fma(p, z, 1.0);
    p = fma(p, z, 1.0);
    return __builtin_ldexp(p, static_cast<int>(n));
}

// exp((x - top) / temperature) of x <= top; c = log2(e) / temperature
__device__ __forceinline__ double weight_of(float x, float top, double c) {
    const double a = fmax((static_cast<double>(x) - static_cast<double>(top)) * c, -1100.0);
    return x == top ? 1.0 : exp2_of(a);
}

// in whole units of 2^-44, rounded to nearest: the low bits of w * 2^44 + 2^52
__device__ __forceinline__ u64 units_of(double w) {
    constexpr double kUnit = 17592186044416.0, kShift = 4503599627370496.0;
    return __builtin_bit_cast(u64, fma(w, kUnit, kShift)) - __builtin_bit_cast(u64, kShift);
}

// the order of floats as that of numbers (-0 as 0)
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == 0.f ? 0.f : x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __builtin_bit_cast(float, (k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// What a row asks for.
struct Asked {
    float temperature, min_p;
    double top_p;
    uint32_t top_k;  // vocab: all
    bool valid, greedy;
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

// A wave a chunk, kPer chunks of a row in turn with their loads in flight together.
template <bool kWide, int kPer>
__global__ __launch_bounds__(256) void sample_chunks_kernel(const SampleArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.y, c0 = (blockIdx.x * 4 + wave) * kPer;
    const float* x = a.logits + row * a.stride;
    const Asked ask = asked_of(a, row);
    const bool mass = ask.valid && !ask.greedy && ask.top_k == static_cast<uint32_t>(a.vocab);
    const double c = 1.4426950408889634 / static_cast<double>(ask.temperature);
    bool odd = false;
    if (a.chunk == 256) {
        f32x4 v[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] = four_of<kWide>(x, (c0 + k) * 256 + 4 * lane, a.vocab, odd);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (c0 + k >= a.chunks) break;
            float m = fmaxf(fmaxf(v[k][0], v[k][1]), fmaxf(v[k][2], v[k][3]));
            for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            const size_t at = static_cast<size_t>(row) * a.chunks + c0 + k;
            if (lane == 0) a.chunk_max[at] = m;
            if (!mass) continue;
            double sum = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += v[k][e] == -INFINITY ? 0.0 : weight_of(v[k][e], m, c);
            for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
            if (lane == 0) a.chunk_mass[at] = sum;
        }
    } else {
        for (int k = 0; k < kPer && c0 + k < a.chunks; ++k) {
            const int from = (c0 + k) * a.chunk, to = min(from + a.chunk, a.vocab);
            float m = -INFINITY;
            for (int i = from + 4 * lane; i < to; i += 256) {
                const f32x4 v = four_of<kWide>(x, i, a.vocab, odd);
                m = fmaxf(m, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
            }
            for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            const size_t at = static_cast<size_t>(row) * a.chunks + c0 + k;
            if (lane == 0) a.chunk_max[at] = m;
            if (!mass) continue;
            double sum = 0;
            for (int i = from + 4 * lane; i < to; i += 256) {
                const f32x4 v = four_of<kWide>(x, i, a.vocab, odd);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += v[e] == -INFINITY ? 0.0 : weight_of(v[e], m, c);
            }
            for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
            if (lane == 0) a.chunk_mass[at] = sum;
        }
    }
    if (__any(odd) && lane == 0) a.err[0] = 1;
}

// --------------------------------------------------- the second launch

struct Candidate {
    uint32_t key, index;  // of the logit's order; in the row
};

struct Shared {
    float chunk_max[kSampleChunks];
    u64 chunk_mass[kSampleChunks];
    uint32_t chunk_ties[kSampleChunks];
    uint32_t count[kBins];
    u64 mass[kBins];
    Candidate list[kList];
    u64 wave_sums[kWaves];
    u64 found_before;  // find(): sums up to the place found
    int found, size;
    uint32_t active;
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

// The first of n places (two a thread) up to which the values' sum reaches `need` (1 or
// more), and the sum before it; n where they do not reach it.
template <class F>
__device__ __forceinline__ int find(Shared& s, int n, u64 need, F&& value, u64& before) {
    const int i = 2 * threadIdx.x;
    const u64 v0 = i < n ? value(i) : 0, v1 = i + 1 < n ? value(i + 1) : 0;
    if (threadIdx.x == 0) s.found = n;
    const u64 upto = block_scan(s, v0 + v1), b0 = upto - v1 - v0, b1 = upto - v1;
    if (b0 < need && b1 >= need) {
        s.found = i;
        s.found_before = b0;
    } else if (b1 < need && upto >= need) {
        s.found = i + 1;
        s.found_before = b1;
    }
    __syncthreads();
    before = s.found_before;
    const int at = s.found;
    __syncthreads();
    return at;
}

// A row's candidates: logits in bins 0 .. last of their distance to the maximum.
struct Row {
    const float* x;
    int vocab, chunk, chunks;
    float top, scale;  // scale: bins for two units of a logit
    double c;
    double min_p;

    __device__ __forceinline__ int bin(float v) const {  // kBins: zero weight
        const float d = v == top ? 0.f : 0.5f * top - 0.5f * v;  // (top - v may be beyond f32)
        return static_cast<int>(fminf(d * scale, static_cast<float>(kBins)));
    }
    __device__ __forceinline__ double weight(float v) const { return weight_of(v, top, c); }
    __device__ __forceinline__ u64 units(float v) const { return units_of(weight(v)); }
};

// f(x, index) for the logits of every chunk whose maximum's bin is at most `last`: a
// wave a chunk
template <bool kWide, class F>
__device__ __forceinline__ void each_logit(const Shared& s, const Row& r, int last, F&& f) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int c = wave; c < r.chunks; c += kWaves) {
        if (s.chunk_max[c] == -INFINITY || r.bin(s.chunk_max[c]) > last) continue;
        for (int i = c * r.chunk + 4 * lane; i < min((c + 1) * r.chunk, r.vocab); i += 256) {
            bool odd = false;
            const f32x4 v = four_of<kWide>(r.x, i, r.vocab, odd);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[e] != -INFINITY) f(v[e], i + e);
        }
    }
}

// Which logits are kept: bins before `bin`, and in it those above `key`; of those at
// `key` the first `ties` by index.
struct Border {
    int bin;
    uint32_t key;
    u64 ties;
    u64 above_count, above_mass;  // what lies above the ties
};

// The place in the order, from the largest down, at which `need` is reached, by counts
// or masses (by_mass), among the logits of bin b; `count` and `mass` are what the bins
// before hold.  They come from the list, or (listed false) from memory.
template <bool kWide>
__device__ __forceinline__ Border place(Shared& s, const Row& r, int b, bool listed, int listed_n, bool by_mass, u64 need, u64 count,
                                        u64 mass) {
    // exact, by the bits of the keys: 11, 11 and 10 at a time
    uint32_t prefix = 0, mask = 0;
    for (int shift = 21; shift >= 0; shift -= shift == 21 ? 11 : 10) {
        const int bits = shift ? 11 : 10, n = 1 << bits;
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            s.count[i] = 0;
            s.mass[i] = 0;
        }
        __syncthreads();
        auto take = [&](uint32_t key, float x) {
            if ((key & mask) != prefix) return;
            const int at = n - 1 - static_cast<int>(key >> shift & (n - 1));
            atomicAdd(&s.count[at], 1u);
            const u64 w = r.units(x);
            if (w) atomicAdd(&s.mass[at], w);
        };
        if (listed) {
            for (int i = threadIdx.x; i < listed_n; i += kThreads) {
                const uint32_t key = s.list[i].key;
                if (r.bin(unordered(key)) == b) take(key, unordered(key));
            }
        } else {
            each_logit<kWide>(s, r, b, [&](float x, int) {
                if (r.bin(x) == b) take(ordered(x), x);
            });
        }
        __syncthreads();
        u64 before = 0;
        int at;
        if (by_mass)
            at = find(s, n, need - mass, [&](int i) { return s.mass[i]; }, before);
        else
            at = find(s, n, need - count, [&](int i) { return static_cast<u64>(s.count[i]); }, before);
        // sums of the other kind before the place
        u64 other = 0;
        for (int i = threadIdx.x; i < at && i < n; i += kThreads) other += by_mass ? s.count[i] : s.mass[i];
        other = block_scan(s, other);
        __syncthreads();
        if (threadIdx.x == kThreads - 1) s.found_before = other;
        __syncthreads();
        other = s.found_before;
        __syncthreads();
        count += by_mass ? other : before;
        mass += by_mass ? before : other;
        mask |= static_cast<uint32_t>(n - 1) << shift;
        prefix |= static_cast<uint32_t>(n - 1 - min(at, n - 1)) << shift;
    }
    Border o;
    o.bin = b;
    o.key = prefix;
    o.above_count = count;
    o.above_mass = mass;
    const u64 each = r.units(unordered(prefix));
    o.ties = by_mass ? (each ? (need - mass + each - 1) / each : 0) : need - count;
    return o;
}

template <bool kWide>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(const SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const Asked ask = asked_of(a, row);
    const float u = a.uniforms[row];
    const uint32_t vocab = a.vocab;
    auto answer = [&](uint32_t token, float p) {
        a.tokens[row] = token;
        if (a.probability) a.probability[row] = p;
    };
    if (!ask.valid || !(u >= 0.f && u < 1.f)) {
        if (tid == 0) {
            a.err[1] = 1;
            answer(kNone, 0.f);
        }
        return;
    }
    Row r;
    r.x = a.logits + row * a.stride;
    r.vocab = a.vocab;
    r.chunk = a.chunk;
    r.chunks = a.chunks;
    const size_t at0 = static_cast<size_t>(row) * a.chunks;
    // the row's maximum
    float mine = -INFINITY;
    if (tid < a.chunks) s.chunk_max[tid] = mine = a.chunk_max[at0 + tid];
    float top = mine;
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) s.wave_sums[tid >> 6] = __builtin_bit_cast(uint32_t, top);
    if (tid == 0) s.size = 0;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, __builtin_bit_cast(float, static_cast<uint32_t>(s.wave_sums[w])));
    r.top = top;
    if (top == -INFINITY) {  // nothing to draw
        if (tid == 0) {
            a.err[0] = 1;
            answer(kNone, 0.f);
        }
        return;
    }
    if (ask.greedy) {  // the lowest index of the maximum, in the first chunk that has it
        if (tid == 0) s.found = a.chunks;
        __syncthreads();
        if (mine == top) atomicMin(&s.found, tid);
        __syncthreads();
        const int c = s.found;
        if (tid >= 64) return;
        for (int i = c * a.chunk; i < min((c + 1) * a.chunk, a.vocab); i += 64) {
            const u64 hit = __ballot(i + lane < a.vocab && r.x[min(i + lane, a.vocab - 1)] == top);
            if (!hit) continue;
            if (lane == 0) answer(static_cast<uint32_t>(i + __builtin_ctzll(hit)), 1.f);
            return;
        }
        return;
    }
    r.c = 1.4426950408889634 / static_cast<double>(ask.temperature);
    r.scale = fminf(2.f * kBins / kSpan / ask.temperature, 3e38f);
    r.min_p = ask.min_p;
    const bool by_k = ask.top_k < vocab, by_p = ask.top_p < 1.0;
    // the chunks' masses, and all of it (where top-k does not leave that open)
    u64 total = 0;
    if (!by_k) {
        u64 units = 0;
        if (mine != -INFINITY) units = static_cast<u64>(__builtin_rint(a.chunk_mass[at0 + tid] * r.weight(mine) * 17592186044416.0));
        if (tid < a.chunks) s.chunk_mass[tid] = units;
        total = block_scan(s, units);
        __syncthreads();
        if (tid == kThreads - 1) s.found_before = total;
        __syncthreads();
        total = s.found_before;
        __syncthreads();
    }
    const u64 need_p = by_p && !by_k ? max(static_cast<u64>(__builtin_ceil(ask.top_p * static_cast<double>(total))), u64(1)) : 0;

    Border kept{kBins, 0, 0, 0, 0};  // everything
    bool all = !by_k && !by_p && r.min_p == 0.0;
    if (!all) {
        // The last bin that can hold a kept logit.
        int last = kBins - 1;
        auto down_to = [&](double w) {  // the bin of a weight, or the one behind it
            last = min(last, static_cast<int>(fminf(-__log2f(static_cast<float>(w)) * 0.693147181f * (kBins / kSpan), 2.f * kBins)) + 1);
        };
        if (!by_k && r.min_p > 0.0) down_to(r.min_p);
        // weights below (1 - p) of the mean weigh less than 1 - p together
        if (need_p) down_to(fmin((1.0 - ask.top_p) * static_cast<double>(total) / 17592186044416.0 / vocab, 1.0));
        // the chunks' maxima alone reach k, or p of the mass
        if (need_p || (by_k && ask.top_k <= static_cast<uint32_t>(a.chunks))) {
            for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0;
            __syncthreads();
            if (mine != -INFINITY) {
                const int b = r.bin(mine);
                if (b < kBins) atomicAdd(&s.mass[b], by_k ? u64(1) : r.units(mine));
            }
            __syncthreads();
            u64 before;
            last = min(last, find(s, kBins, by_k ? ask.top_k : need_p, [&](int i) { return s.mass[i]; }, before));
        }
        // The candidates: into the list while there is room, and into the bins.
        for (int i = tid; i < kBins; i += kThreads) {
            s.count[i] = 0;
            s.mass[i] = 0;
        }
        __syncthreads();
        each_logit<kWide>(s, r, last, [&](float x, int i) {
            const int b = r.bin(x);
            if (b > last) return;
            const int at = atomicAdd(&s.size, 1);
            if (at < kList) s.list[at] = {ordered(x), static_cast<uint32_t>(i)};
            if (by_k) atomicAdd(&s.count[b], 1u);
            if (!by_p) return;
            const u64 w = r.units(x);
            if (w) atomicAdd(&s.mass[b], w);
        });
        __syncthreads();
        const int size = s.size;
        bool listed = size <= kList;
        // what is collected of a bin, where the list does not hold them all
        auto collect = [&](int b) {
            if (listed) return size;
            __syncthreads();
            if (tid == 0) s.size = 0;
            __syncthreads();
            each_logit<kWide>(s, r, b, [&](float x, int i) {
                if (r.bin(x) != b) return;
                const int at = atomicAdd(&s.size, 1);
                if (at < kList) s.list[at] = {ordered(x), static_cast<uint32_t>(i)};
            });
            __syncthreads();
            return s.size;
        };
        kept.bin = last;  // (no key is 0: all of it)
        int in_list = size;
        bool bin_listed = listed;
        // (the bins' counts and masses are overwritten by place(): both bins first)
        u64 count_before = 0, mass_before = 0;
        int bk = kBins;
        if (by_k && static_cast<u64>(size) > ask.top_k) {
            u64 before;
            bk = find(s, kBins, ask.top_k, [&](int i) { return static_cast<u64>(s.count[i]); }, before);
            count_before = before;
        }
        // masses up to each bin stay in registers: two bins a thread
        const u64 m0 = s.mass[2 * tid], m1 = s.mass[2 * tid + 1];
        const u64 upto = block_scan(s, m0 + m1);
        auto mass_up_to = [&](int b) {  // of the bins before b
            __syncthreads();
            if (2 * tid == b) s.found_before = upto - m0 - m1;
            if (2 * tid + 1 == b) s.found_before = upto - m1;
            if (b == kBins && tid == kThreads - 1) s.found_before = upto;
            __syncthreads();
            const u64 v = s.found_before;
            __syncthreads();
            return v;
        };
        if (bk < kBins) {
            mass_before = mass_up_to(bk);
            in_list = collect(bk);
            bin_listed = in_list <= kList;
            kept = place<kWide>(s, r, bk, bin_listed, in_list, false, ask.top_k, count_before, mass_before);
        }
        if (by_p) {
            u64 need = need_p;
            if (by_k) {
                total = bk < kBins ? kept.above_mass + kept.ties * r.units(unordered(kept.key)) : mass_up_to(kBins);
                need = max(static_cast<u64>(__builtin_ceil(ask.top_p * static_cast<double>(total))), u64(1));
            }
            // the bin at which the mass is reached
            __syncthreads();
            if (tid == 0) s.found = kBins;
            __syncthreads();
            if (upto - m0 - m1 < need && upto - m1 >= need) s.found = 2 * tid;
            if (upto - m1 < need && upto >= need) s.found = 2 * tid + 1;
            __syncthreads();
            const int bp = s.found;
            __syncthreads();
            if (bp < kBins && bp <= kept.bin) {
                const u64 before = mass_up_to(bp);
                if (bp != bk) {
                    in_list = collect(bp);
                    bin_listed = in_list <= kList;
                }
                const Border p = place<kWide>(s, r, bp, bin_listed, in_list, true, need, 0, before);
                // (top-k's border lies behind, or leaves fewer of the same ties)
                if (bk == kBins || p.bin < kept.bin || p.key > kept.key || (p.key == kept.key && p.ties < kept.ties)) kept = p;
            }
        }
        // what is kept, by chunks
        __syncthreads();
        if (tid < a.chunks) {
            s.chunk_mass[tid] = 0;
            s.chunk_ties[tid] = 0;
        }
        __syncthreads();
        auto add = [&](float x, int i, int b) {
            const double w = r.weight(x);
            if (w < r.min_p) return;
            const uint32_t key = ordered(x);
            if (b == kept.bin && key <= kept.key) {
                if (key == kept.key) atomicAdd(&s.chunk_ties[i / a.chunk], 1u);
                return;
            }
            const u64 units = units_of(w);
            if (units) atomicAdd(&s.chunk_mass[i / a.chunk], units);
        };
        if (listed) {
            for (int k = tid; k < size; k += kThreads) {
                const float x = unordered(s.list[k].key);
                const int b = r.bin(x);
                if (b <= kept.bin) add(x, static_cast<int>(s.list[k].index), b);
            }
        } else {
            each_logit<kWide>(s, r, min(kept.bin, last), [&](float x, int i) {
                const int b = r.bin(x);
                if (b <= kept.bin && b <= last) add(x, i, b);
            });
        }
        __syncthreads();
    }
    // ties by index, then the chunk and the token that the random number falls on
    const u64 each = kept.bin < kBins ? r.units(unordered(kept.key)) : 0;
    u64 ties = 0, ties_before = 0, units = 0;
    if (!all) {
        ties = tid < a.chunks ? s.chunk_ties[tid] : 0;
        ties_before = block_scan(s, ties) - ties;
    }
    if (tid < a.chunks) {
        units = s.chunk_mass[tid];
        if (ties_before < kept.ties) units += min(ties, kept.ties - ties_before) * each;
    }
    const u64 upto = block_scan(s, units);
    __syncthreads();
    if (tid == kThreads - 1) s.found_before = upto;
    if (tid == 0) s.found = a.chunks - 1;
    __syncthreads();
    const u64 sum = s.found_before;
    const u64 target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(sum));
    __syncthreads();
    if (upto - units <= target && upto > target) {
        s.found = tid;
        s.mass[0] = target - (upto - units);
        s.mass[1] = ties_before;
    }
    __syncthreads();
    if (tid >= 64) return;
    const int c = s.found;
    u64 left = s.mass[0], rank = s.mass[1];
    uint32_t token = kNone;
    float x_token = top;
    int last_kept = -1;
    for (int i0 = c * a.chunk; i0 < min((c + 1) * a.chunk, a.vocab); i0 += 256) {
        bool odd = false;
        const int i = i0 + 4 * lane;
        const f32x4 v = four_of<kWide>(r.x, i, a.vocab, odd);
        u64 w[4];
        uint32_t tied = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = 0;
            if (v[e] == -INFINITY) continue;
            const int b = r.bin(v[e]);
            const double weight = r.weight(v[e]);
            if (b > kept.bin || b >= kBins || weight < r.min_p) continue;
            const uint32_t key = ordered(v[e]);
            if (b == kept.bin && key == kept.key) tied |= 1u << e;
            if (b < kept.bin || key > kept.key) w[e] = units_of(weight);
        }
        const u64 tied_upto = wave_scan(__builtin_popcount(tied));
        u64 before = rank + tied_upto - __builtin_popcount(tied);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (tied >> e & 1) {
                if (before < kept.ties) w[e] = each;
                ++before;
            }
        rank += __shfl(tied_upto, 63);
        const u64 own = w[0] + w[1] + w[2] + w[3], upto_here = wave_scan(own);
        const u64 any = __ballot(own != 0);
        if (any) last_kept = i0 + 4 * (63 - __builtin_clzll(any));
        const u64 hit = __ballot(upto_here > left);
        if (hit) {
            const int who = __builtin_ctzll(hit);
            u64 from = upto_here - own;
            int e = 0;
            while (e < 3 && from + w[e] <= left) from += w[e++];
            token = __shfl(static_cast<uint32_t>(i + e), who);
            x_token = __shfl(e == 0 ? v[0] : e == 1 ? v[1] : e == 2 ? v[2] : v[3], who);
            break;
        }
        left -= __shfl(upto_here, 63);
    }
    if (token == kNone) {
        // the chunk's mass was summed before it was rounded: its last kept token, or,
        // where each alone rounds to nothing, its maximum
        const float want = s.chunk_max[c];
        for (int i = c * a.chunk + lane; i < min((c + 1) * a.chunk, a.vocab) && token == kNone; i += 64) {
            const u64 hit = __ballot(last_kept >= 0 ? i >= last_kept && r.bin(r.x[i]) < kBins && r.units(r.x[i]) : r.x[i] == want);
            if (hit) token = static_cast<uint32_t>(i - lane + __builtin_ctzll(hit));
        }
        token = __builtin_amdgcn_readfirstlane(token);
        if (token < vocab) x_token = r.x[token];
    }
    if (lane == 0) answer(token, static_cast<float>(r.weight(x_token) / (static_cast<double>(sum) / 17592186044416.0)));
}

}  // namespace

void launch_sample(const SampleArgs& a, hipStream_t s) {
    const bool wide = a.stride % 4 == 0;
    // four chunks a wave where the waves are many
    const int per = static_cast<size_t>(a.rows) * a.chunks >= 16384 ? 4 : 1;
    const dim3 grid(static_cast<unsigned>((a.chunks + 4 * per - 1) / (4 * per)), static_cast<unsigned>(a.rows));
    auto chunks = [&](auto kernel) { launch("sample_chunks", kernel, grid, dim3(256), 0, s, a); };
    if (wide)
        per == 4 ? chunks(sample_chunks_kernel<true, 4>) : chunks(sample_chunks_kernel<true, 1>);
    else
        per == 4 ? chunks(sample_chunks_kernel<false, 4>) : chunks(sample_chunks_kernel<false, 1>);
    launch("sample_pick", wide ? sample_pick_kernel<true> : sample_pick_kernel<false>, dim3(static_cast<unsigned>(a.rows)),
           dim3(kThreads), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

// Scored attention (score.hip) on the matrix cores, for head_dim 64 and 128 over f32
// or Q8_0 blocks of a power of two from 16 tokens.
//
// An attention row is a (row, query head) pair; the rows of a block share the keys of
// their KV head.  Scores S^T = K Q^T and outputs O^T = V^T P^T both have the row in
// lane % 16, so that what the softmax does to a row stays in its four lanes, and the
// probabilities are the second product's operand where they are.  Steps that some row
// sees only a part of are masked by the rows' ranges; in them a value that is not
// finite is taken out of the product, in which zero times it would reach every row,
// and added to the rows that see it.
#include <type_traits>

#include "score_util.hpp"

namespace tvara_amd {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr float kThreshold = 8.0f;
constexpr int kBufferWord3 = 0x00020000;  // gfx9 buffer descriptor, dword 3

// A workgroup's work (ScoreArgs::work)
struct Item {
    int table, tokens, rows, row0, head, heads, step, end, run, runs, slot, position;
};
__device__ __forceinline__ Item item_of(const ScoreArgs& a, unsigned i) {
    const int4 x = a.work[3 * static_cast<size_t>(i)], y = a.work[3 * static_cast<size_t>(i) + 1], z = a.work[3 * static_cast<size_t>(i) + 2];
    return {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
}

__device__ __forceinline__ bf16x8 both(bf16x4 x, bf16x4 y) { return bf16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}; }
__device__ __forceinline__ bf16x8 eight(f32x4 x, f32x4 y) {
    return both(__builtin_convertvector(x, bf16x4), __builtin_convertvector(y, bf16x4));
}
// Eight values as three parts in bf16, each the rest's nearest.
__device__ __forceinline__ void split3(f32x4 x, f32x4 y, bf16x8 (&p)[3]) {
    bf16x4 part[2][3];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        f32x4 rest = half ? y : x;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            part[half][i] = __builtin_convertvector(rest, bf16x4);
            rest -= __builtin_convertvector(part[half][i], f32x4);
        }
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) p[i] = both(part[0][i], part[1][i]);
}

// max / min over the 16 lanes of a row of a wave, to a scalar
__device__ __forceinline__ int uniform_max(int v) {
    for (int o = 8; o >= 1; o >>= 1) v = max(v, __shfl_xor(v, o));
    return __builtin_amdgcn_readfirstlane(v);
}

// maximum over the n lanes (8 or 16, from a multiple of n) of a key's row
template <int kControl>
__device__ __forceinline__ float moved(float v) {
    const int b = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, kControl, 0xf, 0xf, false));
}
template <int n>
__device__ __forceinline__ float row_max(float v) {
    constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;
    v = fmaxf(v, moved<kSwap1>(v));
    v = fmaxf(v, moved<kSwap2>(v));
    v = fmaxf(v, moved<kHalfMirror>(v));
    return n == 16 ? fmaxf(v, moved<kMirror>(v)) : v;
}

// ------------------------------------------------------------- few rows

constexpr int kFewStep = 32, kFewWaves = 4;

// Up to 16 attention rows in f32 (v_mfma_f32_16x16x4_f32): four waves take steps of
// 32 keys in turn, with no barrier until the end, where their results meet in LDS.
// Bound: HBM; keys of f32 blocks come as whole rows into the wave's own part of LDS
// without passing registers (as operands they take four times as long through the CU's
// cache), values straight into registers as the product has them.  48 contexts of 100
// to 3,000 tokens, 32 heads on 8 of 64 (315 MB): 68 us, 4.6 TB/s, nearly a large copy's
// rate; one of 700, nine heads on three: 7 us, a chain of three reads.
template <int D>
__global__ __launch_bounds__(64 * kFewWaves, 2) void score_tile_kernel(const ScoreArgs a) {
    constexpr int WK = kFewWaves, C = D / 16, H = D / 64;
    constexpr int W = D / 4;  // 16-byte parts of a row
    __shared__ f32x4 staged[WK][kFewStep * W];
    auto result = [&](int w, int i) -> f32x4& { return staged[w][i * 64 + static_cast<int>(threadIdx.x & 63)]; };
    __shared__ float2 stats[WK][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    const Item it = item_of(a, blockIdx.x);
    if (!it.rows) return;  // the list's padding
    const int kh = it.head / a.group, kvw = a.lay.kv_width, tokens = it.tokens;

    // this lane's row
    const int index = r16 / it.heads, head = it.head + r16 - index * it.heads;
    const bool live = index < it.rows;
    const int position = it.position + index;
    const size_t row = static_cast<size_t>(it.row0) + index;
    const int2 range = live ? a.ranges[row] : make_int2(0, 0);
    const float slope = a.slopes && live ? a.slopes[head] : 0.f;
    const int lo = uniform_max(range.x), hi = -uniform_max(live ? -range.y : -0x7fffffff);  // keys that all rows see: [lo, hi)

    // column of element 0 of a lane's c-th four of a key, and of the h-th four of
    // a value (r: the loading lane's r16, or an output row of the tiles)
    auto kcol = [&](int c) { return 16 * c + 4 * g; };
    auto vcol = [](int h, int r) { return 64 * h + 4 * r; };

    const int tpb = a.lay.tpb, tsh = __builtin_ctz(static_cast<unsigned>(tpb));
    const int32_t* tab = a.tables + it.table;
    const size_t kbytes = (static_cast<size_t>(a.layer) * 2 * tpb * kvw + static_cast<size_t>(kh) * D) * sizeof(float);
    const size_t vsec = static_cast<size_t>(tpb) * kvw * sizeof(float);
    const int rowb = kvw * static_cast<int>(sizeof(float));  // from one slot to the next
    const unsigned koff = static_cast<unsigned>(lane / W * rowb + (lane % W ^ lane / W) * 16);
    const unsigned voff = static_cast<unsigned>(4 * g * rowb + vcol(0, r16) * 4);
    int step = it.step + wave;
    const int last = max(tokens - 1, 0) >> 4;  // 16 keys a table lookup; past the end the last again
    // lane 2i + mt: the block of the wave's i-th step from here
    auto lookup = [&](int from) { return tokens ? tab[min(2 * (from + (lane >> 1) * WK) + (lane & 1), last) << 4 >> tsh] : 0; };
    int ids = lookup(step), more = lookup(step + 32 * WK), at = 0;
    auto block = [&](int mt, int stp) {
        const int id = __builtin_amdgcn_readlane(ids, 2 * at + mt);
        const int slot = (min(2 * stp + mt, last) << 4) & (tpb - 1);
        return a.pool + static_cast<size_t>(id) * a.lay.stride + kbytes + static_cast<size_t>(slot) * rowb;
    };
    f32x4 qf[C];
    f32x4 v[2][4][H];
    auto load_k = [&](int stp) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const char* b = block(mt, stp);
            // straight into LDS, lane after lane; what a lane loads is permuted by its
            // row, so that the operands' reads meet no bank twice
            const __amdgpu_buffer_rsrc_t rows =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(b), 0, 15 * rowb + 4 * D, kBufferWord3);
#pragma unroll
            for (int c = 0; c < C; ++c)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (__attribute__((address_space(3))) void*)&staged[wave][(mt * C + c) * 64],
                                                         16, koff ^ 1024 / W * c, 64 / W * c * rowb, 0, 0);
        }
    };
    auto load_v = [&](int stp) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const char* b = block(mt, stp) + vsec;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int h = 0; h < H; ++h)
                    v[mt][i][h] = *reinterpret_cast<const f32x4*>(b + static_cast<size_t>(i) * rowb + voff + 256 * h);
        }
    };
    {
        const float* qp = a.q + (row * a.heads + head) * D;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            qf[c] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (live) qf[c] = *reinterpret_cast<const f32x4*>(qp + kcol(c));
        }
    }
    if (step < it.end) {
        load_k(step);
        asm volatile("" ::: "memory");
        load_v(step);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) qf[c] *= a.qscale;

    f32x4 acc[4 * H];  // tile (h, j) at 4h + j
    float m = -INFINITY, l = 0.f, rounded = 0.f, nonfinite = 0.f;  // nonfinite: NaN once a score is not finite
#pragma unroll
    for (int dt = 0; dt < 4 * H; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 s[2];  // scores, then probabilities, of keys 16mt + 4g + i
    auto key_part = [&](int mt, int c) __attribute__((always_inline)) { return staged[wave][(16 * mt + r16) * W + ((4 * c + g) ^ r16)]; };
    auto value = [&](int mt, int i, int h, auto j) __attribute__((always_inline)) { return v[mt][i][h][j.value]; };
    auto every_tile = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            f(h, std::integral_constant<int, 0>{});
            f(h, std::integral_constant<int, 1>{});
            f(h, std::integral_constant<int, 2>{});
            f(h, std::integral_constant<int, 3>{});
        }
    };
    // the lane's columns of key 16mt + 4g + i
    auto finite_value = [&](int mt, int i) __attribute__((always_inline)) {
        bool fine = true;
#pragma unroll
        for (int h = 0; h < H; ++h) fine &= all_finite(v[mt][i][h]);
        return fine;
    };
    auto drop_odd = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[mt][i][h][j] = __builtin_isfinite(v[mt][i][h][j]) ? v[mt][i][h][j] : 0.f;
            }
    };
    for (; step < it.end; step += WK) {
        const int next = step + WK, key0 = kFewStep * step;
        wait_until_left<8 * H>();  // the values'
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            s[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const f32x4 k = key_part(mt, c);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i], qf[c][i], s[mt], 0, 0, 0);
            }
        }
        wait_for_lds();
        // the loads of the next step go out as soon as there is room (past the end the
        // last step's again: its blocks are there)
        if (++at == 32) {
            at = 0;
            ids = more;
            more = lookup(next + 32 * WK);
        }
        load_k(next);
        asm volatile("" ::: "memory");
        const bool whole = key0 >= lo && key0 + kFewStep <= hi;  // every row sees every key
        const int first = range.x - key0 - 4 * g, end = range.y - key0 - 4 * g;  // of the lane's keys 16mt + i
        if (whole) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) nonfinite = fmaf(s[mt][i], 0.f, nonfinite);
        } else {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool on = 16 * mt + i >= first && 16 * mt + i < end;
                    s[mt][i] = on ? s[mt][i] : 0.f;
                    nonfinite = fmaf(s[mt][i], 0.f, nonfinite);
                }
        }
        if (a.cap != 0.f) {
            float most = 0.f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) most = fmaxf(most, __builtin_fabsf(s[mt][i]));
            const bool small = !__any(most > kSmallTanh);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt][i] = a.cap * (small ? small_tanh(s[mt][i]) : both_tanh(s[mt][i]));
        }
        if (a.slopes) {
            const int away = position - key0 - 4 * g;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt][i] = fmaf(-slope, static_cast<float>(abs(away - 16 * mt - i)), s[mt][i]);
        }
        if (!whole) {
            bool odd = false;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (16 * mt + i < first || 16 * mt + i >= end) s[mt][i] = -INFINITY;
                    odd |= !finite_value(mt, i);
                }
            if (__any(odd)) {
                // A row that sees such a value has a column that is not finite: their
                // product as ones and zeros counts them.
                auto count = [&](int h, auto j) __attribute__((always_inline)) {
                    f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool on = 16 * mt + i >= first && 16 * mt + i < end;
                            part = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_isfinite(value(mt, i, h, j)) ? 0.f : 1.f, on ? 1.f : 0.f,
                                                                        part, 0, 0, 0);
                        }
#pragma unroll
                    for (int o = 0; o < 4; ++o) acc[4 * h + j.value][o] += part[o] != 0.f ? NAN : 0.f;
                };
                every_tile(count);
                drop_odd();
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[mt][i]);
        if (__any(mx > m + kThreshold)) {
            const float mn = fmaxf(m, cross_row_max(mx));
            const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mn);
            m = mn;
            l *= alpha;
            rounded *= alpha;
#pragma unroll
            for (int dt = 0; dt < 4 * H; ++dt) acc[dt] *= alpha;
        }
        const float base = m == -INFINITY ? 0.f : m;  // (no key seen yet: probabilities 0)
        float sum = 0.f;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[mt][i] = fast_exp2(s[mt][i] - base);
                sum += s[mt][i];
            }
        add_to(l, rounded, sum);
        // a step's part is a chain of eight from zero, added to the rest: as short as a
        // long context's sums need it
        auto tile = [&](int h, auto j) __attribute__((always_inline)) {
            f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) part = __builtin_amdgcn_mfma_f32_16x16x4f32(value(mt, i, h, j), s[mt][i], part, 0, 0, 0);
            acc[4 * h + j.value] += part;
        };
        every_tile(tile);
        load_v(next);
    }
    wait_until_left<0>();  // (LDS is used again)

    // ---- the waves that shared these rows' keys, together
    float total = cross_row_sum(l);
    nonfinite = fmaf(total, 0.f, nonfinite);  // (a score and its bias may be finite and their sum not)
    if (__any(nonfinite != 0.f) && lane == 0) *a.err = 1;
    if (g == 0) stats[wave][r16] = make_float2(m, total);
    __syncthreads();
    {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, stats[w][r16].x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WK; ++w) sum = fmaf(fast_exp2(stats[w][r16].x - base), stats[w][r16].y, sum);
        const float scale = fast_exp2(m - base);
#pragma unroll
        for (int dt = 0; dt < 4 * H; ++dt) acc[dt] *= scale;
        m = top;
        total = sum;
    }
    // four columns of output row 4g + i of the tiles
#pragma unroll
    for (int h = 0; h < H; ++h) {
        if (h) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) result(wave, i) = f32x4{acc[4 * h][i], acc[4 * h + 1][i], acc[4 * h + 2][i], acc[4 * h + 3][i]};
        __syncthreads();
        f32x4 x = result(0, wave);
#pragma unroll
        for (int w = 1; w < WK; ++w) x += result(w, wave);
        if (!live) continue;
        if (it.runs == 1) {
            *reinterpret_cast<f32x4*>(a.out + (row * a.heads + head) * D + vcol(h, 4 * g + wave)) = x / (total != 0.f ? total : 1.f);
        } else {
            const size_t p = (static_cast<size_t>(it.slot) + static_cast<size_t>(index) * it.runs + it.run) * a.heads + head;
            *reinterpret_cast<f32x4*>(a.part_acc + p * D + vcol(h, 4 * g + wave)) = x;
            if (h == 0 && wave == 0 && g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * p) = make_float2(m, total);
        }
    }
}

// The same over Q8_0 blocks, whose bytes are operands as they are: 16x16x32 products of
// bf16, which holds a byte exactly, with queries and probabilities in three bf16 parts
// (24 bits, f32's range).  A product over 32 columns is one group's: scores are multiplied
// by the group's scale behind it, probabilities before, one column group after the other.
// A wave's bytes go straight into LDS, the next step's keys once the scores have read
// these, its values behind the products; the queries' parts are there too, for registers
// of three waves on a SIMD: eight contexts of 16,000 to 32,768 tokens, 32 heads on 8 of 128
// (390 MB), take 95 us (4.1 TB/s), bound by the 850 vector instructions of a step, and 140 us
// with the next step's bytes in registers and two waves.  (In f32 products the matrix
// instructions bound it, at 224 us.)
template <int D>
__global__ __launch_bounds__(64 * kFewWaves, 3) void score_tile_q8_kernel(const ScoreArgs a) {
    constexpr int WK = kFewWaves, KC = D / 32, H = D / 64;
    // a wave's keys, values and scales of a step, straight from memory: the next step's keys are
    // loaded once the scores have read them, its values behind the products.  At the end the
    // wave's results, for the others.
    struct alignas(16) Step {
        char rows[2][kFewStep * D];     // keys, values; 16 bytes at p hold those at p ^ row % 8 (128 columns)
        char scales[2][kFewStep * KC * 2];
    };
    __shared__ union {
        Step step;
        f32x4 result[4 * 64];
    } staged[WK];
    auto result = [&](int w, int i) -> f32x4& { return staged[w].result[i * 64 + static_cast<int>(threadIdx.x & 63)]; };
    __shared__ float2 stats[WK][16];
    __shared__ u32x4 queries[KC][3][64];  // in three parts, the same for all waves
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    const Item it = item_of(a, blockIdx.x);
    if (!it.rows) return;  // the list's padding
    const int kh = it.head / a.group, tokens = it.tokens;

    // this lane's row
    const int index = r16 / it.heads, head = it.head + r16 - index * it.heads;
    const bool live = index < it.rows;
    const int position = it.position + index;
    const size_t row = static_cast<size_t>(it.row0) + index;
    const int2 range = live ? a.ranges[row] : make_int2(0, 0);
    const float slope = a.slopes && live ? a.slopes[head] : 0.f;
    const int lo = uniform_max(range.x), hi = -uniform_max(live ? -range.y : -0x7fffffff);  // keys that all rows see: [lo, hi)

    const int tpb = a.lay.tpb, tsh = __builtin_ctz(static_cast<unsigned>(tpb));
    const int32_t* tab = a.tables + it.table;
    const size_t kbytes = static_cast<size_t>(a.layer) * 2 * a.lay.section + static_cast<size_t>(kh) * a.lay.head_bytes, vsec = a.lay.section;
    int step = it.step + wave;
    const int last = max(tokens - 1, 0) >> 4;  // 16 keys a table lookup; past the end the last again
    // lane 2i + mt: the block of the wave's i-th step from here
    auto lookup = [&](int from) { return tokens ? tab[min(2 * (from + (lane >> 1) * WK) + (lane & 1), last) << 4 >> tsh] : 0; };
    int ids = lookup(step), more = lookup(step + 32 * WK), at = 0;
    constexpr int P = D / 16;            // 16-byte parts of a row
    constexpr int kLoads = 2 * D / 64 + 1;  // of a step's keys or values
    const int swap = P - 1;                 // of a part's place, by row
    unsigned part_at[D / 64];
#pragma unroll
    for (int n = 0; n < D / 64; ++n) {  // 64 / P keys a load
        const int row = 64 / P * n + lane / P;
        part_at[n] = row * D + ((lane % P) ^ (row & swap)) * 16;
    }
    auto load = [&](int kind, int stp) __attribute__((always_inline)) {
        typedef __attribute__((address_space(1))) const void* global;
        typedef __attribute__((address_space(3))) void* shared;
        const char* scales[2];
        Step& to = staged[wave].step;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const int id = __builtin_amdgcn_readlane(ids, 2 * at + mt), slot = (min(2 * stp + mt, last) << 4) & (tpb - 1);
            const char* b = a.pool + static_cast<size_t>(id) * a.lay.stride + kbytes + kind * vsec;
            const char* from = b + static_cast<size_t>(slot) * D;
            scales[mt] = b + static_cast<size_t>(tpb) * D + static_cast<size_t>(slot) * KC * 2;
#pragma unroll
            for (int n = 0; n < D / 64; ++n)
                __builtin_amdgcn_global_load_lds((global)(from + part_at[n]), (shared)(to.rows[kind] + (16 * mt) * D + 1024 * n), 16, 0, 0);
        }
        // (of 64 columns half of the lanes are enough)
        const char* x = (lane / (8 * KC) & 1 ? scales[1] : scales[0]) + lane % (8 * KC) * 4;
        if (lane < 16 * KC) __builtin_amdgcn_global_load_lds((global)x, (shared)to.scales[kind], 4, 0, 0);
    };
    // bytes of key 16 mt + r16, columns 32 kc + 8 g on; of keys 16 mt + 4 g + i, columns 32 kc + 2 r16 on
    auto key_bytes = [&](int mt, int kc) __attribute__((always_inline)) {
        return *reinterpret_cast<const u32x2*>(staged[wave].step.rows[0] + (16 * mt + r16) * D + ((2 * kc + (g >> 1)) ^ (r16 & swap)) * 16 + 8 * (g & 1));
    };
    auto value_bytes = [&](int mt, int i, int kc) __attribute__((always_inline)) {
        const int row = 4 * g + i;
        return static_cast<unsigned>(*reinterpret_cast<const uint16_t*>(staged[wave].step.rows[1] + (16 * mt + row) * D +
                                                                         ((2 * kc + (r16 >> 3)) ^ (row & swap)) * 16 + 2 * (r16 & 7)));
    };
    auto query = [&](int kc, int part) __attribute__((always_inline)) { return __builtin_bit_cast(bf16x8, queries[kc][part][lane]); };
    struct Scales {
        _Float16 d[4][KC];
    };
    // (read as vectors: a read of a struct waits for every load into LDS that is on its way)
    auto scales_of = [&](int kind, int mt) __attribute__((always_inline)) {
        const f32x4* x = reinterpret_cast<const f32x4*>(staged[wave].step.scales[kind] + (16 * mt + 4 * g) * KC * 2);
        struct {
            f32x4 v[KC / 2];
        } all;
#pragma unroll
        for (int i = 0; i < KC / 2; ++i) all.v[i] = x[i];
        return __builtin_bit_cast(Scales, all);
    };
    if (wave < KC) {
        const float* qp = a.q + (row * a.heads + head) * D + 8 * g + 32 * wave;
        f32x4 x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (live) x[i] = *reinterpret_cast<const f32x4*>(qp + 4 * i);
        }
        bf16x8 q[3];
        split3(x[0] * a.qscale, x[1] * a.qscale, q);
#pragma unroll
        for (int i = 0; i < 3; ++i) queries[wave][i][lane] = __builtin_bit_cast(u32x4, q[i]);
    }
    static_assert(KC <= WK);
    __syncthreads();
    f32x4 acc[2 * KC];  // columns 32 kc + 2 m + e at 2 kc + e, m being the tile's row
    float m = -INFINITY, l = 0.f, rounded = 0.f, nonfinite = 0.f;  // nonfinite: NaN once a score is not finite
#pragma unroll
    for (int dt = 0; dt < 2 * KC; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto advance = [&](int next) {
        if (++at == 32) {
            at = 0;
            ids = more;
            more = lookup(next + 32 * WK);
            wait_until_left<0>();
            asm volatile("" : "+v"(more));  // (its load ends here, not at a use among loads into LDS)
        }
    };
    if (step < it.end) {
        wait_until_left<0>();
        asm volatile("" : "+v"(ids), "+v"(more));
        load(0, step);
        load(1, step);
    }
    for (; step < it.end; step += WK) {
        const int key0 = kFewStep * step;
        const bool another = step + WK < it.end;
        wait_until_left<kLoads>();  // the values
        Scales kd[2], vd[2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) kd[mt] = scales_of(0, mt);
        f32x4 s[2];  // scores, then probabilities, of keys 16mt + 4g + i
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            s[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                const u32x2 w = key_bytes(mt, kc);
                const unsigned w0 = w[0], w1 = w[1];
                const bf16x8 k = eight(f32x4{sbyte_to_float<0>(w0), sbyte_to_float<1>(w0), sbyte_to_float<2>(w0), sbyte_to_float<3>(w0)},
                                       f32x4{sbyte_to_float<0>(w1), sbyte_to_float<1>(w1), sbyte_to_float<2>(w1), sbyte_to_float<3>(w1)});
                f32x4 part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, query(kc, 2), f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, query(kc, 1), part, 0, 0, 0);
                part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, query(kc, 0), part, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt][i] = fmaf(part[i], static_cast<float>(kd[mt].d[i][kc]), s[mt][i]);
            }
        }
        wait_for_lds();
        advance(step + WK);
        if (another) {
            load(0, step + WK);
            wait_until_left<kLoads>();  // the next keys
        } else {
            wait_until_left<0>();
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) vd[mt] = scales_of(1, mt);
        const bool whole = key0 >= lo && key0 + kFewStep <= hi;  // every row sees every key
        const int first = range.x - key0 - 4 * g, end = range.y - key0 - 4 * g;  // of the lane's keys 16mt + i
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!whole) s[mt][i] = 16 * mt + i >= first && 16 * mt + i < end ? s[mt][i] : 0.f;
                nonfinite = fmaf(s[mt][i], 0.f, nonfinite);
            }
        if (a.cap != 0.f) {
            float most = 0.f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) most = fmaxf(most, __builtin_fabsf(s[mt][i]));
            const bool small = !__any(most > kSmallTanh);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt][i] = a.cap * (small ? small_tanh(s[mt][i]) : both_tanh(s[mt][i]));
        }
        if (a.slopes) {
            const int away = position - key0 - 4 * g;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt][i] = fmaf(-slope, static_cast<float>(abs(away - 16 * mt - i)), s[mt][i]);
        }
        if (!whole) {
            // (a scale that is not finite does not reach the rows that do not see it)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (16 * mt + i < first || 16 * mt + i >= end) {
                        s[mt][i] = -INFINITY;
#pragma unroll
                        for (int kc = 0; kc < KC; ++kc) vd[mt].d[i][kc] = static_cast<_Float16>(0.f);
                    }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[mt][i]);
        if (__any(mx > m + kThreshold)) {
            const float mn = fmaxf(m, cross_row_max(mx));
            const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mn);
            m = mn;
            l *= alpha;
            rounded *= alpha;
#pragma unroll
            for (int dt = 0; dt < 2 * KC; ++dt) acc[dt] *= alpha;
        }
        const float base = m == -INFINITY ? 0.f : m;  // (no key seen yet: probabilities 0)
        float sum = 0.f;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[mt][i] = fast_exp2(s[mt][i] - base);
                sum += s[mt][i];
            }
        add_to(l, rounded, sum);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            f32x4 d[2];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) d[mt][i] = s[mt][i] * static_cast<float>(vd[mt].d[i][kc]);
            bf16x8 p[3];
            split3(d[0], d[1], p);
            unsigned w[2][4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[mt][i] = value_bytes(mt, i, kc);
            auto tile = [&](auto e) __attribute__((always_inline)) {
                f32x4 x[2];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[mt][i] = sbyte_to_float<e.value>(w[mt][i]);
                const bf16x8 v = eight(x[0], x[1]);
                f32x4 part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[2], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[1], part, 0, 0, 0);
                acc[2 * kc + e.value] += __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[0], part, 0, 0, 0);
            };
            tile(std::integral_constant<int, 0>{});
            tile(std::integral_constant<int, 1>{});
        }
        wait_for_lds();
        if (another) load(1, step + WK);
    }
    wait_until_left<0>();  // (LDS is used again)

    // ---- the waves that shared these rows' keys, together
    float total = cross_row_sum(l);
    nonfinite = fmaf(total, 0.f, nonfinite);  // (a score and its bias may be finite and their sum not)
    if (__any(nonfinite != 0.f) && lane == 0) *a.err = 1;
    if (g == 0) stats[wave][r16] = make_float2(m, total);
    __syncthreads();
    {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, stats[w][r16].x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WK; ++w) sum = fmaf(fast_exp2(stats[w][r16].x - base), stats[w][r16].y, sum);
        const float scale = fast_exp2(m - base);
#pragma unroll
        for (int dt = 0; dt < 2 * KC; ++dt) acc[dt] *= scale;
        m = top;
        total = sum;
    }
    // the n-th four columns of a lane, from 32 (n / 2) + 8 g + 4 (n % 2) on
#pragma unroll
    for (int h = 0; h < H; ++h) {
        if (h) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int kc = 2 * h + i / 2, o = 2 * (i % 2);
            result(wave, i) = f32x4{acc[2 * kc][o], acc[2 * kc + 1][o], acc[2 * kc][o + 1], acc[2 * kc + 1][o + 1]};
        }
        __syncthreads();
        f32x4 x = result(0, wave);
#pragma unroll
        for (int w = 1; w < WK; ++w) x += result(w, wave);
        const int column = 32 * (2 * h + wave / 2) + 8 * g + 4 * (wave % 2);
        if (!live) continue;
        if (it.runs == 1) {
            *reinterpret_cast<f32x4*>(a.out + (row * a.heads + head) * D + column) = x / (total != 0.f ? total : 1.f);
        } else {
            const size_t p = (static_cast<size_t>(it.slot) + static_cast<size_t>(index) * it.runs + it.run) * a.heads + head;
            *reinterpret_cast<f32x4*>(a.part_acc + p * D + column) = x;
            if (h == 0 && wave == 0 && g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * p) = make_float2(m, total);
        }
    }
}

// ------------------------------------------------------------ many rows

constexpr int kManyWaves = 8;

// ds_read_b64_tr_b16: within 16 lanes, lane i receives element i % 4 of the four that
// lane 4j + i / 4 addresses, as its element j
__device__ __forceinline__ f16x4 transposed_read(const _Float16* p) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p));
    return __builtin_bit_cast(f16x4, v);
}

// Eight values as two fp16 parts, hi + lo = x to 22 bits.
struct Parts {
    u32x4 hi, lo;
    __device__ __forceinline__ f16x8 high() const { return __builtin_bit_cast(f16x8, hi); }
    __device__ __forceinline__ f16x8 low() const { return __builtin_bit_cast(f16x8, lo); }
};
__device__ __forceinline__ Parts split8(f32x4 x, f32x4 y) {
    Parts p;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        unsigned hi, lo;
        split2(x[2 * e], x[2 * e + 1], hi, lo);
        p.hi[e] = hi;
        p.lo[e] = lo;
        split2(y[2 * e], y[2 * e + 1], hi, lo);
        p.hi[2 + e] = hi;
        p.lo[2 + e] = lo;
    }
    return p;
}

// Rows go into parts multiplied by a power of two that brings their largest element to
// 2^14 .. 2^15: then an element is off by 2^-23 of itself or 2^-39 of the row's largest,
// whatever the row's size (plans in f32 keep all rows from here: ScorePlan::build).  The
// exponent (0 for 2^0 .. 2^1) of a magnitude, kept where both that power and its inverse,
// times 2^15 more, are normal numbers.
__device__ __forceinline__ int exponent_of(float most) {
    return max(static_cast<int>(__builtin_bit_cast(unsigned, most) >> 23 & 255) - 127, -97);
}
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }
constexpr int kHigh = 14;  // the exponent of a row's largest element in parts

// Up to 256 attention rows, eight waves of 32.  f32 products as three of fp16 parts
// (16x16x32, 16 times the f32 instruction's rate): lo hi + hi lo + hi hi, of rows
// brought to one size by powers of two (queries by lanes, keys and values when they are
// staged), which the scores, and the probabilities before their own parts, are multiplied
// by again.  All waves load and split a step's keys and values once, into the other of two
// buffers in LDS; one barrier a step.  Bound: the vector instructions of the softmax and of
// the probabilities' split beside the products, with two waves a SIMD (256 registers, and of
// 128 columns 10 to 16 more in scratch memory, of which a step reads one): 2 x 2,048 rows
// after 2,048, 32 heads on 8 of 128, capped (206 GFLOP): 793 us, 260 TFLOP/s, 1.7 times what
// f32's products reach at their best, and 1,727 us with six products of bf16 parts.
template <int D, bool kQ8>
__global__ __launch_bounds__(64 * kManyWaves) void score_shared_kernel(const ScoreArgs a) {
    constexpr int NT = 2, KC = D / 32, DT = D / 16;
    constexpr int KEYS = 4096 / D, MT = KEYS / 16;  // keys of a step: eight columns a thread
    constexpr int LPR = D / 8;                      // lanes of a key's row
    constexpr int STR = D + 16;                     // LDS row pitch: no bank twice
    __shared__ __attribute__((aligned(16))) _Float16 kparts[2][2][KEYS * STR];
    __shared__ __attribute__((aligned(16))) _Float16 vparts[2][2][KEYS * STR];
    __shared__ __attribute__((aligned(16))) float kscale[2][KEYS];  // what a key's scores are multiplied by
    __shared__ __attribute__((aligned(16))) float vscale[2][KEYS];  // and its probability
    // the queries' low parts, where registers do not hold them beside 128 columns of output
    constexpr bool kFar = D == 128;
    __shared__ u32x4 qlow[kFar ? kManyWaves : 1][kFar ? NT * KC : 1][64];
    __shared__ float stored_max[NT][64 * kManyWaves];  // a lane's rows' maxima when their sums last went to memory
    __shared__ int odd_values;   // some value is not finite
    __shared__ int most_query;   // the exponent of the queries' largest element, scaled
    __shared__ int large_keys;   // some score may be 2^17 or more, or leave f32
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    const Item it = item_of(a, blockIdx.x);
    if (!it.rows) return;  // the list's padding
    const int kh = it.head / a.group, kvw = a.lay.kv_width, tokens = it.tokens;

    auto row_of = [&](int nt, int& head) {  // of the block's rows; behind them there are none
        const int r = 32 * wave + 16 * nt + r16, row = r / it.heads;
        head = it.head + r - row * it.heads;
        return row;
    };
    int position[NT];
    int2 range[NT];
    float slope[NT];
    int all_lo = 0, all_hi = 0x7fffffff, from = 0x7fffffff;  // keys that all rows of the wave see; its first position
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        int head;
        const int row = row_of(nt, head);
        const bool live = row < it.rows;
        position[nt] = it.position + row;
        range[nt] = live ? a.ranges[static_cast<size_t>(it.row0) + row] : make_int2(0, 0);
        slope[nt] = a.slopes && live ? a.slopes[head] : 0.f;
        if (live) {
            all_lo = max(all_lo, range[nt].x);
            all_hi = min(all_hi, range[nt].y);
            from = min(from, position[nt]);
        }
    }
    all_lo = uniform_max(all_lo);
    all_hi = -uniform_max(-all_hi);
    from = -uniform_max(-from);
    if (tid == 0) {
        odd_values = 0;
        large_keys = 0;
        most_query = -1000;
    }
    __syncthreads();

    u32x4 qh[NT][KC], ql[kFar ? 1 : NT][kFar ? 1 : KC];
    float qsize[NT];  // what a row's scores are multiplied by
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        f32x4 x[KC][2];
        float most = 0.f;
        int head;
        const int row = row_of(nt, head);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x[kc][i] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (row < it.rows)
                    x[kc][i] = *reinterpret_cast<const f32x4*>(a.q + ((static_cast<size_t>(it.row0) + row) * a.heads + head) * D +
                                                               32 * kc + 8 * g + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) most = fmaxf(most, __builtin_fabsf(x[kc][i][e]));
            }
        const int size = exponent_of(cross_row_max(most));
        const float up = power_of_two(kHigh - size);
        qsize[nt] = fmaxf(power_of_two(size - kHigh) * a.qscale, 1.17549435e-38f);
        atomicMax(&most_query, size + exponent_of(fmaxf(a.qscale, a.qscale * a.cap)) + 1);  // (before a cap, and behind it)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            const Parts p = split8(x[kc][0] * up, x[kc][1] * up);
            qh[nt][kc] = p.hi;
            if constexpr (kFar)
                qlow[wave][nt * KC + kc][lane] = p.lo;
            else
                ql[nt][kc] = p.lo;
        }
    }

    // staging: eight columns of a key; a wave's keys lie in one block
    const int skey = tid / LPR, col = 8 * (tid % LPR);
    const int tpb = a.lay.tpb, tsh = __builtin_ctz(static_cast<unsigned>(tpb));
    const int32_t* tab = a.tables + it.table;
    const size_t kbytes = kQ8 ? static_cast<size_t>(a.layer) * 2 * a.lay.section + static_cast<size_t>(kh) * a.lay.head_bytes
                              : (static_cast<size_t>(a.layer) * 2 * tpb * kvw + static_cast<size_t>(kh) * D) * sizeof(float);
    const size_t vsec = kQ8 ? a.lay.section : static_cast<size_t>(tpb) * kvw * sizeof(float);
    // (past the last key: its block again, whose slots are there whatever they hold)
    const int wkey = __builtin_amdgcn_readfirstlane(skey);  // the wave's first
    // (constant to the compiler too: a scalar load, which waits for no other, though sums are
    // stored between)
    const auto ids = reinterpret_cast<__attribute__((address_space(4))) const int32_t*>(reinterpret_cast<uintptr_t>(tab));
    auto lookup = [&](int stp) { return ids[min(KEYS * stp + wkey, tokens - 1) >> tsh]; };
    const unsigned in_row = kQ8 ? (skey - wkey) * D + col : ((skey - wkey) * kvw + col) * static_cast<unsigned>(sizeof(float));
    const unsigned in_scales = ((skey - wkey) * (D / 32) + col / 32) * 2;
    f32x4 kreg[2], vreg[2];
    u32x2 kraw, vraw;
    unsigned kdraw, vdraw;
    auto load = [&](int stp, int id) __attribute__((always_inline)) {
        const int slot = (KEYS * stp + wkey) & (tpb - 1);
        const char* block = a.pool + static_cast<size_t>(id) * a.lay.stride + kbytes;
        if constexpr (kQ8) {
            const char *k = block + static_cast<size_t>(slot) * D, *sc = block + static_cast<size_t>(tpb) * D + static_cast<size_t>(slot * (D / 32)) * 2;
            kraw = *reinterpret_cast<const u32x2*>(k + in_row);
            kdraw = *reinterpret_cast<const uint16_t*>(sc + in_scales);
            vraw = *reinterpret_cast<const u32x2*>(k + vsec + in_row);
            vdraw = *reinterpret_cast<const uint16_t*>(sc + vsec + in_scales);
        } else {
            const char *k = block + static_cast<size_t>(slot) * kvw * sizeof(float), *v = k + vsec;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                kreg[i] = *reinterpret_cast<const f32x4*>(k + in_row + 16 * i);
                vreg[i] = *reinterpret_cast<const f32x4*>(v + in_row + 16 * i);
            }
        }
    };
    auto stage = [&](int buf) __attribute__((always_inline)) {
        if constexpr (kQ8) {
            const float kd = half_bits_to_float(static_cast<uint16_t>(kdraw)), vd = half_bits_to_float(static_cast<uint16_t>(vdraw));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const unsigned kw = kraw[i], vw = vraw[i];
                kreg[i] = f32x4{sbyte_to_float<0>(kw) * kd, sbyte_to_float<1>(kw) * kd, sbyte_to_float<2>(kw) * kd, sbyte_to_float<3>(kw) * kd};
                vreg[i] = f32x4{sbyte_to_float<0>(vw) * vd, sbyte_to_float<1>(vw) * vd, sbyte_to_float<2>(vw) * vd, sbyte_to_float<3>(vw) * vd};
            }
        }
        float kmost = 0.f, vmost = 0.f;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool fine = __builtin_isfinite(vreg[i][e]);
                odd |= !fine;
                vreg[i][e] = fine ? vreg[i][e] : 0.f;
                kmost = fmaxf(kmost, __builtin_fabsf(kreg[i][e]));
                vmost = fmaxf(vmost, __builtin_fabsf(vreg[i][e]));
            }
        if (odd) odd_values = 1;
        // over the row's lanes: 8, or 16
        kmost = row_max<LPR>(kmost);
        vmost = row_max<LPR>(vmost);
        const int ksize = exponent_of(kmost), size = exponent_of(vmost);
        if (ksize + most_query >= 16) large_keys = 1;
        if (tid % LPR == 0) {
            kscale[buf][skey] = power_of_two(ksize - kHigh);
            vscale[buf][skey] = power_of_two(size);
        }
        const int at = skey * STR + col;
        const float kup = power_of_two(kHigh - min(ksize, 127)), vup = power_of_two(kHigh - size);
        const Parts k = split8(kreg[0] * kup, kreg[1] * kup), v = split8(vreg[0] * vup, vreg[1] * vup);
        *reinterpret_cast<u32x4*>(&kparts[buf][0][at]) = k.hi;
        *reinterpret_cast<u32x4*>(&kparts[buf][1][at]) = k.lo;
        *reinterpret_cast<u32x4*>(&vparts[buf][0][at]) = v.hi;
        *reinterpret_cast<u32x4*>(&vparts[buf][1][at]) = v.lo;
    };

    f32x4 acc[DT][NT];
    float m[NT], l[NT], rounded[NT], nonfinite = 0.f;
    int asize[NT];  // acc is in units of 2^(asize - 2 kHigh)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = rounded[nt] = 0.f;
        asize[nt] = -97;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // the products of two parts each, small ones first
    auto three = [](const Parts& x, const Parts& y, f32x4 c) __attribute__((always_inline)) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.low(), y.high(), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.high(), y.low(), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(x.high(), y.high(), c, 0, 0, 0);
    };
    f32x4 s[MT][NT];  // scores, then probabilities, of keys 16mt + 4g + i
    auto scores = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
        // (operands are read from LDS one ahead of their products)
        auto key_parts = [&](int o) __attribute__((always_inline)) {
            const int at = (16 * (o % MT) + r16) * STR + 32 * (o / MT) + 8 * g;
            return Parts{*reinterpret_cast<const u32x4*>(&kparts[buf][0][at]), *reinterpret_cast<const u32x4*>(&kparts[buf][1][at])};
        };
        u32x4 low[NT];
        auto query_parts = [&](int kc) __attribute__((always_inline)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if constexpr (kFar)
                    low[nt] = qlow[wave][nt * KC + kc][lane];
                else
                    low[nt] = ql[nt][kc];
            }
        };
        Parts k = key_parts(0);
        query_parts(0);
#pragma unroll
        for (int o = 0; o < KC * MT; ++o) {
            const Parts now = k;
            if (o + 1 < KC * MT) k = key_parts(o + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[o % MT][nt] = three(now, Parts{qh[nt][o / MT], low[nt]}, s[o % MT][nt]);
            if (o % MT == MT - 1 && o + 1 < KC * MT) query_parts(o / MT + 1);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto output = [&](int buf, int stp) __attribute__((always_inline)) {
        const int key0 = KEYS * stp;
        const bool whole = key0 >= all_lo && key0 + KEYS <= all_hi;
        const bool large = __builtin_amdgcn_readfirstlane(large_keys);
        float alpha[NT];
        Parts p[NT][MT / 2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int first = range[nt].x - key0 - 4 * g, end = range[nt].y - key0 - 4 * g;
            // scores are s * by
            float by = qsize[nt];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][nt] *= *reinterpret_cast<const f32x4*>(&kscale[buf][16 * mt + 4 * g]);
            if (large) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        nonfinite = fmaf(16 * mt + i >= first && 16 * mt + i < end ? s[mt][nt][i] * by : 0.f, 0.f, nonfinite);
            }
            if (a.cap != 0.f) {
                float top = 0.f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    s[mt][nt] *= by;
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fabsf(s[mt][nt][i]));
                }
                by = a.cap;
                if (!__any(top > kSmallTanh)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[mt][nt][i] = small_tanh(s[mt][nt][i]);
                } else {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[mt][nt][i] = any_tanh(s[mt][nt][i]);
                }
            }
            if (large) {
                // (the maximum below is a rounded one: its product with `by` inside an
                // exponential's argument would be off by half an ulp of the score)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][nt] *= by;
                by = 1.f;
            }
            if (a.slopes) {
                const int away = position[nt] - key0 - 4 * g;
                if (key0 + KEYS <= from) {  // every key lies before every row
                    const float far = -slope[nt] * static_cast<float>(away);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[mt][nt][i] = fmaf(s[mt][nt][i], by, fmaf(slope[nt], static_cast<float>(16 * mt + i), far));
                } else {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[mt][nt][i] = fmaf(s[mt][nt][i], by, -slope[nt] * static_cast<float>(abs(away - 16 * mt - i)));
                }
                by = 1.f;
            }
            if (!whole) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (16 * mt + i < first || 16 * mt + i >= end) s[mt][nt][i] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[mt][nt][i]);
            const float mn = fmaxf(m[nt], cross_row_max(mx) * by), base = mn == -INFINITY ? 0.f : mn;
            alpha[nt] = fast_exp2(m[nt] - base);
            m[nt] = mn;
            // probabilities times their values' sizes, brought to one size in turn: the
            // largest one's, or that of what was added before
            float sum = 0.f, most = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const f32x4 sizes = *reinterpret_cast<const f32x4*>(&vscale[buf][16 * mt + 4 * g]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[mt][nt][i] = fast_exp2(fmaf(s[mt][nt][i], by, -base));
                    sum += s[mt][nt][i];
                    s[mt][nt][i] *= sizes[i];
                    most = fmaxf(most, s[mt][nt][i]);
                }
            }
            l[nt] *= alpha[nt];
            rounded[nt] *= alpha[nt];
            add_to(l[nt], rounded[nt], sum);
            const int size = max(exponent_of(cross_row_max(most)), max(asize[nt] + exponent_of(alpha[nt]), -97));
            alpha[nt] *= power_of_two(max(asize[nt] - size, -126));
            asize[nt] = size;
            const float up = power_of_two(kHigh - size);
#pragma unroll
            for (int h = 0; h < MT / 2; ++h) p[nt][h] = split8(s[2 * h][nt] * up, s[2 * h + 1][nt] * up);
        }
        // lane (g, i): column 16dt + i of keys 4g .. 4g + 3 and 16 + 4g .. of each 32, as the
        // probabilities have them; a step's part from zero, then added to the rest
        auto value_parts = [&](int o) __attribute__((always_inline)) {
            const int at = (32 * (o % (MT / 2)) + 4 * g + (r16 >> 2)) * STR + 16 * (o / (MT / 2)) + 4 * (r16 & 3);
            auto both = [&](int part) __attribute__((always_inline)) {
                const f16x4 x = transposed_read(&vparts[buf][part][at]), y = transposed_read(&vparts[buf][part][at + 16 * STR]);
                return __builtin_bit_cast(u32x4, f16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
            };
            return Parts{both(0), both(1)};
        };
        Parts v = value_parts(0);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            f32x4 part[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) part[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < MT / 2; ++h) {
                const Parts now = v;
                if (dt * (MT / 2) + h + 1 < DT * (MT / 2)) v = value_parts(dt * (MT / 2) + h + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) part[nt] = three(now, p[nt][h], part[nt]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[dt][nt][i] = fmaf(acc[dt][nt][i], alpha[nt], part[nt][i]);
        }
    };

    // The sums to their rows' place (a result, a run's partial), onto those that are there
    // already from kScoreManyChain steps before; `last`: divided.  A lane its own.
    auto put = [&](bool again, bool last) __attribute__((always_inline)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float total = last ? cross_row_sum(l[nt]) : 0.f;
            int r = 32 * wave + 16 * nt + r16;
            asm("" : "+v"(r));  // (worked out here, not kept through the loop)
            const int row = r / it.heads, head = it.head + r - row * it.heads;
            if (row >= it.rows) continue;
            const bool whole = it.runs == 1;
            const size_t at = (whole ? static_cast<size_t>(it.row0) + row
                                     : static_cast<size_t>(it.slot) + static_cast<size_t>(row) * it.runs + it.run) * a.heads + head;
            float* o = (whole ? a.out : a.part_acc) + at * D + 4 * g;
            const float unit = power_of_two(asize[nt] - 2 * kHigh);
            const float before = again ? fast_exp2(stored_max[nt][tid] - (m[nt] == -INFINITY ? 0.f : m[nt])) : 0.f;
            float div = 1.f;
            if (last) {
                nonfinite = fmaf(total, 0.f, nonfinite);  // (a score that is NaN is in its row's sum)
                if (whole && total != 0.f) div = total;
                if (!whole && g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(m[nt], total);
            } else {
                stored_max[nt][tid] = m[nt];
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                f32x4 x = acc[dt][nt] * unit;
                if (again) x += *reinterpret_cast<const f32x4*>(o + 16 * dt) * before;
                *reinterpret_cast<f32x4*>(o + 16 * dt) = last ? x / div : x;
                acc[dt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            asize[nt] = -97;
        }
    };

    int step = it.step, buf = 0, id = 0;
    if (step < it.end) {
        load(step, lookup(step));
        id = lookup(step + 1);
        __syncthreads();
        stage(0);
        __syncthreads();
    }
    for (bool again = false;; again = true) {
        for (const int until = min(it.end, step + kScoreManyChain); step < until; ++step, buf ^= 1) {
            scores(buf);
            load(step + 1, id);
            id = lookup(step + 2);
            output(buf, step);
            stage(buf ^ 1);
            __syncthreads();
        }
        put(again, step >= it.end);
        if (step >= it.end) break;
    }
    if (nonfinite != 0.f) *a.err = 1;
    if (it.step >= it.end || !odd_values) return;
    // Values that are not finite were zeros above: a row that sees one is given a column that
    // is not finite, over what was written.
    __threadfence_block();
    __syncthreads();
    const int keys = min(KEYS * it.end, tokens) - KEYS * it.step;
    for (int i = tid; i < keys * D; i += 64 * kManyWaves) {
        const int key = KEYS * it.step + i / D, c = i % D;
        if (__builtin_isfinite(score_element(a, tab[key >> tsh], 1, key & (tpb - 1), kh * D + c))) continue;
        for (int row = 0; row < it.rows; ++row) {
            const int2 seen = a.ranges[static_cast<size_t>(it.row0) + row];
            if (key < seen.x || key >= seen.y) continue;
            const size_t at = it.runs == 1 ? static_cast<size_t>(it.row0) + row
                                           : static_cast<size_t>(it.slot) + static_cast<size_t>(row) * it.runs + it.run;
            for (int head = it.head; head < it.head + it.heads; ++head)
                (it.runs == 1 ? a.out : a.part_acc)[(at * a.heads + head) * D + c] = NAN;
        }
    }
}

}  // namespace

int score_step(const BlockLayout& lay, int block) { return block == kScoreFew ? kFewStep : 4096 / lay.head_dim; }

// (us with 1, 2 and 3 for few rows, eight contexts of 4,000 to 9,000, 32 heads on 8: f32 of 64
// 45, 47 and 50, of 128 92, 93 and 95; Q8_0 of 64 35, 27 and 25, of 128 48, 40 and 38)
int score_units(const BlockLayout& lay, int block) {
    return block == kScoreMany || lay.format != kQ8 ? 1 : 3;
}

void launch_score_tiles(const ScoreArgs& a, int block, int workgroups, hipStream_t s) {
    const bool q8 = a.lay.format == kQ8;
    auto go = [&](const char* name, auto kernel, int waves) { launch(name, kernel, dim3(workgroups), dim3(64 * waves), 0, s, a); };
    if (block == kScoreFew) {
        const char* name = "score_attention_tiles";
        if (a.lay.head_dim == 128)
            q8 ? go(name, score_tile_q8_kernel<128>, kFewWaves) : go(name, score_tile_kernel<128>, kFewWaves);
        else
            q8 ? go(name, score_tile_q8_kernel<64>, kFewWaves) : go(name, score_tile_kernel<64>, kFewWaves);
    } else {
        const char* name = "score_attention_shared";
        if (a.lay.head_dim == 128)
            q8 ? go(name, score_shared_kernel<128, true>, kManyWaves) : go(name, score_shared_kernel<128, false>, kManyWaves);
        else
            q8 ? go(name, score_shared_kernel<64, true>, kManyWaves) : go(name, score_shared_kernel<64, false>, kManyWaves);
    }
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

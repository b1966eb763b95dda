// Attention of token trees on the matrix cores, for head_dim 64 and 128 over f32
// or Q8_0 blocks of a power of two from 16 tokens.
//
// A row is a (node, query head) pair; the rows of one (tree, KV head) share its
// keys.  A wave takes 16 * NT rows, whose queries, output and statistics stay in its
// registers, and walks keys 32 at a time ("a step"), with no barrier until they are done.
//  S^T = K Q^T: the lane (g, r) = (l / 16, l % 16) has four columns at a time of key r
//    as operands, in an order of its own, since the numbering of a contraction's terms
//    is free as long as Q has the same.  Q8_0 bytes are loaded so; keys of f32 blocks
//    go as whole rows from memory into the wave's own part of LDS and are read from
//    there so.
//  O^T = V^T P^T: lane (g, r) loads four columns of the keys 4g + i of each 16 into
//    registers, so it holds V^T's operand for four output tiles (tile j: column j of
//    every lane's four) and its own scores are P^T's.
// Steps are dealt in turn to the workgroup's waves, whose results meet in LDS.  A
// long context is cut into runs, a workgroup each, that leave partials for a merge.
// After the cached steps come those over the tree's own nodes, with a mask word a row.
//
// f32: v_mfma_f32_16x16x4_f32.  f32x3 (kX3): 16x16x32 on operands in two fp16
// parts, hi * hi + hi * lo + lo * hi.  Softmax in log2 units with a
// running maximum that moves only where a step exceeds it by 2^8 (f32x3: 2^4).
//
// MI355X: f32, 16 contexts of 123 to 2,793 tokens with 6 to 24 nodes, 32 heads on 8
// of 64: 45.6 us with the merge (floor 21: one read of K and V at a copy's rate), bound
// by the longest workgroups and the f32 products (25 us, padded to 16 rows: the matrix
// pipe is busy 58% of the time, the CUs' caches 88%).
// f32x3, 16 contexts of 2,048 with 16 nodes, head_dim 128: 58.2 us, 4.6 TB/s.
#include <algorithm>
#include <limits>

#include "common.hpp"
#include "device_util.hpp"
#include "q8.hpp"
#include "tree.hpp"

namespace tvara_amd {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kThreshold = 8.0f;
// f32x3: what two fp16 parts hold of a probability ends at 2^-25, and a row may have
// its largest one beside thousands of small ones that count together (the first token
// of a text draws such weight, and may have little value itself).  So m is kept 2^11
// below the running maximum, which every probability, sum and partial is then relative
// to, and the maximum may pass it by 2^4: the largest lies between 2^11 and 2^15, fp16
// ends at 2^16, and a small one is off by 2^-36 of it.  MI355X, one key without value 18
// above 32,768 of N(0,1): 2-norm 0.19 (m the maximum, which may move by 2^8),
// 1.6e-3 (2^7 and 2^8), 1e-4 so (128 rows a workgroup: 2e-4).
constexpr float kPartsThreshold = 4.0f, kPartsLift = 11.0f;
constexpr int kStep = kTreeStep, kWaves = kTreeWaves;
constexpr int kBufferWord3 = 0x00020000;  // gfx9 buffer descriptor, dword 3

// Whether a product with x passes zeros on: x is finite, and (kParts) so is the nearest
// fp16 number, x's first part.
template <bool kParts>
__device__ __forceinline__ bool fits(float x) {
    return kParts ? __builtin_fabsf(x) < 65520.f : __builtin_isfinite(x);
}
// What a row that sees such a value is given of it: in parts, something that is not
// finite, which the launch reports.
template <bool kParts>
__device__ __forceinline__ float unfit(float x) {
    return kParts ? x * INFINITY : x;
}

// Where 64 runs of bytes start and how far they go, one a lane.
struct Spans {
    unsigned lo, hi;
    int range;
    __device__ __forceinline__ void set(const char* base, int bytes) {
        const uint64_t b = reinterpret_cast<uint64_t>(base);
        lo = static_cast<unsigned>(b);
        hi = static_cast<unsigned>(b >> 32);
        range = bytes;
    }
    // lane i's as a buffer descriptor, in scalar registers
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(int i) const {
        const uint64_t b = static_cast<uint64_t>(static_cast<unsigned>(__builtin_amdgcn_readlane(hi, i))) << 32 |
                           static_cast<unsigned>(__builtin_amdgcn_readlane(lo, i));
        return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(b), 0, __builtin_amdgcn_readlane(range, i), kBufferWord3);
    }
};

// Ends a rare branch that loads: where it joins the common path nothing of it is in
// flight, so that no wait for it is put there, which would wait for the loads
// ahead too (they return in order).
__device__ __forceinline__ void wait_for_loads() { __builtin_amdgcn_s_waitcnt(0); }

// Two elements of Q8_0 blocks as hi + lo in fp16: bytes i and j (4 to 7: of w1) of a
// pair of words times the fp16 scales d.  A byte in the low end of 1024 is q + 1152
// exactly, and the scale times q less its rounding is exact as well: five
// instructions a pair, eight by way of f32.
template <int i, int j>
__device__ __forceinline__ void scaled2(unsigned w0, unsigned w1, f16x2 d, unsigned& hi, unsigned& lo) {
    const unsigned u = __builtin_amdgcn_perm(w1, w0, 0x0c000c00u | j << 16 | i) ^ 0x64806480u;
    const f16x2 q = __builtin_bit_cast(f16x2, u) - f16x2{1152, 1152}, h = q * d;
    hi = __builtin_bit_cast(unsigned, h);
    lo = __builtin_bit_cast(unsigned, __builtin_elementwise_fma(q, d, -h));
}

// A workgroup's work: a tree (TreeArgs::trees), the KV head and first row of a row
// block, and a run of its steps; the partials of the tree's node j are slot + j *
// runs on.
struct Item {
    int4 tree;
    int head, row0, step, end, run, runs, slot;
};
__device__ __forceinline__ Item item_of(const TreeArgs& a, unsigned i) {
    const int4 t = a.work[3 * static_cast<size_t>(i)], x = a.work[3 * static_cast<size_t>(i) + 1], y = a.work[3 * static_cast<size_t>(i) + 2];
    return {t, x.x, x.y, x.z, x.w, y.x, y.y, y.z};
}

template <int D, int NT, bool kQ8, bool kX3, bool kAlone = false>
__global__ __launch_bounds__(64 * kWaves, D == 64 || !kX3 ? 2 : 1) void tree_tile_kernel(const TreeArgs a) {
    constexpr int WK = kWaves, C = D / 16, KC = D / 32, H = D / 64;
    constexpr int W = D / 4;  // 16-byte parts of a row
    // f32 keys come as whole rows, W lanes each, and turn into operands (16 lanes, 16
    // rows) by way of LDS: read from memory as operands they take four times as long
    // to come through the CU's cache.  They go there without passing registers, so
    // that 128 columns leave room for two waves a SIMD (16 contexts of 2048, 32 heads on
    // 8: f32 and head_dim 64, 64 rows 63.7 us as operands, 56.9 by way of registers and
    // LDS, 55.0 so; head_dim 128, 32 rows 63, 73, 58.7; f32x3 and head_dim 128, 64 rows
    // 65.8, 60.6, 58.7).
    constexpr bool kStaged = !kQ8;
    // a wave's keys of a step; at the end its results, for the others
    __shared__ f32x4 staged[WK][kStaged ? kStep * W : 4 * NT * 64];
    auto result = [&](int w, int i, int nt) -> f32x4& { return staged[w][(i * NT + nt) * 64 + static_cast<int>(threadIdx.x & 63)]; };
    __shared__ float2 stats[WK][16 * NT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    // one entry of work a workgroup, whose steps the waves share, or (kAlone) one a wave
    constexpr int stride = kAlone ? 1 : WK;
    const Item it = item_of(a, kAlone ? blockIdx.x * WK + wave : blockIdx.x);
    if (!it.tree.z) return;  // the list's padding
    const int4 tree = it.tree;
    const int cached = tree.y, nodes = tree.z, kh = it.head, G = a.group, kvw = a.lay.kv_width;
    const int row0 = it.row0;

    // this lane's row of each row tile
    int node[NT], head[NT];
    bool live[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + 16 * nt + r16;
        node[nt] = r / G;
        head[nt] = kh * G + r - node[nt] * G;
        live[nt] = node[nt] < nodes;
    }
    // column of element 0 of a lane's c-th four of a key, and of the h-th four of
    // a value (r: the loading lane's r16, or an output row of the tiles)
    auto kcol = [&](int c) { return kQ8 ? 64 * (c / 4) + 16 * g + 4 * (c % 4) : 16 * c + 4 * g; };
    auto vcol = [](int h, int r) { return kQ8 ? (D / 16) * r + 4 * h : 64 * h + 4 * r; };

    const int csteps = (cached + kStep - 1) / kStep, end = min(it.end, csteps);
    const int tpb = a.lay.tpb, tsh = __builtin_ctz(static_cast<unsigned>(tpb));
    const int32_t* tab = a.tables + tree.x;
    const size_t kbytes = kQ8 ? static_cast<size_t>(a.layer) * 2 * a.lay.section + static_cast<size_t>(kh) * a.lay.head_bytes
                              : (static_cast<size_t>(a.layer) * 2 * tpb * kvw + static_cast<size_t>(kh) * D) * sizeof(float);
    const size_t vsec = kQ8 ? a.lay.section : static_cast<size_t>(tpb) * kvw * sizeof(float);
    const int rowb = kQ8 ? D : kvw * static_cast<int>(sizeof(float));  // from one slot to the next
    const unsigned koff = static_cast<unsigned>(kStaged ? lane / W * rowb + (lane % W ^ lane / W) * 16 : r16 * rowb + kcol(0));
    const unsigned voff = static_cast<unsigned>(4 * g * rowb + vcol(0, r16) * (kQ8 ? 1 : 4));
    int step = it.step + (kAlone ? 0 : wave);
    const int last = max(cached - 1, 0) >> 4;  // 16 keys a table lookup; past the end the last again
    // lane 2i + mt: the block of the wave's i-th step from here
    auto lookup = [&](int from) { return cached ? tab[min(2 * (from + (lane >> 1) * stride) + (lane & 1), last) << 4 >> tsh] : 0; };
    int ids = lookup(step), more = lookup(step + 32 * stride), at = 0;
    auto block = [&](int mt, int stp) {
        const int id = __builtin_amdgcn_readlane(ids, 2 * at + mt);
        const int slot = (min(2 * stp + mt, last) << 4) & (tpb - 1);
        return a.pool + static_cast<size_t>(id) * a.lay.stride + kbytes + static_cast<size_t>(slot) * rowb;
    };
    // A workgroup's start is a chain of waits for memory: table, then keys.  With
    // head_dim 64 the first keys are asked for before the queries are waited for (16
    // ragged contexts 50.2 -> 48.3 us).
    f32x4 qf[NT][C];
    auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float* qp = a.q + (static_cast<size_t>(tree.w + node[nt]) * a.heads + head[nt]) * D;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                qf[nt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (live[nt]) qf[nt][c] = *reinterpret_cast<const f32x4*>(qp + kcol(c));
            }
        }
    };
    // f32 rows, or Q8_0 bytes and scales, which become values where they are used
    f32x4 v[kQ8 ? 1 : 2][4][H];
    u32x4 kw[kQ8 ? 2 : 1][H];
    unsigned kd[kQ8 ? 2 : 1][H], vw[kQ8 ? 2 : 1][4][H], vd[kQ8 ? 2 : 1][4];
    auto scales = [&](const char* b, int mt, int stp) {  // of the block's rows from the tile's first on
        const int slot = (min(2 * stp + mt, last) << 4) & (tpb - 1);
        return b + static_cast<size_t>(tpb - slot) * D + static_cast<size_t>(slot) * (D / 32) * 2;
    };
    auto load_k = [&](int stp) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const char* b = block(mt, stp);
            if constexpr (kQ8) {
                const char* sc = scales(b, mt, stp);
#pragma unroll
                for (int u = 0; u < H; ++u) {
                    kw[mt][u] = *reinterpret_cast<const u32x4*>(b + koff + 64 * u);
                    kd[mt][u] = *reinterpret_cast<const uint16_t*>(sc + (r16 * (D / 32) + 2 * u + (g >> 1)) * 2);
                }
            } else {
                // straight into LDS, lane after lane; what a lane loads is permuted by its
                // row, so that the operands' reads meet no bank twice
                const __amdgpu_buffer_rsrc_t rows =
                    __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(b), 0, 15 * rowb + 4 * D, kBufferWord3);
#pragma unroll
                for (int c = 0; c < C; ++c)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (__attribute__((address_space(3))) void*)&staged[wave][(mt * C + c) * 64],
                                                             16, koff ^ 1024 / W * c, 64 / W * c * rowb, 0, 0);
            }
        }
    };
    auto staged_k = [&](int mt, int c) __attribute__((always_inline)) {
        return staged[wave][(16 * mt + r16) * W + ((4 * c + g) ^ r16)];
    };
    auto load_v = [&](int stp) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const char* b = block(mt, stp) + vsec;
            if constexpr (kQ8) {
                const char* sc = scales(b, mt, stp);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vd[mt][i] = *reinterpret_cast<const uint16_t*>(sc + ((4 * g + i) * (D / 32) + (D / 16) * r16 / 32) * 2);
#pragma unroll
                    for (int h = 0; h < H; ++h) vw[mt][i][h] = *reinterpret_cast<const unsigned*>(b + voff + i * D + 4 * h);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < H; ++h)
                        v[mt][i][h] = *reinterpret_cast<const f32x4*>(b + static_cast<size_t>(i) * rowb + voff + 256 * h);
            }
        }
    };
    constexpr bool kEarly = D == 64;
    load_q();
    if (kEarly && step < end) {
        load_k(step);
        if constexpr (kStaged) asm volatile("" ::: "memory");
        load_v(step);
    }
    u32x4 qh[kX3 ? NT : 1][kX3 ? KC : 1], ql[kX3 ? NT : 1][kX3 ? KC : 1];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            qf[nt][c] *= a.qscale;
            if constexpr (kX3) {
                const f32x4 x = qf[nt][c];
                unsigned h0, h1, l0, l1;
                split2(x[0], x[1], h0, l0);
                split2(x[2], x[3], h1, l1);
                qh[nt][c / 2][2 * (c % 2)] = h0;
                qh[nt][c / 2][2 * (c % 2) + 1] = h1;
                ql[nt][c / 2][2 * (c % 2)] = l0;
                ql[nt][c / 2][2 * (c % 2) + 1] = l1;
            }
        }

    f32x4 acc[4 * H][NT];  // tile (h, j) at 4h + j
    constexpr float kLift = kX3 ? kPartsLift : 0.f, kMove = (kX3 ? kPartsThreshold : kThreshold) + kLift;
    float m[NT], l[NT], rounded[NT], nonfinite = 0.f;  // m: the maximum less kLift; nonfinite: NaN once a score is not finite
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = rounded[nt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 4 * H; ++dt) acc[dt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    f32x4 s[2][NT];  // scores, then probabilities, of keys 16mt + 4g + i
    // key(mt, c): the lane's c-th four columns; key(mt, kc, hi, lo): eight in parts
    auto scores = [&](auto&& key) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (kX3) {
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    u32x4 hi, lo;
                    key(mt, kc, hi, lo);
                    const f16x8 kh8 = __builtin_bit_cast(f16x8, hi), kl8 = __builtin_bit_cast(f16x8, lo);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const f16x8 q8 = __builtin_bit_cast(f16x8, qh[nt][kc]);
                        s[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl8, q8, s[mt][nt], 0, 0, 0);
                        s[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh8, __builtin_bit_cast(f16x8, ql[nt][kc]),
                                                                           s[mt][nt], 0, 0, 0);
                        s[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh8, q8, s[mt][nt], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const f32x4 k = key(mt, c);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            s[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i], qf[nt][c][i], s[mt][nt], 0, 0, 0);
                }
            }
        }
    };
    // f32 keys k(mt, c), and values in registers, given so
    auto from_f32 = [](auto&& k) __attribute__((always_inline)) {
        if constexpr (kX3)
            return [&k](int mt, int kc, u32x4& hi, u32x4& lo) __attribute__((always_inline)) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const f32x4 x = k(mt, 2 * kc + half);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        unsigned h1, l1;
                        split2(x[2 * e], x[2 * e + 1], h1, l1);
                        hi[2 * half + e] = h1;
                        lo[2 * half + e] = l1;
                    }
                }
            };
        else
            return [&k](int mt, int c) __attribute__((always_inline)) { return k(mt, c); };
    };
    auto values_from_f32 = [](const f32x4 (&v)[2][4][H]) __attribute__((always_inline)) {
        if constexpr (kX3)
            return [&v](int h, auto j, u32x4& hi, u32x4& lo) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned h1, l1;
                    split2(v[e / 2][2 * (e % 2)][h][j.value], v[e / 2][2 * (e % 2) + 1][h][j.value], h1, l1);
                    hi[e] = h1;
                    lo[e] = l1;
                }
            };
        else
            return [&v](int mt, int i, int h, auto j) __attribute__((always_inline)) { return v[mt][i][h][j.value]; };
    };
    // seen(mt, i, nt): whether the row sees the key
    auto softmax = [&](auto masked, auto&& seen) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = s[mt][nt][i];
                    if constexpr (decltype(masked)::value) {
                        const bool on = seen(mt, i, nt);
                        nonfinite = fmaf(on ? x : 0.f, 0.f, nonfinite);
                        x = on ? x : -INFINITY;
                        s[mt][nt][i] = x;
                    } else {
                        nonfinite = fmaf(x, 0.f, nonfinite);
                    }
                    mx = fmaxf(mx, x);
                }
            if (__any(mx > m[nt] + kMove)) {
                const float mn = fmaxf(m[nt], cross_row_max(mx) - kLift);
                const float alpha = m[nt] == -INFINITY ? 0.f : fast_exp2(m[nt] - mn);
                m[nt] = mn;
                l[nt] *= alpha;
                rounded[nt] *= alpha;
#pragma unroll
                for (int dt = 0; dt < 4 * H; ++dt) acc[dt][nt] *= alpha;
            }
            const float base = m[nt] == -INFINITY ? 0.f : m[nt];  // (no key seen yet: probabilities 0)
            float sum = 0.f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = fast_exp2(s[mt][nt][i] - base);
                    s[mt][nt][i] = p;
                    sum += p;
                }
            add_to(l[nt], rounded[nt], sum);
        }
    };
    // value(mt, i, h, j): column j of the h-th four of key 16mt + 4g + i;
    // value(h, j, hi, lo): of the lane's eight keys in parts
    auto output = [&](auto&& value) __attribute__((always_inline)) {
        u32x4 ph[NT], pl[NT];
        if constexpr (kX3) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned h1, l1;
                    split2(s[e / 2][nt][2 * (e % 2)], s[e / 2][nt][2 * (e % 2) + 1], h1, l1);
                    ph[nt][e] = h1;
                    pl[nt][e] = l1;
                }
        }
        auto tile = [&](int h, auto j) __attribute__((always_inline)) {
            if constexpr (kX3) {
                u32x4 hi, lo;
                value(h, j, hi, lo);
                const f16x8 vh = __builtin_bit_cast(f16x8, hi), vl = __builtin_bit_cast(f16x8, lo);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    f32x4& o = acc[4 * h + j][nt];
                    const f16x8 p8 = __builtin_bit_cast(f16x8, ph[nt]);
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, p8, o, 0, 0, 0);
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, __builtin_bit_cast(f16x8, pl[nt]), o, 0, 0, 0);
                    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, p8, o, 0, 0, 0);
                }
            } else {
                // a step's part is a chain of eight from zero, added to the rest: as
                // short as a long context's sums need it
                f32x4 part[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) part[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = value(mt, i, h, j);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            part[nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[mt][nt][i], part[nt], 0, 0, 0);
                    }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[4 * h + j][nt] += part[nt];
            }
        };
#pragma unroll
        for (int h = 0; h < H; ++h) {
            tile(h, std::integral_constant<int, 0>{});
            tile(h, std::integral_constant<int, 1>{});
            tile(h, std::integral_constant<int, 2>{});
            tile(h, std::integral_constant<int, 3>{});
        }
    };

    // ---- cached steps
    if (step < end) {
        auto cached_scores = [&]() __attribute__((always_inline)) {
            if constexpr (kStaged)
                scores(from_f32(staged_k));
            else if constexpr (kX3)
                scores([&](int mt, int kc, u32x4& hi, u32x4& lo) __attribute__((always_inline)) {
                    const unsigned one = kd[mt][kc / 2];
                    const f16x2 d = __builtin_bit_cast(f16x2, one | one << 16);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const unsigned w = kw[mt][kc / 2][2 * (kc % 2) + e];
                        unsigned h0, h1, l0, l1;
                        scaled2<0, 1>(w, 0, d, h0, l0);
                        scaled2<2, 3>(w, 0, d, h1, l1);
                        hi[2 * e] = h0;
                        hi[2 * e + 1] = h1;
                        lo[2 * e] = l0;
                        lo[2 * e + 1] = l1;
                    }
                });
            else
                scores([&](int mt, int c) __attribute__((always_inline)) {
                    const float d = half_bits_to_float(static_cast<uint16_t>(kd[mt][c / 4]));
                    const unsigned w = kw[mt][c / 4][c % 4];
                    return f32x4{sbyte_to_float<0>(w) * d, sbyte_to_float<1>(w) * d, sbyte_to_float<2>(w) * d, sbyte_to_float<3>(w) * d};
                });
        };
        auto cached_output = [&]() __attribute__((always_inline)) {
            if constexpr (!kQ8)
                output(values_from_f32(v));
            else if constexpr (kX3)
                output([&](int h, auto j, u32x4& hi, u32x4& lo) __attribute__((always_inline)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int mt = e / 2, i = 2 * (e % 2);
                        unsigned h1, l1;
                        scaled2<j, 4 + j>(vw[mt][i][h], vw[mt][i + 1][h],
                                          __builtin_bit_cast(f16x2, vd[mt][i] | vd[mt][i + 1] << 16), h1, l1);
                        hi[e] = h1;
                        lo[e] = l1;
                    }
                });
            else
                output([&](int mt, int i, int h, auto j) __attribute__((always_inline)) {
                    return sbyte_to_float<j>(vw[mt][i][h]) * half_bits_to_float(static_cast<uint16_t>(vd[mt][i]));
                });
        };
        if constexpr (!kEarly) {
            load_k(step);
            if constexpr (kStaged) asm volatile("" ::: "memory");
            load_v(step);
        }
        for (; step < end; step += stride) {
            const int next = step + stride;
            if constexpr (kStaged) wait_until_left<8 * H>();  // the values'
            cached_scores();
            if constexpr (kStaged) wait_for_lds();
            // the loads of the next step go out as soon as there is room (past the end the
            // last step's again: its blocks are there)
            if (++at == 32) {
                at = 0;
                ids = more;
                more = lookup(next + 32 * stride);
            }
            load_k(next);
            if constexpr (kStaged) asm volatile("" ::: "memory");
            if (kStep * step + kStep <= cached) {
                softmax(std::false_type{}, [](int, int, int) { return true; });
            } else {  // the last keys: what lies behind them is not seen, and its values are zeros
                softmax(std::true_type{}, [&](int mt, int i, int) { return kStep * step + 16 * mt + 4 * g + i < cached; });
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (kStep * step + 16 * mt + 4 * g + i >= cached) {
                            if constexpr (kQ8) vd[mt][i] = 0;
#pragma unroll
                            for (int h = 0; h < H; ++h)
                                if constexpr (kQ8)
                                    vw[mt][i][h] = 0;
                                else
                                    v[mt][i][h] = f32x4{0.f, 0.f, 0.f, 0.f};
                        }
            }
            cached_output();
            load_v(next);
        }
        if constexpr (kStaged) wait_until_left<0>();  // (LDS is used again)
    }

    // ---- the tree's own nodes
    for (; step < it.end; step += stride) {
        const int n0 = kStep * (step - csteps);
        const float* kb = a.keys + static_cast<size_t>(tree.w) * a.row_stride + static_cast<size_t>(kh) * D;
        const float* vb = a.values + static_cast<size_t>(tree.w) * a.row_stride + static_cast<size_t>(kh) * D;
        f32x4 k[2][C], v[2][4][H];
        uint32_t mask[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            mask[nt] = live[nt] ? a.mask[static_cast<size_t>(tree.w + node[nt]) * a.words + (step - csteps)] : 0u;
        bool odd = false;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const float* kr = kb + static_cast<size_t>(min(n0 + 16 * mt + r16, nodes - 1)) * a.row_stride;
#pragma unroll
            for (int c = 0; c < C; ++c) k[mt][c] = *reinterpret_cast<const f32x4*>(kr + kcol(c));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float* vr = vb + static_cast<size_t>(min(n0 + 16 * mt + 4 * g + i, nodes - 1)) * a.row_stride;
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    v[mt][i][h] = *reinterpret_cast<const f32x4*>(vr + vcol(h, r16));
#pragma unroll
                    for (int j = 0; j < 4; ++j) odd |= !fits<kX3>(v[mt][i][h][j]);
                }
            }
        }
        scores(from_f32([&](int mt, int c) __attribute__((always_inline)) { return k[mt][c]; }));
        softmax(std::true_type{}, [&](int mt, int i, int nt) { return (mask[nt] >> (16 * mt + 4 * g + i) & 1u) != 0; });
        const bool plain = !__any(odd);
        if (!plain) {
            // Zero times such a value would reach rows that do not see it: it is
            // zero in the product, and added below to the rows that do.
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[mt][i][h][j] = fits<kX3>(v[mt][i][h][j]) ? v[mt][i][h][j] : 0.f;
        }
        output(values_from_f32(v));
        if (plain) continue;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll 1
            for (int e = 0; e < 16; ++e) {
                const int key = n0 + 16 * mt + e, i = e & 3;
                if (key >= nodes) break;
                const float* vr = vb + static_cast<size_t>(key) * a.row_stride;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float own = i == 0 ? s[mt][nt][0] : i == 1 ? s[mt][nt][1] : i == 2 ? s[mt][nt][2] : s[mt][nt][3];
                    const float p = __shfl(own, r16 + 16 * (e >> 2));
                    const bool on = (mask[nt] >> (16 * mt + e) & 1u) != 0;
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int o = 0; o < 4; ++o) {
                            const f32x4 x = *reinterpret_cast<const f32x4*>(vr + vcol(h, 4 * g + o));
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (on && !fits<kX3>(x[j]))
                                    acc[4 * h + j][nt][o] = fmaf(p, unfit<kX3>(x[j]), acc[4 * h + j][nt][o]);
                        }
                }
            }
    }
    if (__any(nonfinite != 0.f) && lane == 0) *a.err = 1;

    // ---- the waves that shared these rows' keys, together
    float total[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) total[nt] = cross_row_sum(l[nt]);
    if constexpr (!kAlone) {
        if (g == 0)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) stats[wave][16 * nt + r16] = make_float2(m[nt], total[nt]);
        __syncthreads();
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if constexpr (kAlone) continue;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, stats[w][16 * nt + r16].x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            const float2 x = stats[w][16 * nt + r16];
            sum = fmaf(fast_exp2(x.x - base), x.y, sum);
        }
        const float scale = fast_exp2(m[nt] - base);
#pragma unroll
        for (int dt = 0; dt < 4 * H; ++dt) acc[dt][nt] *= scale;
        m[nt] = top;
        total[nt] = sum;
    }
    // four columns of output row 4g + i of the tiles, of a row tile's row r16
    bool bad = false;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        auto mine = [&](int i, int nt) {
            return f32x4{acc[4 * h][nt][i], acc[4 * h + 1][nt][i], acc[4 * h + 2][nt][i], acc[4 * h + 3][nt][i]};
        };
        auto put = [&](int i, int nt, f32x4 x) __attribute__((always_inline)) {
            if (!live[nt]) return;
            const size_t row = static_cast<size_t>(tree.w) + node[nt];
            if (it.runs == 1) {
                x /= total[nt];
                bad |= kX3 && !all_finite(x);
                *reinterpret_cast<f32x4*>(a.out + (row * a.heads + head[nt]) * D + vcol(h, 4 * g + i)) = x;
            } else {
                const size_t p = (static_cast<size_t>(it.slot) + static_cast<size_t>(node[nt]) * it.runs + it.run) * a.heads + head[nt];
                *reinterpret_cast<f32x4*>(a.part_acc + p * D + vcol(h, 4 * g + i)) = x;
                if (h == 0 && i == 0 && g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * p) = make_float2(m[nt], total[nt]);
            }
        };
        if constexpr (kAlone) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) put(i, nt, mine(i, nt));
            continue;
        }
        if (h) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) result(wave, i, nt) = mine(i, nt);
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            f32x4 x = result(0, wave, nt);
#pragma unroll
            for (int w = 1; w < WK; ++w) x += result(w, wave, nt);
            put(wave, nt, x);
        }
    }
    if (bad) *a.err = 1;
}

// Many rows of a (tree, KV head), f32x3: four waves of up to 32 rows each share every
// key.  A wave in turn is given 16 keys, or the values of 32, of a step to come: it
// loads them an iteration ahead into registers, splits them once for all the rows
// and leaves the parts in LDS in the order in which the products' lanes read them
// (lane l its own 16 bytes: no conflicts), in the other of two buffers; one barrier
// an iteration of S steps.  Loads go through descriptors that end with the last
// key, so that what lies behind it reads as zeros.
//
// MI355X, 16 contexts of 4,096 with 32 nodes, 32 heads on 8 of 128: 140 us with the
// merge, 4.0 TB/s (a copy reads and writes 4.8); 8 contexts of 4,096 with 64 nodes, 64
// heads on 8: 224 us, 3 x 308 TFLOP/s of fp16 products: the matrix pipe is busy half
// of the time, and the vector instructions of two waves a SIMD (250 a step, beside
// 96 products) do not hide behind it.
template <int D, bool kQ8>
__global__ __launch_bounds__(64 * kWaves, 2) void tree_shared_kernel(const TreeArgs a) {
    constexpr int NT = 2, C = D / 16, KC = D / 32, H = D / 64;
    constexpr int S = 128 / D;       // steps an iteration: eight float4 a thread
    constexpr int KW = kWaves / 2;   // waves that take keys; the others take values
    constexpr int TK = 128 / D;      // key tiles of 16 a wave takes
    constexpr int VO = 4 * KC, OPS = VO + 8 * H;  // operands of a step: hi, lo of [mt][kc] keys, then of the value tiles
    __shared__ u32x4 parts[2][S][OPS][64];
    __shared__ int odds[2][S][H];    // the tree's own values: some do not fit
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    const Item it = item_of(a, blockIdx.x);
    if (!it.tree.z) return;  // the list's padding
    const int4 tree = it.tree;
    const int cached = tree.y, nodes = tree.z, kh = it.head, G = a.group, kvw = a.lay.kv_width;
    // 16 rows a tile, dealt to the waves in turn; a wave without any still stages
    const int row0 = it.row0 + wave * 16, left_rows = nodes * G - row0;
    const int tiles = left_rows > 16 * kWaves ? 2 : left_rows > 0 ? 1 : 0;
    auto row_of = [&](int nt) { return row0 + 16 * kWaves * nt + r16; };
    auto node_of = [&](int nt) { return row_of(nt) / G; };

    // the lane's c-th four columns of a key: as the staging lane holds them.  Of f32
    // blocks that one loads parts of whole rows, two for each operand: part X of the
    // row's first half and of its second make eight columns for the lane group X % 4
    // of the products over X / 4.
    constexpr int X = D / 8;  // lanes that load a row's half
    auto kcol = [&](int c) { return kQ8 ? 64 * (c / 4) + 16 * g + 4 * (c % 4) : 16 * (c / 2) + 4 * g + D / 2 * (c % 2); };
    // f32: where the operand of part x of row r goes among the 16 of its lane group, so
    // that neither the lanes of a row nor those of a group meet a bank twice
    auto swizzle = [&](int r, int x) { return kQ8 ? r : r ^ (16 / X * x); };
    u32x4 qh[NT][KC], ql[NT][KC];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int node = node_of(nt), head = kh * G + row_of(nt) - node * G;
        const float* qp = a.q + (static_cast<size_t>(tree.w + node) * a.heads + head) * D;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
            if (node < nodes) x = *reinterpret_cast<const f32x4*>(qp + kcol(c));
            x *= a.qscale;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                unsigned hi, lo;
                split2(x[2 * e], x[2 * e + 1], hi, lo);
                qh[nt][c / 2][2 * (c % 2) + e] = hi;
                ql[nt][c / 2][2 * (c % 2) + e] = lo;
            }
        }
    }
    f32x4 acc[4 * H][NT];
    float m[NT], l[NT], rounded[NT];  // m: the maximum less kPartsLift
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = rounded[nt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < 4 * H; ++dt) acc[dt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // ---- staging: TK key tiles of 16 from mt0 on, or the value half vh, of step
    // `sub` of the iteration
    const bool takes_keys = wave < KW;
    const int mt0 = wave * TK % 2, vh = (wave - KW) % H;
    const int sub = takes_keys ? wave * TK / 2 : (wave - KW) / H;
    const int csteps = (cached + kStep - 1) / kStep;
    const int tpb = a.lay.tpb, tsh = __builtin_ctz(static_cast<unsigned>(tpb));
    const int32_t* tab = a.tables + tree.x;
    const size_t section = kQ8 ? a.lay.section : static_cast<size_t>(tpb) * kvw * sizeof(float);
    const size_t kbytes = (static_cast<size_t>(a.layer) * 2 + (takes_keys ? 0 : 1)) * section +
                          (kQ8 ? static_cast<size_t>(kh) * a.lay.head_bytes : static_cast<size_t>(kh) * D * sizeof(float));
    const int rowb = kQ8 ? D : kvw * static_cast<int>(sizeof(float));
    const int last = max(cached - 1, 0) >> 4;  // the last 16 cached keys
    const char* own = reinterpret_cast<const char*>((takes_keys ? a.keys : a.values) +
                                                    static_cast<size_t>(tree.w) * a.row_stride + static_cast<size_t>(kh) * D);
    const int ownb = static_cast<int>(a.row_stride * sizeof(float));
    f32x4 raw[8];                     // eight float4
    u32x4 rawq[kQ8 ? 2 : 1];          // Q8_0: their bytes and scales
    unsigned rawd[kQ8 ? 8 : 1];
    // Lane 2i + mt has key tile mt (16 keys) of this wave's step in the i-th
    // iteration from here: its block, and where its rows start and how many bytes
    // there are to the end of the last key, zero behind it.
    auto lookup = [&](int step) __attribute__((always_inline)) {
        return cached ? tab[min(2 * min(step + (lane >> 1) * S, csteps) + (lane & 1), last) << 4 >> tsh] : 0;
    };
    Spans rows16, scales16;
    auto spans = [&](int step, int id) __attribute__((always_inline)) {
        const int mine = step + (lane >> 1) * S, key = 16 * (2 * mine + (lane & 1)), n = key - kStep * csteps;
        const char* block = a.pool + static_cast<size_t>(id) * a.lay.stride + kbytes;
        const int slot = key & (tpb - 1), left = min(cached - key, 16), own_left = min(nodes - n, 16);
        if (kQ8 || mine < csteps)
            rows16.set(block + static_cast<size_t>(slot) * rowb, left > 0 ? (left - 1) * rowb + (kQ8 ? D : 4 * D) : 0);
        else
            rows16.set(own + static_cast<size_t>(n) * ownb, own_left > 0 ? (own_left - 1) * ownb + 4 * D : 0);
        if constexpr (kQ8)
            scales16.set(block + static_cast<size_t>(tpb) * D + static_cast<size_t>(slot) * (D / 32) * 2, max(left, 0) * (D / 32) * 2);
    };
    int more = lookup(it.step + 32 * S + sub), at = 0;
    spans(it.step + sub, lookup(it.step + sub));
    auto load = [&](int step) __attribute__((always_inline)) {
        // the key tiles of a thread's first and second half of the loads
        const int ia = 2 * at + (takes_keys && D == 128 ? mt0 : 0), ib = 2 * at + (takes_keys && D == 128 ? mt0 : 1);
        const __amdgpu_buffer_rsrc_t t0 = rows16.descriptor(ia), t1 = rows16.descriptor(ib);
        if constexpr (!kQ8) {
            const int pitch = step < csteps ? rowb : ownb;
            const int off = takes_keys ? lane / X * pitch + lane % X * 16 : 4 * g * pitch + 256 * vh + 16 * r16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // (keys: 64 / X rows an instruction)
                const int n = D == 128 ? i : i / 2, half = D == 128 ? 0 : i % 2;
                const int at0 = takes_keys ? 64 / X * n * pitch + 2 * D * half : i * pitch;
                raw[i] = __builtin_amdgcn_raw_buffer_load_b128(t0, off, at0, 0);
                raw[4 + i] = __builtin_amdgcn_raw_buffer_load_b128(t1, off, at0 + (takes_keys && D == 128 ? 2 * D : 0), 0);
            }
        } else {
            const __amdgpu_buffer_rsrc_t s0 = scales16.descriptor(ia), s1 = scales16.descriptor(ib);
            const int off = takes_keys ? r16 * D + 16 * g : 4 * g * D + 64 * vh + 4 * r16;
            const int soff = takes_keys ? (r16 * (D / 32) + (g >> 1)) * 2 : (4 * g * (D / 32) + 2 * vh + (r16 >> 3)) * 2;
            if (takes_keys) {
                const int far = D == 128 ? 1 : 0;
                rawq[0] = __builtin_amdgcn_raw_buffer_load_b128(t0, off, 0, 0);
                rawq[1] = __builtin_amdgcn_raw_buffer_load_b128(t1, off, 64 * far, 0);
                rawd[0] = __builtin_amdgcn_raw_buffer_load_b16(s0, soff, 0, 0);
                rawd[1] = __builtin_amdgcn_raw_buffer_load_b16(s1, soff, 4 * far, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    rawq[i / 4][i % 4] = __builtin_amdgcn_raw_buffer_load_b32(i < 4 ? t0 : t1, off, i % 4 * D, 0);
                    rawd[i] = __builtin_amdgcn_raw_buffer_load_b16(i < 4 ? s0 : s1, soff, i % 4 * (D / 32) * 2, 0);
                }
            }
        }
        if (++at == 32) {
            at = 0;
            spans(step + S, more);
            more = lookup(step + 33 * S);
            wait_for_loads();
        }
    };
    auto stage = [&](int buf, int step, const f32x4 (&x)[8]) __attribute__((always_inline)) {
        if (takes_keys) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {  // an operand: two float4
                u32x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f32x4 y = x[kQ8 || D == 64 ? 2 * p + e / 2 : p + 4 * (e / 2)];
                    unsigned h1, l1;
                    split2(y[2 * (e % 2)], y[2 * (e % 2) + 1], h1, l1);
                    hi[e] = h1;
                    lo[e] = l1;
                }
                u32x4* to;
                if constexpr (kQ8) {
                    const int o = D == 128 ? mt0 * KC + p : p;  // [mt][kc]
                    to = &parts[buf][sub][2 * o][lane];
                } else {
                    const int part = lane % X, row = 64 / X * (D == 128 ? p : p % 2) + lane / X, mt = D == 128 ? mt0 : p / 2;
                    to = &parts[buf][sub][2 * (mt * KC + part / 4)][16 * (part % 4) + swizzle(row, part)];
                }
                to[0] = hi;
                to[64] = lo;
            }
        } else {
            const bool tail = step >= csteps;
            bool odd = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 y[2] = {{x[0][j], x[1][j], x[2][j], x[3][j]}, {x[4][j], x[5][j], x[6][j], x[7][j]}};
                if (tail) {
                    // Zero times a value that does not fit would reach rows that do not
                    // see it: it is zero in the product, and added to the rows that do.
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const bool in = fits<true>(y[e / 4][e % 4]);
                        odd |= !in;
                        y[e / 4][e % 4] = in ? y[e / 4][e % 4] : 0.f;
                    }
                }
                u32x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned h1, l1;
                    split2(y[e / 2][2 * (e % 2)], y[e / 2][2 * (e % 2) + 1], h1, l1);
                    hi[e] = h1;
                    lo[e] = l1;
                }
                parts[buf][sub][VO + 2 * (4 * vh + j)][lane] = hi;
                parts[buf][sub][VO + 2 * (4 * vh + j) + 1][lane] = lo;
            }
            if (tail) {
                const bool any = __any(odd);
                if (lane == 0) odds[buf][sub][vh] = any;
            }
        }
    };
    auto put = [&](int buf, int step) __attribute__((always_inline)) {
        if constexpr (!kQ8) {
            stage(buf, step, raw);
        } else if (takes_keys) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {  // (words 0 to 3 are of the first key or half, 4 to 7 of the second)
                const f16x2 d = __builtin_bit_cast(f16x2, rawd[p / 2] | rawd[p / 2] << 16);
                u32x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const unsigned w = rawq[p / 2][2 * (p % 2) + e];
                    unsigned h0, h1, l0, l1;
                    scaled2<0, 1>(w, 0, d, h0, l0);
                    scaled2<2, 3>(w, 0, d, h1, l1);
                    hi[2 * e] = h0;
                    hi[2 * e + 1] = h1;
                    lo[2 * e] = l0;
                    lo[2 * e + 1] = l1;
                }
                const int o = D == 128 ? mt0 * KC + p : p;
                parts[buf][sub][2 * o][lane] = hi;
                parts[buf][sub][2 * o + 1][lane] = lo;
            }
        } else {
            auto tile = [&](auto j) __attribute__((always_inline)) {
                u32x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x2 d = __builtin_bit_cast(f16x2, rawd[2 * e] | rawd[2 * e + 1] << 16);
                    unsigned h1, l1;
                    scaled2<j, 4 + j>(rawq[e / 2][2 * (e % 2)], rawq[e / 2][2 * (e % 2) + 1], d, h1, l1);
                    hi[e] = h1;
                    lo[e] = l1;
                }
                parts[buf][sub][VO + 2 * (4 * vh + j)][lane] = hi;
                parts[buf][sub][VO + 2 * (4 * vh + j) + 1][lane] = lo;
            };
            tile(std::integral_constant<int, 0>{});
            tile(std::integral_constant<int, 1>{});
            tile(std::integral_constant<int, 2>{});
            tile(std::integral_constant<int, 3>{});
        }
    };

    f32x4 s[2][NT];  // scores, then probabilities, of keys 16mt + 4g + i
    auto operands = [&](int buf, int t) __attribute__((always_inline)) {
        unsigned at16 = static_cast<unsigned>((buf * S + t) * OPS * 64 + lane);
        asm("" : "+v"(at16));  // one address, the operands at constant offsets from it
        return &parts[0][0][0][0] + at16;
    };
    // (operands are read from LDS one ahead of their products)
    auto scores = [&](int buf, int t) __attribute__((always_inline)) {
        unsigned base = static_cast<unsigned>((buf * S + t) * OPS * 64 + 16 * g + swizzle(r16, g));
        asm("" : "+v"(base));
        auto operand = [&](int o) __attribute__((always_inline)) {  // (swizzle(r16, 4 kc + g): an exclusive or by 4 kc more)
            return &parts[0][0][0][0] + (kQ8 ? base : base ^ (16 / X * 4 * (o % KC))) + 128 * o;
        };
        u32x4 hi = operand(0)[0], lo = operand(0)[64];
#pragma unroll
        for (int o = 0; o < 2 * KC; ++o) {
            const int mt = o / KC, kc = o % KC;
            const f16x8 kh8 = __builtin_bit_cast(f16x8, hi), kl8 = __builtin_bit_cast(f16x8, lo);
            if (o + 1 < 2 * KC) {
                hi = operand(o + 1)[0];
                lo = operand(o + 1)[64];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                s[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl8, __builtin_bit_cast(f16x8, qh[nt][kc]),
                                                                   kc ? s[mt][nt] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                s[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh8, __builtin_bit_cast(f16x8, ql[nt][kc]), s[mt][nt], 0, 0, 0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                s[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh8, __builtin_bit_cast(f16x8, qh[nt][kc]), s[mt][nt], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    u32x4 ph[NT], pl[NT];
    auto softmax = [&](int buf, int t, int step) __attribute__((always_inline)) {
        // what a row does not see: keys behind the last cached one, other branches' nodes
        const bool tail = step >= csteps;
        if (tail || kStep * step + kStep > cached) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int node = node_of(nt);
                uint32_t mask = tail ? 0u : (1u << (cached - kStep * step)) - 1;
                if (tail && node < nodes) mask = a.mask[static_cast<size_t>(tree.w + node) * a.words + (step - csteps)];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(mask >> (16 * mt + 4 * g + i) & 1u)) s[mt][nt][i] = -INFINITY;
            }
            wait_for_loads();
        }
        // (a score that is not finite is NaN here, and so is its row's sum: an input
        // beyond fp16 is infinite in one part and its opposite in the other)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[mt][nt][i]);
            if (__any(mx > m[nt] + (kPartsThreshold + kPartsLift))) {
                const float mn = fmaxf(m[nt], cross_row_max(mx) - kPartsLift);
                const float alpha = m[nt] == -INFINITY ? 0.f : fast_exp2(m[nt] - mn);
                m[nt] = mn;
                l[nt] *= alpha;
                rounded[nt] *= alpha;
#pragma unroll
                for (int dt = 0; dt < 4 * H; ++dt) acc[dt][nt] *= alpha;
            }
            const float base = m[nt] == -INFINITY ? 0.f : m[nt];  // (no key seen yet: probabilities 0)
            float sum = 0.f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = fast_exp2(s[mt][nt][i] - base);
                    s[mt][nt][i] = p;
                    sum += p;
                }
            add_to(l[nt], rounded[nt], sum);
        }
        bool odd = false;
        if (tail)
#pragma unroll
            for (int h = 0; h < H; ++h) odd |= odds[buf][t][h] != 0;
        if (odd) {
            const int n0 = kStep * (step - csteps);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int node = node_of(nt);
                const uint32_t mask = node < nodes ? a.mask[static_cast<size_t>(tree.w + node) * a.words + (step - csteps)] : 0u;
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll 1
                    for (int e = 0; e < 16; ++e) {
                        const int key = n0 + 16 * mt + e, i = e & 3;
                        if (key >= nodes) break;
                        const float* vr = a.values + static_cast<size_t>(tree.w + key) * a.row_stride + static_cast<size_t>(kh) * D;
                        const float mine = i == 0 ? s[mt][nt][0] : i == 1 ? s[mt][nt][1] : i == 2 ? s[mt][nt][2] : s[mt][nt][3];
                        const float p = __shfl(mine, r16 + 16 * (e >> 2));
                        const bool on = (mask >> (16 * mt + e) & 1u) != 0;
#pragma unroll
                        for (int h = 0; h < H; ++h)
#pragma unroll
                            for (int o = 0; o < 4; ++o) {
                                const f32x4 y = *reinterpret_cast<const f32x4*>(vr + 64 * h + 4 * (4 * g + o));
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    if (on && !fits<true>(y[j]))
                                        acc[4 * h + j][nt][o] = fmaf(p, unfit<true>(y[j]), acc[4 * h + j][nt][o]);
                            }
                    }
            }
            wait_for_loads();
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned h1, l1;
                split2(s[e / 2][nt][2 * (e % 2)], s[e / 2][nt][2 * (e % 2) + 1], h1, l1);
                ph[nt][e] = h1;
                pl[nt][e] = l1;
            }
    };
    auto output = [&](int buf, int t) __attribute__((always_inline)) {
        const u32x4* op = operands(buf, t) + 64 * VO;
        u32x4 hi = op[0], lo = op[64];
#pragma unroll
        for (int dt = 0; dt < 4 * H; ++dt) {
            const f16x8 vh8 = __builtin_bit_cast(f16x8, hi), vl8 = __builtin_bit_cast(f16x8, lo);
            if (dt + 1 < 4 * H) {
                hi = op[64 * (2 * dt + 2)];
                lo = op[64 * (2 * dt + 3)];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                acc[dt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl8, __builtin_bit_cast(f16x8, ph[nt]), acc[dt][nt], 0, 0, 0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                acc[dt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh8, __builtin_bit_cast(f16x8, pl[nt]), acc[dt][nt], 0, 0, 0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                acc[dt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh8, __builtin_bit_cast(f16x8, ph[nt]), acc[dt][nt], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Q8_0 blocks: the tree's own f32 rows are not in the pipeline of the cached ones
    const int end = kQ8 ? min(it.end, csteps) : it.end;
    if (it.step < end) {
        load(it.step + sub);
        put(0, it.step + sub);
        load(it.step + S + sub);
        __syncthreads();
        int buf = 0;
        for (int step = it.step; step < end; step += S, buf ^= 1) {
            put(buf ^ 1, step + S + sub);
            load(step + 2 * S + sub);
            if (tiles)
#pragma unroll 1
                for (int t = 0; t < S && step + t < end; ++t) {
                    scores(buf, t);
                    softmax(buf, t, step + t);
                    output(buf, t);
                }
            __syncthreads();
        }
    }
    if constexpr (kQ8) {
#pragma unroll 1
        for (int step = max(it.step, csteps); step < it.end; step += S) {
            const int n0 = kStep * (step + sub - csteps);
            f32x4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = n0 + (takes_keys ? 16 * (D == 128 ? mt0 : i / 4) + r16 : 16 * (i / 4) + 4 * g + i % 4);
                const int col = takes_keys ? kcol(D == 128 ? i : i % 4) : 64 * vh + 4 * r16;
                x[i] = *reinterpret_cast<const f32x4*>(own + static_cast<size_t>(min(key, nodes - 1)) * ownb + 4 * col);
            }
            stage(0, step + sub, x);
            __syncthreads();
            if (tiles)
#pragma unroll 1
                for (int t = 0; t < S && step + t < it.end; ++t) {
                    scores(0, t);
                    softmax(0, t, step + t);
                    output(0, t);
                }
            __syncthreads();
        }
    }

    float total[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) total[nt] = cross_row_sum(l[nt]);
    bool bad = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int node = node_of(nt), head = kh * G + row_of(nt) - node * G;
        if (node >= nodes) continue;
        const bool whole = it.runs == 1;
        const size_t to = (whole ? static_cast<size_t>(tree.w) + node
                                 : static_cast<size_t>(it.slot) + static_cast<size_t>(node) * it.runs + it.run) * a.heads + head;
        float* o = (whole ? a.out : a.part_acc) + to * D + 16 * g;
        const float inv = whole ? total[nt] : 1.f;
        if (!whole && g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * to) = make_float2(m[nt], total[nt]);
        bad |= !__builtin_isfinite(total[nt]);
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 x = f32x4{acc[4 * h][nt][i], acc[4 * h + 1][nt][i], acc[4 * h + 2][nt][i], acc[4 * h + 3][nt][i]} / inv;
                bad |= !all_finite(x);
                *reinterpret_cast<f32x4*>(o + 64 * h + 4 * i) = x;
            }
    }
    if (bad) *a.err = 1;
}

template <int D, bool kQ8, bool kX3>
void launch_shape(const TreeArgs& a, int rows, int workgroups, hipStream_t s) {
    auto go = [&](auto kernel) { launch("tree_attention_tiles", kernel, dim3(workgroups), dim3(64 * kWaves), 0, s, a); };
    if constexpr (!kX3)
        if (a.alone) return go(tree_tile_kernel<D, 1, kQ8, false, true>);
    if (rows == 16)
        go(tree_tile_kernel<D, 1, kQ8, kX3>);
    else if constexpr (kX3)
        rows == 32 ? go(tree_tile_kernel<D, 2, kQ8, kX3>) : go(tree_shared_kernel<D, kQ8>);
    else
        throw std::logic_error("no f32 tree kernel for these rows");
}

}  // namespace

bool tree_tiles_supported(const BlockLayout& lay) {
    return (lay.head_dim == 64 || lay.head_dim == 128) && lay.tpb >= 16 && (lay.tpb & (lay.tpb - 1)) == 0 &&
           lay.stride <= static_cast<size_t>(1) << 31;
}

// Workgroups that a CU is dealt: what its registers (f32x3 of 128 columns one, of 64
// two) or LDS (128 rows: two) hold.  f32 holds more than pay for their merges: of 64
// columns (four) three (MI355X, 16 ragged contexts 2: 47.1 us  3: 45.4  4: 46.9), of
// 128 (two) over f32 blocks one (16 contexts of 2048, 32 rows 1: 58.7  2: 67.0), over
// Q8_0 two (1: 70.0  2: 63.2).
// Where workgroups are many and their steps few, the waves of f32 take an entry of work
// each (alone): a workgroup's start, not its steps, is what passes then (60 trees of 24
// nodes after 3 tokens, head_dim 128: 57.6 us shared  31.5 alone; after 250: 118 and 89,
// but 16 of 12 nodes 22.2 and 30.7; over Q8_0, whose steps wait less, 61 trees of 11 nodes
// after 295, head_dim 64: 29.3 and 41.3).
// A run has at least a step a wave, and no more where there are CUs: a wave's second
// step waits for memory again (one context of 512 tokens in runs of 4 steps: 12.7,
// of 8: 14.0, of 12: 15.3, each with its merge).
TreeTileShape tree_tile_shape(const BlockLayout& lay, int rows, bool x3) {
    TreeTileShape t{};
    t.rows = rows;
    if (x3)
        t.units = rows == 128 || lay.head_dim == 64 ? 2 : 1;
    else
        t.units = lay.head_dim == 64 ? 3 : lay.format == kQ8 ? 2 : 1;
    t.least = kWaves;
    t.alone_from = x3 ? std::numeric_limits<int>::max() : lay.head_dim == 64 ? 4 : 3;
    t.alone_to = lay.format == kQ8 ? 4 : 12;
    return t;
}

void launch_tree_tiles(const TreeArgs& a, int rows, int workgroups, bool x3, hipStream_t s) {
    const bool q8 = a.lay.format == kQ8;
    if (a.lay.head_dim == 128) {
        if (x3)
            q8 ? launch_shape<128, true, true>(a, rows, workgroups, s) : launch_shape<128, false, true>(a, rows, workgroups, s);
        else
            q8 ? launch_shape<128, true, false>(a, rows, workgroups, s) : launch_shape<128, false, false>(a, rows, workgroups, s);
    } else {
        if (x3)
            q8 ? launch_shape<64, true, true>(a, rows, workgroups, s) : launch_shape<64, false, true>(a, rows, workgroups, s);
        else
            q8 ? launch_shape<64, true, false>(a, rows, workgroups, s) : launch_shape<64, false, false>(a, rows, workgroups, s);
    }
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

// Rows on their way into the cache, and out of it.
//
// Into it: of each head x of a token's queries and keys
//   y_c = x_c w_c / sqrt(mean_c x_c^2 + eps)          (where weights are given)
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_a sin t + y_b cos t),  t = position * freq_j
// for the pairs j of its first `rotary` columns; queries go to rows, keys and values
// into the token's slot, as f32 or quantised as appends quantise them.  One pass: a
// row is read once and written once.
//
// In f64 until the one rounding to f32 (its rate is f32's here): an angle of a far
// position needs it, and a key's byte in a Q8_0 block is then that of the exact value,
// however the sums were ordered.
#include <algorithm>

#include "common.hpp"
#include "q8.hpp"
#include "tree.hpp"

namespace tvara_amd {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kMaxDim = 512;

struct Turn {
    double c, s;
};

// cos and sin of position * freq: the rest of a quarter turn by two fused steps (the
// first is exact where the multiple of pi / 2 is below 2^31), then Taylor's series up to
// the terms below 1e-16.
__device__ __forceinline__ Turn turn_of(int position, float freq) {
    const double t = static_cast<double>(position) * static_cast<double>(freq);
    const double k = __builtin_rint(t * 0.63661977236758134308);
    double r = fma(-k, 1.57079632679489655800, t);
    r = fma(-k, 6.12323399573676603587e-17, r);
    const double y = r * r;
    double s = 1.0 / 6227020800.0 - y * (1.0 / 1307674368000.0);
    s = fma(-s, y, 1.0 / 39916800.0);
    s = fma(-s, y, 1.0 / 362880.0);
    s = fma(-s, y, 1.0 / 5040.0);
    s = fma(-s, y, 1.0 / 120.0);
    s = fma(-s, y, 1.0 / 6.0);
    s = fma(-s * y, r, r);
    double c = 1.0 / 87178291200.0 - y * (1.0 / 20922789888000.0);
    c = fma(-c, y, 1.0 / 479001600.0);
    c = fma(-c, y, 1.0 / 3628800.0);
    c = fma(-c, y, 1.0 / 40320.0);
    c = fma(-c, y, 1.0 / 720.0);
    c = fma(-c, y, 1.0 / 24.0);
    c = fma(-c, y, 0.5);
    c = fma(-c, y, 1.0);
    const int quarter = static_cast<int>(k - 4.0 * __builtin_floor(k * 0.25));
    const double a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
    return {quarter == 1 || quarter == 2 ? -a : a, quarter >= 2 ? -b : b};
}

// where a slot's element lies in its block: the bytes before the layer's section of K
// (kind 0) or V
__device__ __forceinline__ size_t section_at(const BlockLayout& lay, int layer, int kind) {
    const size_t sec = static_cast<size_t>(layer) * 2 + kind;
    return lay.format == kF32 ? sec * lay.tpb * lay.kv_width * sizeof(float) : sec * lay.section;
}

// a token's slot: false where it has none
template <class Args>
__device__ __forceinline__ bool slot_of(const Args& a, size_t t, int64_t& block, int& slot) {
    const int64_t to = a.slots[t];
    if (to < 0) return false;
    if (to >= a.slot_count) {
        *a.err = 1;
        return false;
    }
    block = to / a.lay.tpb;
    slot = static_cast<int>(to - block * a.lay.tpb);
    return true;
}

// eight values of a group of 32 that four lanes hold, into a Q8_0 section
__device__ __forceinline__ void put_eight(char* section, const BlockLayout& lay, int slot, int column, const float (&x)[8]) {
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, __builtin_fabsf(x[e]));
    amax = fmaxf(amax, __shfl_xor(amax, 1));
    amax = fmaxf(amax, __shfl_xor(amax, 2));
    uint16_t d;
    u32x2 bytes = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        int8_t q;
        q8_encode_element(x[e], amax, &d, &q);
        bytes[e / 4] |= static_cast<unsigned>(static_cast<uint8_t>(q)) << 8 * (e % 4);
    }
    *reinterpret_cast<u32x2*>(section + q8_byte_offset(lay, slot, column)) = bytes;
    if (column % 32 == 0) *reinterpret_cast<uint16_t*>(section + q8_scale_offset(lay, slot, column / 32)) = d;
}

// Head sizes of eight columns times a power of two: a lane has eight columns, whole
// pairs of them.  Bound: HBM (4,000 tokens, 32 heads on 8 of 128, with norms: 41 us for 197 MB,
// 4.8 TB/s; 32 us over the same rows again and again, out of the last-level cache); a launch
// where tokens are few (one: 3 us).  grid.x: token, grid.y: a share of its heads (of queries,
// then keys, then values).
template <bool kQ8>
__global__ __launch_bounds__(kThreads) void rotate_kernel(const RotateArgs a, int turns) {
    __shared__ Turn angles[kMaxDim / 2];
    __shared__ float heads_of[kQ8 ? kThreads * 8 : 1];
    const size_t t = blockIdx.x;
    const int tid = threadIdx.x, D = a.lay.head_dim, lanes = D / 8, half = a.rotary / 2;
    const int units = a.heads + 2 * a.lay.kv_heads, each = kThreads / lanes, c = tid % lanes;
    int64_t block = 0;
    int slot = 0;
    const bool placed = a.slots && slot_of(a, t, block, slot);
    char* base = a.pool + block * a.lay.stride;
    for (int j = tid; j < half; j += kThreads) angles[j] = turn_of(a.positions[t], a.freqs[j]);
    __syncthreads();
    // columns of the lane's two fours, and the pair of the first
    const bool turning = a.interleaved ? 8 * c < a.rotary : 4 * c < half;
    const bool apart = !a.interleaved && turning;
    const int col0 = apart ? 4 * c : a.interleaved || !turning ? 8 * c : 0, col1 = apart ? half + 4 * c : col0 + 4;
    for (int i = 0; i < turns; ++i) {
        const int unit = (blockIdx.y * turns + i) * each + tid / lanes;
        const int kind = unit < a.heads ? 0 : unit < a.heads + a.lay.kv_heads ? 1 : 2;  // queries, keys, values
        const bool in = unit < units && (kind == 0 ? a.q_out != nullptr : placed || (kind == 1 && a.k_out));
        const int head = kind == 0 ? unit : kind == 1 ? unit - a.heads : unit - a.heads - a.lay.kv_heads;
        const float* from = kind == 0 ? a.q + t * a.q_stride : (kind == 1 ? a.keys : a.values) + t * a.kv_stride;
        const float* weight = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
        float out[8] = {};
        if (in) {
            const f32x4 x0 = *reinterpret_cast<const f32x4*>(from + head * D + col0);
            const f32x4 x1 = *reinterpret_cast<const f32x4*>(from + head * D + col1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                out[e] = x0[e];
                out[4 + e] = x1[e];
            }
        }
        if (kind < 2) {
            double x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = out[e];
            if (weight) {
                double sum = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fma(x[e], x[e], sum);
                for (int m = lanes / 2; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
                const double inv = 1.0 / __builtin_sqrt(sum / D + static_cast<double>(a.eps));
                const f32x4 w0 = *reinterpret_cast<const f32x4*>(weight + col0), w1 = *reinterpret_cast<const f32x4*>(weight + col1);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] *= inv * w0[e];
                    x[4 + e] *= inv * w1[e];
                }
            }
            if (turning) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const Turn u = angles[4 * c + e];
                    double& p = x[a.interleaved ? 2 * e : e];
                    double& q = x[a.interleaved ? 2 * e + 1 : 4 + e];
                    const double y = p;
                    p = fma(y, u.c, -(q * u.s));
                    q = fma(y, u.s, q * u.c);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = static_cast<float>(x[e]);
        }
        const f32x4 y0 = {out[0], out[1], out[2], out[3]}, y1 = {out[4], out[5], out[6], out[7]};
        float* row = kind == 0 ? a.q_out + (a.q_out ? t * a.heads * D : 0) : a.k_out + (a.k_out ? t * a.lay.kv_width : 0);
        if (in && kind < 2 && (kind == 0 ? a.q_out : a.k_out)) {
            *reinterpret_cast<f32x4*>(row + head * D + col0) = y0;
            *reinterpret_cast<f32x4*>(row + head * D + col1) = y1;
        }
        if constexpr (kQ8) {
            // a head's columns in order, by way of LDS
            float* mine = heads_of + (tid - c) * 8;
            __syncthreads();
            *reinterpret_cast<f32x4*>(mine + col0) = y0;
            *reinterpret_cast<f32x4*>(mine + col1) = y1;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = mine[8 * c + e];
            if (in && kind && placed) put_eight(base + section_at(a.lay, a.layer, kind - 1), a.lay, slot, head * D + 8 * c, out);
        } else if (in && kind && placed) {
            float* to = reinterpret_cast<float*>(base + section_at(a.lay, a.layer, kind - 1)) + static_cast<size_t>(slot) * a.lay.kv_width + head * D;
            *reinterpret_cast<f32x4*>(to + col0) = y0;
            *reinterpret_cast<f32x4*>(to + col1) = y1;
        }
    }
}

// Any even head size: a wave a (token, head), which passes over its columns by pairs.
template <bool kQ8>
__global__ __launch_bounds__(64) void rotate_rows_kernel(const RotateArgs a) {
    __shared__ float head_of[kQ8 ? kMaxDim : 1];
    const size_t t = blockIdx.x;
    const int lane = threadIdx.x, unit = blockIdx.y, D = a.lay.head_dim, half = a.rotary / 2;
    const int kind = unit < a.heads ? 0 : unit < a.heads + a.lay.kv_heads ? 1 : 2;
    const int head = kind == 0 ? unit : kind == 1 ? unit - a.heads : unit - a.heads - a.lay.kv_heads;
    const float* from = (kind == 0 ? a.q + t * a.q_stride : (kind == 1 ? a.keys : a.values) + t * a.kv_stride) + static_cast<size_t>(head) * D;
    const float* weight = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    float* rows = kind == 0 ? a.q_out : kind == 1 ? a.k_out : nullptr;
    if (rows) rows += t * (kind == 0 ? static_cast<size_t>(a.heads) * D : a.lay.kv_width) + static_cast<size_t>(head) * D;
    int64_t block = 0;
    int slot = 0;
    const bool placed = kind && a.slots && slot_of(a, t, block, slot);
    if (!rows && !placed) return;
    char* section = a.pool + block * a.lay.stride + section_at(a.lay, a.layer, kind ? kind - 1 : 0);
    float* to = kQ8 || !placed ? nullptr : reinterpret_cast<float*>(section) + static_cast<size_t>(slot) * a.lay.kv_width + static_cast<size_t>(head) * D;
    double inv = 1;
    if (weight) {
        double sum = 0;
        for (int c = lane; c < D; c += 64) sum = fma(static_cast<double>(from[c]), static_cast<double>(from[c]), sum);
        for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
        inv = 1.0 / __builtin_sqrt(sum / D + static_cast<double>(a.eps));
    }
    auto put = [&](int c, float y) {
        if (rows) rows[c] = y;
        if (to) to[c] = y;
        if constexpr (kQ8) head_of[c] = y;
    };
    for (int j = lane; j < D / 2; j += 64) {
        const bool turning = kind < 2 && j < half;
        const int c0 = turning ? (a.interleaved ? 2 * j : j) : j < half ? j : a.rotary + 2 * (j - half);
        const int c1 = turning && !a.interleaved ? j + half : j < half && !turning ? j + half : c0 + 1;
        const float f0 = from[c0], f1 = from[c1];
        if (kind == 2) {
            put(c0, f0);
            put(c1, f1);
            continue;
        }
        double x = f0, y = f1;
        if (weight) {
            x *= inv * weight[c0];
            y *= inv * weight[c1];
        }
        if (turning) {
            const Turn u = turn_of(a.positions[t], a.freqs[j]);
            const double z = x;
            x = fma(z, u.c, -(y * u.s));
            y = fma(z, u.s, y * u.c);
        }
        put(c0, static_cast<float>(x));
        put(c1, static_cast<float>(y));
    }
    if constexpr (kQ8) {
        if (!kind) return;
        __syncthreads();
        if (!placed) return;
        for (int c = lane; c < D; c += 64) {  // (whole groups of 32 lanes)
            float amax = __builtin_fabsf(head_of[c]);
            for (int m = 16; m >= 1; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m));
            uint16_t d;
            int8_t q;
            q8_encode_element(head_of[c], amax, &d, &q);
            const int column = head * D + c;
            *reinterpret_cast<int8_t*>(section + q8_byte_offset(a.lay, slot, column)) = q;
            if (c % 32 == 0) *reinterpret_cast<uint16_t*>(section + q8_scale_offset(a.lay, slot, column / 32)) = d;
        }
    }
}

// Slots back to rows: grid.x: token, grid.y: a share of its rows of every (layer, kind),
// kVec floats a thread.  Bound: HBM (1,500 tokens, four layers, 8 heads of 128 out of Q8_0:
// 14 to 16 us for 62 MB, 4.3 TB/s).
template <bool kQ8, int kVec>
__global__ __launch_bounds__(kThreads) void slot_read_kernel(const ReadArgs a) {
    int64_t block;
    int slot;
    const size_t t = blockIdx.x;
    if (!slot_of(a, t, block, slot)) return;
    const unsigned w = a.lay.kv_width / kVec, units = 2 * a.layers * w;
    const unsigned u = blockIdx.y * kThreads + threadIdx.x;
    if (u >= units) return;
    const unsigned r = u / w, c = (u - r * w) * kVec;  // r: layer * 2 + kind
    const char* section = a.pool + block * a.lay.stride + section_at(a.lay, a.layer + static_cast<int>(r >> 1), r & 1);
    float* to = ((r & 1) ? a.values : a.keys) + t * a.row_stride + (r >> 1) * a.layer_stride + c;
    if constexpr (kQ8) {
        const u32x2 bytes = *reinterpret_cast<const u32x2*>(section + q8_byte_offset(a.lay, slot, static_cast<int>(c)));
        const float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(section + q8_scale_offset(a.lay, slot, static_cast<int>(c / 32))));
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = d * static_cast<float>(static_cast<int8_t>(bytes[e / 4] >> 8 * (e % 4)));
        __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4*>(to));
        __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4*>(to + 4));
    } else {
        typedef float vec __attribute__((ext_vector_type(kVec)));
        const float* from = reinterpret_cast<const float*>(section) + static_cast<size_t>(slot) * a.lay.kv_width + c;
        __builtin_nontemporal_store(*reinterpret_cast<const vec*>(from), reinterpret_cast<vec*>(to));
    }
}

}  // namespace

void launch_rotate(const RotateArgs& a, hipStream_t s) {
    const int D = a.lay.head_dim, units = a.heads + 2 * a.lay.kv_heads;
    const bool q8 = a.lay.format == kQ8;
    const bool wide = D % 8 == 0 && (D & (D - 1)) == 0 && a.rotary % 8 == 0 && a.q_stride % 4 == 0 && a.kv_stride % 4 == 0;
    if (wide) {
        const int each = kThreads / (D / 8), shares = (units + each - 1) / each;
        // all of a token's heads in one workgroup, which takes their angles once, where
        // tokens are many (32 heads on 8 of 128, over the same rows again and again, which the
        // last-level cache holds, us with all heads and with a share: 256 tokens 5.3 and 4.9,
        // 1,024 9.3 and 10.1, 4,096 27.6 and 28.7)
        const int turns = a.n >= 1024 ? shares : 1;
        launch("rotate", q8 ? rotate_kernel<true> : rotate_kernel<false>,
               dim3(static_cast<unsigned>(a.n), static_cast<unsigned>((shares + turns - 1) / turns)), dim3(kThreads), 0, s, a, turns);
    } else {
        launch("rotate", q8 ? rotate_rows_kernel<true> : rotate_rows_kernel<false>,
               dim3(static_cast<unsigned>(a.n), static_cast<unsigned>(units)), dim3(64), 0, s, a);
    }
    TVARA_HIP(hipGetLastError());
}

void launch_slot_read(const ReadArgs& a, hipStream_t s) {
    const bool q8 = a.lay.format == kQ8, wide = a.lay.kv_width % 4 == 0 && a.row_stride % 4 == 0 && a.layer_stride % 4 == 0;
    const size_t units = static_cast<size_t>(2) * a.layers * a.lay.kv_width / (q8 ? 8 : wide ? 4 : 1);
    const dim3 grid(static_cast<unsigned>(a.n), static_cast<unsigned>((units + kThreads - 1) / kThreads));
    launch("slot_read", q8 ? slot_read_kernel<true, 8> : wide ? slot_read_kernel<false, 4> : slot_read_kernel<false, 1>, grid,
           dim3(kThreads), 0, s, a);
    TVARA_HIP(hipGetLastError());
}

}  // namespace tvara_amd

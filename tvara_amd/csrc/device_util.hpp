// Device-only helpers shared by the HIP kernels (included by .hip files).
#pragma once

#include <cstdint>

namespace tvara_amd {

// Signed byte B of w to float in one instruction (SDWA byte select with sign
// extension); the compiler's own lowering takes a shift, a bit-field extract
// and a conversion.
template <int B>
__device__ __forceinline__ float sbyte_to_float(uint32_t w) {
    float r;
    if constexpr (B == 0)
        asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(r) : "v"(w));
    else if constexpr (B == 1)
        asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(r) : "v"(w));
    else if constexpr (B == 2)
        asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(r) : "v"(w));
    else
        asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(r) : "v"(w));
    return r;
}

// Cross-row reductions with gfx950's permlane swaps.  permlane32_swap(x, y)
// returns (x.lo | y.lo, x.hi | y.hi) by 32-lane half and permlane16_swap
// returns (x.r0, y.r0, x.r2, y.r2 | x.r1, y.r1, x.r3, y.r3) by 16-lane row, so
// with y = x the two results hold a lane's value and its partner's.  (The
// results are copied to scalars before the bit cast: __builtin_bit_cast of a
// vector element reads element 0 with this compiler.)
template <class Op>
__device__ __forceinline__ float cross_row_reduce(float v, Op op) {
    const unsigned a = __builtin_bit_cast(unsigned, v);
    const auto h = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    const unsigned h0 = h[0], h1 = h[1];
    v = op(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1));
    const unsigned b = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return op(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}

// sum / max over lanes l%16 + 16r (the four 16-lane rows); every lane gets
// the same bits
__device__ __forceinline__ float cross_row_sum(float v) {
    return cross_row_reduce(v, [](float x, float y) { return x + y; });
}

__device__ __forceinline__ float cross_row_max(float v) {
    return cross_row_reduce(v, [](float x, float y) { return fmaxf(x, y); });
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Until at most n loads are on their way (they return in order), or every read of LDS
// is done; no access to memory moves across either.
template <int n>
__device__ __forceinline__ void wait_until_left() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((n & 15) | n >> 4 << 14 | 0xf70);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_for_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    asm volatile("" ::: "memory");
}

// A step's probabilities join a row's normaliser, with what the additions before have
// rounded away (Kahan's sum): beside one large probability each step's part may be
// less than half an ulp, and they are all of one sign.  MI355X, one key 19.5 above 131,072
// of N(0,1), f32: every output off by 2.4e-5 of itself without, 7e-7 with it.
__device__ __forceinline__ void add_to(float& l, float& rounded, float sum) {
    const float y = sum - rounded, t = l + y;
    rounded = (t - l) - y;
    l = t;
}

__device__ __forceinline__ bool all_finite(f32x4 x) {
    return __builtin_isfinite(x[0]) && __builtin_isfinite(x[1]) && __builtin_isfinite(x[2]) && __builtin_isfinite(x[3]);
}

// Two values as hi + lo in fp16, each rounded to nearest (22 bits; beyond fp16's
// range one is infinite and the other its opposite).  `one` is 1, hidden from the
// compiler, so that x - hi stays a mixed-precision fma: four instructions a pair
// where converting hi back takes six.
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) {
    float one = 1.f;
    asm("" : "+s"(one));
    const f32x2 v = {x, y};
    const f16x2 h = __builtin_convertvector(v, f16x2);
    const f32x2 rest = {fmaf(-static_cast<float>(h[0]), one, x), fmaf(-static_cast<float>(h[1]), one, y)};
    hi = __builtin_bit_cast(unsigned, h);
    lo = __builtin_bit_cast(unsigned, __builtin_convertvector(rest, f16x2));
}

}  // namespace tvara_amd

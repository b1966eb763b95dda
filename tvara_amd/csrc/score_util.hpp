// Device helpers of the scored attention kernels.
#pragma once

#include "common.hpp"

#include "device_util.hpp"
#include "q8.hpp"
#include "score.hpp"

namespace tvara_amd {

// element `column` of a cached K (kind 0) or V row
__device__ __forceinline__ float score_element(const ScoreArgs& a, int block, int kind, int slot, int column) {
    const char* base = a.pool + static_cast<size_t>(block) * a.lay.stride;
    const size_t sec = static_cast<size_t>(a.layer) * 2 + kind;
    if (a.lay.format == kF32)
        return reinterpret_cast<const float*>(base)[(sec * a.lay.tpb + slot) * a.lay.kv_width + column];
    const char* s = base + sec * a.lay.section;
    const int8_t q = reinterpret_cast<const int8_t*>(s)[q8_byte_offset(a.lay, slot, column)];
    return half_bits_to_float(*reinterpret_cast<const uint16_t*>(s + q8_scale_offset(a.lay, slot, column / 32))) *
           static_cast<float>(q);
}

// tanh, odd in x.  Up to 5/8 a polynomial in x^2 fitted at Chebyshev's nodes (9e-8 of
// the result, rounding and all), where the other form loses bits: above, 1 - 2 / (e^2x + 1).
__device__ __forceinline__ float small_tanh(float x) {
    const float y = x * x;
    float p = fmaf(-0.0061049391f, y, 0.0210036337f);
    p = fmaf(p, y, -0.0538524948f);
    p = fmaf(p, y, 0.1333278269f);
    p = fmaf(p, y, -0.3333332837f);
    return fmaf(x * y, p, x);
}
__device__ __forceinline__ float large_tanh(float x) {
    const float e = fast_exp2(__builtin_fabsf(x) * 2.8853900817779268f);
    return __builtin_copysignf(fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f), x);
}

constexpr float kSmallTanh = 0.625f;
__device__ __forceinline__ float any_tanh(float x) {
    return __builtin_fabsf(x) <= kSmallTanh ? small_tanh(x) : large_tanh(x);
}
// the same without branches by lane, for more registers
__device__ __forceinline__ float both_tanh(float x) {
    const float small = small_tanh(x), large = large_tanh(x);
    return __builtin_fabsf(x) <= kSmallTanh ? small : large;
}

}  // namespace tvara_amd

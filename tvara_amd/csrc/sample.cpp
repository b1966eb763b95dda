// Plans of sampling (sample.hpp): what the host checks and lays out.
#include "sample.hpp"

#include <algorithm>
#include <bit>
#include <cmath>
#include <limits>
#include <stdexcept>
#include <type_traits>

namespace tvara_amd {

void SamplePlan::build(size_t n, size_t v) {
    constexpr size_t kIntMax = static_cast<size_t>(std::numeric_limits<int32_t>::max());
    if (!n || !v) throw std::invalid_argument("empty sample plan");
    // (rows are a grid's second dimension)
    if (v > kIntMax / 2 || n > 65535 || n > (size_t(1) << 33) / v) throw std::invalid_argument("sample plan too large");
    TVARA_HIP(hipGetDevice(&device));
    rows = static_cast<int>(n);
    vocab = static_cast<int>(v);
    chunk = 256;
    while (v > static_cast<size_t>(chunk) * kSampleChunks) chunk *= 2;
    chunks = static_cast<int>((v + chunk - 1) / chunk);
    room = static_cast<int>(std::min<size_t>(v, kSampleList));
    // A row's mass is at most v times the largest weight, and stays below 2^64 units: 2^44 of
    // them to that weight up to 2^20 - 1 logits, half as many for each doubling from there.
    one = std::ldexp(1.0, std::min(44, 64 - static_cast<int>(std::bit_width(v))));
    carve(nullptr, nullptr);
    space.ensure(bytes);
    auto* f = static_cast<volatile int*>(flag.acquire(2 * sizeof(int)));
    f[0] = 0;
    f[1] = 0;
}

// the workspace's parts, into `a` where it is given; bytes: all of them
void SamplePlan::carve(char* base, SampleArgs* a) {
    bytes = 0;
    auto part = [&](auto*& p, size_t each) {
        if (a) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + bytes);
        bytes = (bytes + each * rows * sizeof(*p) + 255) / 256 * 256;
    };
    SampleArgs none{}, &to = a ? *a : none;
    part(to.group_mass, kSampleGroups);
    part(to.chunk_mass, chunks);
    part(to.chunk_max, chunks);
    part(to.list, room);
    part(to.rows_state, 1);
    if (vocab <= kSampleList) return;
    part(to.bin_mass, kSampleBins);
    part(to.bin_count, kSampleBins);
}

void SamplePlan::launch(size_t n, const float* logits, size_t stride, const float* uniforms, const float* temperature,
                        const int32_t* top_k, const float* top_p, const float* min_p, uint32_t* tokens, float* probability,
                        hipStream_t s) {
    if (n > static_cast<size_t>(rows)) throw std::invalid_argument("more rows than the sample plan has");
    if (!stride) stride = vocab;
    if (stride < static_cast<size_t>(vocab) || (n && stride > (size_t(1) << 59) / n)) throw std::invalid_argument("logit rows overlap");
    if (!n) return;
    int dev = 0;
    TVARA_HIP(hipGetDevice(&dev));
    if (dev != device) throw std::invalid_argument("the sample plan is on another device");
    SampleArgs a{};
    a.logits = logits;
    a.stride = stride;
    a.rows = static_cast<int>(n);
    a.vocab = vocab;
    a.chunk = chunk;
    a.chunks = chunks;
    a.one = one;
    a.uniforms = uniforms;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.tokens = tokens;
    a.probability = probability;
    a.room = room;
    carve(static_cast<char*>(space.ptr), &a);
    a.err = static_cast<int*>(flag.ptr);
    launch_sample(a, s);
    last = s;
}

void SamplePlan::check() {
    TVARA_HIP(hipStreamSynchronize(last));
    auto* f = static_cast<volatile int*>(flag.ptr);
    const bool logits = f[0], asked = f[1];
    f[0] = 0;
    f[1] = 0;
    if (asked) throw std::invalid_argument("invalid sampling parameters");
    if (logits) throw std::invalid_argument("invalid logits to sample from");
}

}  // namespace tvara_amd

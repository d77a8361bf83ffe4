// Device-side helpers of the 8-bit KV cache (kv8.hpp has its layout).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8.hpp"

namespace ribn_amd {

typedef _Float16 kv8_half2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv8_half8 __attribute__((ext_vector_type(8)));

// f16 as a cache takes it: round to nearest even, +-65504 at most, NaN as 0.
__device__ __forceinline__ _Float16 kv8_half(float v) {
    const float c = fminf(fmaxf(v, -65504.0f), 65504.0f);
    return (_Float16)(v == v ? c : 0.0f);
}

__device__ __forceinline__ float kv8_power(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

// A block's exponent from its largest magnitude (an f16 value, so normal in f32, or 0).
__device__ __forceinline__ int kv8_exponent(float a) {
    const int e = (int)(__builtin_bit_cast(uint32_t, a) >> 23) - 127 - 6;
    return e < -24 ? -24 : e;
}

__device__ __forceinline__ uint32_t kv8_code(float v, float inv) {
    return (uint32_t)(int)(fminf(fmaxf(__builtin_rintf(v * inv), -127.0f), 127.0f) + 128.0f);
}

// Two codes of a word as the whole numbers they are, in f16: the byte under
// 0x64 is 1024 + code + 128 (exact), one permute and one packed add for two.
template <int HI>
__device__ __forceinline__ kv8_half2 kv8_pair(uint32_t w) {
    const uint32_t h = __builtin_amdgcn_perm(0x64646464u, w, HI ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(kv8_half2, h) - kv8_half2{(_Float16)1152.0f, (_Float16)1152.0f};
}

// Eight codes (two words) as whole numbers.
__device__ __forceinline__ kv8_half8 kv8_whole(uint32_t w0, uint32_t w1) {
    const kv8_half2 a = kv8_pair<0>(w0), b = kv8_pair<1>(w0), c = kv8_pair<0>(w1), d = kv8_pair<1>(w1);
    return kv8_half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight codes as the values they stand for.
__device__ __forceinline__ kv8_half8 kv8_values(uint32_t w0, uint32_t w1, _Float16 scale) {
    const kv8_half2 s{scale, scale};
    const kv8_half2 a = kv8_pair<0>(w0) * s, b = kv8_pair<1>(w0) * s, c = kv8_pair<0>(w1) * s, d = kv8_pair<1>(w1) * s;
    return kv8_half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The parts of a (layer, KV head) region.
struct Kv8Head {
    uint8_t* codes;
    _Float16* tail_k;
    _Float16* tail_v;
    float2* scales;
    int32_t* end;
};

__device__ __forceinline__ Kv8Head kv8_head(const AttnMember& m, int layer, int kvh) {
    uint8_t* const base = reinterpret_cast<uint8_t*>(m.keys) + (size_t)layer * m.layer_elems + (size_t)kvh * kv8_head_bytes(m.capacity);
    Kv8Head h;
    h.codes = base;
    h.tail_k = reinterpret_cast<_Float16*>(base + kv8_tail_offset(m.capacity));
    h.tail_v = h.tail_k + kKv8TailElems;
    h.scales = reinterpret_cast<float2*>(base + kv8_scales_offset(m.capacity));
    h.end = reinterpret_cast<int32_t*>(base + kv8_end_offset(m.capacity));
    return h;
}

}  // namespace ribn_amd

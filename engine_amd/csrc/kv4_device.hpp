// Device-side helpers of the 4-bit KV cache (kv4.hpp has its layout).
#pragma once

#include "kv4.hpp"
#include "kv8_device.hpp"

namespace ribn_amd {

typedef uint32_t kv4_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ KvHead kv4_head(const AttnMember& m, int layer, int kvh) {
    uint8_t* const base = reinterpret_cast<uint8_t*>(m.keys) + (size_t)layer * m.layer_elems + (size_t)kvh * kv4_head_bytes(m.capacity);
    KvHead h;
    h.codes = base;
    h.tail_k = reinterpret_cast<_Float16*>(base + kv4_tail_offset(m.capacity));
    h.tail_v = h.tail_k + kKv8TailElems;
    h.scales = nullptr;
    h.end = reinterpret_cast<int32_t*>(base + kv4_end_offset(m.capacity));
    return h;
}

// Eight codes as the values they stand for, with a scale and a low each: a nibble under 0x64 is 1024 + code
// (exact), less 1024, then one fused multiply-add in f16.
__device__ __forceinline__ kv8_half8 kv4_values(uint32_t w, kv4_u4 scale, kv4_u4 low) {
    kv8_half8 x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const kv8_half2 c = __builtin_bit_cast(kv8_half2, ((w >> (4 * j)) & 0x000f000fu) | 0x64006400u) - kv8_half2{(_Float16)1024.0f, (_Float16)1024.0f};
        const uint32_t sw = scale[j], lw = low[j];
        const kv8_half2 v = __builtin_elementwise_fma(c, __builtin_bit_cast(kv8_half2, sw), __builtin_bit_cast(kv8_half2, lw));
        x[2 * j] = v[0];
        x[2 * j + 1] = v[1];
    }
    return x;
}

// A group's scale, and its reciprocal in f32.
struct Kv4Scale {
    _Float16 s;
    float inv;
    __device__ __forceinline__ Kv4Scale(_Float16 lo, _Float16 hi) {
        const float wide = ((float)hi - (float)lo) * (1.0f / 15.0f);
        s = __builtin_bit_cast(kv8_half2, __builtin_amdgcn_cvt_pkrtz(wide, 0.0f))[0];
        inv = s > (_Float16)0.0f ? 1.0f / (float)s : 0.0f;
    }
};

__device__ __forceinline__ uint32_t kv4_code(_Float16 x, _Float16 lo, float inv) {
    return (uint32_t)fminf(rintf(((float)x - (float)lo) * inv), 15.0f);
}

// Where element e of a word's eight lies.
__device__ __forceinline__ constexpr int kv4_shift(int e) { return 16 * (e & 1) + 4 * (e >> 1); }

// Smaller (larger) halves of two pairs, over a row of 16 lanes, or over four of them.
__device__ __forceinline__ kv8_half2 kv4_min(kv8_half2 a, kv8_half2 b) { return __builtin_elementwise_min(a, b); }
template <int CTRL>
__device__ __forceinline__ kv8_half2 kv4_min_step(kv8_half2 v) {
    return kv4_min(v, __builtin_bit_cast(kv8_half2, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ kv8_half2 kv4_quad_min(kv8_half2 v) { return kv4_min_step<0x4e>(kv4_min_step<0xb1>(v)); }
__device__ __forceinline__ kv8_half2 kv4_row_min(kv8_half2 v) { return kv4_min_step<0x140>(kv4_min_step<0x141>(kv4_quad_min(v))); }

}  // namespace ribn_amd

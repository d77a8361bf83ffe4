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

// Eight codes as the values they stand for, with a scale and a low each: a nibble under 0x64 is 1024 + code, one
// four bits up under 0x54 is 64 + code (exact), less that, then one fused multiply-add in f16. Thirteen instructions:
// the two patterns are kept in vector registers (hidden from the compiler, which would take an and and an or for each pair).
// HERE: formed where it is used, two registers less across a loop that has none left.
template <bool HERE = false> struct Kv4Patterns {
    uint32_t low = 0x64006400u, high = 0x54005400u;
    __device__ __forceinline__ Kv4Patterns() {
        if constexpr (HERE) asm volatile("" : "+v"(low), "+v"(high));
        else asm("" : "+v"(low), "+v"(high));
    }
};
using Kv4Bias = Kv4Patterns<>;

template <bool HERE>
__device__ __forceinline__ kv8_half8 kv4_values(uint32_t w, kv4_u4 scale, kv4_u4 low, const Kv4Patterns<HERE>& bias) {
    const uint32_t u = w >> 8;
    const uint32_t biased[4] = {(w & 0x000f000fu) | bias.low, (w & 0x00f000f0u) | bias.high, (u & 0x000f000fu) | bias.low, (u & 0x00f000f0u) | bias.high};
    kv8_half8 x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const _Float16 one = (j & 1) ? (_Float16)64.0f : (_Float16)1024.0f;
        const kv8_half2 c = __builtin_bit_cast(kv8_half2, biased[j]) - kv8_half2{one, one};
        const uint32_t sw = scale[j], lw = low[j];
        const kv8_half2 v = __builtin_elementwise_fma(c, __builtin_bit_cast(kv8_half2, sw), __builtin_bit_cast(kv8_half2, lw));
        x[2 * j] = v[0];
        x[2 * j + 1] = v[1];
    }
    return x;
}

// A group's scale, and its reciprocal in f32 (1 for a scale of 0: a group that narrow, under 15 * 2^-24, gets codes of 0 by it).
struct Kv4Scale {
    _Float16 s;
    float inv;
    __device__ __forceinline__ Kv4Scale(_Float16 lo, _Float16 hi) {
        const float wide = ((float)hi - (float)lo) * (1.0f / 15.0f);
        s = __builtin_bit_cast(kv8_half2, __builtin_amdgcn_cvt_pkrtz(wide, 0.0f))[0];
        inv = 1.0f / (s > (_Float16)0.0f ? (float)s : 1.0f);
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

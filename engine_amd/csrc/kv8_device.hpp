// Device-side helpers of the 8-bit KV cache (kv8.hpp has its layout).
#pragma once

#include <float.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kquant_device.hpp"
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

// Largest magnitudes of pairs, and of a pair.
__device__ __forceinline__ kv8_half2 kv8_top(kv8_half2 top, kv8_half2 x) {
    return __builtin_elementwise_max(top, __builtin_bit_cast(kv8_half2, __builtin_bit_cast(uint32_t, x) & 0x7fff7fffu));
}

// A scale's reciprocal 2^-e as two factors f16 holds (e is -24 .. 9).
struct Kv8Inverse {
    kv8_half2 a, b;
    __device__ __forceinline__ explicit Kv8Inverse(int e) {
        const int h = -e / 2;
        const _Float16 x = (_Float16)kv8_power(h), y = (_Float16)kv8_power(-e - h);
        a = kv8_half2{x, x};
        b = kv8_half2{y, y};
    }
};

// Four values to the word of their codes, in packed f16: the products with powers of two
// are exact (or far below half a code), and 1536 + x is rounded to a whole
// number, ties to even, whose low byte is that number's.
__device__ __forceinline__ uint32_t kv8_word(kv8_half2 x, kv8_half2 y, const Kv8Inverse& inv) {
    const kv8_half2 lim{(_Float16)127.0f, (_Float16)127.0f}, bias{(_Float16)1536.0f, (_Float16)1536.0f};
    x = __builtin_elementwise_min(__builtin_elementwise_max(x * inv.a * inv.b, -lim), lim) + bias;
    y = __builtin_elementwise_min(__builtin_elementwise_max(y * inv.a * inv.b, -lim), lim) + bias;
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x06040200u) ^ 0x80808080u;
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

// Reductions over a wave by row rotations and lane reads: no LDS round trips,
// which follow one another on the way from a launch's first load to its products.
template <int CTRL>
__device__ __forceinline__ double dpp_add64(double v) {
    const uint2 w = __builtin_bit_cast(uint2, v);
    const uint2 moved = make_uint2((uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, CTRL, 0xf, 0xf, false),
                                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, CTRL, 0xf, 0xf, false));
    return v + __builtin_bit_cast(double, moved);
}

// Sum over a row of 16 lanes, in all of them.
__device__ __forceinline__ double row_sum64(double v) {
    v = dpp_add64<0xb1>(v);   // quad_perm [1,0,3,2]
    v = dpp_add64<0x4e>(v);   // quad_perm [2,3,0,1]
    v = dpp_add64<0x141>(v);  // row_half_mirror
    return dpp_add64<0x140>(v);  // row_mirror
}

__device__ __forceinline__ double wave_sum64(double v) {
    const uint2 w = __builtin_bit_cast(uint2, row_sum64(v));
    double r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = __builtin_bit_cast(double, make_uint2((uint32_t)__builtin_amdgcn_readlane((int)w.x, 16 * i),
                                                     (uint32_t)__builtin_amdgcn_readlane((int)w.y, 16 * i)));
    }
    return (r[0] + r[1]) + (r[2] + r[3]);
}

__device__ __forceinline__ float wave_max(float v) {
    v = dpp_max_step<0xb1>(v);
    v = dpp_max_step<0x4e>(v);
    v = dpp_max_step<0x141>(v);
    v = dpp_max_step<0x140>(v);
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 16 * i));
    return fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
}

// Softmax numerators as the matrix-core kernels form them, 2^(x - m) of scores x in log2
// units, each as two f16 pieces. f16 ends at 2^-24: smaller parts of a numerator are rounded, and one
// below 2^-25 is lost, while the denominator's f32 sum has it whole. With the largest at 2^0, an early key
// far above 131,072 others took 3e-3 off the output. So the reference m is set
// kTopExponent below the largest score (N keys then lose at most N 2^-33 of it), and moves
// when a score passes it by kMaxExponent, the pieces being still in f16's range. The room between the
// two keeps moves rare: 1,999 tokens after 6,203 take 437 us with 15 (m at the top), 443 with 7, 448 with 3.
constexpr float kTopExponent = 8.0f;
constexpr float kMaxExponent = 15.0f;

// A query head is taken in two f16 pieces too, divided by 2^e, which leaves its largest magnitude `top`
// just below 2: whatever the norm's weights are, no piece overflows and small heads keep their
// bits. 2^e goes into the f32 scale of its scores (both products are exact).
__device__ __forceinline__ int query_exponent(float top) {
    return max(-100, min(100, (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127));
}

// Two values as f16, to nearest even (one instruction here). The pieces of a numerator are
// rounded so: cut off toward zero they leave lower pieces that are all positive, and what of those
// a large sum on the matrix cores cannot take (it rounds after every eight products) is lost to
// one side (1.5e-4 with the 131,072 keys above in one sum).
typedef float kv8_float2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ kv8_half2 kv8_halfs(float a, float b) { return __builtin_convertvector((kv8_float2{a, b}), kv8_half2); }

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

// One row's partials (kPartStride floats each: 128 sums, their maximum in log2
// units, their denominator) merged by a workgroup of 128 threads:
//   o = sum_s O_s 2^(m_s - M) / sum_s L_s 2^(m_s - M).
// 32 lanes hold a partial's sums (four each) and take the slots s, s + 4, ... of NC
// or fewer (`slots` in memory, the others are not read), all loaded at once; `live()`,
// called after the loads are out, says how many count. The four runs meet in LDS in
// order. A slot that does not count adds exact zeros, so the bits do not depend on NC. No slots: zeros.
template <int NC, class LIVE>
__device__ __forceinline__ void merge_row(const float* partials, int slots, LIVE live, float* out) {
    constexpr int kRun = NC / 4;
    __shared__ float4 so[4][32];
    __shared__ float2 sml[4];
    const int run = (int)threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const __amdgpu_buffer_rsrc_t pr = make_rsrc(partials, (uint32_t)(slots * kPartStride * 4));
    float4 o[kRun];
    float2 ml[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const uint32_t row = (uint32_t)((4 * i + run) * kPartStride) * 4u;
        o[i] = __builtin_bit_cast(float4, load_b128(pr, row + 16u * (uint32_t)lane));
        ml[i] = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(pr, (int)(row + kHeadDim * 4), 0, 0));
    }
    const int count = live();
    float mx = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const bool counts = 4 * i + run < count;
        ml[i] = counts ? ml[i] : make_float2(-FLT_MAX, 0.f);
        o[i] = counts ? o[i] : make_float4(0.f, 0.f, 0.f, 0.f);
        mx = fmaxf(mx, ml[i].x);
    }
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const float f = __builtin_amdgcn_exp2f(ml[i].x - mx);
        l = __builtin_fmaf(ml[i].y, f, l);
        acc.x = __builtin_fmaf(o[i].x, f, acc.x);
        acc.y = __builtin_fmaf(o[i].y, f, acc.y);
        acc.z = __builtin_fmaf(o[i].z, f, acc.z);
        acc.w = __builtin_fmaf(o[i].w, f, acc.w);
    }
    so[run][lane] = acc;
    if (lane == 0) sml[run] = make_float2(mx, l);
    __syncthreads();
    const int d = threadIdx.x;
    mx = fmaxf(fmaxf(sml[0].x, sml[1].x), fmaxf(sml[2].x, sml[3].x));
    l = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float f = __builtin_amdgcn_exp2f(sml[r].x - mx);
        l = __builtin_fmaf(sml[r].y, f, l);
        sum = __builtin_fmaf(reinterpret_cast<const float*>(so[r])[d], f, sum);
    }
    out[d] = count > 0 ? sum / l : 0.f;
}

}  // namespace ribn_amd

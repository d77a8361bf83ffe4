// Rotary positions of query and key rows (rope_neox, model_ops.rs:393-425, in the
// reference: half layout, unscaled, f32 angles).
//
// For the pair (a, b) with angle p = position * turns (64 bits, rope_device.hpp):
//   a' = a cos p - b sin p,  b' = a sin p + b cos p
// A thread takes one group of pairs of a token, forms their angles once and
// turns that group in every slices-th head of every tensor of the call. Bound by
// memory: each value is read and written once, in 16-byte pieces (a wave
// covers whole heads), kUnroll heads in flight; the angles, some 50
// instructions a pair, are spread over the heads a thread takes. Few tokens: the
// heads are spread over threads instead (slices), down to one each.
#include "rope.hpp"

#include <algorithm>

#include "rope_device.hpp"

namespace ribn_amd {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;

template <typename T, int E> struct Piece { T v[E]; };

// E elements at p, as one access where they make 16 bytes.
template <typename T, int E>
__device__ __forceinline__ Piece<T, E> load_piece(const T* p) {
    if constexpr (E * sizeof(T) == 16) {
        return __builtin_bit_cast(Piece<T, E>, *reinterpret_cast<const uint4*>(p));
    } else {
        Piece<T, E> r;
#pragma unroll
        for (int i = 0; i < E; ++i) r.v[i] = p[i];
        return r;
    }
}

template <typename T, int E>
__device__ __forceinline__ void store_piece(T* p, const Piece<T, E>& r) {
    if constexpr (E * sizeof(T) == 16) {
        *reinterpret_cast<uint4*>(p) = __builtin_bit_cast(uint4, r);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] = r.v[i];
    }
}

template <typename T>
__device__ __forceinline__ void turn(T& a, T& b, float c, float s) {
    const float x = (float)a, y = (float)b;
    a = (T)__builtin_fmaf(x, c, -(y * s));
    b = (T)__builtin_fmaf(x, s, y * c);
}

// E: elements a thread moves at a time. Half layout: E pairs, two pieces half
// the rotary part apart. Interleaved: E / 2 pairs, one piece. Dims past the rotary part: one piece, as it is.
template <typename T, int E, bool HALF>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
    constexpr int kPairs = HALF ? E : E / 2;
    const int pairs = a.rotary_dim / 2;
    const uint32_t turning = (uint32_t)(pairs / kPairs);
    const uint32_t groups = turning + (uint32_t)((a.head_dim - a.rotary_dim) / E);
    const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t group = id % groups;
    const uint32_t slice = (id / groups) % (uint32_t)a.slices;
    const size_t t = id / groups / (uint32_t)a.slices;
    if (t >= a.tokens) return;
    const bool turns = group < turning;
    const int dim = turns ? (int)group * E : a.rotary_dim + (int)(group - turning) * E;
    float c[kPairs], s[kPairs];
    if (turns) {
        const int position = a.positions[t];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const Rot64 r = table_rot(a.table, pairs, (int)group * kPairs + i, position);
            c[i] = (float)r.c;
            s[i] = (float)r.s;
        }
    }
    for (int n = 0; n < a.count; ++n) {
        const RopeRows& r = a.rows[n];
        const T* x = static_cast<const T*>(r.x) + t * r.x_token + dim;
        T* y = static_cast<T*>(r.y) + t * r.y_token + dim;
        // heads are dealt out over the tensors' heads in a row
        const int ahead = r.before % a.slices;
        const int first = ((int)slice >= ahead ? 0 : a.slices) + (int)slice - ahead;
        if (turns) {
            for (int h0 = first; h0 < r.heads; h0 += kUnroll * a.slices) {
                Piece<T, E> lo[kUnroll], hi[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int h = h0 + u * a.slices;
                    if (h < r.heads) {
                        lo[u] = load_piece<T, E>(x + (size_t)h * r.x_head);
                        if constexpr (HALF) hi[u] = load_piece<T, E>(x + (size_t)h * r.x_head + pairs);
                    }
                }
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int h = h0 + u * a.slices;
                    if (h < r.heads) {
#pragma unroll
                        for (int i = 0; i < kPairs; ++i) {
                            if constexpr (HALF) turn(lo[u].v[i], hi[u].v[i], c[i], s[i]);
                            else turn(lo[u].v[2 * i], lo[u].v[2 * i + 1], c[i], s[i]);
                        }
                        store_piece<T, E>(y + (size_t)h * r.y_head, lo[u]);
                        if constexpr (HALF) store_piece<T, E>(y + (size_t)h * r.y_head + pairs, hi[u]);
                    }
                }
            }
        } else if (x != y) {
            for (int h = first; h < r.heads; h += a.slices)
                store_piece<T, E>(y + (size_t)h * r.y_head, load_piece<T, E>(x + (size_t)h * r.x_head));
        }
    }
}

template <typename T, int E, bool HALF>
hipError_t launch(RopeArgs a, int cu_count, hipStream_t stream) {
    constexpr int kPairs = HALF ? E : E / 2;
    const size_t groups = (size_t)(a.rotary_dim / 2 / kPairs + (a.head_dim - a.rotary_dim) / E);
    int most = 1;
    for (int i = 0; i < a.count; ++i) most = std::max(most, a.rows[i].before + a.rows[i].heads);
    // as many threads as keep the CUs full (1,024 each), if the heads allow it
    const size_t wanted = (size_t)cu_count * 1024;
    a.slices = (int)std::max<size_t>(1, std::min<size_t>((size_t)most, wanted / std::max<size_t>(1, a.tokens * groups)));
    // tokens a launch's 32-bit thread ids cover
    const size_t span = ((size_t)1 << 31) / (groups * (size_t)a.slices);
    RopeArgs b = a;
    for (size_t t0 = 0; t0 < a.tokens; t0 += span) {
        b.tokens = std::min(span, a.tokens - t0);
        b.positions = a.positions + t0;
        for (int i = 0; i < a.count; ++i) {
            b.rows[i].x = static_cast<const T*>(a.rows[i].x) + t0 * a.rows[i].x_token;
            b.rows[i].y = static_cast<T*>(a.rows[i].y) + t0 * a.rows[i].y_token;
        }
        const size_t threads = b.tokens * groups * (size_t)a.slices;
        hipLaunchKernelGGL((rope_kernel<T, E, HALF>), dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, b);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// 16-byte pieces need every row's start, every stride and both parts of the head in whole pieces.
template <typename T>
hipError_t launch_type(const RopeArgs& a, bool half, int cu_count, hipStream_t stream) {
    constexpr int E = 16 / sizeof(T);
    bool wide = (half ? a.rotary_dim / 2 : a.rotary_dim) % E == 0 && (a.head_dim - a.rotary_dim) % E == 0;
    for (int i = 0; i < a.count; ++i) {
        const RopeRows& r = a.rows[i];
        wide = wide && ((reinterpret_cast<uintptr_t>(r.x) | reinterpret_cast<uintptr_t>(r.y)) & 15) == 0 &&
               (r.x_token | r.x_head | r.y_token | r.y_head) % E == 0;
    }
    if (half) return wide ? launch<T, E, true>(a, cu_count, stream) : launch<T, 1, true>(a, cu_count, stream);
    return wide ? launch<T, E, false>(a, cu_count, stream) : launch<T, 2, false>(a, cu_count, stream);
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, uint32_t dtype, uint32_t layout, int cu_count, hipStream_t stream) {
    if (a.tokens < 1 || a.count < 1 || a.count > kRopeMaxTensors || a.table == nullptr || a.positions == nullptr) return hipErrorInvalidValue;
    const bool half = layout == RIBN_AMD_ROPE_HALF;
    switch (dtype) {
    case RIBN_AMD_F32: return launch_type<float>(a, half, cu_count, stream);
    case RIBN_AMD_BF16: return launch_type<__bf16>(a, half, cu_count, stream);
    case RIBN_AMD_F16: return launch_type<_Float16>(a, half, cu_count, stream);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace ribn_amd

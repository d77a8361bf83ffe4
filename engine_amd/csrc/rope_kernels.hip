// Rotary positions of query and key rows (rope_neox, model_ops.rs:393-425, in the
// reference: half layout, unscaled, f32 angles).
//
// For the pair (a, b) with angle p = position * turns (64 bits, rope_device.hpp):
//   a' = a cos p - b sin p,  b' = a sin p + b cos p
// A workgroup takes a few tokens. Its threads form each of their angles once (some
// 50 instructions each), into LDS, while their first rows are on the way; then a
// thread turns one group of pairs in every slices-th head of every tensor of the
// call. Bound by memory: each value is read and written once, in 16-byte pieces (a
// wave covers whole heads), kUnroll heads in flight: 32,768 tokens of 40 f32 heads of 128
// (1.34 GB) take 230 us, 5.8 TB/s. One token takes 3 us, a launch and one load's way.
#include "rope.hpp"

#include <algorithm>

#include "rope_device.hpp"

namespace ribn_amd {

namespace {

constexpr int kThreads = 256;     // of a workgroup, or what one head takes: up to 1,023 single elements
constexpr int kMaxThreads = 1024;
static_assert(kRopeMaxDim <= kMaxThreads, "a head fits a workgroup");
// Heads a thread has in flight and takes where tokens are many: 32,768 tokens (above) with
// 1 / 3 / 4 / 8 heads 238 / 232 / 233 / 248 us, with workgroups of 512 239.
constexpr int kUnroll = 3;
constexpr int kHeads = kUnroll;
// Below this many threads a CU a token's heads are spread over more of them: 2,047 tokens of 32
// bf16 heads, half of each turning, with 512 / 1,024 / 2,048 threads 7.8 / 7.9 / 10.0 us.
constexpr int kThreadsPerCu = 1024;

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
__global__ __launch_bounds__(kMaxThreads) void rope_kernel(RopeArgs a) {
    constexpr int kPairs = HALF ? E : E / 2;
    extern __shared__ __attribute__((aligned(16))) float2 angles[];  // [tokens of the workgroup][pairs] cosine, sine
    const int pairs = a.rotary_dim / 2;
    const int turning = pairs / kPairs;
    const int groups = turning + (a.head_dim - a.rotary_dim) / E;
    const int group = (int)threadIdx.x % groups;
    const int inside = a.slices / (int)gridDim.y;  // slices of this workgroup
    const int slice = (int)blockIdx.y * inside + (int)threadIdx.x / groups % inside;
    const int local = (int)threadIdx.x / (groups * inside);
    const size_t t0 = (size_t)blockIdx.x * a.per_group;
    const size_t t = t0 + local;
    const bool mine = local < a.per_group && t < a.tokens;
    const bool turns = group < turning;
    const int dim = turns ? group * E : a.rotary_dim + (group - turning) * E;

    Piece<T, E> lo[kUnroll], hi[kUnroll];
    auto load = [&](const RopeRows& r, int h0) {
        const T* x = static_cast<const T*>(r.x) + t * r.x_token + dim;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = h0 + u * a.slices;
            if (h < r.heads) {
                lo[u] = load_piece<T, E>(x + (size_t)h * r.x_head);
                if constexpr (HALF) {
                    if (turns) hi[u] = load_piece<T, E>(x + (size_t)h * r.x_head + pairs);
                }
            }
        }
    };
    if (mine) load(a.rows[0], slice);
    const int here = (int)min((size_t)a.per_group, a.tokens - t0);
    for (int i = threadIdx.x; i < here * pairs; i += blockDim.x) {
        const int token = i / pairs, pair = i - token * pairs;
        const Rot64 r = table_rot(a.table, pairs, pair, a.positions[t0 + token]);
        angles[i] = make_float2((float)r.c, (float)r.s);
    }
    __syncthreads();
    if (!mine) return;
    float c[kPairs], s[kPairs];
    if (turns) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const float2 r = angles[local * pairs + group * kPairs + i];
            c[i] = r.x;
            s[i] = r.y;
        }
    }
    for (int n = 0; n < a.count; ++n) {
        const RopeRows& r = a.rows[n];
        T* y = static_cast<T*>(r.y) + t * r.y_token + dim;
        // heads are dealt out over the tensors' heads in a row
        const int ahead = r.before % a.slices;
        for (int h0 = (slice >= ahead ? 0 : a.slices) + slice - ahead; h0 < r.heads; h0 += kUnroll * a.slices) {
            if (n > 0 || h0 != slice) load(r, h0);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int h = h0 + u * a.slices;
                if (h < r.heads) {
                    T* to = y + (size_t)h * r.y_head;
                    if (turns) {
#pragma unroll
                        for (int i = 0; i < kPairs; ++i) {
                            if constexpr (HALF) turn(lo[u].v[i], hi[u].v[i], c[i], s[i]);
                            else turn(lo[u].v[2 * i], lo[u].v[2 * i + 1], c[i], s[i]);
                        }
                        if constexpr (HALF) store_piece<T, E>(to + pairs, hi[u]);
                    }
                    store_piece<T, E>(to, lo[u]);
                }
            }
        }
    }
}

template <typename T, int E, bool HALF>
hipError_t launch(RopeArgs a, int cu_count, hipStream_t stream) {
    constexpr int kPairs = HALF ? E : E / 2;
    const int groups = a.rotary_dim / 2 / kPairs + (a.head_dim - a.rotary_dim) / E;
    int heads = 0;
    for (int i = 0; i < a.count; ++i) heads = std::max(heads, a.rows[i].before + a.rows[i].heads);
    // Threads that share a token's heads: a head each where the tokens are few (then
    // over several workgroups, if it takes more than one), else kHeads each.
    const size_t wanted = (size_t)cu_count * kThreadsPerCu / (a.tokens * (size_t)groups) + 1;
    const int fit = std::max(1, kThreads / groups);  // slices a workgroup holds
    const int shared = std::min(fit, (heads + kHeads - 1) / kHeads);
    const int inside = wanted > (size_t)shared ? (int)std::min<size_t>(std::min<size_t>(wanted, (size_t)heads), (size_t)fit) : shared;
    const int parts = wanted > (size_t)inside ? (int)std::min<size_t>((wanted + inside - 1) / inside, (size_t)(heads + inside - 1) / inside) : 1;
    a.slices = inside * parts;
    a.per_group = std::max(1, kThreads / (groups * inside));
    const int threads = (a.per_group * groups * inside + 63) / 64 * 64;
    const size_t lds = (size_t)a.per_group * (a.rotary_dim / 2) * sizeof(float2);
    // a launch has fewer than 2^32 threads
    const size_t span = (((size_t)1 << 31) / ((size_t)threads * parts)) * (size_t)a.per_group;
    RopeArgs b = a;
    for (size_t t0 = 0; t0 < a.tokens; t0 += span) {
        b.tokens = std::min(span, a.tokens - t0);
        b.positions = a.positions + t0;
        for (int i = 0; i < a.count; ++i) {
            b.rows[i].x = static_cast<const T*>(a.rows[i].x) + t0 * a.rows[i].x_token;
            b.rows[i].y = static_cast<T*>(a.rows[i].y) + t0 * a.rows[i].y_token;
        }
        const size_t blocks = (b.tokens + a.per_group - 1) / a.per_group;
        hipLaunchKernelGGL((rope_kernel<T, E, HALF>), dim3((unsigned)blocks, (unsigned)parts), dim3((unsigned)threads), (unsigned)lds, stream, b);
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

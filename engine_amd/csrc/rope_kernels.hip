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

// The angles of a workgroup's tokens.
__device__ __forceinline__ void form_angles(const RopeArgs& a, size_t t0, float2* angles) {
    const int pairs = a.rotary_dim / 2;
    const int here = (int)min((size_t)a.per_group, a.tokens - t0);
    for (int i = threadIdx.x; i < here * pairs; i += blockDim.x) {
        const int token = i / pairs, pair = i - token * pairs;
        const Rot64 r = table_rot(a.table, pairs, pair, a.positions[t0 + token]);
        angles[i] = make_float2((float)r.c, (float)r.s);
    }
}

// E: elements a thread moves at a time. Half layout: E pairs, two pieces half
// the rotary part apart; dims past the rotary part: one piece, as it is. Interleaved: one
// piece, the pairs of it that turn.
template <int E, bool HALF>
__host__ __device__ inline int rope_groups(const RopeArgs& a) {
    return HALF ? (a.rotary_dim / 2 + a.head_dim - a.rotary_dim) / E : a.head_dim / E;
}

template <typename T, int E, bool HALF>
__global__ __launch_bounds__(kMaxThreads) void rope_kernel(RopeArgs a) {
    constexpr int kPairs = HALF ? E : E / 2;
    extern __shared__ __attribute__((aligned(16))) float2 angles[];  // [tokens of the workgroup][pairs] cosine, sine
    const int pairs = a.rotary_dim / 2;
    const int turning = (pairs + kPairs - 1) / kPairs;
    const int groups = rope_groups<E, HALF>(a);
    const int group = (int)threadIdx.x % groups;
    const int inside = a.slices / (int)gridDim.y;  // slices of this workgroup
    const int slice = (int)blockIdx.y * inside + (int)threadIdx.x / groups % inside;
    const int local = (int)threadIdx.x / (groups * inside);
    const size_t t0 = (size_t)blockIdx.x * a.per_group;
    const size_t t = t0 + local;
    const bool mine = local < a.per_group && t < a.tokens;
    const bool turns = group < turning;
    const int dim = HALF && !turns ? a.rotary_dim + (group - turning) * E : group * E;

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
    form_angles(a, t0, angles);
    __syncthreads();
    if (!mine) return;
    const int live = HALF ? kPairs : min(kPairs, pairs - group * kPairs);  // pairs of the piece that turn
    float c[kPairs], s[kPairs];
    if (turns) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            if (i < live) {
                const float2 r = angles[local * pairs + group * kPairs + i];
                c[i] = r.x;
                s[i] = r.y;
            }
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
                            else if (i < live) turn(lo[u].v[2 * i], lo[u].v[2 * i + 1], c[i], s[i]);
                        }
                        if constexpr (HALF) store_piece<T, E>(to + pairs, hi[u]);
                    }
                    store_piece<T, E>(to, lo[u]);
                }
            }
        }
    }
}

// The half layout where the rotary part's halves do not fall into whole pieces: rows go
// through LDS, so that memory is still read and written in whole 16-byte pieces of the head, and a
// thread finds the other element of each of its pairs there. (All of a head's threads are of one workgroup, and its
// rows are read before any is written: in place is safe.) 16,759 tokens of 8 f16 heads of
// 96, 42 dims turning, take 16.5 us, by single elements 33.9; 25,896 of 4 f32 heads of 128, 14 turning,
// 23.7 and 54.6; 4,096 of 40 bf16 heads of 128, 126 turning, 22.3 and 23.0.
template <typename T, int E>
__global__ __launch_bounds__(kThreads) void rope_across_kernel(RopeArgs a, int angle_bytes) {
    extern __shared__ __attribute__((aligned(16))) char room[];
    float2* const angles = reinterpret_cast<float2*>(room);
    const int half = a.rotary_dim / 2;
    const int groups = a.head_dim / E;
    const int slot = (int)threadIdx.x / groups;  // (token, slice) of the workgroup
    const int inside = a.slices / (int)gridDim.y;
    const int slots = a.per_group * inside;
    const int slice = (int)blockIdx.y * inside + slot % inside;
    const int local = slot / inside;
    const size_t t0 = (size_t)blockIdx.x * a.per_group;
    const size_t t = t0 + local;
    const bool mine = slot < slots && t < a.tokens;
    const int dim = (int)threadIdx.x % groups * E;
    const bool turns = dim < a.rotary_dim;
    T* const held = reinterpret_cast<T*>(room + angle_bytes) + (size_t)min(slot, slots - 1) * a.head_dim;  // [kUnroll][slots][head_dim]
    const int apart = slots * a.head_dim;

    Piece<T, E> x[kUnroll];
    auto load = [&](const RopeRows& r, int h0) {
        const T* from = static_cast<const T*>(r.x) + t * r.x_token + dim;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = h0 + u * a.slices;
            if (h < r.heads) x[u] = load_piece<T, E>(from + (size_t)h * r.x_head);
        }
    };
    if (mine) load(a.rows[0], slice);
    form_angles(a, t0, angles);
    __syncthreads();
    float c[E], s[E];
    int other[E];  // the pair's other element
    if (mine && turns) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int d = dim + i;
            other[i] = d < half ? d + half : d < a.rotary_dim ? d - half : d;
            const float2 r = angles[local * half + min(min(d, other[i]), half - 1)];
            c[i] = r.x;
            s[i] = r.y;
        }
    }
    for (int n = 0; n < a.count; ++n) {
        const RopeRows& r = a.rows[n];
        T* const y = static_cast<T*>(r.y) + t * r.y_token + dim;
        const int ahead = r.before % a.slices;
        const int first = (slice >= ahead ? 0 : a.slices) + slice - ahead;
        // (as many rounds for every slice, so that all meet at the barriers)
        for (int h0 = first; h0 - first < r.heads; h0 += kUnroll * a.slices) {
            if (mine) {
                if (n > 0 || h0 != slice) load(r, h0);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
                    if (h0 + u * a.slices < r.heads) store_piece<T, E>(held + u * apart + dim, x[u]);
            }
            __syncthreads();
            if (mine) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int h = h0 + u * a.slices;
                    if (h < r.heads) {
                        if (turns) {
#pragma unroll
                            for (int i = 0; i < E; ++i) {
                                const int d = dim + i;
                                const float own = (float)x[u].v[i], b = (float)held[u * apart + other[i]];
                                const float lower = __builtin_fmaf(own, c[i], -(b * s[i])), upper = __builtin_fmaf(b, s[i], own * c[i]);
                                if (d < a.rotary_dim) x[u].v[i] = (T)(d < half ? lower : upper);
                            }
                        }
                        store_piece<T, E>(y + (size_t)h * r.y_head, x[u]);
                    }
                }
            }
            __syncthreads();
        }
    }
}

// How a launch's threads are dealt out: `groups` of them a head.
struct RopeGrid {
    int threads;
    int parts;  // workgroups that share a token's heads
};

RopeGrid deal(RopeArgs& a, int groups, int cu_count) {
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
    return {(a.per_group * groups * inside + 63) / 64 * 64, parts};
}

// `go` launches the rows that one launch (fewer than 2^32 threads) takes, in turn.
template <typename T, class GO>
hipError_t launch_spans(const RopeArgs& a, const RopeGrid& g, GO go) {
    const size_t span = (((size_t)1 << 31) / ((size_t)g.threads * g.parts)) * (size_t)a.per_group;
    RopeArgs b = a;
    for (size_t t0 = 0; t0 < a.tokens; t0 += span) {
        b.tokens = std::min(span, a.tokens - t0);
        b.positions = a.positions + t0;
        for (int i = 0; i < a.count; ++i) {
            b.rows[i].x = static_cast<const T*>(a.rows[i].x) + t0 * a.rows[i].x_token;
            b.rows[i].y = static_cast<T*>(a.rows[i].y) + t0 * a.rows[i].y_token;
        }
        go(b, dim3((unsigned)((b.tokens + a.per_group - 1) / a.per_group), (unsigned)g.parts));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <typename T, int E, bool HALF>
hipError_t launch(RopeArgs a, int cu_count, hipStream_t stream) {
    const RopeGrid g = deal(a, rope_groups<E, HALF>(a), cu_count);
    const size_t lds = (size_t)a.per_group * (a.rotary_dim / 2) * sizeof(float2);
    return launch_spans<T>(a, g, [&](const RopeArgs& b, dim3 grid) {
        hipLaunchKernelGGL((rope_kernel<T, E, HALF>), grid, dim3((unsigned)g.threads), (unsigned)lds, stream, b);
    });
}

template <typename T, int E>
hipError_t launch_across(RopeArgs a, int cu_count, hipStream_t stream) {
    static_assert(kRopeMaxDim / E <= kThreads, "a head fits a workgroup");
    const RopeGrid g = deal(a, a.head_dim / E, cu_count);
    const int angle_bytes = (int)(((size_t)a.per_group * (a.rotary_dim / 2) * sizeof(float2) + 15) / 16 * 16);
    const size_t slots = (size_t)a.per_group * (a.slices / g.parts);
    const size_t lds = (size_t)angle_bytes + kUnroll * slots * a.head_dim * sizeof(T);
    return launch_spans<T>(a, g, [&](const RopeArgs& b, dim3 grid) {
        hipLaunchKernelGGL((rope_across_kernel<T, E>), grid, dim3((unsigned)g.threads), (unsigned)lds, stream, b, angle_bytes);
    });
}

// 16-byte pieces need every row's start, every stride and the head in whole pieces (else single
// elements, or pairs); in the half layout also both halves of the rotary part, or the rows go through LDS.
template <typename T>
hipError_t launch_type(const RopeArgs& a, bool half, int cu_count, hipStream_t stream) {
    constexpr int E = 16 / sizeof(T);
    bool wide = a.head_dim % E == 0;
    for (int i = 0; i < a.count; ++i) {
        const RopeRows& r = a.rows[i];
        wide = wide && ((reinterpret_cast<uintptr_t>(r.x) | reinterpret_cast<uintptr_t>(r.y)) & 15) == 0 &&
               (r.x_token | r.x_head | r.y_token | r.y_head) % E == 0;
    }
    if (!half) return wide ? launch<T, E, false>(a, cu_count, stream) : launch<T, 2, false>(a, cu_count, stream);
    if (!wide) return launch<T, 1, true>(a, cu_count, stream);
    return a.rotary_dim / 2 % E == 0 ? launch<T, E, true>(a, cu_count, stream) : launch_across<T, E>(a, cu_count, stream);
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

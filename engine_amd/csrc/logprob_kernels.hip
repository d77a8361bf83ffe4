// Log probabilities of given tokens, the entropy of their distributions and the likeliest
// alternatives, from rows of logits, in one pass over them (gfx950).
//
// With M a row's largest logit, t = (x - M) log2 e, R = sum of 2^t over all tokens but one
// at M, and E = sum t 2^t:
//   log p(x) = (x - M) - log1p(R),   entropy = log1p(R) - ln 2 E / (1 + R).
// The token at M is left out of R, and log1p taken of the rest, since a certain model's log
// probability is R itself, which a sum with the 1 in it rounds away. A lane's sums are f32 (some hundred
// terms of at most 1), those over lanes, waves and workgroups f64.
//
// NaN and -inf have probability 0: t is raised to -160, where 2^t is 0 and so is t 2^t, and a maximum takes
// the operand that is a number. A row of nothing else has no M (-inf): its log probabilities are -inf and
// its entropy 0. Of +inf the limit is taken: the tokens at it share the probability.
//
// A workgroup takes a row, or one of `splits` parts of it; its four waves take 1,024 logits in turn, 16 a
// lane in 16-byte loads (those before the row's first and after its last such piece are the first
// workgroup's, one a lane), the next ones under way meanwhile. Each wave has its own M and its own alternatives, so
// the loop has no barrier. An iteration whose logits all lie below both M and the wave's last alternative
// (most of them, after the first ones) costs about ten VALU slots a logit. Others move M, or
// hand their candidates to the wave's Best.
#include "logprob.hpp"

#include <algorithm>

#include "kv8_device.hpp"

namespace ribn_amd {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kValues = 16;                    // logits a lane and iteration
constexpr int kIteration = kThreads * kValues;
constexpr int kBest = 128;                     // candidates a wave holds
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLeast = -160.0f;              // 2^kLeast is 0 in f32

// Orders as (logit, lower token first): larger keys are better, 0 is none. x is a number, and no negative zero.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
    return ((uint64_t)order_of(x == x ? x : -INFINITY) << 32) | (uint32_t)~token;
}
__device__ __forceinline__ uint32_t token_of(uint64_t key) { return ~(uint32_t)key; }

// LDS written by some lanes of a wave and read by others of it: in order as issued.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The best `top` of n <= kBest distinct keys, in order, by counting: a key's place is the number of larger ones.
__device__ __forceinline__ void sort_best(uint64_t* keys, int n, int top) {
    const int lane = threadIdx.x & 63;
    wave_sync();
    const uint64_t a = lane < n ? keys[lane] : 0, b = lane + 64 < n ? keys[lane + 64] : 0;
    int ra = 0, rb = 0;
    for (int i = 0; i < n; ++i) {
        const uint64_t k = keys[i];
        ra += k > a;
        rb += k > b;
    }
    wave_sync();
    if (lane < n && ra < top) keys[ra] = a;
    if (lane + 64 < n && rb < top) keys[rb] = b;
    wave_sync();
}

// A wave's best `top` keys so far: candidates are appended, and sorted out when more than 64 are there.
struct Best {
    uint64_t* keys;      // LDS [kBest]
    int top;
    int count = 0;
    uint64_t least = 0;  // keys up to this one are none of the best

    __device__ __forceinline__ Best(uint64_t* room, int n) : keys(room), top(n) {}
    __device__ __forceinline__ float least_logit() const { return top == 0 ? INFINITY : least == 0 ? -INFINITY : logit_of(least); }
    __device__ __forceinline__ void sort() {
        sort_best(keys, count, top);
        count = min(count, top);
        if (count == top && top > 0) least = keys[top - 1];
    }
    // One candidate a lane (0: none).
    __device__ __forceinline__ void add(uint64_t key) {
        const bool has = key > least;
        const uint64_t who = __ballot(has);
        if (who == 0) return;
        if (has) keys[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = key;
        count += __popcll(who);
        if (count > kBest - 64) sort();
    }
    // From each lane's best key: what the top-th of them bounds from below.
    __device__ __forceinline__ void bound(uint32_t order) {
        uint32_t v = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t up = v | (1u << bit);
            if (__popcll(__ballot(order >= up)) >= top) v = up;
        }
        // (the order before v's is a logit's while v is not that of -inf, below which nothing is)
        if (v > order_of(-INFINITY)) least = ((uint64_t)v << 32) - 1;
    }
};

// A part's sums: M, R without the token at M, E in log2 units.
struct Sums {
    float m;
    double r, e;
};

// Parts i of `count` lanes (the others hold m = -inf, 0, 0), merged over a wave: every part's own token
// at its m counts but one at the largest.
__device__ __forceinline__ Sums merge_sums(Sums s) {
    const float m = wave_max(s.m);
    if (m == -INFINITY) return Sums{m, 0.0, 0.0};
    const uint64_t at = __ballot(s.m == m);
    const bool left_out = (threadIdx.x & 63) == (unsigned)(__ffsll((long long)at) - 1);
    double r = 0.0, e = 0.0;
    if (s.m != -INFINITY) {
        const double d = s.m == m ? 0.0 : fmax(((double)s.m - (double)m) * 1.4426950408889634074, -1100.0);
        const double f = exp2(d);
        r = f * (s.r + (left_out ? 0.0 : 1.0));
        e = f * (s.e + d * (s.r + 1.0));
    }
    return Sums{m, wave_sum64(r), wave_sum64(e)};
}

template <int DT> __device__ __forceinline__ float load_logit(const void* p, size_t i) {
    if constexpr (DT == kLogitF32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == kLogitF16) return (float)static_cast<const _Float16*>(p)[i];
    else return __builtin_bit_cast(float, (uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}

// A row's results by a wave, from its sums and its best keys in order.
template <int DT>
__device__ __forceinline__ void finish(const LogprobArgs& a, size_t row, const Sums& s, const uint64_t* best) {
    const int lane = threadIdx.x & 63;
    const double rest = log1p(s.r);
    auto logprob = [&](float x) {
        if (!(x > -INFINITY)) return -INFINITY;  // (or no number)
        return (float)((x == s.m ? 0.0 : (double)x - (double)s.m) - rest);
    };
    if (lane == 0) {
        if (a.logprobs != nullptr) {
            const size_t t = a.targets[row];
            a.logprobs[row] = t < a.length ? logprob(load_logit<DT>(a.logits, row * a.stride + t)) : -INFINITY;
        }
        if (a.entropy != nullptr) a.entropy[row] = s.m == -INFINITY ? 0.f : (float)fmax(rest - 0.69314718055994530942 * s.e / (1.0 + s.r), 0.0);
    }
    if (lane < a.top) {
        const uint64_t key = best[lane];
        a.top_tokens[row * a.top + lane] = token_of(key);
        a.top_logprobs[row * a.top + lane] = logprob(logit_of(key));
    }
}

// What a wave has seen: a lane's sums relative to the wave's m.
struct Wave {
    float m = -INFINITY, l = 0.f, e = 0.f;

    // 16 logits a lane (-inf: none); key(i): the i-th's key, 0: none.
    template <class KEY>
    __device__ __forceinline__ void take(float (&x)[kValues], Best& best, KEY key) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) x[i] += 0.0f;  // one zero, and no signaling NaN
        float top = x[0];
#pragma unroll
        for (int i = 1; i < kValues; ++i) top = fmaxf(top, x[i]);
        top = fmaxf(top, -INFINITY);  // (a number, if all are none)
        if (__any(top > m || top >= best.least_logit())) {
            if (best.top > 0) {
                if (best.count < best.top) best.bound(order_of(top));
                const float least = best.least_logit();
                uint32_t slots = 0;  // with a candidate in some lane
#pragma unroll
                for (int i = 0; i < kValues; ++i) slots |= __ballot(!(x[i] < least)) != 0 ? 1u << i : 0u;
                while (slots != 0) {
                    const int i = __ffs(slots) - 1;
                    slots &= slots - 1;
                    float v = x[0];
#pragma unroll
                    for (int j = 1; j < kValues; ++j) v = i == j ? x[j] : v;
                    best.add(key(v, i));
                }
            }
            const float most = wave_max(top);
            if (most > m) {
                if (m > -INFINITY) {
                    if ((threadIdx.x & 63) == 0) l += 1.0f;
                    const float d = fmaxf((m - most) * kLog2e, kLeast), f = __builtin_amdgcn_exp2f(d);
                    e = f * __builtin_fmaf(d, l, e);
                    l *= f;
                }
                m = most;
                bool found = false;  // one of those at m is left out
#pragma unroll
                for (int i = 0; i < kValues; ++i) {
                    const uint64_t at = __ballot(x[i] == m);
                    if (!found && at != 0) {
                        if ((threadIdx.x & 63) == (unsigned)(__ffsll((long long)at) - 1)) x[i] = -INFINITY;
                        found = true;
                    }
                }
            }
        }
        if (m == -INFINITY) return;
        if (__builtin_expect(m == INFINITY, 0)) {
#pragma unroll
            for (int i = 0; i < kValues; ++i) l += x[i] == m ? 1.0f : 0.0f;
            return;
        }
        float l16 = 0.f, e16 = 0.f;  // (an iteration's first: a lane's rounding errors are those of 16 + 40 terms, not of 600)
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            const float t = fmaxf((x[i] - m) * kLog2e, kLeast);
            const float p = __builtin_amdgcn_exp2f(t);
            l16 += p;
            e16 = __builtin_fmaf(t, p, e16);
        }
        l += l16;
        e += e16;
    }
};

// Grid (row, split).
template <int DT>
__global__ __launch_bounds__(kThreads) void logprob_kernel(LogprobArgs a) {
    constexpr int kSize = DT == kLogitF32 ? 4 : 2;
    constexpr int kPer = 16 / kSize;            // logits a piece
    constexpr int kPieces = kValues / kPer;     // pieces a lane and iteration
    __shared__ uint64_t keys[kWaves][kBest];
    __shared__ float part_m[kWaves];
    __shared__ double part_r[kWaves], part_e[kWaves];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const size_t row = blockIdx.x;
    const int split = blockIdx.y;
    const char* const base = static_cast<const char*>(a.logits) + row * a.stride * kSize;
    // the row's pieces: 16-byte aligned and whole; the first `head` logits and those after the last piece are single
    const size_t head = std::min<size_t>(a.length, ((16 - ((uintptr_t)base & 15)) & 15) / kSize);
    const size_t pieces = (a.length - head) / kPer;
    const uint4* const body = reinterpret_cast<const uint4*>(base + head * kSize);
    const size_t first = pieces * (size_t)split / (size_t)a.splits, last = pieces * ((size_t)split + 1) / (size_t)a.splits;

    Best best(keys[wave], a.top);
    Wave w;
    uint4 raw[kPieces];
    auto load = [&](size_t at) {
#pragma unroll
        for (int u = 0; u < kPieces; ++u)
            if (at + 64u * u + lane < last) raw[u] = body[at + 64u * u + lane];
    };
    size_t at = first + (size_t)wave * 64 * kPieces;
    load(at);
    if (split == 0 && wave == 0) {  // the single ones
        const size_t end = head + pieces * kPer, singles = head + (a.length - end);
        float x[kValues];
#pragma unroll
        for (int i = 0; i < kValues; ++i) x[i] = -INFINITY;
        const size_t token = (size_t)lane < head ? (size_t)lane : end + ((size_t)lane - head);
        if ((size_t)lane < singles) x[0] = load_logit<DT>(base, token);
        if (singles > 0) w.take(x, best, [&](float v, int i) { return i == 0 && (size_t)lane < singles ? key_of(v, (uint32_t)token) : 0; });
    }
    for (; at < last; at += (size_t)kThreads * kPieces) {
        float x[kValues];
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const bool live = at + 64u * u + lane < last;
            const uint32_t words[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                float v;
                if constexpr (DT == kLogitF32) v = __builtin_bit_cast(float, words[j]);
                else if constexpr (DT == kLogitF16) v = half_bits_to_float((words[j >> 1] >> (16 * (j & 1))) & 0xffffu);
                else v = __builtin_bit_cast(float, (j & 1) ? words[j >> 1] & 0xffff0000u : words[j >> 1] << 16);
                x[kPer * u + j] = live ? v : -INFINITY;
            }
        }
        const size_t now = at;
        load(at + (size_t)kThreads * kPieces);
        w.take(x, best, [&](float v, int i) {
            const size_t piece = now + 64u * (unsigned)(i / kPer) + lane;
            return piece < last ? key_of(v, (uint32_t)(head + piece * kPer + (unsigned)(i % kPer))) : 0;
        });
    }
    best.sort();
    if (lane == 0) part_m[wave] = w.m;
    const double r = wave_sum64((double)w.l), e = wave_sum64((double)w.e);
    if (lane == 0) {
        part_r[wave] = r;
        part_e[wave] = e;
    }
    // the waves' lists one after another
    __shared__ int counts[kWaves];
    if (lane == 0) counts[wave] = best.count;
    __syncthreads();
    if (wave != 0) return;
    Sums s{-INFINITY, 0.0, 0.0};
    if (lane < kWaves) s = Sums{part_m[lane], part_r[lane], part_e[lane]};
    s = merge_sums(s);
    int n = best.count;
    for (int i = 1; i < kWaves; ++i) {
        if (lane < counts[i]) keys[0][n + lane] = keys[i][lane];
        n += counts[i];
    }
    sort_best(keys[0], n, a.top);
    if (a.splits == 1) {
        finish<DT>(a, row, s, keys[0]);
        return;
    }
    uint64_t* part = a.partials + (row * (size_t)a.splits + (size_t)split) * (size_t)(3 + a.top);
    if (lane == 0) {
        part[0] = __builtin_bit_cast(uint32_t, s.m);
        part[1] = __builtin_bit_cast(uint64_t, s.r);
        part[2] = __builtin_bit_cast(uint64_t, s.e);
    }
    if (lane < a.top) part[3 + lane] = lane < n ? keys[0][lane] : 0;
}

// A row's parts, one a lane.
template <int DT>
__global__ __launch_bounds__(64) void logprob_merge_kernel(LogprobArgs a) {
    __shared__ uint64_t keys[kBest];
    const int lane = threadIdx.x;
    const size_t row = blockIdx.x;
    const bool live = lane < a.splits;
    const uint64_t* part = a.partials + (row * (size_t)a.splits + (size_t)lane) * (size_t)(3 + a.top);
    Sums s{-INFINITY, 0.0, 0.0};
    if (live) s = Sums{__builtin_bit_cast(float, (uint32_t)part[0]), __builtin_bit_cast(double, part[1]), __builtin_bit_cast(double, part[2])};
    Best best(keys, a.top);
    constexpr int kAhead = 4;
    for (int j = 0; j < a.top; j += kAhead) {
        uint64_t k[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) k[i] = live && j + i < a.top ? part[3 + j + i] : 0;
        if (j == 0) best.bound((uint32_t)(k[0] >> 32));
        if (!__any(k[0] > best.least)) break;  // (lists are in order)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) best.add(k[i]);
    }
    best.sort();
    finish<DT>(a, row, merge_sums(s), keys);
}

template <int DT>
hipError_t launch(const LogprobArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(logprob_kernel<DT>, dim3((unsigned)a.rows, (unsigned)a.splits), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL(logprob_merge_kernel<DT>, dim3((unsigned)a.rows), dim3(64), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_logprobs(const LogprobArgs& args, int dtype, int cu_count, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    if (args.rows == 0 || args.rows > 0x7fffffffu || args.length == 0 || args.top < 0 || args.top > kLogprobMaxTop || args.top > (long long)args.length) return hipErrorInvalidValue;
    LogprobArgs a = args;
    // parts: until four workgroups a CU are there, of an iteration at least
    const size_t most = std::min<size_t>({kLogprobMaxSplits, (a.length + kIteration - 1) / kIteration,
                                          scratch_bytes / (a.rows * (size_t)(3 + a.top) * sizeof(uint64_t))});
    a.splits = (int)std::max<size_t>(1, std::min<size_t>(most, 4 * (size_t)cu_count / a.rows));
    a.partials = static_cast<uint64_t*>(scratch);
    switch (dtype) {
    case kLogitF32: return launch<kLogitF32>(a, stream);
    case kLogitBf16: return launch<kLogitBf16>(a, stream);
    case kLogitF16: return launch<kLogitF16>(a, stream);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace ribn_amd

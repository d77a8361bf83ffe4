// Log probabilities of given tokens, the entropy of their distributions and the likeliest
// alternatives, from rows of logits, in one pass over them (gfx950).
//
// With c = log2 e (as f32), M a row's largest logit and M2 = f32(M c), t = x c - M2 by one multiply-add, and over all
// tokens but one at M: R = sum 2^t, E = sum t 2^t. With w = 2^(M c - M2) (nearly 1: what M2 was rounded by), R and E
// are brought to M itself at the end, R' = R / w and E' likewise, and
//   log p(x) = (x - M) - log1p(R'),   entropy = log1p(R') - ln 2 E' / (1 + R').
// The token at M is left out of R, and log1p taken of the rest, since a certain model's log
// probability is R itself, which a sum with the 1 in it rounds away. A lane's sums are f32, 16 terms
// first; those over lanes, waves and workgroups f64. A term is off by t's rounding, up to 6e-8 |x - M| of it, either way; what c is
// short of log2 e would add 1.3e-8 |x - M| to each, always up, and is taken back at the end (finish).
//
// NaN and -inf have probability 0: where an iteration's E is no number it is formed again with t raised to -160, where
// 2^t is 0 and so is t 2^t (and a maximum takes the operand that is a number). A row of nothing else has no M (-inf):
// its log probabilities are -inf and its entropy 0. Of +inf the limit is taken: the tokens at it share the probability.
// An M past 65,536 either way, whose M2 would be off by much of a power of two, takes t = (x - M) c, two roundings (Wave::wide).
//
// A workgroup takes a row, or one of `splits` parts of it; its four waves take 1,024 logits in turn, 16 a
// lane in 16-byte loads (those before the row's first and after its last such piece are the first
// workgroup's, one a lane), the next ones under way meanwhile. Each wave has its own M and its own alternatives, so
// the loop has no barrier. An iteration whose logits all lie below both M and what the row's alternatives are known to
// reach (most of them, after the first ones) costs eight and a half VALU slots a logit, four of which are the exponential. Others move M, or
// hand their candidates to the wave's Best.
//
// What a row's alternatives reach: each wave publishes a logit that a fourth of `top` of its own are no less than, of
// its first iteration from the lanes' largest ones, later from its sorted list. All four are no less than the least of these.
// (When a wave sees what the others publish is a matter of time, and decides which logits it looks at as candidates, never a result: the
// sums take either way by the wave's own M.)
//
// Memory bounds many rows: 2,047 of 151,936 f32 logits (1.24 GB) with one alternative 217 us, 5.7 TB/s; bf16 without
// alternatives 119 (5.2 TB/s), with 1, 5, 20 of them 138, 146, 164: at 37 iterations a wave, nearly half hold one
// of the row's best so far. Of few rows, launches and round trips: one row of 151,936 with 5 10.5 us (7 and 3.5
// on the card), 33 of 32,001 bf16 with 20 12.3 (9 and 4). A wave of one iteration takes 12,200 cycles for 20
// alternatives: 1,100 until its logits are there, 1,200 what they reach, 1,100 for the others' and again the logits, 2,000 its
// candidates, 2,400 M and the sums, 900 sorting eight candidates, 900 for the others', 1,200 the waves' lists into one, 1,200 the sums' merge.
// (18,600, and 15.7 us of the 12.3, with each wave bounding its own 20, candidates taken register by register, keys compared one by
// one and twice, and the token at M found by branches.)
#include "logprob.hpp"

#include <algorithm>

#include "kv8_device.hpp"

namespace ribn_amd {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kValues = 16;                    // logits a lane and iteration
constexpr int kIteration = kThreads * kValues;
typedef float Logits __attribute__((ext_vector_type(kValues)));  // (a vector: of an array, a choice by lane is a load from scratch)
constexpr int kBest = 128;                     // candidates a wave holds
constexpr float kLog2e = 1.44269504088896341f;
constexpr double kLn2 = 0.69314718055994530942;
constexpr double kShort = 1.0 - (double)kLog2e * kLn2;  // 1.335e-8: what c is short of log2 e, of itself
constexpr float kLeast = -160.0f;              // 2^kLeast is 0 in f32
constexpr float kWide = 65536.0f;
// Candidates a wave takes between two sorts. 8 / 12 / 24: 2,047 rows of 151,936 bf16 with 1 alternative 136.6 / 139.5 / 144.0 us, with 5
// 144.7 / 146.8 / 152.7, with 20 165.4 / 165.0 / 166.7; 64 f32 rows with 20 25.0 / 24.8 / 24.0; 33 of 32,001 12.6 / 12.3 / 12.1.
constexpr int kRoom = 12;

// A number's place among all, a negative zero not among them.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
// Orders as (logit, lower token first): larger keys are better, 0 is none.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
    return ((uint64_t)order_of(x == x ? x + 0.0f : -INFINITY) << 32) | (uint32_t)~token;
}
// The number after x (any but NaN; -inf: the lowest one).
__device__ __forceinline__ float above_next(float x) {
    const uint32_t o = order_of(x + 0.0f) + (x < INFINITY ? 1u : 0u);
    return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint32_t token_of(uint64_t key) { return ~(uint32_t)key; }

// LDS written by some lanes of a wave and read by others of it: in order as issued.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ uint64_t key_of_lane(uint64_t key, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(key >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, lane);
}

// The best `top` of n <= kBest distinct keys, in order, by counting: a key's place is the number of larger ones. (The others
// come by lane reads: from LDS each took its latency, 4 us for 80 keys. Eight at a time: one by one 1.2 us for 24, now 0.4.)
__device__ __forceinline__ void sort_best(uint64_t* keys, int n, int top) {
    const int lane = threadIdx.x & 63;
    wave_sync();
    const uint64_t a = lane < n ? keys[lane] : 0, b = lane + 64 < n ? keys[lane + 64] : 0;
    int ra = 0, rb = 0;
    if (n <= 64) {
#pragma unroll 1
        for (int i = 0; i < n; i += 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) ra += key_of_lane(a, i + j) > a;
    } else {
#pragma unroll 1
        for (int i = 0; i < 64; i += 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint64_t k = key_of_lane(a, i + j);
                ra += k > a;
                rb += k > b;
            }
#pragma unroll 1
        for (int i = 0; i < n - 64; i += 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint64_t k = key_of_lane(b, i + j);
                ra += k > a;
                rb += k > b;
            }
    }
    wave_sync();
    if (lane < n && ra < top) keys[ra] = a;
    if (lane + 64 < n && rb < top) keys[rb] = b;
    wave_sync();
}

// What the n-th largest of a wave's `order`s is at least, by its upper 18 bits; 0 if that is no number.
__device__ __forceinline__ uint32_t bound_of(uint32_t order, int n) {
    uint32_t v = 0;
    for (int bit = 31; bit >= 14; --bit) {
        const uint32_t up = v | (1u << bit);
        if (__popcll(__ballot(order >= up)) >= n) v = up;
    }
    return v > order_of(-INFINITY) ? v : 0;
}

// A wave's best `top` keys so far: candidates are appended, and sorted out when kRoom new ones are there.
struct Best {
    uint64_t* keys;      // LDS [kBest]
    int top;
    int count = 0;
    int sorted = 0;      // keys in order
    uint64_t least = 0;  // keys up to this one are none of the best

    __device__ __forceinline__ Best(uint64_t* room, int n) : keys(room), top(n) {}
    __device__ __forceinline__ float least_logit() const { return top == 0 ? INFINITY : least == 0 ? -INFINITY : logit_of(least); }
    __device__ __forceinline__ void sort() {
        if (sorted == count) return;
        sort_best(keys, count, top);
        sorted = count = min(count, top);
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
    // From each lane's best logit: what the top-th of them bounds from below.
    __device__ __forceinline__ void bound(uint32_t order) {
        const uint32_t v = bound_of(order, top);
        if (v != 0) least = ((uint64_t)v << 32) - 1;  // (the order before v's is a logit's)
    }
};

// A part's sums: its M, R and E over the tokens but one at M, relative to the reference `ref` (log2 units).
struct Sums {
    float m;
    double ref, r, e;
};

// A row's: R' and E' relative to M.
struct Row {
    float m;
    double r, e;
};

// Parts, one a lane (the others hold m = -inf), merged over a wave. Every part's own token at its m counts
// but one at the largest.
__device__ __forceinline__ Row merge_sums(const Sums& s) {
    constexpr double c = kLog2e;
    const float m = wave_max(s.m);
    if (m == -INFINITY) return Row{m, 0.0, 0.0};
    const uint64_t at = __ballot(s.m == m);
    const bool left_out = (threadIdx.x & 63) == (unsigned)(__ffsll((long long)at) - 1);
    double r = 0.0, e = 0.0;
    if (s.m != -INFINITY) {
        // the part's reference and its M above the row's M (both 0 where all are infinite)
        const double d = s.m == m && !(fabsf(m) < INFINITY) ? 0.0 : fmax(s.ref - (double)m * c, -1100.0);
        const double own = s.m == m ? 0.0 : fmax(((double)s.m - (double)m) * c, -1100.0);
        const double f = __builtin_amdgcn_exp2f((float)d), w = left_out ? 0.0 : (double)__builtin_amdgcn_exp2f((float)own);
        r = f * s.r + w;
        e = f * (s.e + d * s.r) + w * own;
    }
    return Row{m, wave_sum64(r), wave_sum64(e)};
}

template <int DT> __device__ __forceinline__ float load_logit(const void* p, size_t i) {
    if constexpr (DT == kLogitF32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == kLogitF16) return (float)static_cast<const _Float16*>(p)[i];
    else return __builtin_bit_cast(float, (uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}

// The given token's logit, -inf for one outside the row (loaded ahead of what it is used after).
template <int DT> __device__ __forceinline__ float given_logit(const LogprobArgs& a, size_t row) {
    if (a.logprobs == nullptr) return 0.f;
    const size_t t = a.targets[row];
    return t < a.length ? load_logit<DT>(a.logits, row * a.stride + t) : -INFINITY;
}

// A row's results by a wave, from its sums and its best keys in order.
__device__ __forceinline__ void finish(const LogprobArgs& a, size_t row, const Row& s, float given, const uint64_t* best) {
    const int lane = threadIdx.x & 63;
    // e^(x - M) = 2^t (1 + kShort ln2 t) to first order, so that E times kShort ln 2 is what R' lacks; what E' lacks is the
    // second moment's, which is E'^2 / R' of tokens that lie equally far below M, and more of others by their variance.
    double r = s.r, e = s.e;
    if (r > 0.0) {  // (R may be 0 in f32 where E is not)
        r = __builtin_fma(kShort * kLn2, s.e, s.r);
        e = __builtin_fma(kShort * s.e, __builtin_fma(kLn2 * s.e, __builtin_amdgcn_rcp(s.r), 1.0), s.e);  // (an estimate is enough)
    }
    const double rest = log1pf((float)r);  // (all of a result's parts have its sign: f32 is as good as its own rounding)
    auto logprob = [&](float x) {
        if (!(x > -INFINITY)) return -INFINITY;  // (or no number)
        return (float)((x == s.m ? 0.0 : (double)x - (double)s.m) - rest);
    };
    if (lane == 0) {
        if (a.logprobs != nullptr) a.logprobs[row] = logprob(given);
        if (a.entropy != nullptr) a.entropy[row] = s.m == -INFINITY ? 0.f : (float)fmax(rest - kLn2 * e / (1.0 + r), 0.0);
    }
    if (lane < a.top) {
        const uint64_t key = best[lane];
        a.top_tokens[row * a.top + lane] = token_of(key);
        a.top_logprobs[row * a.top + lane] = logprob(logit_of(key));
    }
}

// What a wave has seen: a lane's sums relative to the wave's reference.
struct Wave {
    float m = -INFINITY, ref = 0.f;
    float l = 0.f, e = 0.f;
    bool wide = false;  // |m| past kWide: the reference is m c exactly, t = (x - m) c

    // m moves to the largest of the lanes' `most`, and one of the logits at it (x is set to -inf) is left out; the one left
    // out so far counts.
    __device__ __forceinline__ void move(float to, float most, Logits& x) {
        const int lane = threadIdx.x & 63;
        const bool was_wide = wide;
        const float old = m, old_ref = ref;
        if (m > -INFINITY && lane == 0) {
            const float t = wide ? 0.f : __builtin_fmaf(m, kLog2e, -ref), w = __builtin_amdgcn_exp2f(t);
            l += w;
            e = __builtin_fmaf(t, w, e);
        }
        m = to;
        wide = !(fabsf(m) < kWide);
        ref = wide ? 0.f : m * kLog2e;
        if (old > -INFINITY) {
            // between what the sums are relative to: with |m| past kWide m c itself, else its f32
            float d = old_ref - ref;
            if (__builtin_expect(wide || was_wide, 0)) {
                d = (float)((was_wide ? (double)old * (double)kLog2e : (double)old_ref) - (wide ? (double)m * (double)kLog2e : (double)ref));
            }
            d = fmaxf(d, kLeast);
            const float f = __builtin_amdgcn_exp2f(d);
            e = f * __builtin_fmaf(d, l, e);
            l *= f;
        }
        bool here = lane == __ffsll((long long)__ballot(most == m)) - 1;
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            const bool at = here && x[i] == m;
            x[i] = at ? -INFINITY : x[i];
            here = here && !at;
        }
    }

    // The t from which a logit is past m (without an m any: the lowest numbers' t is -inf too).
    __device__ __forceinline__ float past() const { return m == -INFINITY ? m : above_next(__builtin_fmaf(m, kLog2e, -ref)); }

    // 16 logits a lane (-inf: none), none of them past m.
    __device__ __forceinline__ void add(const Logits& t) {
        float l16 = 0.f, e16 = 0.f;
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            const float p = __builtin_amdgcn_exp2f(t[i]);
            l16 += p;
            e16 = __builtin_fmaf(t[i], p, e16);
        }
        if (__builtin_expect(__any(!(e16 == e16)), 0)) {  // -inf, NaN
            l16 = e16 = 0.f;
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                const float raised = fmaxf(t[i], kLeast), p = __builtin_amdgcn_exp2f(raised);
                l16 += p;
                e16 = __builtin_fmaf(raised, p, e16);
            }
        }
        l += l16;
        e += e16;
    }

    // 16 logits a lane, some of which may be past m.
    __device__ __forceinline__ void take(Logits x, float most) {
        const float to = wave_max(most);
        if (to > m) move(to, most, x);
        if (m == -INFINITY) return;
        if (m == INFINITY) {
#pragma unroll
            for (int i = 0; i < kValues; ++i) l += x[i] == m ? 1.0f : 0.0f;
            return;
        }
        Logits t;
        if (wide) {
#pragma unroll
            for (int i = 0; i < kValues; ++i) t[i] = (x[i] - m) * kLog2e;
        } else {
#pragma unroll
            for (int i = 0; i < kValues; ++i) t[i] = __builtin_fmaf(x[i], kLog2e, -ref);
        }
        add(t);
    }
};

__device__ __forceinline__ float most_of(const Logits& x) {
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kValues; ++i) most = fmaxf(most, x[i] + 0.0f);  // (of a signaling NaN, a quiet one)
    return most;
}

// The candidates among 16 logits a lane, those of `least` or more: each lane's first ones, its second ones and so on.
// key(x, i): the i-th's key, 0: none.
template <class KEY>
__device__ __forceinline__ void collect(Best& best, const Logits& x, float least, KEY key) {
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kValues; ++i) mine |= x[i] >= least ? 1u << i : 0u;
    if (least == -INFINITY) mine = (1u << kValues) - 1;  // (any, NaN too)
    while (__any(mine != 0)) {
        const int i = __ffs(mine) - 1;
        float v = x[0];
#pragma unroll
        for (int j = 1; j < kValues; ++j) v = i == j ? x[j] : v;
        best.add(mine != 0 ? key(v, i) : 0);
        mine &= mine - 1;
    }
}

// Grid (row, split).
template <int DT>
__global__ __launch_bounds__(kThreads) void logprob_kernel(LogprobArgs a) {
    constexpr int kSize = DT == kLogitF32 ? 4 : 2;
    constexpr int kPer = 16 / kSize;            // logits a piece
    constexpr int kPieces = kValues / kPer;     // pieces a lane and iteration
    __shared__ uint64_t keys[kWaves][kBest];
    __shared__ uint64_t merged[kLogprobMaxTop];
    __shared__ int counts[kWaves];
    __shared__ float reached[kWaves];  // each wave's (top / 4)-th best logit: all four reach the least of them
    __shared__ float part_m[kWaves];
    __shared__ double part_ref[kWaves], part_r[kWaves], part_e[kWaves];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const size_t row = blockIdx.x;
    const int split = blockIdx.y;
    const char* const base = static_cast<const char*>(a.logits) + row * a.stride * kSize;
    // the row's pieces: 16-byte aligned and whole; the first `head` logits and those after the last piece are single
    const uint32_t length = (uint32_t)a.length;
    const uint32_t head = std::min<uint32_t>(length, (uint32_t)((16 - ((uintptr_t)base & 15)) & 15) / kSize);
    const uint32_t pieces = (length - head) / kPer;
    const uint4* const body = reinterpret_cast<const uint4*>(base + head * kSize);
    const uint32_t first = (uint32_t)((uint64_t)pieces * (unsigned)split / (unsigned)a.splits);
    const uint32_t last = (uint32_t)((uint64_t)pieces * ((unsigned)split + 1) / (unsigned)a.splits);

    Best best(keys[wave], a.top);
    Wave w;
    uint4 raw[kPieces];
    uint32_t at = first + (uint32_t)wave * 64 * kPieces;
    // (without a branch: past the part's end its last piece once more, a single line)
    auto load = [&] {
#pragma unroll
        for (int u = 0; u < kPieces; ++u) raw[u] = body[min(at + 64 * u + lane, last - 1)];
    };
    if (at < last) load();
    auto unpack = [&](uint32_t now) {
        Logits x;
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const uint32_t words[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                if constexpr (DT == kLogitF32) x[kPer * u + j] = __builtin_bit_cast(float, words[j]);
                else if constexpr (DT == kLogitF16) x[kPer * u + j] = half_bits_to_float((words[j >> 1] >> (16 * (j & 1))) & 0xffffu);
                else x[kPer * u + j] = __builtin_bit_cast(float, (j & 1) ? words[j >> 1] & 0xffff0000u : words[j >> 1] << 16);
            }
        }
        if (now + 64 * kPieces > last) {
#pragma unroll
            for (int i = 0; i < kValues; ++i) x[i] = now + 64 * (unsigned)(i / kPer) + lane < last ? x[i] : -INFINITY;
        }
        return x;
    };
    const float given = wave == 0 && a.splits == 1 ? given_logit<DT>(a, row) : 0.f;
    const int share = (a.top + kWaves - 1) / kWaves;
    if (a.top > 0) {
        const uint32_t v = at < last ? bound_of(order_of(most_of(unpack(at))), share) : 0;
        if (lane == 0) reached[wave] = v != 0 ? logit_of((uint64_t)v << 32) : -INFINITY;
    }
    __syncthreads();
    auto sort = [&] {
        best.sort();
        if (best.count >= share && lane == 0) __hip_atomic_store(&reached[wave], logit_of(keys[wave][share - 1]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    // What a candidate is at least: past the wave's own (its tokens rise, so that of equals the earlier is in), and
    // what the four waves reach together. `past` and `from`: the t past m, and that of such a candidate too.
    float shared = INFINITY, least = INFINITY, past = -INFINITY, from = -INFINITY;
    auto thresholds = [&] {
        if (a.top > 0) {
            shared = INFINITY;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) shared = fminf(shared, __hip_atomic_load(&reached[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            least = best.least != 0 ? fmaxf(shared, above_next(logit_of(best.least))) : shared;
        }
        from = least <= w.m ? fminf(past, __builtin_fmaf(least, kLog2e, -w.ref)) : past;
    };
    // the single ones: a last iteration of the first wave, one a lane (of equals, a token before the others' wins)
    const uint32_t end = head + pieces * kPer, singles = split == 0 && wave == 0 ? head + (length - end) : 0;
    const uint32_t token = (uint32_t)lane < head ? (uint32_t)lane : end + ((uint32_t)lane - head);
    const float one = (uint32_t)lane < singles ? load_logit<DT>(base, token) : -INFINITY;
    bool single = false;
    thresholds();
    for (uint32_t round = 0;; ++round) {
        Logits x;
        const uint32_t now = at;
        if (at < last) {
            x = unpack(now);
            at += kThreads * kPieces;
            load();
        } else {
            if (single || singles == 0) break;
            single = true;
            x = -INFINITY;
            x[0] = one;
        }
        Logits t;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            t[i] = __builtin_fmaf(x[i], kLog2e, -w.ref);
            top = fmaxf(top, t[i]);
        }
        bool changed = (round & 3) == 3, taken = false;
        if (w.wide || single || __any(top >= from)) {
            if (a.top > 0) {
                if (best.count < a.top && least == -INFINITY) best.bound(order_of(most_of(x)));
                collect(best, x, fmaxf(single ? shared : least, best.least_logit()), [&](float v, int i) {
                    if (single) return i == 0 && (uint32_t)lane < singles ? key_of(v, token) : 0;
                    const uint32_t piece = now + 64 * (unsigned)(i / kPer) + lane;
                    return piece < last ? key_of(v, head + piece * kPer + (unsigned)(i % kPer)) : 0;
                });
                if (best.count >= best.sorted + kRoom) {
                    sort();
                    changed = true;
                }
            }
            if (w.wide || __any(top >= past)) {
                w.take(x, most_of(x));
                past = w.past();
                changed = taken = true;
            }
        }
        if (!taken) w.add(t);
        if (changed) thresholds();
    }
    best.sort();
    const double r = wave_sum64((double)w.l), e = wave_sum64((double)w.e);
    if (lane == 0) {
        part_m[wave] = w.m;
        part_ref[wave] = w.wide ? (double)w.m * (double)kLog2e : (double)w.ref;
        part_r[wave] = r;
        part_e[wave] = e;
        counts[wave] = best.count;
    }
    __syncthreads();
    // the waves' lists in one: a key's place is its own and the larger ones of the three others
    {
        const uint64_t key = lane < best.count ? keys[wave][lane] : 0;
        int larger[kWaves - 1] = {};
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) {
            uint64_t k[kWaves - 1];
#pragma unroll
            for (int i = 0; i < kWaves - 1; ++i) k[i] = keys[(wave + 1 + i) % kWaves][larger[i] + step - 1];  // (at most 62)
#pragma unroll
            for (int i = 0; i < kWaves - 1; ++i)
                if (larger[i] + step <= counts[(wave + 1 + i) % kWaves] && k[i] > key) larger[i] += step;
        }
        const int place = lane + larger[0] + larger[1] + larger[2];
        if (lane < best.count && place < a.top) merged[place] = key;
    }
    __syncthreads();
    if (wave != 0) return;
    Sums s{-INFINITY, 0.0, 0.0, 0.0};
    if (lane < kWaves) s = Sums{part_m[lane], part_ref[lane], part_r[lane], part_e[lane]};
    const Row all = merge_sums(s);
    if (a.splits == 1) {
        finish(a, row, all, given, merged);
        return;
    }
    const int n = counts[0] + counts[1] + counts[2] + counts[3];
    uint64_t* part = a.partials + (row * (size_t)a.splits + (size_t)split) * (size_t)(3 + a.top);
    if (lane == 0) {
        part[0] = __builtin_bit_cast(uint32_t, all.m);
        part[1] = __builtin_bit_cast(uint64_t, all.r);
        part[2] = __builtin_bit_cast(uint64_t, all.e);
    }
    if (lane < a.top) part[3 + lane] = lane < n ? merged[lane] : 0;
}

// A row's parts: sums one a lane, keys one after another.
template <int DT>
__global__ __launch_bounds__(64) void logprob_merge_kernel(LogprobArgs a) {
    __shared__ uint64_t keys[kBest];
    constexpr int kAhead = 12;  // keys a lane under way
    const int lane = threadIdx.x;
    const size_t row = blockIdx.x;
    const uint64_t* parts = a.partials + row * (size_t)a.splits * (size_t)(3 + a.top);
    const int total = a.splits * a.top;
    uint64_t k[kAhead];
    auto load = [&](int e0) {  // key e: the (e / splits)-th best of part e % splits
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int e = e0 + 64 * i + lane;
            k[i] = e < total ? parts[(unsigned)e % (unsigned)a.splits * (unsigned)(3 + a.top) + 3u + (unsigned)e / (unsigned)a.splits] : 0;
        }
    };
    load(0);
    Sums s{-INFINITY, 0.0, 0.0, 0.0};
    if (lane < a.splits) {
        const uint64_t* part = parts + (size_t)lane * (size_t)(3 + a.top);
        const float m = __builtin_bit_cast(float, (uint32_t)part[0]);
        s = Sums{m, (double)m * (double)kLog2e, __builtin_bit_cast(double, part[1]), __builtin_bit_cast(double, part[2])};
    }
    const float given = given_logit<DT>(a, row);
    Best best(keys, a.top);
    for (int e = 0; e < total; e += 64 * kAhead) {
        if (e > 0) load(e);
        if (e == 0) {
            uint64_t most = k[0];
#pragma unroll
            for (int i = 1; i < kAhead; ++i) most = max(most, k[i]);
            best.bound((uint32_t)(most >> 32));
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) best.add(k[i]);
    }
    best.sort();
    finish(a, row, merge_sums(s), given, keys);
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
    if (args.rows == 0 || args.rows > 0xffffffffu / kThreads || args.length == 0 || args.top < 0 || args.top > kLogprobMaxTop || args.top > (long long)args.length) return hipErrorInvalidValue;
    LogprobArgs a = args;
    // Parts: until four workgroups a CU are there, of an iteration at least. With one, two, three, four, six a CU: 500 rows of
    // 151,936 bf16 with 20 alternatives 64.2, 64.3, 64.4, 63.5, 67.5 us; 64 of f32 31.1, 26.0, 26.4, 26.3, 30.0, without
    // alternatives 19.3, 16.6, 17.0, 17.4, 18.7; 33 of 32,001 15.0 by one, 13.1 by others.
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

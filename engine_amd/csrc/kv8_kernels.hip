// Kernels of the 8-bit KV cache for gfx950 (kv8.hpp has the layout and the
// arithmetic of a code): the append of new tokens, decode attention over the
// cache, and rows moved in and out of it.
#include "kv8.hpp"

#include <float.h>

#include <algorithm>

#include "kquant_device.hpp"
#include "kv8_device.hpp"
#include "rope_device.hpp"

namespace ribn_amd {

namespace {

// Buffer offset past any head's codes (2^28 bytes with the largest capacity), and still past them with
// a block's piece added: loads return 0 and fetch nothing.
constexpr uint32_t kOOR = 0x80000000u;
static_assert((uint64_t)kOOR >= ((uint64_t)1 << 20) / kKv8Block * kKv8BlockBytes && (uint64_t)kOOR + kKv8BlockBytes <= UINT32_MAX);
constexpr int kRowHalfs = kHeadDim + 8;  // LDS row of a staged token (272 B: 16-byte reads of 8 rows fall in distinct banks)

// ------------------------------------------------------------------- append
//
// One workgroup a (KV head, block of 32 positions). The block's new rows are
// staged in LDS as f16; a block that is whole after the append has its earlier
// rows added (from the tail, or from the codes of a block taken back into), its
// two scales found and its codes written, 16 of keys or of values a thread. The
// last block's workgroup writes what the tail holds after the call (its rows)
// and `end`, unless workgroup 0 may read the tail as it was (an append into the middle
// of a block): then that one does both, after its own block. Traffic is the rows in
// and a byte a value out: 32,768 f16 rows of 8 heads (134 MB in, 67 out) take 48 us, 4.2 TB/s.
// Short appends are the latency of one row's chain (load, sum of squares, angles, LDS,
// maximum, codes): 37 prompt tokens 7.0 us, 2,047 (17 MB in, 4 out) 8.8.

constexpr int kAppendThreads = 512;  // 16 lanes a row, a block's rows at once
__device__ __forceinline__ int append_tid() { return threadIdx.x & (kAppendThreads - 1); }

struct Rows {
    const void* k;    // the head's first row
    const void* v;
    size_t stride;    // values between tokens
};

// How rows arrive: raw projections (keys to be normalised and rotated), or as they are.
constexpr int kRowsRaw = 0, kRowsF32 = 1, kRowsF16 = 2;

struct Stage {
    _Float16 k[kKv8Block][kRowHalfs];
    _Float16 v[kKv8Block][kRowHalfs];
    float amax[8];
};

// The value of lane ^ 8 within a row of 16 lanes (row_ror 8).
__device__ __forceinline__ double other_half64(double v) {
    const uint2 w = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2((uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, 0x128, 0xf, 0xf, false),
                                                 (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, 0x128, 0xf, 0xf, false)));
}

// Eight values of a row as a cache takes them.
__device__ __forceinline__ kv8_half8 cache_halfs(const float (&x)[8]) {
    kv8_half8 h;
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = kv8_half(x[j]);
    return h;
}
__device__ __forceinline__ kv8_half8 cache_halfs(uint4 w) {
    auto special = [](uint32_t v) { return ((v & 0x7fff7fffu) + 0x04000400u) & 0x80008000u; };  // a half that is not finite
    kv8_half8 h = __builtin_bit_cast(kv8_half8, w);
    if (__builtin_expect((special(w.x) | special(w.y) | special(w.z) | special(w.w)) != 0, 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = kv8_half((float)h[j]);
    }
    return h;
}

// 1 / sqrt(x) of a normal x in 64 bits: the hardware's estimate (about 2^-23) and
// two Newton steps, y (3 - x y^2) / 2, where sqrt and a division take some 50 instructions.
__device__ __forceinline__ double inverse_root(double x) {
    double y = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) y = y * __builtin_fma(-0.5 * x * y, y, 1.5);
    return y;
}

// 16 lanes a row: lane c holds dims 8c .. 8c + 7 of row threadIdx / 16.
template <int ROWS>
__device__ __forceinline__ void stage_rows(Stage& st, const Rows& in, int first, int count, int row0, const float* k_norm,
                                           double eps, const double* rope, int position) {
    constexpr int kWords = ROWS == kRowsF16 ? 1 : 2;  // 16-byte pieces of a lane's eight values
    const int c = append_tid() & 15;
    const int i = append_tid() >> 4;
    if (i >= count) return;
    uint4 kw[kWords], vw[kWords];
    const size_t at = ((size_t)(first + i) * in.stride + 8 * c) * (ROWS == kRowsF16 ? 2 : 4);
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
        kw[w] = reinterpret_cast<const uint4*>(static_cast<const char*>(in.k) + at)[w];
        vw[w] = reinterpret_cast<const uint4*>(static_cast<const char*>(in.v) + at)[w];
    }
    if constexpr (ROWS == kRowsF16) {
        *reinterpret_cast<kv8_half8*>(&st.k[row0 + i][8 * c]) = cache_halfs(kw[0]);
        *reinterpret_cast<kv8_half8*>(&st.v[row0 + i][8 * c]) = cache_halfs(vw[0]);
    } else {
        float k[8], v[8];
        __builtin_memcpy(k, kw, 32);
        __builtin_memcpy(v, vw, 32);
        if constexpr (ROWS == kRowsRaw) {
            // 64 bits up to the one rounding to f32: where a key falls between two
            // codes then does not depend on the order of a sum. Lanes c and c ^ 8 hold the
            // two dims of the same eight pairs and form four of their angles each.
            const int upper = c >> 3;
            Rot64 mine[4], theirs[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mine[j] = turn_sincos((double)(position + i) * rope[8 * (c & 7) + 4 * upper + j]);
                theirs[j].s = other_half64(mine[j].s);
                theirs[j].c = other_half64(mine[j].c);
            }
            double ssq = 0.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) ssq = __builtin_fma((double)k[j], (double)k[j], ssq);
            const double inv = inverse_root(row_sum64(ssq) * (1.0 / kHeadDim) + eps) * rope[kHeadDim / 2];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const Rot64 r = (j >> 2) == upper ? mine[j & 3] : theirs[j & 3];
                const double y = (double)k[j] * inv * (double)k_norm[8 * c + j];
                const double o = other_half64(y) * r.s;
                k[j] = (float)__builtin_fma(y, r.c, upper ? o : -o);
            }
        }
        *reinterpret_cast<kv8_half8*>(&st.k[row0 + i][8 * c]) = cache_halfs(k);
        *reinterpret_cast<kv8_half8*>(&st.v[row0 + i][8 * c]) = cache_halfs(v);
    }
}

// Rows 0 .. count - 1 of block b as the cache has them, from its tail or its codes.
__device__ __forceinline__ void stage_held(Stage& st, const Kv8Head& h, int b, int count, bool tail) {
    const int tid = append_tid();
    if (tail) {
        if (tid < count * 16) *reinterpret_cast<uint4*>(&st.k[tid >> 4][8 * (tid & 15)]) = reinterpret_cast<const uint4*>(h.tail_k)[tid];
        const int dim = tid >> 2, key = 8 * (tid & 3);  // eight keys of a dim
        const kv8_half8 x = *reinterpret_cast<const kv8_half8*>(h.tail_v + dim * kKv8Block + key);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (key + j < count) st.v[key + j][dim] = x[j];
        return;
    }
    // a thread's piece: 256 of keys, then 256 of values, as the codes lie
    const uint4 w = reinterpret_cast<const uint4*>(h.codes + (size_t)b * kKv8BlockBytes)[tid];
    const float2 sc = h.scales[b];
    const bool keys = tid < 256;
    const int lane = tid & 63, u = (tid >> 6) & 3, g = lane >> 4, m = lane & 15;
    const _Float16 scale = (_Float16)(keys ? sc.x : sc.y);
    const kv8_half8 x0 = kv8_values(w.x, w.y, scale), x1 = kv8_values(w.z, w.w, scale);
    if (keys) {
        const int row = kv8_key_row(u >> 1, m);
        if (row < count) {
            kv8_half8* k = reinterpret_cast<kv8_half8*>(&st.k[row][64 * (u & 1) + 16 * g]);
            k[0] = x0;
            k[1] = x1;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (8 * g + j < count) *reinterpret_cast<kv8_half2*>(&st.v[8 * g + j][32 * u + 2 * m]) = kv8_half2{x0[j], x1[j]};
    }
}

// The staged block's 32 rows into codes and scales, a piece a thread.
__device__ __forceinline__ void quantise(Stage& st, const Kv8Head& h, int b) {
    const int tid = append_tid(), lane = tid & 63, wave = tid >> 6, u = wave & 3, g = lane >> 4, m = lane & 15;
    const bool keys = tid < 256;
    kv8_half2 x[8], top{};
    const kv8_half2* kr = reinterpret_cast<const kv8_half2*>(&st.k[kv8_key_row(u >> 1, m)][64 * (u & 1) + 16 * g]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = keys ? kr[j] : *reinterpret_cast<const kv8_half2*>(&st.v[8 * g + j][32 * u + 2 * m]);
        top = kv8_top(top, x[j]);
    }
    const float wave_top = wave_max(fmaxf((float)top[0], (float)top[1]));
    if (lane == 0) st.amax[wave] = wave_top;
    __syncthreads();
    const float* parts = st.amax + (wave & 4);
    const int e = kv8_exponent(fmaxf(fmaxf(parts[0], parts[1]), fmaxf(parts[2], parts[3])));
    const Kv8Inverse inv(e);
    if (!keys) {  // pairs of dims to pairs of keys: the first dim's eight, then the second's
        kv8_half2 y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = kv8_half2{x[2 * (j & 3)][j >> 2], x[2 * (j & 3) + 1][j >> 2]};
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = y[j];
    }
    reinterpret_cast<uint4*>(h.codes + (size_t)b * kKv8BlockBytes)[tid] =
        make_uint4(kv8_word(x[0], x[1], inv), kv8_word(x[2], x[3], inv), kv8_word(x[4], x[5], inv), kv8_word(x[6], x[7], inv));
    if (lane == 0 && u == 0) reinterpret_cast<float*>(h.scales + b)[keys ? 0 : 1] = kv8_power(e);
}

__device__ __forceinline__ void store_tail(const Stage& st, const Kv8Head& h, int row0, int rows) {
    const int i = row0 * 16 + append_tid();
    if (i < rows * 16) reinterpret_cast<uint4*>(h.tail_k)[i] = *reinterpret_cast<const uint4*>(&st.k[i >> 4][8 * (i & 15)]);
    const int d = append_tid() & 127;
    for (int r = row0 + (append_tid() >> 7); r < rows; r += 4) h.tail_v[d * kKv8Block + r] = st.v[r][d];
}

// Block p0 / 32 + j of an append of `tokens` rows at p0 (0 <= p0, p0 + tokens <= capacity).
// Where workgroup 0 keeps the tail besides a block of its own, it has two halves of
// kAppendThreads: the second one stages the last block meanwhile, and stores it
// once the first has read the tail.
template <int ROWS>
__device__ __forceinline__ void append_block(Stage (&stages)[2], const Kv8Head& h, const Rows& in, int p0, int tokens, int j,
                                             const float* k_norm, double eps, const double* rope) {
    const int end = p0 + tokens;
    const int own = p0 / kKv8Block + j;
    const int last = (end - 1) / kKv8Block;
    const bool apart = p0 % kKv8Block == 0;  // nobody reads the old tail: the last block's workgroup may write it
    const bool keeper = apart ? own == last : j == 0;
    const bool second = threadIdx.x >= kAppendThreads;
    if (second && !(keeper && own != last)) return;
    if (!keeper && end - own * kKv8Block < kKv8Block) return;  // the last block, not whole: workgroup 0's
    const int b = second ? last : own;
    Stage& st = stages[second ? 1 : 0];
    const int first = max(p0, b * kKv8Block);             // this block's new positions
    const int fill = min(end - b * kKv8Block, kKv8Block);  // rows it holds afterwards
    const bool whole = fill == kKv8Block;
    const int row0 = first - b * kKv8Block;
    stage_rows<ROWS>(st, in, first - p0, fill - row0, row0, k_norm, eps, rope, first);
    int kept = row0;  // rows of the tail that stay as they are
    if (row0 != 0) {
        const int old = *h.end;
        const bool held = old > 0 && (old - 1) / kKv8Block == b;
        if (whole || !held) stage_held(st, h, b, row0, held);
        if (!held) kept = 0;
    }
    __syncthreads();
    if (second) {
        __syncthreads();  // (quantise's)
    } else if (whole) {
        quantise(st, h, b);
    }
    if (!keeper || b != last) return;
    store_tail(st, h, kept, fill);
    if (append_tid() == 0) *h.end = end;
}

// Threads of an append's workgroups.
int append_threads(int p0, int tokens) {
    const bool twice = p0 % kKv8Block != 0 && (p0 + tokens - 1) / kKv8Block != p0 / kKv8Block;
    return twice ? 2 * kAppendThreads : kAppendThreads;
}

// Members that share a cache, at consecutive positions. Grid (KV head, block).
__global__ __launch_bounds__(2 * kAppendThreads) void kv8_append_kernel(AttnArgs a, int members) {
    __shared__ Stage st[2];
    const int kvh = blockIdx.x;
    const AttnMember mb = a.mem[0];
    const int pos = a.positions[0];
    if (pos < 0 || pos > mb.capacity - members) return;
    const int j = blockIdx.y;
    if (pos / kKv8Block + j > (pos + members - 1) / kKv8Block) return;
    const size_t at = (size_t)kvh * kHeadDim;
    const Rows in{a.k + at, a.v + at, (size_t)a.kv_heads * kHeadDim};
    append_block<kRowsRaw>(st, kv8_head(mb, a.layer, kvh), in, pos, members, j, a.k_norm, a.eps, mb.rope);
}

__global__ __launch_bounds__(2 * kAppendThreads) void kv8_append_seq_kernel(PrefillAttnArgs a) {
    __shared__ Stage st[2];
    const int kvh = blockIdx.x;
    const size_t at = (size_t)kvh * kHeadDim;
    const Rows in{a.k + at, a.v + at, (size_t)a.kv_heads * kHeadDim};
    append_block<kRowsRaw>(st, kv8_head(a.mem, a.layer, kvh), in, a.p0, a.tokens, blockIdx.y, a.k_norm, a.eps, a.mem.rope);
}

template <int ROWS>
__global__ __launch_bounds__(2 * kAppendThreads) void kv8_write_kernel(KvMoveArgs a) {
    __shared__ Stage st[2];
    const int kvh = blockIdx.x;
    const size_t at = (size_t)kvh * kHeadDim * (ROWS == kRowsF16 ? 2 : 4);
    const Rows in{static_cast<const char*>(a.keys) + at, static_cast<const char*>(a.values) + at, (size_t)a.kv_heads * kHeadDim};
    append_block<ROWS>(st, kv8_head(a.mem, a.layer, kvh), in, a.p0, a.tokens, blockIdx.y, nullptr, 0.0, nullptr);
}

// Eight values of a row in memory, as f16.
__device__ __forceinline__ kv8_half8 load_row(const _Float16* p) { return *reinterpret_cast<const kv8_half8*>(p); }
__device__ __forceinline__ kv8_half8 load_row(const float* p) {
    kv8_half8 h;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float4 x = reinterpret_cast<const float4*>(p)[i];
        h[4 * i] = (_Float16)x.x;
        h[4 * i + 1] = (_Float16)x.y;
        h[4 * i + 2] = (_Float16)x.z;
        h[4 * i + 3] = (_Float16)x.w;
    }
    return h;
}
__device__ __forceinline__ void store_row(_Float16* p, kv8_half8 h) { *reinterpret_cast<kv8_half8*>(p) = h; }
__device__ __forceinline__ void store_row(float* p, kv8_half8 h) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        reinterpret_cast<float4*>(p)[i] = make_float4((float)h[4 * i], (float)h[4 * i + 1], (float)h[4 * i + 2], (float)h[4 * i + 3]);
}

// Rows out of an 8-bit cache, grid (KV head, block): the values its codes stand
// for, the tail's f16 values of the block that is not whole, zeros past `end`. Through
// LDS, so that rows leave whole: 32,768 rows of 8 heads (67 MB in, 134 out) in 30.6 us, 6.6 TB/s
// (the codes had just been written).
template <typename T>
__global__ __launch_bounds__(kAppendThreads, 4) void kv8_read_kernel(KvMoveArgs a) {
    __shared__ Stage st;
    const int kvh = blockIdx.x;
    const int b = a.p0 / kKv8Block + (int)blockIdx.y;
    const Kv8Head h = kv8_head(a.mem, a.layer, kvh);
    const int end = *h.end;
    const int rows = max(0, min(end - b * kKv8Block, kKv8Block));
    stage_held(st, h, b, rows, rows < kKv8Block);
    __syncthreads();
    const int lo = max(a.p0, b * kKv8Block) - b * kKv8Block, hi = min(a.p0 + a.tokens, (b + 1) * kKv8Block) - b * kKv8Block;
    const int c = threadIdx.x & 15;
    const int r = (int)threadIdx.x >> 4;
    if (r < lo || r >= hi) return;
    const size_t at = ((size_t)(b * kKv8Block + r - a.p0) * a.kv_heads + kvh) * kHeadDim + 8 * c;
    kv8_half8 k{}, v{};
    if (r < rows) {
        k = *reinterpret_cast<const kv8_half8*>(&st.k[r][8 * c]);
        v = *reinterpret_cast<const kv8_half8*>(&st.v[r][8 * c]);
    }
    store_row(static_cast<T*>(a.keys) + at, k);
    store_row(static_cast<T*>(a.values) + at, v);
}

// An f16 cache's rows ([kv_head][token][128]), in and out: 16 lanes a row, grid
// (16 tokens, KV head). (f16 overflow gives infinities here, as the appends of f16 caches do.)
template <typename T>
__global__ __launch_bounds__(256) void kv16_write_kernel(KvMoveArgs a) {
    const int kvh = blockIdx.y, c = threadIdx.x & 15, t = (int)blockIdx.x * 16 + ((int)threadIdx.x >> 4);
    if (t >= a.tokens) return;
    const size_t to = (size_t)a.layer * a.mem.layer_elems + ((size_t)kvh * a.mem.capacity + (size_t)(a.p0 + t)) * kHeadDim + 8 * c;
    const size_t at = ((size_t)t * a.kv_heads + kvh) * kHeadDim + 8 * c;
    store_row(reinterpret_cast<_Float16*>(a.mem.keys) + to, load_row(static_cast<const T*>(a.keys) + at));
    store_row(reinterpret_cast<_Float16*>(a.mem.values) + to, load_row(static_cast<const T*>(a.values) + at));
}

template <typename T>
__global__ __launch_bounds__(256) void kv16_read_kernel(KvMoveArgs a) {
    const int kvh = blockIdx.y, c = threadIdx.x & 15, t = (int)blockIdx.x * 16 + ((int)threadIdx.x >> 4);
    if (t >= a.tokens) return;
    const size_t from = (size_t)a.layer * a.mem.layer_elems + ((size_t)kvh * a.mem.capacity + (size_t)(a.p0 + t)) * kHeadDim + 8 * c;
    const size_t at = ((size_t)t * a.kv_heads + kvh) * kHeadDim + 8 * c;
    store_row(static_cast<T*>(a.keys) + at, load_row(reinterpret_cast<const _Float16*>(a.mem.keys) + from));
    store_row(static_cast<T*>(a.values) + at, load_row(reinterpret_cast<const _Float16*>(a.mem.values) + from));
}

struct CacheInit {
    double table[kHeadDim / 2 + 1];
    double* table_dst;
    char* regions;
    size_t stride;  // bytes a region
    size_t codes;   // its code bytes, left as they are
};

__global__ __launch_bounds__(256) void cache_init_kernel(CacheInit a) {
    const int tid = threadIdx.x;
    if (blockIdx.x == 0 && tid <= kHeadDim / 2) a.table_dst[tid] = a.table[tid];
    if (a.regions == nullptr) return;
    uint4* p = reinterpret_cast<uint4*>(a.regions + (size_t)blockIdx.x * a.stride + a.codes);
    for (size_t i = tid; i < (a.stride - a.codes) / sizeof(uint4); i += 256) p[i] = make_uint4(0, 0, 0, 0);
}

// ---------------------------------------------------------- decode attention
//
// kv8_attn_kernel: one layer's attention of decode members over their caches,
// the new token's key and value appended on the way, on the f16 matrix cores: the
// cache's values are f16 exactly, and converting and multiplying a byte for eight
// query heads would leave the VALU behind the memory. Memory bounds the long cases
// (131,071 tokens, 269 MB: 49.5 us, 5.4 TB/s), latency the short ones: 5.6 us pass
// between a launch and its output however little it reads (40 tokens), and 8 members of 3,000
// (36 MB) take 11, 24 of 1,501 with 64 heads (58 MB) 16, their merge 2 to 3 more.
//
// Split as attn_decode_kernel's: grid (chunk, KV head, member), a chunk one
// contiguous run of whole blocks; its waves take the blocks in turn. A block is
// 8 KB of codes, eight 16-byte loads a lane, each of them contiguous over
// the wave (the codes lie in that order), one block in flight a wave, up to three
// workgroups a CU. (Two blocks in flight: 8 members of 3,000 16.1 us for 13.9, 24 of 1,501
// 20.4 for 19.3, 131,071 tokens 52.8 for 52.1; with two KV heads, where a wave has its SIMD to itself, 30.2 for 31.4.)
//
// The chunks are merged by a launch of its own. The last workgroup of a row to arrive could
// do it, but handing partials over between XCDs costs as much: with write-through
// stores and loads 8 members of 3,000 took 14.4 us for 13.9, 131,071 tokens 55.0
// for 52.3, 8 members of 15,000 53 for 40 (with fences, which write back an XCD's whole L2, 70, 74 and 387).
//
// S^T = K Q^T (v_mfma_f32_16x16x32_f16: M = 16 keys, N = 16 columns, K = 32
// dims): the columns are the QPK query heads of the KV head twice, the upper
// f16 piece of each in columns 0..7 and the lower one in 8..15, so one product
// carries 22 bits of q and the two halves of a score are one row rotation apart.
// Row 4g + i of tile t is key 8g + 4t + i: lane group g ends up with eight
// consecutive keys, which is the B operand's share of O^T += V^T P^T (M = 16
// dims, K = 32 keys), the probabilities again in two pieces by column half.
// Codes enter the scores as whole numbers, the block's key scale being applied to
// the f32 score; values are scaled as f16 (both exact). The softmax's reference is
// the column's and moves as kTopExponent says; denominators are f32 sums of f32
// numerators, a block's first, so that many small ones do not each meet a large sum.
//
// The block the sequence stands in is the last wave's: it has the tail's rows in
// the operands' order, puts the new token's row in from LDS, and, when the block is whole,
// finds its scales and writes its codes from there, going on with what these stand for.
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;

// Tokens of a chunk: two blocks a wave at least, four where there are many members (more than
// 8, as for f16 caches: a member's bits do not depend on the others within either range).
// Whole calls with 128 / 256 / 512 tokens: one member of 2,047 11.0 / 11.4 / 12.2 us, 8
// of 3,000 15.8 / 14.0 / 13.7; with 256 / 512 / 1,024: 24 of 1,501 20.9 / 19.4 / 21.3.
constexpr int kMinChunk = 256;
constexpr int kMinChunkWide = 512;
constexpr int kFewMembers = 8;
int kv8_min_chunk(int members) { return members > kFewMembers ? kMinChunkWide : kMinChunk; }

__device__ __forceinline__ int kv8_chunk_tokens(int tokens, int chunks, int min_chunk) {
    const int len = max((tokens + chunks - 1) / chunks, min_chunk);
    return (len + kKv8Block - 1) / kKv8Block * kKv8Block;
}

// The value of lane ^ 8.
__device__ __forceinline__ float other_half(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false));
}

typedef float kv8_float4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv8_u4 __attribute__((ext_vector_type(4)));

// The tail's block in the operands' order: keys (tile t, step s) at 4 t + s, values
// (u, i) at 2 u + i (kv8.hpp's code order, a piece being two of these).
struct TailBlock {
    kv8_u4 (&k)[8];
    kv8_u4 (&v)[8];

    __device__ __forceinline__ static int key_at(int i, int lane) {
        return kv8_key_row(i >> 2, lane & 15) * kHeadDim + 64 * ((i >> 1) & 1) + 16 * (lane >> 4) + 8 * (i & 1);
    }
    __device__ __forceinline__ static int value_at(int i, int lane) {
        return (32 * (i >> 1) + 2 * (lane & 15) + (i & 1)) * kKv8Block + 8 * (lane >> 4);
    }
    __device__ __forceinline__ void load(const Kv8Head& h, int lane) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k[i] = *reinterpret_cast<const kv8_u4*>(h.tail_k + key_at(i, lane));
            v[i] = *reinterpret_cast<const kv8_u4*>(h.tail_v + value_at(i, lane));
        }
    }
    __device__ __forceinline__ static void expand(kv8_u4 w, float scale, kv8_u4& x, kv8_u4& y) {
        x = __builtin_bit_cast(kv8_u4, kv8_values(w.x, w.y, (_Float16)scale));
        y = __builtin_bit_cast(kv8_u4, kv8_values(w.z, w.w, (_Float16)scale));
    }
    // What the codes of block b stand for.
    __device__ __forceinline__ void load_codes(const Kv8Head& h, int b, int lane) {
        const kv8_u4* c = reinterpret_cast<const kv8_u4*>(h.codes + (size_t)b * kKv8BlockBytes) + lane;
        const float2 sc = h.scales[b];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            expand(c[64 * i], sc.x, k[2 * i], k[2 * i + 1]);
            expand(c[64 * (4 + i)], sc.y, v[2 * i], v[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void store(const Kv8Head& h, int rows, int lane) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (kv8_key_row(i >> 2, lane & 15) < rows) *reinterpret_cast<kv8_u4*>(h.tail_k + key_at(i, lane)) = k[i];
            *reinterpret_cast<kv8_u4*>(h.tail_v + value_at(i, lane)) = v[i];
        }
    }
    // Row r from `row_k`, `row_v` [128].
    __device__ __forceinline__ void insert(int r, const _Float16* row_k, const _Float16* row_v, int lane) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (kv8_key_row(i >> 2, lane & 15) == r) k[i] = *reinterpret_cast<const kv8_u4*>(row_k + (key_at(i, lane) & (kHeadDim - 1)));
            const uint32_t y = 0x10001u * __builtin_bit_cast(uint16_t, row_v[value_at(i, lane) / kKv8Block]);
            const uint32_t half = (lane >> 4) == (r >> 3) ? ((r & 1) ? 0xffff0000u : 0xffffu) : 0u;
            uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t mask = j == ((r & 7) >> 1) ? half : 0u;
                w[j] = (w[j] & ~mask) | (y & mask);
            }
            v[i] = kv8_u4{w[0], w[1], w[2], w[3]};
        }
    }
    __device__ __forceinline__ static void quantise_part(kv8_u4 (&x)[8], kv8_u4* codes, float& scale) {
        auto pair = [](uint32_t w) { return __builtin_bit_cast(kv8_half2, w); };
        kv8_half2 top{};
#pragma unroll
        for (int i = 0; i < 8; ++i) top = kv8_top(kv8_top(kv8_top(kv8_top(top, pair(x[i].x)), pair(x[i].y)), pair(x[i].z)), pair(x[i].w));
        const int e = kv8_exponent(wave_max(fmaxf((float)top[0], (float)top[1])));
        const Kv8Inverse inv(e);
        scale = kv8_power(e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const kv8_u4 a = x[2 * i], b = x[2 * i + 1];
            const kv8_u4 w = kv8_u4{kv8_word(pair(a.x), pair(a.y), inv), kv8_word(pair(a.z), pair(a.w), inv),
                                  kv8_word(pair(b.x), pair(b.y), inv), kv8_word(pair(b.z), pair(b.w), inv)};
            codes[64 * i] = w;
            expand(w, scale, x[2 * i], x[2 * i + 1]);
        }
    }
    // Codes and scales of the whole block; its values become what these stand for.
    __device__ __forceinline__ void quantise(const Kv8Head& h, int b, int lane) {
        kv8_u4* c = reinterpret_cast<kv8_u4*>(h.codes + (size_t)b * kKv8BlockBytes) + lane;
        float2 sc;
        quantise_part(k, c, sc.x);
        quantise_part(v, c + 256, sc.y);
        if (lane == 0) h.scales[b] = sc;
    }
};

// The members' descriptors: in device memory (a captured step's), or in the
// launch's own arguments, which saves a call the launch that would put them there and
// the kernel a load that everything else waits for.
template <bool INLINE> struct Members {
    __device__ __forceinline__ AttnMember get(const AttnArgs& a, int m) const { return a.mem[m]; }
};
template <> struct Members<true> {
    AttnMember mem[kAttnMaxMembers];
    __device__ __forceinline__ AttnMember get(const AttnArgs&, int m) const { return mem[m]; }
};

// How many tokens a member attends: its position's and those before it, or, where
// the append was dropped or done for several members at once, what the cache holds.
__device__ __forceinline__ int kv8_tokens(const AttnArgs& a, const AttnMember& mb, const Kv8Head& head, int pos, int& end) {
    const int reach = min(pos, mb.capacity) + 1;  // (any int32 is a position)
    end = reach;
    if (a.appended || pos >= mb.capacity) end = *head.end;
    return min(reach, end);
}

template <int QPK, bool INLINE>
__global__ __launch_bounds__(kThreads, 3) void kv8_attn_kernel(AttnArgs a, Members<INLINE> members) {
    constexpr int kHeadsPerWave = (QPK + kWaves - 1) / kWaves;
    __shared__ __attribute__((aligned(16))) _Float16 qs[2][QPK][kRowHalfs];
    __shared__ __attribute__((aligned(16))) _Float16 fresh[2][kHeadDim];  // the new token's key and value
    __shared__ float qfac[QPK];
    __shared__ float2 st_ml[kWaves][QPK];
    __shared__ float st_o[kWaves][QPK][kHeadDim];

    const int chunk = blockIdx.x;
    const int kvh = blockIdx.y;
    const int m = blockIdx.z;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4;
    const int n = lane & 15;
    const AttnMember mb = members.get(a, m);
    const int pos = a.positions[m];
    // loads that need neither go first: the query heads, the norm weights, the new token's row
    const float* qm = a.q + ((size_t)m * a.q_heads + (size_t)kvh * QPK) * kHeadDim;
    float qx[kHeadsPerWave][2];
#pragma unroll
    for (int i = 0; i < kHeadsPerWave; ++i) {
        const int h = min(wave + kWaves * i, QPK - 1);
        qx[i][0] = qm[h * kHeadDim + lane];
        qx[i][1] = qm[h * kHeadDim + 64 + lane];
    }
    const float qw0 = a.q_norm[lane], qw1 = a.q_norm[lane + 64];
    float nx0 = 0.f, nx1 = 0.f, kw0 = 0.f, kw1 = 0.f;
    if (wave < 2) {
        const float* src = (wave == 0 ? a.k : a.v) + ((size_t)m * a.kv_heads + kvh) * kHeadDim;
        nx0 = src[lane];
        nx1 = src[lane + 64];
        kw0 = a.k_norm[lane];
        kw1 = a.k_norm[lane + 64];
    }

    const Kv8Head head = kv8_head(mb, a.layer, kvh);
    int end;
    const int tokens = kv8_tokens(a, mb, head, pos, end);
    const bool append = !a.appended && pos < mb.capacity;
    const int len = kv8_chunk_tokens(tokens, a.chunks, a.min_chunk);
    const int t0 = chunk * len;
    if (t0 >= tokens) {
        if (a.chunks == 1) {  // a member without tokens: zeros
            for (int i = tid; i < QPK * kHeadDim; i += kThreads) a.out[((size_t)m * a.q_heads + (size_t)kvh * QPK) * kHeadDim + i] = 0.f;
        }
        return;
    }
    const int t1 = min(t0 + len, tokens);

    // ---- blocks of this wave: b0 + wave, + kWaves, ... below `coded`, whose codes are
    // in the cache; the one after them, if the chunk reaches it, is the last wave's first
    const int b0 = t0 / kKv8Block;
    const int coded = min((t1 + kKv8Block - 1) / kKv8Block, (append ? pos : end) / kKv8Block);
    const bool has_tail = t1 > coded * kKv8Block;
    const bool tail = has_tail && wave == kWaves - 1;
    const __amdgpu_buffer_rsrc_t cr = make_rsrc(head.codes, (uint32_t)kv8_tail_offset(mb.capacity));
    const __amdgpu_buffer_rsrc_t sr = make_rsrc(head.scales, (uint32_t)(kv8_blocks(mb.capacity) * sizeof(float2)));
    // A block's keys (or values) and their scale, 0 or kKv8PartBytes of it.
    auto issue = [&](int b, int part, kv8_u4 (&w)[8], float& scale) {
        const uint32_t at = b < coded ? (uint32_t)b * kKv8BlockBytes + (uint32_t)part + 16u * (uint32_t)lane : kOOR;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(kv8_u4, load_b128(cr, at + 1024u * i));
        scale = __builtin_bit_cast(float, load_b32(sr, b < coded ? 8u * (uint32_t)b + (part ? 4u : 0u) : kOOR));
    };
    kv8_u4 kq[8], vq[8];  // a block's codes (the first four), or the tail's block
    float ks = 0.f, vs = 0.f;
    TailBlock tb{kq, vq};
    int old_end = 0;
    if (tail) {
        old_end = *head.end;
        tb.load(head, lane);
    } else {
        issue(b0 + wave, 0, kq, ks);
        issue(b0 + wave, kKv8PartBytes, vq, vs);
    }

    // ---- query heads: norm and rope, scaled by a power of two (query_exponent), in pieces
    const Rot64 rot = turn_sincos((double)pos * mb.rope[lane]);
    const double gain = mb.rope[kHeadDim / 2];
    const float rc = (float)(rot.c * gain), rs = (float)(rot.s * gain);
#pragma unroll
    for (int i = 0; i < kHeadsPerWave; ++i) {
        const int h = wave + kWaves * i;
        if (h < QPK) {
            const float ssq = wave_sum_uniform(qx[i][0] * qx[i][0] + qx[i][1] * qx[i][1]);
            const float inv = 1.0f / sqrtf(ssq / (float)kHeadDim + a.eps);
            const float y0 = qx[i][0] * inv * qw0, y1 = qx[i][1] * inv * qw1;
            const float q0 = y0 * rc - y1 * rs, q1 = y0 * rs + y1 * rc;
            const float top = wave_max(fmaxf(fabsf(q0), fabsf(q1)));
            const int e = query_exponent(top);
            const float p0 = q0 * kv8_power(-e), p1 = q1 * kv8_power(-e);
            qs[0][h][lane] = (_Float16)p0;
            qs[0][h][lane + 64] = (_Float16)p1;
            qs[1][h][lane] = (_Float16)(p0 - (float)(_Float16)p0);
            qs[1][h][lane + 64] = (_Float16)(p1 - (float)(_Float16)p1);
            if (lane == 0) qfac[h] = a.scale * kv8_power(e);
        }
    }
    const int row = pos & (kKv8Block - 1);
    if (append && has_tail && wave < 2) {  // the new token: wave 0 its key (64 bits), wave 1 its value
        if (wave == 0) {
            const double x0 = nx0, x1 = nx1;
            const double ssq = wave_sum64(__builtin_fma(x0, x0, x1 * x1));
            const double inv = inverse_root(ssq * (1.0 / kHeadDim) + (double)a.eps) * gain;
            const double y0 = x0 * inv * (double)kw0, y1 = x1 * inv * (double)kw1;
            nx0 = (float)__builtin_fma(y0, rot.c, -y1 * rot.s);
            nx1 = (float)__builtin_fma(y0, rot.s, y1 * rot.c);
        }
        const _Float16 h0 = kv8_half(nx0), h1 = kv8_half(nx1);
        fresh[wave][lane] = h0;
        fresh[wave][lane + 64] = h1;
        if (wave == 0) {
            head.tail_k[row * kHeadDim + lane] = h0;
            head.tail_k[row * kHeadDim + 64 + lane] = h1;
        } else {
            head.tail_v[lane * kKv8Block + row] = h0;
            head.tail_v[(lane + 64) * kKv8Block + row] = h1;
        }
    }
    __syncthreads();
    const int hn = n & 7;
    kv8_half8 qb[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        qb[s] = kv8_half8{};
        if (hn < QPK) qb[s] = *reinterpret_cast<const kv8_half8*>(&qs[n >> 3][hn][64 * (s >> 1) + 16 * g + 8 * (s & 1)]);
    }
    const float fac = hn < QPK ? qfac[hn] : 0.f;

    float mrun = -FLT_MAX, lrun = 0.f;
    kv8_float4 o[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) o[d] = kv8_float4{0.f, 0.f, 0.f, 0.f};

    // Scores of a block's two key tiles to probabilities in pieces (s in f32, `scaled` by the key scale).
    auto soften = [&](kv8_float4 (&s)[2], float scaled, int b, kv8_half8& pb) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (s[j >> 2][j & 3] + other_half(s[j >> 2][j & 3])) * scaled;
        if (b * kKv8Block + kKv8Block > tokens) {  // keys past the member's position
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (b * kKv8Block + 8 * g + j >= tokens) x[j] = -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
        if (__any(top > mrun + kMaxExponent)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float mn = top > mrun + kMaxExponent ? top - kTopExponent : mrun;
            const float corr = __builtin_amdgcn_exp2f(mrun - mn);
            mrun = mn;
            lrun *= corr;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[d] *= corr;
        }
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float p0 = __builtin_amdgcn_exp2f(x[j] - mrun), p1 = __builtin_amdgcn_exp2f(x[j + 1] - mrun);
            sum += p0;
            sum += p1;
            const kv8_half2 hi = kv8_halfs(p0, p1);
            const kv8_half2 lo = kv8_halfs(p0 - (float)hi[0], p1 - (float)hi[1]);
            const uint32_t hw = __builtin_bit_cast(uint32_t, hi), lw = __builtin_bit_cast(uint32_t, lo);
            const kv8_half2 p = __builtin_bit_cast(kv8_half2, n < 8 ? hw : lw);
            pb[j] = p[0];
            pb[j + 1] = p[1];
        }
        lrun += sum;
    };

    if (tail) {
        const int b = coded;
        if (append) {
            // rows before the new one, if the tail has another block's: what the block's codes stand for
            const bool held = row == 0 || (old_end > 0 && (old_end - 1) / kKv8Block == b);
            if (__builtin_expect(!held, 0)) tb.load_codes(head, b, lane);
            tb.insert(row, fresh[0], fresh[1], lane);
            if (__builtin_expect(!held, 0)) tb.store(head, row + 1, lane);
            if (__builtin_expect(row == kKv8Block - 1, 0)) tb.quantise(head, b, lane);
            if (lane == 0) *head.end = pos + 1;
        }
        kv8_float4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(kv8_half8, kq[4 * t + i]), qb[i], s[t], 0, 0, 0);
        kv8_half8 pb;
        soften(s, fac, b, pb);
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(kv8_half8, vq[d]), pb, o[d], 0, 0, 0);
        issue(b0 + wave, 0, kq, ks);
        issue(b0 + wave, kKv8PartBytes, vq, vs);
    }
    // (the next block's keys are under way as soon as this one's are used, its values likewise)
    for (int b = b0 + wave; b < coded; b += kWaves) {
        kv8_float4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const kv8_u4 w = kq[2 * t + (i >> 1)];
                const kv8_half8 k = (i & 1) ? kv8_whole(w.z, w.w) : kv8_whole(w.x, w.y);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qb[i], s[t], 0, 0, 0);
            }
        }
        const float scaled = fac * ks;
        issue(b + kWaves, 0, kq, ks);
        kv8_half8 pb;
        soften(s, scaled, b, pb);
        const _Float16 value_scale = (_Float16)vs;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const kv8_u4 w = vq[d >> 1];
            const kv8_half8 v = (d & 1) ? kv8_values(w.z, w.w, value_scale) : kv8_values(w.x, w.y, value_scale);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb, o[d], 0, 0, 0);
        }
        issue(b + kWaves, kKv8PartBytes, vq, vs);
    }

    // ---- the waves' states meet in LDS: the chunk's partial in attn_decode_kernel's
    // layout, or the output where a launch has one chunk
    lrun += __shfl_xor(lrun, 16, 64);
    lrun += __shfl_xor(lrun, 32, 64);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = o[d][i] + other_half(o[d][i]);
            if (n < QPK) st_o[wave][n][32 * (d >> 1) + 2 * (4 * g + i) + (d & 1)] = v;
        }
    }
    if (g == 0 && n < QPK) st_ml[wave][n] = make_float2(mrun, lrun);
    __syncthreads();
    float* const own = a.partials != nullptr ? a.partials + (size_t)m * a.partial_floats : mb.partials;
    for (int i = tid; i < QPK * kHeadDim; i += kThreads) {
        const int h = i >> 7, d = i & 127;
        float mx = -FLT_MAX;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, st_ml[w][h].x);
        float l = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(st_ml[w][h].x - mx);
            l = __builtin_fmaf(st_ml[w][h].y, f, l);
            acc = __builtin_fmaf(st_o[w][h][d], f, acc);
        }
        if (a.chunks == 1) {
            a.out[((size_t)m * a.q_heads + (size_t)kvh * QPK) * kHeadDim + i] = acc / l;
            continue;
        }
        float* part = own + ((size_t)(kvh * QPK + h) * kAttnChunks + chunk) * kPartStride;
        part[d] = acc;
        if (d == 0) {
            part[kHeadDim] = mx;
            part[kHeadDim + 1] = l;
        }
    }
}

// The chunks' partials of a (query head, member) merged; every slot the launch can
// hold is loaded before the position says which are live (the others hold stale
// memory). A member without tokens (a negative position) gets zeros.
template <int NC, bool INLINE>
__global__ __launch_bounds__(128) void kv8_combine_kernel(AttnArgs a, Members<INLINE> members) {
    const int qh = blockIdx.x;
    const int m = blockIdx.y;
    const AttnMember mb = members.get(a, m);
    const float* own = a.partials != nullptr ? a.partials + (size_t)m * a.partial_floats : mb.partials;
    auto live = [&] {
        int end;
        const int tokens = kv8_tokens(a, mb, kv8_head(mb, a.layer, qh / (a.q_heads / a.kv_heads)), a.positions[m], end);
        const int len = kv8_chunk_tokens(tokens, a.chunks, a.min_chunk);
        return tokens > 0 ? (tokens + len - 1) / len : 0;
    };
    merge_row<NC>(own + (size_t)qh * kAttnChunks * kPartStride, a.chunks, live, a.out + ((size_t)m * a.q_heads + qh) * kHeadDim);
}

}  // namespace

int kv8_grid_chunks(int max_capacity, int members) {
    const int min_chunk = kv8_min_chunk(members);
    return std::max(1, std::min(kAttnChunks, (max_capacity + min_chunk - 1) / min_chunk));
}

hipError_t launch_cache_init(void* regions, size_t count, int capacity, const double* table, double* table_dst,
                             hipStream_t stream) {
    CacheInit a;
    std::copy(table, table + kHeadDim / 2 + 1, a.table);
    a.table_dst = table_dst;
    a.regions = static_cast<char*>(regions);
    a.stride = kv8_head_bytes(capacity);
    a.codes = kv8_tail_offset(capacity);
    hipLaunchKernelGGL(cache_init_kernel, dim3(regions != nullptr ? (unsigned)count : 1u), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_kv8_append(const AttnArgs& a, int members, hipStream_t stream) {
    if (members < 1 || members > kAttnMaxMembers || a.kv_heads < 1 || a.mem == nullptr) return hipErrorInvalidValue;
    // consecutive positions touch at most one block more than they fill
    const int blocks = (members + kKv8Block - 2) / kKv8Block + 1;
    hipLaunchKernelGGL(kv8_append_kernel, dim3((unsigned)a.kv_heads, (unsigned)blocks), dim3(blocks > 1 ? 2 * kAppendThreads : kAppendThreads), 0,
                       stream, a, members);
    return hipGetLastError();
}

hipError_t launch_kv8_append_seq(const PrefillAttnArgs& a, hipStream_t stream) {
    if (a.tokens < 1 || a.kv_heads < 1 || a.p0 < 0 || (long long)a.p0 + a.tokens > a.mem.capacity) return hipErrorInvalidValue;
    const int blocks = (a.p0 + a.tokens - 1) / kKv8Block - a.p0 / kKv8Block + 1;
    hipLaunchKernelGGL(kv8_append_seq_kernel, dim3((unsigned)a.kv_heads, (unsigned)blocks), dim3(append_threads(a.p0, a.tokens)), 0, stream, a);
    return hipGetLastError();
}

namespace {
template <bool INLINE>
hipError_t launch_members(const AttnArgs& b, const Members<INLINE>& mem, int members, hipStream_t stream) {
    const dim3 grid((unsigned)b.chunks, (unsigned)b.kv_heads, (unsigned)members);
    switch (b.q_heads / b.kv_heads) {
    case 1: hipLaunchKernelGGL((kv8_attn_kernel<1, INLINE>), grid, dim3(kThreads), 0, stream, b, mem); break;
    case 2: hipLaunchKernelGGL((kv8_attn_kernel<2, INLINE>), grid, dim3(kThreads), 0, stream, b, mem); break;
    case 4: hipLaunchKernelGGL((kv8_attn_kernel<4, INLINE>), grid, dim3(kThreads), 0, stream, b, mem); break;
    case 8: hipLaunchKernelGGL((kv8_attn_kernel<8, INLINE>), grid, dim3(kThreads), 0, stream, b, mem); break;
    default: return hipErrorInvalidValue;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || b.chunks == 1) return e;
    const dim3 rows((unsigned)b.q_heads, (unsigned)members);
    static_assert(kAttnChunks == 32, "the merge's forms cover the grid's chunks");
    if (b.chunks <= 8) hipLaunchKernelGGL((kv8_combine_kernel<8, INLINE>), rows, dim3(128), 0, stream, b, mem);
    else hipLaunchKernelGGL((kv8_combine_kernel<32, INLINE>), rows, dim3(128), 0, stream, b, mem);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_kv8_attention(const AttnArgs& args, const AttnMember* host_mem, int members, hipStream_t stream) {
    if (members < 1 || members > kAttnMaxMembers || args.kv_heads < 1 || args.q_heads % args.kv_heads != 0 ||
        args.chunks < 1 || args.chunks > kAttnChunks || (args.mem == nullptr && (host_mem == nullptr || args.appended))) {
        return hipErrorInvalidValue;
    }
    AttnArgs b = args;
    b.min_chunk = kv8_min_chunk(members);
    if (host_mem == nullptr) return launch_members<false>(b, Members<false>{}, members, stream);
    Members<true> mem;
    std::copy(host_mem, host_mem + members, mem.mem);
    return launch_members<true>(b, mem, members, stream);
}

namespace {
bool move_fits(const KvMoveArgs& a) {
    return a.tokens >= 1 && a.kv_heads >= 1 && a.p0 >= 0 && (long long)a.p0 + a.tokens <= a.mem.capacity && a.mem.keys != nullptr;
}
dim3 move_grid(const KvMoveArgs& a, bool kv8) {
    if (!kv8) return dim3((unsigned)(a.tokens + 15) / 16, (unsigned)a.kv_heads);
    return dim3((unsigned)a.kv_heads, (unsigned)((a.p0 + a.tokens - 1) / kKv8Block - a.p0 / kKv8Block + 1));
}
}  // namespace

hipError_t launch_kv_write(const KvMoveArgs& a, bool half, bool kv8, hipStream_t stream) {
    if (!move_fits(a)) return hipErrorInvalidValue;
    const dim3 grid = move_grid(a, kv8);
    if (kv8 && half) hipLaunchKernelGGL(kv8_write_kernel<kRowsF16>, grid, dim3(append_threads(a.p0, a.tokens)), 0, stream, a);
    else if (kv8) hipLaunchKernelGGL(kv8_write_kernel<kRowsF32>, grid, dim3(append_threads(a.p0, a.tokens)), 0, stream, a);
    else if (half) hipLaunchKernelGGL(kv16_write_kernel<_Float16>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(kv16_write_kernel<float>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvMoveArgs& a, bool half, bool kv8, hipStream_t stream) {
    if (!move_fits(a)) return hipErrorInvalidValue;
    const dim3 grid = move_grid(a, kv8);
    if (kv8 && half) hipLaunchKernelGGL(kv8_read_kernel<_Float16>, grid, dim3(kAppendThreads), 0, stream, a);
    else if (kv8) hipLaunchKernelGGL(kv8_read_kernel<float>, grid, dim3(kAppendThreads), 0, stream, a);
    else if (half) hipLaunchKernelGGL(kv16_read_kernel<_Float16>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(kv16_read_kernel<float>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ribn_amd

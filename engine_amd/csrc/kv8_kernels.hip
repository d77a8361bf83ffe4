// Kernels of the 8-bit KV cache for gfx950 (kv8.hpp has the layout and the
// arithmetic of a code, kvq_device.hpp what other formats share): the append of new tokens, decode attention over the
// cache, and rows moved in and out of it.
#include "kv8.hpp"

#include <algorithm>

#include "kvq_device.hpp"

namespace ribn_amd {

namespace {

struct Kv8Format {
    static constexpr bool kFused = false;
    static constexpr bool kTableFirst = false;
    static constexpr int kKeyRegs = 8, kValueRegs = 8;  // (codes take the first four)
    static constexpr int kQuantiseBarriers = 1;
    struct Scratch {
        float amax[8];
    };

    __device__ __forceinline__ static KvHead head(const AttnMember& m, int layer, int kvh) { return kv8_head(m, layer, kvh); }

    // Rows 0 .. count - 1 of block b.
    __device__ __forceinline__ static void stage_codes(StageRows& st, const KvHead& h, int b, int count) {
        const int tid = append_tid();
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
    __device__ __forceinline__ static void quantise(Stage<Kv8Format>& st, const KvHead& h, int b) {
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
        if (lane == 0) st.x.amax[wave] = wave_top;
        __syncthreads();
        const float* parts = st.x.amax + (wave & 4);
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

    // A block's codes, four 16-byte loads a lane of keys and of values, and their scales.
    struct Source {
        __amdgpu_buffer_rsrc_t cr, sr;
        __device__ __forceinline__ Source(const KvHead& h, int capacity)
            : cr(make_rsrc(h.codes, (uint32_t)kv8_tail_offset(capacity))),
              sr(make_rsrc(h.scales, (uint32_t)(kv8_blocks(capacity) * sizeof(float2)))) {}
        __device__ __forceinline__ void part(int b, int end, int part, int lane, kv8_u4 (&w)[8], float& scale) const {
            const uint32_t at = b < end ? (uint32_t)b * kKv8BlockBytes + (uint32_t)part + 16u * (uint32_t)lane : kCacheOOR;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(kv8_u4, load_b128(cr, at + 1024u * i));
            scale = __builtin_bit_cast(float, load_b32(sr, b < end ? 8u * (uint32_t)b + (part ? 4u : 0u) : kCacheOOR));
        }
        __device__ __forceinline__ void keys(int b, int end, int lane, kv8_u4 (&w)[8], float& scale) const { part(b, end, 0, lane, w, scale); }
        __device__ __forceinline__ void values(int b, int end, int lane, kv8_u4 (&w)[8], float& scale) const {
            part(b, end, kKv8PartBytes, lane, w, scale);
        }
    };

    struct Constants {};
    static constexpr bool kSharedQuantise = false;
    struct Parked {};
    struct WaveScratch {};
    __device__ __forceinline__ static void begin(const kv8_u4 (&)[8], WaveScratch&, int) {}
    // Codes enter the scores as whole numbers, the block's key scale being applied to
    // the f32 score; values are scaled as f16 (both exact).
    __device__ __forceinline__ static void scores(const kv8_u4 (&kq)[8], const WaveScratch&, const Constants&, int, const kv8_half8 (&qb)[4], kv8_float4 (&s)[2]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const kv8_u4 w = kq[2 * t + (i >> 1)];
                const kv8_half8 k = (i & 1) ? kv8_whole(w.z, w.w) : kv8_whole(w.x, w.y);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qb[i], s[t], 0, 0, 0);
            }
        }
    }
    __device__ __forceinline__ static float scaled(float fac, float scale) { return fac * scale; }
    __device__ __forceinline__ static void outputs(const kv8_u4 (&vq)[8], float scale, const WaveScratch&, const Constants&, int, kv8_half8 pb, kv8_float4 (&o)[8]) {
        const _Float16 value_scale = (_Float16)scale;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const kv8_u4 w = vq[d >> 1];
            const kv8_half8 v = (d & 1) ? kv8_values(w.z, w.w, value_scale) : kv8_values(w.x, w.y, value_scale);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb, o[d], 0, 0, 0);
        }
    }

    // The block in the tail's registers (TailBlock).

    __device__ __forceinline__ static void expand(kv8_u4 w, float scale, kv8_u4& x, kv8_u4& y) {
        x = __builtin_bit_cast(kv8_u4, kv8_values(w.x, w.y, (_Float16)scale));
        y = __builtin_bit_cast(kv8_u4, kv8_values(w.z, w.w, (_Float16)scale));
    }
    // What the codes of block b stand for.
    __device__ __forceinline__ static void load_tail(const KvHead& h, int b, int lane, kv8_u4 (&k)[8], kv8_u4 (&v)[8]) {
        const kv8_u4* c = reinterpret_cast<const kv8_u4*>(h.codes + (size_t)b * kKv8BlockBytes) + lane;
        const float2 sc = h.scales[b];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            expand(c[64 * i], sc.x, k[2 * i], k[2 * i + 1]);
            expand(c[64 * (4 + i)], sc.y, v[2 * i], v[2 * i + 1]);
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
    __device__ __forceinline__ static void quantise_tail(const KvHead& h, int b, int lane, kv8_u4 (&k)[8], kv8_u4 (&v)[8]) {
        kv8_u4* c = reinterpret_cast<kv8_u4*>(h.codes + (size_t)b * kKv8BlockBytes) + lane;
        float2 sc;
        quantise_part(k, c, sc.x);
        quantise_part(v, c + 256, sc.y);
        if (lane == 0) h.scales[b] = sc;
    }
};

// Traffic of an append is the rows in
// and a byte a value out: 32,768 f16 rows of 8 heads (134 MB in, 67 out) take 48 us, 4.2 TB/s.
// Short appends are the latency of one row's chain (load, sum of squares, angles, LDS,
// maximum, codes): 37 prompt tokens 7.0 us, 2,047 (17 MB in, 4 out) 8.8.
__global__ __launch_bounds__(2 * kAppendThreads) void kv8_append_kernel(AttnArgs a, int members) { append_members<Kv8Format>(a, members); }
__global__ __launch_bounds__(2 * kAppendThreads) void kv8_append_seq_kernel(PrefillAttnArgs a) { append_chunk<Kv8Format>(a); }
template <int ROWS>
__global__ __launch_bounds__(2 * kAppendThreads) void kv8_write_kernel(KvMoveArgs a) { write_rows<Kv8Format, ROWS>(a); }
// 32,768 rows of 8 heads (67 MB in, 134 out) in 30.6 us, 6.6 TB/s (the codes had just been written).
template <typename T>
__global__ __launch_bounds__(kAppendThreads, 4) void kv8_read_kernel(KvMoveArgs a) { read_rows<Kv8Format, T>(a); }

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
    size_t codes;   // its first bytes, left as they are
};

// Grid (region, slice of it).
__global__ __launch_bounds__(256) void cache_init_kernel(CacheInit a) {
    const int tid = threadIdx.x;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid <= kHeadDim / 2) a.table_dst[tid] = a.table[tid];
    if (a.regions == nullptr) return;
    uint4* p = reinterpret_cast<uint4*>(a.regions + (size_t)blockIdx.x * a.stride + a.codes);
    for (size_t i = (size_t)blockIdx.y * 256 + tid; i < (a.stride - a.codes) / sizeof(uint4); i += 256 * (size_t)gridDim.y) p[i] = make_uint4(0, 0, 0, 0);
}

// Decode attention (kvq_device.hpp). Memory bounds the long cases
// (131,071 tokens, 269 MB: 49.5 us, 5.4 TB/s), latency the short ones: 5.6 us pass
// between a launch and its output however little it reads (40 tokens), and 8 members of 3,000
// (36 MB) take 11, 24 of 1,501 with 64 heads (58 MB) 16, their merge 2 to 3 more.
//
// One block in flight a wave. (Two blocks: 8 members of 3,000 16.1 us for 13.9, 24 of 1,501
// 20.4 for 19.3, 131,071 tokens 52.8 for 52.1; with two KV heads, where a wave has its SIMD to itself, 30.2 for 31.4.)
//
// Handing partials over between XCDs, so that the last workgroup of a row merges them: with write-through
// stores and loads 8 members of 3,000 took 14.4 us for 13.9, 131,071 tokens 55.0
// for 52.3, 8 members of 15,000 53 for 40 (with fences, which write back an XCD's whole L2, 70, 74 and 387).
template <int QPK, bool INLINE>
__global__ __launch_bounds__(kAttnThreads, 3) void kv8_attn_kernel(AttnArgs a, Members<INLINE> members) {
    cache_attention<Kv8Format, QPK, INLINE>(a, members);
}
template <int NC, bool INLINE>
__global__ __launch_bounds__(128) void kv8_combine_kernel(AttnArgs a, Members<INLINE> members) {
    combine_chunks<Kv8Format, NC, INLINE>(a, members);
}
template <bool INLINE>
constexpr AttnKernels<INLINE> kKernels{{kv8_attn_kernel<1, INLINE>, kv8_attn_kernel<2, INLINE>, kv8_attn_kernel<4, INLINE>, kv8_attn_kernel<8, INLINE>},
                                       {kv8_combine_kernel<8, INLINE>, kv8_combine_kernel<32, INLINE>}};

}  // namespace

int kv8_grid_chunks(int max_capacity, int members) {
    const int min_chunk = cache_min_chunk(members);
    return std::max(1, std::min(kAttnChunks, (max_capacity + min_chunk - 1) / min_chunk));
}

hipError_t launch_cache_init(void* regions, size_t count, size_t stride, size_t codes, const double* table, double* table_dst,
                             hipStream_t stream) {
    CacheInit a;
    std::copy(table, table + kHeadDim / 2 + 1, a.table);
    a.table_dst = table_dst;
    a.regions = static_cast<char*>(regions);
    a.stride = stride;
    a.codes = codes;
    const unsigned slices = (unsigned)std::min<size_t>(64, (stride - codes) / 65536 + 1);  // of 64 KB or more
    hipLaunchKernelGGL(cache_init_kernel, regions != nullptr ? dim3((unsigned)count, slices) : dim3(1), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_kv8_append(const AttnArgs& a, int members, hipStream_t stream) { return launch_append(kv8_append_kernel, a, members, stream); }
hipError_t launch_kv8_append_seq(const PrefillAttnArgs& a, hipStream_t stream) { return launch_append_chunk(kv8_append_seq_kernel, a, stream); }
hipError_t launch_kv8_attention(const AttnArgs& a, const AttnMember* host_mem, int members, hipStream_t stream) {
    return launch_cache_attention(kKernels<true>, kKernels<false>, a, host_mem, members, stream);
}

hipError_t launch_kv_write(const KvMoveArgs& a, bool half, bool kv8, hipStream_t stream) {
    if (!move_fits(a)) return hipErrorInvalidValue;
    if (kv8) return launch_move(half ? kv8_write_kernel<kRowsF16> : kv8_write_kernel<kRowsF32>, a, append_threads(a.p0, a.tokens), stream);
    const dim3 grid((unsigned)(a.tokens + 15) / 16, (unsigned)a.kv_heads);
    if (half) hipLaunchKernelGGL(kv16_write_kernel<_Float16>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(kv16_write_kernel<float>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvMoveArgs& a, bool half, bool kv8, hipStream_t stream) {
    if (!move_fits(a)) return hipErrorInvalidValue;
    if (kv8) return launch_move(half ? kv8_read_kernel<_Float16> : kv8_read_kernel<float>, a, kAppendThreads, stream);
    const dim3 grid((unsigned)(a.tokens + 15) / 16, (unsigned)a.kv_heads);
    if (half) hipLaunchKernelGGL(kv16_read_kernel<_Float16>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(kv16_read_kernel<float>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ribn_amd

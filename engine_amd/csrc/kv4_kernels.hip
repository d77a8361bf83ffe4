// Kernels of the 4-bit KV cache for gfx950 (kv4.hpp has the layout and the arithmetic of a
// code, kvq_device.hpp what other formats share): the append of new tokens, decode attention over the
// cache, and rows moved in and out of it.
#include "kv4.hpp"

#include "kv4_device.hpp"
#include "kvq_device.hpp"

namespace ribn_amd {

namespace {

struct Kv4Format {
    // Registers of a block: of its keys two of codes, and the block's scales and lows as they lie, 16 bytes a
    // lane; of its values two of codes (and the tail all of them).
    static constexpr int kKeyRegs = 8, kValueRegs = 8;
    static constexpr bool kFused = true;
    static constexpr bool kTableFirst = true;
    static constexpr int kQuantiseBarriers = 2;
    struct Scratch {
        kv8_half2 key_lo[4][64], key_hi[4][64];  // of eight rows each; [0] then of all: low, and
        float2 key_inv[64];
        _Float16 value_lo[2][kKv8Block];
        float value_inv[2][kKv8Block];
    };

    __device__ __forceinline__ static KvHead head(const AttnMember& m, int layer, int kvh) { return kv4_head(m, layer, kvh); }

    // Rows 0 .. count - 1 of block b: eight bytes a thread, 16 dims of a key or two of eight values.
    __device__ __forceinline__ static void stage_codes(StageRows& st, const KvHead& h, int b, int count) {
        const int tid = append_tid(), lane = tid & 63, u = (tid >> 6) & 3, g = lane >> 4, m = lane & 15;
        const uint8_t* block = h.codes + (size_t)b * kKv4BlockBytes;
        const int at = 1024 * (u >> 1) + 16 * lane + 8 * (u & 1);
        const Kv4Bias bias;
        if (tid < 256) {
            const uint2 w = *reinterpret_cast<const uint2*>(block + at);
            const int row = kv8_key_row(u >> 1, m), dim = 64 * (u & 1) + 16 * g;
            const kv4_u4* p = reinterpret_cast<const kv4_u4*>(block + kKv4Params + 2 * dim);
            const kv8_half8 x0 = kv4_values(w.x, p[0], p[16], bias), x1 = kv4_values(w.y, p[1], p[17], bias);
            if (row < count) {
                kv8_half8* k = reinterpret_cast<kv8_half8*>(&st.k[row][dim]);
                k[0] = x0;
                k[1] = x1;
            }
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(block + kKv4Values + at);
            const kv4_u4* p = reinterpret_cast<const kv4_u4*>(block + kKv4Params + kKv4ValueParams + (u >> 1) * kKv4ValueHalf + 16 * g);
            const kv8_half8 x0 = kv4_values(w.x, p[0], p[4], bias), x1 = kv4_values(w.y, p[0], p[4], bias);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * g + j < count) *reinterpret_cast<kv8_half2*>(&st.v[8 * g + j][32 * u + 2 * m]) = kv8_half2{x0[j], x1[j]};
        }
    }

    // The staged block's 32 rows into codes, scales and lows.
    __device__ __forceinline__ static void quantise(Stage<Kv4Format>& st, const KvHead& h, int b) {
        const int tid = append_tid(), lane = tid & 63, u = (tid >> 6) & 3, g = lane >> 4, m = lane & 15;
        const bool keys = tid < 256;
        uint8_t* const block = h.codes + (size_t)b * kKv4BlockBytes;
        if (keys) {  // a pair of dims over eight rows
            kv8_half2 lo = *reinterpret_cast<const kv8_half2*>(&st.k[8 * u][2 * lane]), hi = lo;
#pragma unroll
            for (int r = 1; r < 8; ++r) {
                const kv8_half2 x = *reinterpret_cast<const kv8_half2*>(&st.k[8 * u + r][2 * lane]);
                lo = kv4_min(lo, x);
                hi = __builtin_elementwise_max(hi, x);
            }
            st.x.key_lo[u][lane] = lo;
            st.x.key_hi[u][lane] = hi;
        } else {  // 16 dims of a token, four lanes a group
            const int token = 8 * u + (lane >> 3), half = (lane >> 2) & 1;
            const kv8_half2* row = reinterpret_cast<const kv8_half2*>(&st.v[token][16 * (lane & 7)]);
            kv8_half2 lo = row[0], hi = lo;
#pragma unroll
            for (int j = 1; j < 8; ++j) {
                lo = kv4_min(lo, row[j]);
                hi = __builtin_elementwise_max(hi, row[j]);
            }
            // (the largest as the smallest of its negative, in one reduction)
            const kv8_half2 both = kv4_quad_min(kv8_half2{kv4_min(lo, kv8_half2{lo[1], lo[1]})[0], -__builtin_elementwise_max(hi, kv8_half2{hi[1], hi[1]})[0]});
            if ((lane & 3) == 0) {
                const Kv4Scale s(both[0], -both[1]);
                st.x.value_lo[half][token] = both[0];
                st.x.value_inv[half][token] = s.inv;
                _Float16* p = reinterpret_cast<_Float16*>(block + kKv4Params + kKv4ValueParams + half * kKv4ValueHalf);
                p[token] = s.s;
                p[kKv8Block + token] = both[0];
            }
        }
        __syncthreads();
        if (tid < 64) {
            kv8_half2 lo = st.x.key_lo[0][lane], hi = st.x.key_hi[0][lane];
#pragma unroll
            for (int r = 1; r < 4; ++r) {
                lo = kv4_min(lo, st.x.key_lo[r][lane]);
                hi = __builtin_elementwise_max(hi, st.x.key_hi[r][lane]);
            }
            const Kv4Scale a(lo[0], hi[0]), c(lo[1], hi[1]);
            st.x.key_lo[0][lane] = lo;
            st.x.key_inv[lane] = make_float2(a.inv, c.inv);
            kv8_half2* p = reinterpret_cast<kv8_half2*>(block + kKv4Params);
            p[lane] = kv8_half2{a.s, c.s};
            p[64 + lane] = lo;
        }
        __syncthreads();
        uint32_t w[2] = {0, 0};
        if (keys) {
            const int dim = 64 * (u & 1) + 16 * g;
            const _Float16* row = &st.k[kv8_key_row(u >> 1, m)][dim];
            const _Float16* lo = reinterpret_cast<const _Float16*>(st.x.key_lo[0]) + dim;
            const float* inv = reinterpret_cast<const float*>(st.x.key_inv) + dim;
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j >> 3] |= kv4_code(row[j], lo[j], inv[j]) << kv4_shift(j & 7);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = 8 * g + j;
                const kv8_half2 x = *reinterpret_cast<const kv8_half2*>(&st.v[key][32 * u + 2 * m]);
                const _Float16 lo = st.x.value_lo[u >> 1][key];
                const float inv = st.x.value_inv[u >> 1][key];
                w[0] |= kv4_code(x[0], lo, inv) << kv4_shift(j);
                w[1] |= kv4_code(x[1], lo, inv) << kv4_shift(j);
            }
        }
        *reinterpret_cast<uint2*>(block + (keys ? 0 : kKv4Values) + 1024 * (u >> 1) + 16 * lane + 8 * (u & 1)) = make_uint2(w[0], w[1]);
    }

    // A block's scales and lows, put here by the wave that holds the block: as operands they are 16 bytes each
    // that 16 lanes share, 48 registers a lane if they were loaded so.
    using Constants = Kv4Bias;
    struct WaveScratch {
        kv8_u4 params[64];
    };

    // A block's codes, two 16-byte loads a lane of keys and of values, and its scales and lows.
    struct Source {
        __amdgpu_buffer_rsrc_t r;
        __device__ __forceinline__ Source(const KvHead& h, int capacity) : r(make_rsrc(h.codes, (uint32_t)kv4_tail_offset(capacity))) {}
        __device__ __forceinline__ kv8_u4 load(uint32_t at) const { return __builtin_bit_cast(kv8_u4, load_b128(r, at)); }
        __device__ __forceinline__ void keys(int b, int end, int lane, kv8_u4 (&w)[kKeyRegs], float&) const {
            const uint32_t base = b < end ? (uint32_t)b * kKv4BlockBytes : kCacheOOR;
            w[2] = load(lane < kKv4ParamBytes / 16 ? base + kKv4Params + 16u * (uint32_t)lane : kCacheOOR);
#pragma unroll
            for (int t = 0; t < 2; ++t) w[t] = load(base + 1024u * t + 16u * (uint32_t)lane);
        }
        __device__ __forceinline__ void values(int b, int end, int lane, kv8_u4 (&w)[kValueRegs], float&) const {
            const uint32_t base = b < end ? (uint32_t)b * kKv4BlockBytes : kCacheOOR;
#pragma unroll
            for (int h = 0; h < 2; ++h) w[h] = load(base + kKv4Values + 1024u * h + 16u * (uint32_t)lane);
        }
    };

    // (a wave's LDS accesses come in its order: the block before has read its own)
    __device__ __forceinline__ static void begin(const kv8_u4 (&kq)[kKeyRegs], WaveScratch& ws, int lane) {
        lds_order();
        ws.params[lane] = kq[2];
        lds_order();
    }
    __device__ __forceinline__ static void scores(const kv8_u4 (&kq)[kKeyRegs], const WaveScratch& ws, const Kv4Bias& bias, int g, const kv8_half8 (&qb)[4], kv8_float4 (&s)[2]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // step i: dims 64 (i >> 1) + 16 g + 8 (i & 1)
            const kv8_u4 scale = ws.params[8 * (i >> 1) + 2 * g + (i & 1)], low = ws.params[16 + 8 * (i >> 1) + 2 * g + (i & 1)];
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv4_values(kq[t][i], scale, low, bias), qb[i], s[t], 0, 0, 0);
        }
    }
    __device__ __forceinline__ static float scaled(float fac, float) { return fac; }
    __device__ __forceinline__ static void outputs(const kv8_u4 (&vq)[kValueRegs], float, const WaveScratch& ws, const Kv4Bias& bias, int g, kv8_half8 pb, kv8_float4 (&o)[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const kv8_u4 scale = ws.params[32 + 8 * h + g], low = ws.params[36 + 8 * h + g];
#pragma unroll
            for (int d = 0; d < 4; ++d) o[4 * h + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv4_values(vq[h][d], scale, low, bias), pb, o[4 * h + d], 0, 0, 0);
        }
    }

    // The block in the tail's registers (TailBlock): what the codes of block b stand for.
    __device__ __forceinline__ static void load_tail(const KvHead& h, int b, int lane, kv8_u4 (&k)[kKeyRegs], kv8_u4 (&v)[kValueRegs]) {
        const Kv4Bias bias;
        const uint8_t* block = h.codes + (size_t)b * kKv4BlockBytes;
        const kv8_u4* kp = reinterpret_cast<const kv8_u4*>(block + kKv4Params) + 2 * (lane >> 4);
        const kv8_u4* vp = reinterpret_cast<const kv8_u4*>(block + kKv4Params + kKv4ValueParams) + (lane >> 4);
        const kv8_u4* kc = reinterpret_cast<const kv8_u4*>(block) + lane;
        const kv8_u4* vc = reinterpret_cast<const kv8_u4*>(block + kKv4Values) + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int s = i & 3;  // key step 4 t + s: dims 64 (s >> 1) + 16 g + 8 (s & 1)
            k[i] = __builtin_bit_cast(kv8_u4, kv4_values(kc[64 * (i >> 2)][s], kp[8 * (s >> 1) + (s & 1)], kp[16 + 8 * (s >> 1) + (s & 1)], bias));
            v[i] = __builtin_bit_cast(kv8_u4, kv4_values(vc[64 * (i >> 2)][s], vp[8 * (i >> 2)], vp[8 * (i >> 2) + 4], bias));
        }
    }

    // Codes, scales and lows of the whole block; its values become what these stand for. By way of LDS, where each
    // wave takes a share: a step in 32 comes here, one of a batch's nearly always. One wave took 6.7 us for it, four take
    // 2.1 (a whole call of one member 12.4 and 7.6 us; unrolled over the registers that hold the block it set the kernel's count).
    static constexpr bool kSharedQuantise = true;
    struct Parked {
        kv8_u4 x[8][64];
    };
    __device__ __forceinline__ static void park(Parked (&parked)[2], int lane, const kv8_u4 (&k)[kKeyRegs], const kv8_u4 (&v)[kValueRegs]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            parked[0].x[i][lane] = k[i];
            parked[1].x[i][lane] = v[i];
        }
    }
    __device__ __forceinline__ static void unpark(const Parked (&parked)[2], int lane, kv8_u4 (&k)[kKeyRegs], kv8_u4 (&v)[kValueRegs]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k[i] = parked[0].x[i][lane];
            v[i] = parked[1].x[i][lane];
        }
    }
    __device__ __forceinline__ static void quantise_share(const KvHead& h, int b, int wave, int lane, Parked (&parked)[2]) {
        const Kv4Bias bias;
        uint8_t* const block = h.codes + (size_t)b * kKv4BlockBytes;
        if (wave < 2) quantise_keys(block, 2 * wave, lane, parked[0], bias);
        else quantise_values(block, wave - 2, lane, parked[1], bias);
    }
    __device__ __forceinline__ static kv8_half2 pair(uint32_t w) { return __builtin_bit_cast(kv8_half2, w); }
    __device__ __forceinline__ static uint32_t word(kv8_half2 x) { return __builtin_bit_cast(uint32_t, x); }
    // Steps `step` and the next one of the keys.
    __device__ __forceinline__ static void quantise_keys(uint8_t* block, int step, int lane, Parked& parked, const Kv4Bias& bias) {
        kv8_u4* const kp = reinterpret_cast<kv8_u4*>(block + kKv4Params) + 2 * (lane >> 4);
#pragma unroll 1
        for (int s = step; s < step + 2; ++s) {  // eight dims, of the two tiles
            const kv8_u4 x0 = parked.x[s][lane], x1 = parked.x[4 + s][lane];
            kv8_u4 scale, low;
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // a pair of dims, over the two tiles and the row's 16 keys
                const uint32_t a0 = x0[j], a1 = x1[j];
                const kv8_half2 lo = kv4_row_min(kv4_min(pair(a0), pair(a1))), hi = -kv4_row_min(kv4_min(-pair(a0), -pair(a1)));
                const Kv4Scale a(lo[0], hi[0]), c(lo[1], hi[1]);
                scale[j] = word(kv8_half2{a.s, c.s});
                low[j] = word(lo);
                w[0] |= kv4_code(pair(a0)[0], lo[0], a.inv) << kv4_shift(2 * j) | kv4_code(pair(a0)[1], lo[1], c.inv) << kv4_shift(2 * j + 1);
                w[1] |= kv4_code(pair(a1)[0], lo[0], a.inv) << kv4_shift(2 * j) | kv4_code(pair(a1)[1], lo[1], c.inv) << kv4_shift(2 * j + 1);
            }
            if ((lane & 15) == 0) {
                kp[8 * (s >> 1) + (s & 1)] = scale;
                kp[16 + 8 * (s >> 1) + (s & 1)] = low;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                reinterpret_cast<uint32_t*>(block)[256 * t + 4 * lane + s] = w[t];
                parked.x[4 * t + s][lane] = __builtin_bit_cast(kv8_u4, kv4_values(w[t], scale, low, bias));
            }
        }
    }
    // Half `half` of the values.
    __device__ __forceinline__ static void quantise_values(uint8_t* block, int half, int lane, Parked& parked, const Kv4Bias& bias) {
        kv8_u4 x[4], scale, low, w = kv8_u4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < 4; ++d) x[d] = parked.x[4 * half + d][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // a pair of keys, over four dims and the row's 16 lanes
            kv8_half2 lo, hi;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t a = x[d][j];
                lo = d == 0 ? pair(a) : kv4_min(lo, pair(a));
                hi = d == 0 ? -pair(a) : kv4_min(hi, -pair(a));
            }
            lo = kv4_row_min(lo);
            hi = -kv4_row_min(hi);
            const Kv4Scale a(lo[0], hi[0]), c(lo[1], hi[1]);
            scale[j] = word(kv8_half2{a.s, c.s});
            low[j] = word(lo);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t y = x[d][j];
                w[d] |= kv4_code(pair(y)[0], lo[0], a.inv) << kv4_shift(2 * j) | kv4_code(pair(y)[1], lo[1], c.inv) << kv4_shift(2 * j + 1);
            }
        }
        if ((lane & 15) == 0) {
            kv8_u4* const p = reinterpret_cast<kv8_u4*>(block + kKv4Params + kKv4ValueParams) + (lane >> 4) + 8 * half;
            p[0] = scale;
            p[4] = low;
        }
        reinterpret_cast<kv8_u4*>(block + kKv4Values)[64 * half + lane] = w;
#pragma unroll
        for (int d = 0; d < 4; ++d) parked.x[4 * half + d][lane] = __builtin_bit_cast(kv8_u4, kv4_values(w[d], scale, low, bias));
    }
};

// Appends and writes: 8 KB of rows in LDS a block and part, three passes with a barrier between (smallest and largest,
// scales, codes). 32,768 f16 rows of 8 heads (134 MB in, 39 out) take 42 us, 4.1 TB/s: round trips of the passes at four workgroups a CU (a
// fifth less instructions changed nothing). A prompt's keys are formed in 64 bits first: 29 tokens 5.5 us, 2,047 (17 MB in, 2.4
// out) 8.9, latency both.
__global__ __launch_bounds__(2 * kAppendThreads) void kv4_append_kernel(AttnArgs a, int members) { append_members<Kv4Format>(a, members); }
__global__ __launch_bounds__(2 * kAppendThreads) void kv4_append_seq_kernel(PrefillAttnArgs a) { append_chunk<Kv4Format>(a); }
template <int ROWS>
__global__ __launch_bounds__(2 * kAppendThreads) void kv4_write_kernel(KvMoveArgs a) { write_rows<Kv4Format, ROWS>(a); }
// 32,768 rows (39 MB in, 134 out) in 27 us, 6.4 TB/s (the codes had just been written).
template <typename T>
__global__ __launch_bounds__(kAppendThreads, 4) void kv4_read_kernel(KvMoveArgs a) { read_rows<Kv4Format, T>(a); }

// Decode attention (kvq_device.hpp). Memory bounds the long contexts (131,071 tokens, 159 MB: 35 us, 4.6 TB/s, at one wave a
// SIMD, whose VALU is busy half of that; 30 would be a copy's), round trips and ramp the short ones: 5.4 us pass with
// one block. With 8 members of 4,001 tokens (27 MB) the codes come in about 3 of 12 us; norms, angles and the first loads take 2,
// the waves' meeting 1, the launch and its ramp the rest.
// A block costs some 200 instructions a wave: its codes by the two patterns of kv4_values 13 for eight, the softmax as for 8 bits. What
// has been tried: a lane's own scales and lows as 16-byte loads (12 a block, 48 registers) took 52 us of the 39 of one member
// of 131,071; two blocks in flight a wave 43.0 of 42.9 then; eight waves a workgroup 40.7, but 28 of 17.9 with 8
// members of 4,001; a bound of four workgroups a CU spills (131,071 tokens 57.7 us). LDS shared between the last block's values and the waves' outputs
// would let a fourth workgroup of eight query heads on the CU, but took 13 registers more: 8 members 17.0 of 15.4.
template <int QPK, bool INLINE>
__global__ __launch_bounds__(kAttnThreads, 3) void kv4_attn_kernel(AttnArgs a, Members<INLINE> members) {
    cache_attention<Kv4Format, QPK, INLINE>(a, members);
}
// The chunks' merge: 2 to 4 us, a launch's ramp and one round trip.
template <int NC, bool INLINE>
__global__ __launch_bounds__(128) void kv4_combine_kernel(AttnArgs a, Members<INLINE> members) {
    combine_chunks<Kv4Format, NC, INLINE>(a, members);
}
template <bool INLINE>
constexpr AttnKernels<INLINE> kKernels{{kv4_attn_kernel<1, INLINE>, kv4_attn_kernel<2, INLINE>, kv4_attn_kernel<4, INLINE>, kv4_attn_kernel<8, INLINE>},
                                       {kv4_combine_kernel<8, INLINE>, kv4_combine_kernel<32, INLINE>}};

}  // namespace

hipError_t launch_kv4_append(const AttnArgs& a, int members, hipStream_t stream) { return launch_append(kv4_append_kernel, a, members, stream); }
hipError_t launch_kv4_append_seq(const PrefillAttnArgs& a, hipStream_t stream) { return launch_append_chunk(kv4_append_seq_kernel, a, stream); }
hipError_t launch_kv4_attention(const AttnArgs& a, const AttnMember* host_mem, int members, hipStream_t stream) {
    return launch_cache_attention(kKernels<true>, kKernels<false>, a, host_mem, members, stream);
}

hipError_t launch_kv4_write(const KvMoveArgs& a, bool half, hipStream_t stream) {
    if (!move_fits(a)) return hipErrorInvalidValue;
    return launch_move(half ? kv4_write_kernel<kRowsF16> : kv4_write_kernel<kRowsF32>, a, append_threads(a.p0, a.tokens), stream);
}
hipError_t launch_kv4_read(const KvMoveArgs& a, bool half, hipStream_t stream) {
    if (!move_fits(a)) return hipErrorInvalidValue;
    return launch_move(half ? kv4_read_kernel<_Float16> : kv4_read_kernel<float>, a, kAppendThreads, stream);
}

}  // namespace ribn_amd

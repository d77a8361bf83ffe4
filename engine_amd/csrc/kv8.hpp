// The KV cache in 8 bits: layout, quantisation and launchers (kv8_kernels.hip).
//
// A (layer, KV head) region of a cache holds
//   blocks [ceil(capacity / 32)] of 8192 code bytes, one per 32 tokens: 4096 of
//          keys, 4096 of values, in the order the matrix instructions take them
//   tail   the f16 block the sequence stands in: keys [32][128], values [128][32]
//   scales [blocks] float2: the block's key scale and value scale
//   end    int32: one past the last position appended
// with, for x16 = f16(x) and a = max |x16| over a block's 32 x 128 keys (values):
//   e = max(floor(log2 a) - 6, -24), code = clamp(rint(x16 2^-e), -127, 127)
// stored as the byte code + 128, and the scale 2^e.
//
// A power of two: code * 2^e is then an f16 value, so every reader multiplies on
// the f16 matrix cores what the cache stands for, with no second rounding, and
// a block scaled again from its own values keeps them. It costs half a bit of
// the 8 on average against a / 127. A scale for 32 tokens: the depth of one 16x16x32 product over keys.
//
// What 8 bits cost: a block's largest value sets the step of all 32 x 128, so a value is off by
// 0.29 * 2^e rms, 0.23% to 0.46% of a whatever its own size, and a score by 0.29 * 2^e nats rms for a
// query of rms 1. Where many keys share the weight, the output is off by as much, relatively: with 3,008
// random tokens by 6.3% where 3% of a head's key channels are six times as wide as the others, by 2.1%
// where none is (1.2% from the values). An f16 cache's own error is 0.03% to 0.05% there.
//
// Codes are written when a block's last token arrives; until then its tokens are
// the tail's f16 values, so a token is rounded to 8 bits once and by all 32
// of its block. The tail is block (end - 1) / 32's. An append into another block's
// middle (a sequence taken back) starts from the values that block's codes stand for.
// All tokens of a call read the cache as it stands after the call's appends. So a token's output
// depends on later tokens of its own call (they have a part in a scale), on how a prompt is cut into
// chunks, and, after a sequence was taken back over a block's border, on tokens that it no longer has.
//
// What enters is finite: f16 overflow is held at +-65504 and NaN as 0. A code
// has no infinity, a block's scale is shared by 31 other tokens, and a masked key
// of probability 0 must not make a NaN.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "decode_launch.hpp"

namespace ribn_amd {

constexpr int kKv8Block = 32;                                 // tokens that share a scale
constexpr int kKv8PartBytes = kKv8Block * kHeadDim;           // a block's key (value) codes
constexpr int kKv8BlockBytes = 2 * kKv8PartBytes;
constexpr int kKv8TailElems = kKv8Block * kHeadDim;           // f16 elements of the tail's keys (values)

__host__ __device__ inline size_t kv8_blocks(int capacity) { return ((size_t)capacity + kKv8Block - 1) / kKv8Block; }
// Byte offsets in a region, and its size (a multiple of 256).
__host__ __device__ inline size_t kv8_tail_offset(int capacity) { return kv8_blocks(capacity) * kKv8BlockBytes; }
__host__ __device__ inline size_t kv8_scales_offset(int capacity) { return kv8_tail_offset(capacity) + 2 * kKv8TailElems * sizeof(uint16_t); }
__host__ __device__ inline size_t kv8_end_offset(int capacity) { return kv8_scales_offset(capacity) + kv8_blocks(capacity) * sizeof(float2); }
__host__ __device__ inline size_t kv8_head_bytes(int capacity) { return (kv8_end_offset(capacity) + sizeof(int32_t) + 255) / 256 * 256; }

// Code order within a block's part. Keys: 16 bytes of dims 64 i + 16 g .. + 15
// of the key at row m of product tile t, lane 16 g + m: 64 (2 t + i) + lane.
// Values: 8 keys 8 g .. + 7 of dims 32 u + 2 m and 32 u + 2 m + 1: 64 u + lane.
__host__ __device__ inline int kv8_key_row(int t, int m) { return 8 * (m >> 2) + 4 * t + (m & 3); }

// Sets up a cache: its rotary table (128-wide heads) and, of a cache of blocks (`regions` not
// null), each of the regions of `stride` bytes from byte `codes` on to zeros (an 8-bit cache's tail, scales and
// end: any code is finite; all of a 4-bit cache's), so that it reads as zeros.
hipError_t launch_cache_init(void* regions, size_t count, size_t stride, size_t codes, const double* table, double* table_dst,
                             hipStream_t stream);

// f16 or f32 rows moved into or out of a cache ([tokens][kv_heads][128]).
struct KvMoveArgs {
    AttnMember mem;
    int layer;
    int kv_heads;
    int p0;
    int tokens;
    void* keys;
    void* values;
};

// Keys (RMSNorm and rope in 64 bits, then f32, then f16) and values of new tokens
// into 8-bit caches: rows of members that share one, at positions[0] ..
// positions[0] + members - 1, ahead of an `appended` attention launch; a prompt chunk's.
hipError_t launch_kv8_append(const AttnArgs& args, int members, hipStream_t stream);
hipError_t launch_kv8_append_seq(const PrefillAttnArgs& args, hipStream_t stream);
// Attention of every member over positions 0 .. positions[m], and the merge of
// its chunks. Without `appended`, the members' new tokens go into their caches
// (distinct ones) on the way. `host_mem`: the members' descriptors in host memory,
// instead of args.mem.
hipError_t launch_kv8_attention(const AttnArgs& args, const AttnMember* host_mem, int members, hipStream_t stream);
int kv8_grid_chunks(int max_capacity, int members);

// Rows as they are (keys already normalised and rotated) into a cache, and back
// out of it; `f16` / `f32` by `half`, `kv8` the cache's format.
hipError_t launch_kv_write(const KvMoveArgs& args, bool half, bool kv8, hipStream_t stream);
hipError_t launch_kv_read(const KvMoveArgs& args, bool half, bool kv8, hipStream_t stream);

}  // namespace ribn_amd

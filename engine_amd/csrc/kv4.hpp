// The KV cache in 4 bits: layout, quantisation and launchers (kv4_kernels.hip).
//
// A (layer, KV head) region of a cache holds
//   blocks [ceil(capacity / 32)] of 4864 bytes, one per 32 tokens: 2048 of key codes, 2048 of
//          value codes, the keys' 128 scales and 128 lows (f16), the values' scales and
//          lows [2 halves of the head][scale, low][32 tokens] (f16)
//   tail   the f16 block the sequence stands in: keys [32][128], values [128][32]
//   end    int32: one past the last position appended
// A group shares a scale and a low: 32 tokens of one key dim, 64 dims of one token's value.
// With x16 = f16(x), lo and hi the group's smallest and largest x16:
//   s = (hi - lo) * (1/15) in f32, cut off to f16; inv = 1 / s in f32 (0 where s is 0)
//   code = clamp(rint((x16 - lo) * inv), 0, 15), value = code * s + lo rounded to f16
// Cut off, 15 s + lo does not pass hi: no value leaves its group's range, and none overflows.
//
// Keys by dim, since the dims of a key head differ in size (a norm's weights, and a few wide ones) and
// each dim keeps its own over the tokens; values by token, since they have no such dims and a token's
// own size is what its probability multiplies. A low beside the scale, since a dim that hardly turns
// keeps a mean far from 0. 32 tokens a key group, since that is what a block has together when
// it is quantised; 64 dims a value group: of Gaussian values 32 / 64 / 128 dims are off
// by 7.9% / 9.0% / 10.1% of their deviation at 5 / 4.5 / 4.25 bits. 4.75 bits a value in all, 0.30 of f16's.
//
// Every reader multiplies the same f16 values on the f16 matrix cores, as of an 8-bit cache. What kv8.hpp
// says of the tail, of when a block is quantised and on what an output depends holds here too, but for one
// thing: a block quantised again from its own values (a sequence taken back into it) is rounded again.
// A fresh cache is cleared whole: scales and lows lie among the codes, and what a skipped token reads has to be finite.
#pragma once

#include "kv8.hpp"

namespace ribn_amd {

constexpr int kKv4Group = 64;                                    // dims of a value group
constexpr int kKv4CodeBytes = kKv8Block * kHeadDim / 2;          // a block's key (value) codes
constexpr int kKv4Values = kKv4CodeBytes;                        // byte offsets in a block: value codes
constexpr int kKv4Params = 2 * kKv4CodeBytes;                    // the keys' scales, then lows
constexpr int kKv4ValueParams = 2 * kHeadDim * 2;                // and from there on the values'
constexpr int kKv4ValueHalf = 2 * kKv8Block * 2;                 // bytes of one half's
constexpr int kKv4ParamBytes = kKv4ValueParams + kHeadDim / kKv4Group * kKv4ValueHalf;
constexpr int kKv4BlockBytes = kKv4Params + kKv4ParamBytes;
static_assert(kKv4BlockBytes == 4864);

__host__ __device__ inline size_t kv4_tail_offset(int capacity) { return kv8_blocks(capacity) * kKv4BlockBytes; }
__host__ __device__ inline size_t kv4_end_offset(int capacity) { return kv4_tail_offset(capacity) + 2 * kKv8TailElems * sizeof(uint16_t); }
__host__ __device__ inline size_t kv4_head_bytes(int capacity) { return (kv4_end_offset(capacity) + sizeof(int32_t) + 255) / 256 * 256; }

// Code order within a block's part, 16 bytes a lane 16 g + m. Keys, piece t at 1024 t: dims 16 g .. + 15 (two
// words), then 64 + 16 g .. + 15, of the key at row m of product tile t (kv8_key_row). Values, piece h at
// 1024 h: a word each for dims 64 h + 2 m, + 1, + 32, + 33, of eight keys 8 g .. + 7. A word's
// nibble j is its element 2 j, nibble 4 + j its element 2 j + 1: (w >> 4 j) & 0x000f000f are neighbours.

// As their kv8 counterparts (kv8.hpp).
hipError_t launch_kv4_append(const AttnArgs& args, int members, hipStream_t stream);
hipError_t launch_kv4_append_seq(const PrefillAttnArgs& args, hipStream_t stream);
hipError_t launch_kv4_attention(const AttnArgs& args, const AttnMember* host_mem, int members, hipStream_t stream);
hipError_t launch_kv4_write(const KvMoveArgs& args, bool half, hipStream_t stream);
hipError_t launch_kv4_read(const KvMoveArgs& args, bool half, hipStream_t stream);

}  // namespace ribn_amd

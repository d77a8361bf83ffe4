// Internal API of the rotary positions: spec checks and tables (rope.cpp), the
// operator's launch (rope_kernels.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "ribn_amd.h"

namespace ribn_amd {

constexpr int kRopeMaxDim = 1024;
constexpr int kRopeTableMax = kRopeMaxDim / 2 + 1;  // turns of each pair, then the gain
constexpr int kRopeMaxTensors = 4;

struct RopeRows {
    const void* x;
    void* y;
    size_t x_token, x_head, y_token, y_head;  // strides in elements
    int heads;
    int before;  // heads of the tensors before this one
};

struct RopeArgs {
    const double* table;       // device: turns [rotary_dim / 2], gain
    const int32_t* positions;  // device [tokens]
    RopeRows rows[kRopeMaxTensors];
    size_t tokens;
    int count;
    int head_dim;
    int rotary_dim;
    int slices;     // launch_rope sets it: threads that share a token's heads
    int per_group;  // and this: tokens of a workgroup
};

// `dtype` a RIBN_AMD_F32 / BF16 / F16, `layout` a RIBN_AMD_ROPE_*.
hipError_t launch_rope(const RopeArgs& args, uint32_t dtype, uint32_t layout, int cu_count, hipStream_t stream);

}  // namespace ribn_amd

namespace ribn_amd_abi {

ribn_amd_status check_rope_spec(const ribn_amd_rope_spec* spec);
// The device table of a checked spec: rotary_dim / 2 turns a position adds
// (2 pi radians each), then the gain. Returns how many values were written.
int rope_table(const ribn_amd_rope_spec& spec, double (&table)[ribn_amd::kRopeTableMax]);

}  // namespace ribn_amd_abi

// Internal launcher API of the log-probability kernels (logprob_kernels.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ribn_amd {

constexpr int kLogprobMaxTop = 32;
constexpr uint32_t kLogprobMaxSplits = 64;  // workgroups a row: the merge takes one a lane

// Element types, as in ribn_amd.h.
constexpr int kLogitF32 = 0, kLogitBf16 = 1, kLogitF16 = 2;

struct LogprobArgs {
    const void* logits;       // [rows][stride], the first `length` of each row
    size_t stride;
    size_t length;
    size_t rows;
    const uint32_t* targets;  // [rows], or null
    float* logprobs;          // [rows], or null
    float* entropy;           // [rows], or null
    uint32_t* top_tokens;     // [rows][top], or null
    float* top_logprobs;      // [rows][top], or null
    int top;
    int splits;               // workgroups a row (launch_logprobs sets it)
    uint64_t* partials;       // [rows][splits][3 + top], splits > 1
};

// `scratch`: room of `scratch_bytes` for the partials of split rows.
hipError_t launch_logprobs(const LogprobArgs& args, int dtype, int cu_count, void* scratch, size_t scratch_bytes, hipStream_t stream);

}  // namespace ribn_amd

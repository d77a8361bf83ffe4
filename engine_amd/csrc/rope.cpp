// Rotary positions behind the C ABI: spec checks, frequency tables, the
// operator's handle and call (include/ribn_amd.h, "rotary positions").
#include "rope.hpp"

#include <cmath>
#include <limits>
#include <new>

#include "abi_internal.hpp"

using namespace ribn_amd_abi;

struct ribn_amd_rope {
    ribn_amd_context* ctx;
    uint32_t layout;
    uint32_t head_dim;
    uint32_t rotary_dim;
    double* table;
};

namespace ribn_amd_abi {

ribn_amd_status check_rope_spec(const ribn_amd_rope_spec* s) {
    if (s == nullptr) return fail(RIBN_AMD_INVALID_ARGUMENT, 0, 0, "null rope spec");
    if (s->layout > RIBN_AMD_ROPE_INTERLEAVED) {
        return fail(RIBN_AMD_INVALID_PLAN, RIBN_AMD_ROPE_INTERLEAVED, s->layout, "unknown rope layout %u", s->layout);
    }
    if (s->head_dim < 2 || s->head_dim > (uint32_t)ribn_amd::kRopeMaxDim || s->head_dim % 2 != 0) {
        return fail(RIBN_AMD_INVALID_PLAN, ribn_amd::kRopeMaxDim, s->head_dim, "head_dim must be even, 2..%d (got %u)",
                    ribn_amd::kRopeMaxDim, s->head_dim);
    }
    if (s->rotary_dim < 2 || s->rotary_dim > s->head_dim || s->rotary_dim % 2 != 0) {
        return fail(RIBN_AMD_INVALID_PLAN, s->head_dim, s->rotary_dim, "rotary_dim must be even, 2..%u (got %u)",
                    s->head_dim, s->rotary_dim);
    }
    if (!(s->base > 1.f) || !std::isfinite(s->base)) return fail(RIBN_AMD_INVALID_PLAN, 0, 0, "the rope base must be finite and above 1");
    if (s->scaling > RIBN_AMD_ROPE_YARN) {
        return fail(RIBN_AMD_INVALID_PLAN, RIBN_AMD_ROPE_YARN, s->scaling, "unknown rope scaling %u", s->scaling);
    }
    if (s->scaling != RIBN_AMD_ROPE_UNSCALED && (!(s->factor > 0.f) || !std::isfinite(s->factor))) {
        return fail(RIBN_AMD_INVALID_PLAN, 0, 0, "the rope scaling factor must be finite and positive");
    }
    if (s->scaling == RIBN_AMD_ROPE_YARN) {
        if (s->original_context == 0) return fail(RIBN_AMD_INVALID_PLAN, 1, 0, "YaRN needs the original context length");
        if (!(s->beta_slow > 0.f) || !(s->beta_fast > s->beta_slow) || !std::isfinite(s->beta_fast)) {
            return fail(RIBN_AMD_INVALID_PLAN, 0, 0, "YaRN needs finite beta_fast > beta_slow > 0");
        }
    }
    if (!(s->attention_factor >= 0.f) || !std::isfinite(s->attention_factor)) {
        return fail(RIBN_AMD_INVALID_PLAN, 0, 0, "the attention factor must be finite and not negative");
    }
    if (s->freq_factors != nullptr) {
        for (uint32_t i = 0; i < s->rotary_dim / 2; ++i) {
            if (!(s->freq_factors[i] > 0.f) || !std::isfinite(s->freq_factors[i])) {
                return fail(RIBN_AMD_INVALID_PLAN, 0, i, "frequency factor %u must be finite and positive", i);
            }
        }
    }
    return RIBN_AMD_OK;
}

int rope_table(const ribn_amd_rope_spec& s, double (&table)[ribn_amd::kRopeTableMax]) {
    constexpr double kPi = 3.14159265358979323846;
    const int pairs = (int)s.rotary_dim / 2;
    const double dim = s.rotary_dim, base = s.base;
    double gain = 1.0, low = 0.0, high = 0.0;
    if (s.scaling == RIBN_AMD_ROPE_YARN) {
        // the pair that turns beta times within the original context
        auto pair_of = [&](double beta) { return dim * std::log((double)s.original_context / (2.0 * kPi * beta)) / (2.0 * std::log(base)); };
        low = std::fmax(std::floor(pair_of(s.beta_fast)), 0.0);
        high = std::fmin(std::ceil(pair_of(s.beta_slow)), dim - 1.0);
        if (s.factor > 1.f) gain = 0.1 * std::log((double)s.factor) + 1.0;
    }
    for (int i = 0; i < pairs; ++i) {
        double f = std::pow(base, -2.0 * i / dim);
        if (s.freq_factors != nullptr) f /= (double)s.freq_factors[i];
        if (s.scaling == RIBN_AMD_ROPE_LINEAR) f /= (double)s.factor;
        if (s.scaling == RIBN_AMD_ROPE_YARN) {
            const double ramp = std::fmin(std::fmax((i - low) / std::fmax(high - low, 1e-3), 0.0), 1.0);
            f = f / (double)s.factor * ramp + f * (1.0 - ramp);
        }
        table[i] = f / (2.0 * kPi);
    }
    table[pairs] = s.attention_factor != 0.f ? (double)s.attention_factor : gain;
    return pairs + 1;
}

}  // namespace ribn_amd_abi

namespace {

// The last element of `tokens` x heads rows of `dim`, plus one; false past 64 bits.
bool rows_span(size_t tokens, size_t heads, size_t dim, size_t token_stride, size_t head_stride, size_t* span) {
    size_t a = 0, b = 0;
    return !__builtin_mul_overflow(tokens - 1, token_stride, &a) && !__builtin_mul_overflow(heads - 1, head_stride, &b) &&
           !__builtin_add_overflow(a, b, &a) && !__builtin_add_overflow(a, dim, span);
}

// Whether rows of `dim` lie apart: heads within a token's stride, or tokens within a head's.
bool rows_apart(size_t tokens, size_t heads, size_t dim, size_t token_stride, size_t head_stride) {
    if (heads > 1 && head_stride < dim) return false;
    if (tokens > 1 && token_stride < dim) return false;
    if (tokens == 1 || heads == 1) return true;
    return token_stride >= (heads - 1) * head_stride + dim || head_stride >= (tokens - 1) * token_stride + dim;
}

}  // namespace

extern "C" {

ribn_amd_status ribn_amd_rope_frequencies(const ribn_amd_rope_spec* spec, double* turns, size_t len, double* gain) {
    const ribn_amd_status st = check_rope_spec(spec);
    if (st != RIBN_AMD_OK) return st;
    if (!turns || !gain) return fail(RIBN_AMD_INVALID_ARGUMENT, 0, 0, "null argument");
    const size_t pairs = spec->rotary_dim / 2;
    if (len != pairs) return fail(RIBN_AMD_OUTPUT_LENGTH, pairs, len, "%zu pairs, room for %zu", pairs, len);
    double table[ribn_amd::kRopeTableMax];
    rope_table(*spec, table);
    for (size_t i = 0; i < pairs; ++i) turns[i] = table[i];
    *gain = table[pairs];
    return ok();
}

ribn_amd_status ribn_amd_rope_create(ribn_amd_context* ctx, const ribn_amd_rope_spec* spec, ribn_amd_rope** out) {
    if (!ctx || !out) return fail(RIBN_AMD_INVALID_ARGUMENT, 0, 0, "null argument");
    ribn_amd_status st = check_rope_spec(spec);
    if (st != RIBN_AMD_OK) return st;
    double table[ribn_amd::kRopeTableMax];
    const size_t bytes = (size_t)rope_table(*spec, table) * sizeof(double);
    DeviceGuard guard(ctx->device);
    void* dev = nullptr;
    hipError_t e = hipMalloc(&dev, bytes);
    if (e != hipSuccess) return driver(e, "hipMalloc rope table");
    e = hipMemcpyAsync(dev, table, bytes, hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    auto* r = e == hipSuccess ? new (std::nothrow) ribn_amd_rope{} : nullptr;
    if (!r) {
        hipFree(dev);
        return e != hipSuccess ? driver(e, "upload rope table") : fail(RIBN_AMD_DRIVER, 0, 0, "host allocation failed");
    }
    r->ctx = ctx;
    r->layout = spec->layout;
    r->head_dim = spec->head_dim;
    r->rotary_dim = spec->rotary_dim;
    r->table = static_cast<double*>(dev);
    context_retain(ctx);
    *out = r;
    return ok();
}

void ribn_amd_rope_destroy(ribn_amd_rope* rope) {
    if (!rope) return;
    ribn_amd_context* ctx = rope->ctx;
    {
        DeviceGuard guard(ctx->device);
        hipFree(rope->table);  // waits for outstanding work on the device
    }
    delete rope;
    context_release(ctx);
}

ribn_amd_status ribn_amd_rope_execute(ribn_amd_rope* rope, const int32_t* positions, size_t tokens,
                                      const ribn_amd_rope_rows* rows, size_t count, uint32_t dtype) {
    if (!rope || !rows) return fail(RIBN_AMD_INVALID_ARGUMENT, 0, 0, "null argument");
    if (dtype > RIBN_AMD_F16) return fail(RIBN_AMD_INVALID_ARGUMENT, RIBN_AMD_F16, dtype, "unknown element type %u", dtype);
    if (count == 0 || count > (size_t)ribn_amd::kRopeMaxTensors) {
        return fail(RIBN_AMD_INVALID_ARGUMENT, ribn_amd::kRopeMaxTensors, count, "a rope call takes 1..%d tensors, not %zu",
                    ribn_amd::kRopeMaxTensors, count);
    }
    if (tokens == 0) return fail(RIBN_AMD_EMPTY_INPUT, 1, 0, "a rope call needs at least one token");
    if (tokens > (size_t)std::numeric_limits<int32_t>::max()) return fail(RIBN_AMD_SHAPE_OVERFLOW, 0, 0, "%zu tokens exceed launch limits", tokens);
    ribn_amd_status st = check_device_ptr(rope->ctx, positions, "positions", 4);
    if (st != RIBN_AMD_OK) return st;
    const size_t size = dtype == RIBN_AMD_F32 ? 4 : 2;
    const size_t dim = rope->head_dim;
    ribn_amd::RopeArgs a{};
    size_t heads = 0;
    for (size_t i = 0; i < count; ++i) {
        const ribn_amd_rope_rows& r = rows[i];
        st = check_device_ptr(rope->ctx, r.input, "input", size);
        if (st == RIBN_AMD_OK) st = check_device_ptr(rope->ctx, r.output, "output", size);
        if (st != RIBN_AMD_OK) return st;
        if (r.heads == 0) return fail(RIBN_AMD_EMPTY_INPUT, 1, 0, "tensor %zu has no heads", i);
        heads += r.heads;
        size_t in = 0, out = 0;
        if (r.heads > 65536 || heads > 65536 || !rows_span(tokens, r.heads, dim, r.input_token_stride, r.input_head_stride, &in) ||
            !rows_span(tokens, r.heads, dim, r.output_token_stride, r.output_head_stride, &out)) {
            return fail(RIBN_AMD_SHAPE_OVERFLOW, 0, 0, "the rows of tensor %zu exceed launch limits", i);
        }
        if (in > r.input_len) {
            return fail(RIBN_AMD_INPUT_LENGTH, in, r.input_len, "input %zu has %zu values, its rows take %zu", i, r.input_len, in);
        }
        if (out > r.output_len) {
            return fail(RIBN_AMD_OUTPUT_LENGTH, out, r.output_len, "output %zu has %zu values, its rows take %zu", i, r.output_len, out);
        }
        if (!rows_apart(tokens, r.heads, dim, r.output_token_stride, r.output_head_stride)) {
            return fail(RIBN_AMD_INVALID_ARGUMENT, dim, r.output_head_stride, "output rows of tensor %zu overlap", i);
        }
        if (r.input == r.output && (r.input_token_stride != r.output_token_stride || r.input_head_stride != r.output_head_stride)) {
            return fail(RIBN_AMD_INVALID_ARGUMENT, r.input_token_stride, r.output_token_stride,
                        "tensor %zu is rotated in place with other strides", i);
        }
        a.rows[i] = ribn_amd::RopeRows{r.input, r.output, r.input_token_stride, r.input_head_stride, r.output_token_stride,
                                       r.output_head_stride, (int)r.heads, (int)(heads - r.heads)};
    }
    a.table = rope->table;
    a.positions = positions;
    a.tokens = tokens;
    a.count = (int)count;
    a.head_dim = (int)rope->head_dim;
    a.rotary_dim = (int)rope->rotary_dim;
    DeviceGuard guard(rope->ctx->device);
    const hipError_t e = ribn_amd::launch_rope(a, dtype, rope->layout, rope->ctx->cu_count, rope->ctx->stream);
    return e == hipSuccess ? ok() : driver(e, "rope launch");
}

}  // extern "C"

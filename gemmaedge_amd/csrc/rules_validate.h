// Host-side checks of a call of include/gemmaedge_rules.h, kept apart from the
// HIP launch so that they can be built and run without a device. Nothing here
// reads device memory.
#pragma once

#include <stdint.h>

#include <cmath>

#include "../../include/gemmaedge_rules.h"
#include "sampler_validate.h"

namespace ge {
namespace rules {

constexpr int kMostVocab = 1 << 30;
constexpr int kMostRows = 1 << 24;

inline int size_of(int dtype) { return dtype == GE_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == GE_DTYPE_F32 || dtype == GE_DTYPE_BF16; }
inline bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Bytes from the first to behind the last element of `rows` rows: up to 2^24 rows 2^40 elements apart, more than 63 bits hold.
inline __int128 span(int rows, int vocab, int64_t stride, int size) { return (static_cast<__int128>(rows - 1) * stride + vocab) * size; }

inline bool in_place(const ge_rule_args& x) { return x.out == x.logits; }

inline int check_rules(const ge_rule_args& x, char* msg, size_t n) {
    if (x.rows < 0 || x.vocab < 1) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "rows %d, vocab %d", x.rows, x.vocab);
    if (x.rows > kMostRows || x.vocab > kMostVocab)
        return plan_fail(msg, n, GE_ERR_CAPACITY, "rows %d / vocab %d above %d / %d", x.rows, x.vocab, kMostRows, kMostVocab);
    if (!dtype_ok(x.dtype) || !dtype_ok(x.out_dtype))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "dtype %d, out_dtype %d", x.dtype, x.out_dtype);
    if (!x.row_params) {
        const ge_rule_params& p = x.params;
        if (!std::isfinite(p.softcap) || !std::isfinite(p.repetition_penalty) || !std::isfinite(p.presence_penalty) ||
            !std::isfinite(p.frequency_penalty) || !(p.repetition_penalty > 0.f))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "softcap %g, repetition_penalty %g, presence_penalty %g, frequency_penalty %g",
                             p.softcap, p.repetition_penalty, p.presence_penalty, p.frequency_penalty);
    }
    if (x.ring) {
        if (!x.ring_len || x.ring_capacity < 1)
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "ring needs ring_len and ring_capacity >= 1");
        if (x.history) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "history and ring are exclusive");
    }
    if (x.history && !x.history_offsets) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "history without offsets");
    if (x.bias_ids && (!x.bias_values || !x.bias_offsets))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "bias_ids without values or offsets");
    const int64_t words = (static_cast<int64_t>(x.vocab) + 31) / 32;
    if (x.mask) {
        if (x.masks < 1 || (x.masks > 1 && x.mask_stride < words))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "masks %d of %lld words, %lld apart", x.masks, static_cast<long long>(words),
                             static_cast<long long>(x.mask_stride));
        if (!x.mask_rows && x.masks < x.rows)
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "%d masks for %d rows without mask_rows", x.masks, x.rows);
    } else if (x.mask_rows) {
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "mask_rows without masks");
    }
    if (!aligned_to(x.row_params, 4) || !aligned_to(x.history, 4) || !aligned_to(x.history_offsets, 4) || !aligned_to(x.ring, 4) ||
        !aligned_to(x.ring_len, 4) || !aligned_to(x.prompt_len, 4) || !aligned_to(x.bias_ids, 4) || !aligned_to(x.bias_values, 4) ||
        !aligned_to(x.bias_offsets, 4) || !aligned_to(x.mask, 4) || !aligned_to(x.mask_rows, 4) || !aligned_to(x.flags_out, 4))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "an array is not aligned to its elements");
    if (x.rows == 0) return GE_OK;
    if (!x.logits || !x.out) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "logits or out is NULL");
    if (!aligned_to(x.logits, size_of(x.dtype)) || !aligned_to(x.out, size_of(x.out_dtype)))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "logits or out is not aligned to its elements");
    constexpr int64_t kMost = int64_t{1} << 40;
    if (x.rows > 1 && (x.row_stride < x.vocab || x.out_stride < x.vocab || x.row_stride > kMost || x.out_stride > kMost))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "row_stride %lld or out_stride %lld < vocab %d", static_cast<long long>(x.row_stride),
                         static_cast<long long>(x.out_stride), x.vocab);
    if (in_place(x)) {
        if (x.dtype != x.out_dtype || (x.rows > 1 && x.row_stride != x.out_stride))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "in place with another dtype or stride");
    } else {
        const __int128 a = reinterpret_cast<uintptr_t>(x.logits), b = reinterpret_cast<uintptr_t>(x.out);
        if (a < b + span(x.rows, x.vocab, x.out_stride, size_of(x.out_dtype)) && b < a + span(x.rows, x.vocab, x.row_stride, size_of(x.dtype)))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "out overlaps the logits");
    }
    return GE_OK;
}

}  // namespace rules
}  // namespace ge

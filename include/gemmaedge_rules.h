/*
 * gemmaedge_rules.h — C ABI of the rules on logits on MI355X (gfx950).
 *
 * What a request asks of its answers before the sampler of
 * gemmaedge_sampler.h draws one: penalties for repeated tokens, biases of
 * single tokens and the tokens that a grammar allows. The reference has no
 * counterpart; its softcap (src/generation.cpp:431-437) comes before such
 * rules and can be applied here instead of in the sampler.
 *
 * Conventions are the sampler's: plain C types, status codes (GE_OK or a
 * negative GE_ERR_*), the message in ge_sampler_last_error(), no exceptions
 * across the boundary. The call is stream-ordered and asynchronous, allocates
 * nothing and keeps nothing, so it can be captured into a HIP graph and issued
 * on several streams at once.
 *
 * Per token of a row, in this order, each operation rounded to float32:
 *   v = logit (bf16 widened exactly)
 *   v = softcap * tanh(v / softcap)        if softcap > 0
 *   v = v > 0 ? v / r : v * r              if the history holds the token (r = repetition penalty)
 *   v = v - f * c - p                      if it holds the token c > 0 times behind its prompt
 *                                          (f = frequency, p = presence penalty)
 *   v = v + b                              if the row has a bias for the token
 *   v = -infinity                          if the row's mask does not allow it, whatever v is
 * and v is rounded once more where the output is bf16. Softcap and repetition
 * penalty are the sampler's, bit for bit: sampling a float32 output without
 * them gives what ge_sample gives with them on the input.
 */
#ifndef GEMMAEDGE_RULES_H
#define GEMMAEDGE_RULES_H

#include <stddef.h>
#include <stdint.h>

#include "gemmaedge_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ge_rule_params {
    float softcap;             /* <= 0: no softcap */
    float repetition_penalty;  /* 1: none */
    float presence_penalty;    /* 0: none */
    float frequency_penalty;   /* 0: none */
} ge_rule_params;

/* Per-row output flag: the row's mask allows no token of the vocabulary. */
#define GE_RULE_EMPTY 1

typedef struct ge_rule_args {
    const void* logits;        /* device, row r at logits + r * row_stride elements */
    int32_t dtype;             /* GE_DTYPE_F32 or GE_DTYPE_BF16 */
    int32_t rows;              /* 0 .. 2^24 */
    int32_t vocab;             /* 1 .. 2^30 */
    int64_t row_stride;        /* >= vocab */
    void* out;                 /* device, rows out_stride elements apart: another memory than the
                                  logits, or the logits themselves (same dtype and stride) */
    int32_t out_dtype;
    int64_t out_stride;        /* >= vocab; elements between rows are left as they are */

    /* `params` for every row (finite, repetition_penalty > 0), unless row_params (device
     * array of `rows` entries, 4-byte aligned, not checked) is non-NULL. */
    ge_rule_params params;
    const ge_rule_params* row_params;

    /* The history as in ge_sample_args: CSR or the sampler's ring, which is only read;
     * neither: no history. Duplicates count; ids outside [0, vocab) do not.
     * prompt_len (device int32[rows], or NULL: 0): the first ids of a row that are its
     * prompt, which the presence and frequency penalties do not count. Of a ring that
     * has wrapped, the place of an id is its number among all that were appended. */
    const int32_t* history;
    const int32_t* history_offsets;
    const int32_t* ring;
    const int32_t* ring_len;
    int32_t ring_capacity;
    const int32_t* prompt_len;

    /* Biases (device), CSR: row r's are entries bias_offsets[r] .. bias_offsets[r+1].
     * Of several entries for one token the last counts; ids outside [0, vocab) do not. */
    const int32_t* bias_ids;
    const float* bias_values;
    const int32_t* bias_offsets;

    /* Masks (device): `masks` of them, mask_stride 32-bit words apart, at least
     * ceil(vocab / 32) each; bit t % 32 of word t / 32 is set where token t is
     * allowed. Row r takes mask mask_rows[r], none if that is outside [0, masks);
     * mask_rows NULL: mask r. mask NULL: none. */
    const uint32_t* mask;
    int64_t mask_stride;
    int32_t masks;
    const int32_t* mask_rows;

    int32_t* flags_out;        /* device int32[rows], GE_RULE_* bits; or NULL */
} ge_rule_args;

/* On the calling thread's current device. */
int ge_apply_rules(void* stream, const ge_rule_args* args);

#ifdef __cplusplus
}
#endif

#endif /* GEMMAEDGE_RULES_H */

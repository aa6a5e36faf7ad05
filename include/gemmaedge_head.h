/*
 * gemmaedge_head.h — C ABI of the trainable answer head on MI355X (gfx950).
 *
 * The head is what lies between a model's last hidden state and its next
 * token: the norm, the projection onto the vocabulary with the final-logit
 * softcap (src/generation.cpp:431-437, here with its cross entropy), and the
 * step that updates both. The sampler of gemmaedge_sampler.h answers with the
 * logits; the calls here score given tokens and train. The reference only
 * infers and has no counterpart of the gradients or of the optimiser.
 *
 * Conventions are the sampler's: plain C types, status codes (GE_OK or a
 * negative GE_ERR_*), the message in ge_sampler_last_error(), no exceptions
 * across the boundary. Calls are stream-ordered and asynchronous, allocate
 * nothing and never wait for the device, so they can be captured into a HIP
 * graph. Results do not depend on the order in which workgroups run.
 *
 * Element types are GE_DTYPE_F32 and GE_DTYPE_BF16. Sums, statistics and
 * optimiser arithmetic are float32 or wider whatever the element type.
 */
#ifndef GEMMAEDGE_HEAD_H
#define GEMMAEDGE_HEAD_H

#include <stddef.h>
#include <stdint.h>

#include "gemmaedge_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ge_head ge_head;

#define GE_HEAD_MAX_DIM 65536

/* Create a head on `device` for up to max_rows hidden states of up to max_dim
 * channels and a vocabulary of up to max_vocab, elements of type `dtype`.
 * Allocates every workspace now. train != 0 adds what the backward calls need: the
 * gradient of the logits for a piece of the vocabulary at a time (about 512 MiB for
 * large batches) and the hidden states' gradient in up to 32 parts (256 MiB, or one
 * part if that is more); small handles take less. */
int ge_head_create(int device, int max_rows, int max_dim, int max_vocab, int dtype, int train, ge_head** out);

void ge_head_destroy(ge_head* head);

/* The norm over the channels of each row, and its gradients:
 *   mean = sum(x) / D (0 unless center), rstd = 1 / sqrt(sum((x - mean)^2) / D + eps),
 *   xhat = (x - mean) * rstd, y = xhat * weight + bias;
 *   with a = dy * weight: dx = rstd * (a - [sum(a) / D] - xhat * sum(a * xhat) / D)
 *   (the bracket with center only), dweight = sum over rows of dy * xhat,
 *   dbias = sum over rows of dy.
 * The sums are float32: a row whose squares add up past 3.4e38 has an rstd of 0.
 * center = 1 is the layer norm, center = 0 the root-mean-square norm.
 * Rows may be any stride >= dim apart; channels are contiguous. x, y, dy and
 * dx have the handle's dtype; weight, bias, dweight and dbias weight_dtype. */
typedef struct ge_norm_args {
    const void* x;
    int64_t x_stride;         /* elements from row to row */
    int32_t rows;             /* >= 0 */
    int32_t dim;              /* >= 1 */
    int32_t weight_dtype;
    int32_t center;
    float eps;                /* >= 0 */
    const void* weight;       /* [dim] */
    const void* bias;         /* [dim], or NULL; forward only */
    void* y;                  /* forward: [rows], y_stride */
    int64_t y_stride;
    float* mean;              /* [rows]: written by the forward call, read by the
                                 backward call; may be NULL without center */
    float* rstd;              /* [rows]: likewise */
    const void* dy;           /* backward: [rows], dy_stride */
    int64_t dy_stride;
    void* dx;                 /* backward: [rows], dx_stride; NULL: not wanted */
    int64_t dx_stride;
    void* dweight;            /* backward: [dim]; NULL: not wanted */
    void* dbias;              /* backward: [dim]; NULL: not wanted */
} ge_norm_args;

/* Neither y nor dx may overlap another argument's memory, except that y may be
 * x and dx may be dy (same stride). */
int ge_head_norm(ge_head* head, void* stream, const ge_norm_args* args);
int ge_head_norm_backward(ge_head* head, void* stream, const ge_norm_args* args);

/* Cross entropy of hidden states against their next tokens over the whole
 * vocabulary, without storing the logits:
 *   z_v = hidden . weight_v, l_v = softcap * tanh(z_v / softcap) (l = z if softcap <= 0),
 *   lse = log(sum(exp(l_v))), loss = lse - l_target.
 * A row whose target lies outside [0, vocab) carries no loss: its loss and its
 * dhidden are 0 and it adds nothing to dweight, whatever the row and the weights
 * hold; its lse is computed all the same.
 * The backward call takes grad[r] = d(objective) / d(loss[r]) and the lse of
 * the forward call on the same inputs, and writes
 *   dz_v = grad * (exp(l_v - lse) - [v = target]) * (1 - (l_v / softcap)^2),
 *   dhidden = sum over v of dz_v * weight_v, dweight_v = sum over rows of dz_v * hidden.
 * It computes the logits again, a piece of the vocabulary at a time, and holds
 * dz in the operands' type (bf16: each value rounded once to 8 bits of mantissa,
 * in units of the largest grad's mantissa, before the two products, whose sums
 * are float32; float32 operands are multiplied in three bf16 planes each, 24 bits
 * of magnitudes from 2^-110 to 3.38e38, bf16's largest). With bf16 operands the
 * softcap and the exponentials of both calls use the hardware's exp2 and
 * reciprocal: l is within 4e-7 of the cap for caps up to 64 and within 1e-6 of
 * itself for larger ones, beside the products' own sums. A NaN makes the rows it
 * takes part in NaN; so does an infinity in float32, and in bf16 where a logit
 * becomes +infinity or no number by it. */
typedef struct ge_loss_args {
    const void* hidden;       /* [rows][dim], hidden_stride elements apart */
    int64_t hidden_stride;
    const void* weight;       /* [vocab][dim], weight_stride elements apart */
    int64_t weight_stride;
    int32_t rows;             /* >= 0 */
    int32_t dim;              /* >= 1 */
    int32_t vocab;            /* >= 1 */
    float softcap;
    const int32_t* targets;   /* [rows] */
    float* loss;              /* [rows]: forward output; NULL: not wanted */
    float* lse;               /* [rows]: forward output, backward input */
    const float* grad;        /* [rows]: backward input */
    void* dhidden;            /* [rows][dim], dhidden_stride apart; NULL: not wanted */
    int64_t dhidden_stride;
    void* dweight;            /* [vocab][dim], dweight_stride apart; NULL: not wanted */
    int64_t dweight_stride;
} ge_loss_args;

/* Outputs may not overlap inputs. */
int ge_head_loss(ge_head* head, void* stream, const ge_loss_args* args);
int ge_head_loss_backward(ge_head* head, void* stream, const ge_loss_args* args);

/* One AdamW step over any number of tensors in one launch:
 *   g = grad * grad_scale, m = beta1 m + (1 - beta1) g, v = beta2 v + (1 - beta2) g g,
 *   p = p (1 - lr weight_decay) - (lr / (1 - beta1^step)) m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * in float32, each operation rounded by itself (with 8-bit states the square root
 * and the quotient are within 1 ulp each, unless eps is below
 * 2^-39 / sqrt(1 - beta2^step): then they are rounded correctly). p is the master
 * where there is one (the parameter is then the master rounded), else the parameter.
 *
 * state_bits 32: m and v are float32. state_bits 8: blocks of GE_ADAMW_BLOCK
 * elements share a float32 scale; m is held in e4m3 in units of its scale =
 * largest |m| / 448, v in e5m2 in units of its scale = largest v / 57344. The
 * update uses m and v before they are rounded. Rounding is to one of the two
 * neighbouring codes at random, with the chance that keeps the mean: rounded to
 * the nearest, an average that moves by less than half a code's step would
 * never move. The 32 random bits of element i of block b (blocks counted over
 * the whole list) are a hash of seed, step, b and i, so a step can be repeated
 * exactly. Values of m below the smallest normal code become that code or 0,
 * likewise at random; values of v below it become that code (a denominator
 * never shrinks). A block whose largest value is below 2^-100 is held as
 * zeros. A non-finite value makes its block NaN.
 *
 * Memory that the step writes belongs to one tensor of the list and to nothing else
 * of the call; a float32 parameter may be its own master. */
#define GE_ADAMW_BLOCK 256

typedef struct ge_adamw_tensor {
    void* param;              /* param_dtype [n] */
    const void* grad;         /* grad_dtype [n] */
    float* master;            /* float32 [n], or NULL */
    void* m;                  /* float32 [n], or e4m3 [n] */
    void* v;                  /* float32 [n], or e5m2 [n] */
    float* m_scale;           /* 8-bit states: [ceil(n / GE_ADAMW_BLOCK)] */
    float* v_scale;
    int64_t n;                /* >= 0 */
    int32_t param_dtype;
    int32_t grad_dtype;
} ge_adamw_tensor;

typedef struct ge_adamw_params {
    double lr;
    double beta1;             /* in [0, 1) */
    double beta2;             /* in [0, 1) */
    double eps;               /* >= 0 */
    double weight_decay;
    double grad_scale;
    uint32_t step;            /* this step's number, from 1 */
    uint32_t seed;
} ge_adamw_params;

typedef struct ge_adamw_args {
    const void* table;        /* device copy of what ge_adamw_table wrote */
    int64_t table_bytes;
    int32_t count;            /* tensors in the table */
    int32_t state_bits;       /* 32 or 8, as in ge_adamw_table */
    ge_adamw_params params;
    const ge_adamw_params* device_params; /* device memory, read by the launch instead of
                                             params, for steps replayed from a graph; or NULL.
                                             8-byte aligned; the values are not checked */
} ge_adamw_args;

/* Checks `count` tensors and writes the size of their table to *bytes. */
int ge_adamw_table_bytes(const ge_adamw_tensor* tensors, int count, int state_bits, int64_t* bytes);
/* Writes the table into host memory of that size; the caller copies it to the
 * device (16-byte aligned) and keeps it there while it calls ge_adamw_step. */
int ge_adamw_table(const ge_adamw_tensor* tensors, int count, int state_bits, void* table, int64_t bytes);
/* One step on the calling thread's current device. */
int ge_adamw_step(void* stream, const ge_adamw_args* args);

#ifdef __cplusplus
}
#endif

#endif /* GEMMAEDGE_HEAD_H */

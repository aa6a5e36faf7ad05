/*
 * gemmaedge_projection.h — C ABI of a projection with low-rank adapters on MI355X (gfx950).
 *
 * The product that makes the logits which the sampler of gemmaedge_sampler.h
 * reads (src/generation.cpp:421-430), or any other linear layer: one weight that
 * all rows share, and beside it a low-rank adapter for each row's request, many
 * of them in one call. The backward call trains the adapters; the shared weight
 * is frozen. The reference has no adapters.
 *
 * Conventions are the sampler's: plain C types, status codes (GE_OK or a
 * negative GE_ERR_*), the message in ge_sampler_last_error(), no exceptions
 * across the boundary. Calls are stream-ordered and asynchronous, allocate
 * nothing and never wait for the device, so they can be captured into a HIP
 * graph. A handle must not be used by two streams at once. Results do not
 * depend on the order in which workgroups run.
 */
#ifndef GEMMAEDGE_PROJECTION_H
#define GEMMAEDGE_PROJECTION_H

#include <stddef.h>
#include <stdint.h>

#include "gemmaedge_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ge_projection ge_projection;

#define GE_PROJECT_MAX_DIM 65536
#define GE_PROJECT_MAX_RANK 256
#define GE_PROJECT_MAX_ADAPTERS 65535

/* Create a projection on `device` for up to max_rows rows of up to max_dim
 * channels, weights of up to max_out rows and up to max_adapters adapters of up
 * to max_rank (0: none), elements of type `dtype` (GE_DTYPE_F32 or GE_DTYPE_BF16).
 * Allocates every workspace now; train != 0 adds what the backward call needs. */
int ge_projection_create(int device, int max_rows, int max_dim, int max_out, int max_rank, int max_adapters, int dtype, int train,
                         ge_projection** out);

void ge_projection_destroy(ge_projection* projection);

/* With k = adapter[n], rows whose k is outside [0, adapters) having none:
 *   u[n] = scale[k] A_k hidden[n],  out[n] = weight hidden[n] + B_k u[n];
 * the backward call, for dout[n] = d(objective) / d(out[n]):
 *   du[n] = scale[k] B_k^T dout[n],  dhidden[n] = weight^T dout[n] + A_k^T du[n],
 *   dA_k = sum over its rows of du[n] hidden[n]^T,  dB_k = sum of dout[n] u[n]^T,
 * zeros for adapters without rows. da and db are written, not added to.
 *
 * Sums are float32, and u and du are held in float32's 24 bits (bf16 operands: of
 * magnitudes from 2^-102 on). float32 operands: products with the weight in three
 * bf16 planes each (24 bits of magnitudes from 2^-110 to 3.38e38), those of the
 * adapters in float32. Adapters of a smaller rank are padded with zeros.
 *
 * Infinities and NaN go where the formulas take them, and only there; in float32
 * an infinity in hidden, weight or dout gives NaN in what the product with the weight makes of it. */
typedef struct ge_project_args {
    const void* hidden;       /* [rows][dim], hidden_stride elements apart */
    int64_t hidden_stride;
    const void* weight;       /* [out_dim][dim], weight_stride elements apart */
    int64_t weight_stride;
    int32_t rows;             /* >= 0 */
    int32_t dim;              /* >= 1 */
    int32_t out_dim;          /* >= 1 */
    int32_t rank;             /* >= 1 with adapters */
    int32_t adapters;         /* 0: none, and the next four are not read */
    const void* a;            /* [adapters][rank][dim] */
    const void* b;            /* [adapters][out_dim][rank] */
    const float* scale;       /* [adapters] */
    const int32_t* adapter;   /* [rows] */
    void* out;                /* forward: [rows][out_dim], out_stride apart, out_dtype */
    int64_t out_stride;
    int32_t out_dtype;        /* GE_DTYPE_F32 or GE_DTYPE_BF16 */
    const void* dout;         /* backward: [rows][out_dim], dout_stride apart */
    int64_t dout_stride;
    void* dhidden;            /* backward: [rows][dim], dhidden_stride apart; NULL: not wanted */
    int64_t dhidden_stride;
    void* da;                 /* backward: as a; NULL: not wanted */
    void* db;                 /* backward: as b; NULL: not wanted */
} ge_project_args;

/* Outputs may not overlap inputs or each other (refused; columns of one buffer do not overlap);
 * `out` is not read by the backward call. */
int ge_project(ge_projection* projection, void* stream, const ge_project_args* args);
int ge_project_backward(ge_projection* projection, void* stream, const ge_project_args* args);

#ifdef __cplusplus
}
#endif

#endif /* GEMMAEDGE_PROJECTION_H */

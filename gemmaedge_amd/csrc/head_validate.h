// Host-side checks and geometry of the head's calls (include/gemmaedge_head.h),
// kept apart from the HIP launches so that they can be built and run without a
// device. Nothing here reads device memory.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "../../include/gemmaedge_head.h"
#include "sampler_validate.h"

namespace ge {
namespace head {

constexpr int kUnits = 256;       // compute units
constexpr int kTileM = 256;       // vocabulary (or channels) of a large tile
constexpr int kTile32 = 128;      // of a tile of float32 operands
constexpr int kSmallRows = 64;    // batches up to this take the small tiles
constexpr int kSmallTileM = 128;
constexpr int kSmallTileN = 32;
constexpr int kMaxStride = 1 << 21;  // elements between rows that tiles are fetched from: 256 rows within 31 bits
constexpr int kMostTiles = (1 << 24) - 1;  // of one launch
constexpr int kPadK = 64;         // packed rows are padded to this
constexpr int kPadDz = 64;        // and the logits' gradient's by this: rows a power of two apart share their memory channels
constexpr int kMaxSplits = 32;    // parts of the vocabulary's sum in the hidden states' gradient
constexpr int kNormParts = 512;   // workgroups of the norm's backward pass, whose weight gradients are summed last
constexpr int kNormBlocks = 1280; // and of the forward pass, at most

inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
inline int planes_of(int dtype) { return dtype == GE_DTYPE_F32 ? 2 : 1; }  // of two bytes
inline int elem_size(int dtype) { return dtype == GE_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == GE_DTYPE_F32 || dtype == GE_DTYPE_BF16; }

// What a handle was created for and the workspaces' sizes in bytes.
struct Capacity {
    int max_rows, max_dim, max_vocab;
    int dtype;
    bool train;
    int64_t stats;    // float2 per row and vocabulary tile
    int64_t row;      // forward: the target's logit of each row; backward: the gradient's unit
    int64_t hpack;    // hidden states in padded rows
    int64_t wpack;    // a piece of the weights in padded rows
    int64_t dlogits;  // the logits' gradient of a piece of the vocabulary
    int64_t dhidden;  // float32 parts of the hidden states' gradient
    int64_t norm;     // float32 parts of the norm weights' gradients
};

// Workspace of a handle. Pieces of the vocabulary are as large as fits 512 MB
// of logits' gradient: each piece adds to the hidden states' float32 gradient and
// ends three launches (4,096 rows of 2,816 channels: 0.3 ms for 256 MB). A packed
// piece of weights takes at most 64 MB (bf16).
inline void size_workspace(Capacity& c) {
    const int64_t rows = c.max_rows, dim = round_up(c.max_dim, kPadK), vocab = round_up(c.max_vocab, kTileM);
    const int64_t planes = planes_of(c.dtype), rows_pad = round_up(rows, 256);
    c.stats = 8 * std::max(rows * (vocab / (c.dtype == GE_DTYPE_F32 ? kTile32 : kTileM)),
                           std::min<int64_t>(rows, kSmallRows) * (vocab / kSmallTileM));
    c.row = 8 * rows;
    c.hpack = 2 * planes * rows * dim;
    const int64_t cols = std::min(vocab, std::max<int64_t>(kTileM, ((64LL << 20) / (2 * dim)) / kTileM * kTileM));
    c.wpack = 2 * planes * cols * dim;
    c.dlogits = c.dhidden = c.norm = 0;
    if (!c.train) return;
    const int64_t per_col = 2 * planes * rows_pad;
    c.dlogits = std::min(per_col * (vocab + kPadDz), std::max<int64_t>(per_col * kTileM, 512LL << 20) + per_col * kPadDz);
    const int64_t tiles = (rows_pad / 256) * ((dim + 255) / 256);
    // no call splits its sum into more parts than steps, or 32
    const int64_t parts = std::min<int64_t>(kMaxSplits, vocab / 64);
    c.dhidden = 4 * std::min<int64_t>(256 * 256 * std::max<int64_t>(tiles, 1024), parts * rows * round_up(c.max_dim, 4));
    c.norm = 4LL * 2 * kNormParts * c.max_dim;
}

inline int check_create(int max_rows, int max_dim, int max_vocab, int dtype, char* msg, size_t n) {
    if (max_rows < 1 || max_dim < 1 || max_vocab < 1)
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "max_rows=%d max_dim=%d max_vocab=%d", max_rows, max_dim, max_vocab);
    if (!dtype_ok(dtype)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "dtype %d", dtype);
    if (max_dim > GE_HEAD_MAX_DIM || max_vocab > (1 << 24) || max_rows > (1 << 22))
        return plan_fail(msg, n, GE_ERR_CAPACITY, "max_rows %d / max_dim %d / max_vocab %d above %d / %d / %d", max_rows,
                         max_dim, max_vocab, 1 << 22, GE_HEAD_MAX_DIM, 1 << 24);
    return GE_OK;
}

inline int check_sizes(const Capacity& c, int rows, int dim, char* msg, size_t n) {
    if (rows < 0 || dim < 1) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "rows %d, dim %d", rows, dim);
    if (rows > c.max_rows || dim > c.max_dim)
        return plan_fail(msg, n, GE_ERR_CAPACITY, "rows %d / dim %d above capacity %d / %d", rows, dim, c.max_rows, c.max_dim);
    return GE_OK;
}

// Rows `stride` elements apart of `dim` elements: a single row may carry any stride.
inline bool stride_ok(int64_t stride, int rows, int64_t dim) {
    return rows <= 1 || (stride >= dim && stride <= (int64_t{1} << 40));
}
inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline int check_norm(const Capacity& c, const ge_norm_args& x, bool backward, char* msg, size_t n) {
    if (const int rc = check_sizes(c, x.rows, x.dim, msg, n)) return rc;
    if (!dtype_ok(x.weight_dtype)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "weight_dtype %d", x.weight_dtype);
    if (x.center != 0 && x.center != 1) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "center %d", x.center);
    if (backward && c.norm == 0)
        return plan_fail(msg, n, GE_ERR_CAPACITY, "the handle was created without train");
    if (!backward && !(x.eps >= 0.f)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "eps %g", static_cast<double>(x.eps));
    const size_t es = elem_size(c.dtype), ws = elem_size(x.weight_dtype);
    if (x.rows > 0) {
        if (!x.x || !x.weight || !x.rstd || (x.center && !x.mean))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "x, weight, rstd or (with center) mean is NULL");
        if (!stride_ok(x.x_stride, x.rows, x.dim))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "x_stride %lld < dim %d", static_cast<long long>(x.x_stride), x.dim);
        if (!backward && (!x.y || !stride_ok(x.y_stride, x.rows, x.dim)))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "y is NULL or its rows overlap");
        if (backward && (!x.dy || !stride_ok(x.dy_stride, x.rows, x.dim)))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "dy is NULL or its rows overlap");
        if (backward && x.dx && !stride_ok(x.dx_stride, x.rows, x.dim))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "dx rows overlap");
        if (!aligned_to(x.x, es) || !aligned_to(x.y, es) || !aligned_to(x.dy, es) || !aligned_to(x.dx, es) ||
            !aligned_to(x.mean, 4) || !aligned_to(x.rstd, 4))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "a tensor is not aligned to its elements");
    }
    if (!aligned_to(x.weight, ws) || !aligned_to(x.bias, ws) || !aligned_to(x.dweight, ws) || !aligned_to(x.dbias, ws))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "a weight is not aligned to its elements");
    return GE_OK;
}

// How a loss call runs.
struct LossPlan {
    bool pack_h, pack_w;  // operands copied into padded rows first
    int planes;           // of two bytes: 1 or 2
    int64_t kpad;         // packed rows' length
    int tile_m, tile_n;   // of the logits' product
    int rows_pad;         // rows of the logits' gradient
    int piece;            // vocabulary per piece of the backward (a multiple of kTileM)
    int pack_piece;       // vocabulary per piece of the forward: packed weights, or tiles of a launch
    int splits;           // parts of the vocabulary's sum in dhidden
    int64_t dz_ld;        // elements from row to row of the logits' gradient
};

inline int check_loss(const Capacity& c, const ge_loss_args& x, bool backward, LossPlan& plan, char* msg, size_t n) {
    if (const int rc = check_sizes(c, x.rows, x.dim, msg, n)) return rc;
    if (x.vocab < 1) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "empty vocabulary");
    if (x.vocab > c.max_vocab)
        return plan_fail(msg, n, GE_ERR_CAPACITY, "vocab %d above capacity %d", x.vocab, c.max_vocab);
    if (backward && c.dlogits == 0) return plan_fail(msg, n, GE_ERR_CAPACITY, "the handle was created without train");
    if (!(std::fabs(x.softcap) <= 3.0e38f)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "softcap is not finite");
    const size_t es = elem_size(c.dtype);
    if (x.rows > 0) {
        if (!x.hidden || !x.weight || !x.targets || !x.lse)
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "hidden, weight, targets or lse is NULL");
        if (!stride_ok(x.hidden_stride, x.rows, x.dim) || !stride_ok(x.weight_stride, x.vocab, x.dim))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "hidden_stride %lld or weight_stride %lld < dim %d",
                             static_cast<long long>(x.hidden_stride), static_cast<long long>(x.weight_stride), x.dim);
        if (backward && !x.grad) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "grad is NULL");
        if (!aligned_to(x.targets, 4) || !aligned_to(x.loss, 4) || !aligned_to(x.lse, 4) || !aligned_to(x.grad, 4))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "a tensor is not aligned to its elements");
    }
    if (backward) {
        if (x.dhidden && !stride_ok(x.dhidden_stride, x.rows, x.dim))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "dhidden rows overlap");
        if (x.dweight && !stride_ok(x.dweight_stride, x.vocab, x.dim))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "dweight rows overlap");
    }
    if (!aligned_to(x.hidden, es) || !aligned_to(x.weight, es) || !aligned_to(x.dhidden, es) || !aligned_to(x.dweight, es))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "a tensor is not aligned to its elements");

    plan.planes = planes_of(c.dtype);
    // bf16 tiles are fetched 16 bytes a lane into LDS: other rows are packed first,
    // into rows with zeros behind them. float32 ones pass registers and need no
    // alignment. Offsets in a tile have 31 bits.
    auto direct = [&](const void* p, int64_t stride, int rows) {
        if (rows > 1 && stride > kMaxStride) return false;
        return c.dtype == GE_DTYPE_F32 || (aligned_to(p, 16) && (rows <= 1 || stride % 8 == 0) && x.dim % 8 == 0);
    };
    plan.pack_h = !direct(x.hidden, x.hidden_stride, x.rows);
    plan.pack_w = !direct(x.weight, x.weight_stride, x.vocab);
    plan.kpad = round_up(x.dim, kPadK);
    if (c.dtype == GE_DTYPE_F32) {
        // The widest tile that does not pad the rows much: a tile costs its width and
        // about 20 more. 300 rows: 172 us in tiles of 64 against 186 in tiles of 128;
        // 96 rows: 72 us in tiles of 96 or 128 against 106 in tiles of 64.
        plan.tile_m = kTile32;
        plan.tile_n = 32;
        int64_t best = x.rows <= 32 ? 0 : INT64_MAX;
        for (const int tile : {128, 96, 64}) {
            const int64_t cost = round_up(x.rows, tile) / tile * (tile + 20);
            if (cost < best) {
                best = cost;
                plan.tile_n = tile;
            }
        }
    } else {
        // 100 rows, width 1,024, vocabulary 60,000: 31 us in tiles of 128 rows, 38 in tiles of 256
        const bool small = x.rows <= kSmallRows;
        plan.tile_m = small ? kSmallTileM : kTileM;
        plan.tile_n = small ? kSmallTileN : x.rows <= 128 ? 128 : 256;
    }
    plan.rows_pad = static_cast<int>(round_up(std::max(x.rows, 1), 256));  // whole tiles of any width that is chosen
    const int64_t vpad = round_up(x.vocab, kTileM);
    const int64_t pack_cols = c.wpack / (2 * plan.planes * plan.kpad) / kTileM * kTileM;
    // A launch has less than 2^32 threads, 256 for each tile.
    const int64_t row_tiles = (std::max(x.rows, 1) + plan.tile_n - 1) / plan.tile_n;
    const int64_t launch_cols = kMostTiles / row_tiles * plan.tile_m / kTileM * kTileM;
    plan.pack_piece = static_cast<int>(std::min(std::min(vpad, launch_cols), plan.pack_w ? pack_cols : vpad));
    if (backward) {
        // offsets in a tile of the gradient's rows have 31 bits, as in the operands
        const int64_t cols = std::min<int64_t>(kMaxStride - kTileM, (c.dlogits / (2LL * plan.planes * plan.rows_pad) - kPadDz) / kTileM * kTileM);
        // as few pieces as fit, all of about the same size
        const int64_t most = std::min<int64_t>(std::min<int64_t>(vpad, cols), plan.pack_piece);
        const int64_t pieces = (vpad + most - 1) / most;
        plan.piece = static_cast<int>(std::min(most, round_up((vpad + pieces - 1) / pieces, kTileM)));
        plan.dz_ld = plan.piece + kPadDz;
        // Parts of the sum over the piece: 256 tiles run at a time, one on each compute
        // unit (512 of float32, two on each); a part costs its steps and about 12 more
        // for its beginning and for adding what it has.
        const int64_t tile = c.dtype == GE_DTYPE_F32 ? kTile32 : 256, slots = c.dtype == GE_DTYPE_F32 ? 2 * kUnits : kUnits;
        const int64_t tiles = (x.rows + tile - 1) / tile * ((x.dim + tile - 1) / tile);
        const int64_t steps = plan.piece / 64;
        const int64_t most_bytes = 4 * std::max<int64_t>(x.rows, 1) * round_up(x.dim, 4);
        const int64_t fit = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kMaxSplits, steps), c.dhidden / most_bytes));
        int64_t best = INT64_MAX;
        plan.splits = 1;
        for (int64_t s = 1; s <= fit; ++s) {
            const int64_t cost = (tiles * s + slots - 1) / slots * ((steps + s - 1) / s + 12);
            if (cost < best) {
                best = cost;
                plan.splits = static_cast<int>(s);
            }
        }
    }
    return GE_OK;
}

inline int check_adamw_params(const ge_adamw_params& p, char* msg, size_t n) {
    if (!(p.beta1 >= 0 && p.beta1 < 1 && p.beta2 >= 0 && p.beta2 < 1 && p.eps >= 0) || !std::isfinite(p.lr) ||
        !std::isfinite(p.eps) || !std::isfinite(p.weight_decay) || std::isnan(p.grad_scale) || p.step < 1)
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "lr %g, betas %g and %g, eps %g, weight_decay %g, grad_scale %g, step %u",
                         p.lr, p.beta1, p.beta2, p.eps, p.weight_decay, p.grad_scale, p.step);
    return GE_OK;
}

}  // namespace head
}  // namespace ge

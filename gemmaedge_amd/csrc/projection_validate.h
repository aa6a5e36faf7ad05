// Host-side checks and geometry of the projection's calls (include/gemmaedge_projection.h),
// kept apart from the HIP launches so that they can be built and run without a
// device. Nothing here reads device memory.
#pragma once

#include <stdint.h>

#include <algorithm>

#include "../../include/gemmaedge_projection.h"
#include "head_validate.h"

namespace ge {
namespace projection {

using head::aligned_to;
using head::dtype_ok;
using head::elem_size;
using head::kTile32;
using head::kTileM;
using head::kUnits;
using head::round_up;
using head::stride_ok;

constexpr int kLowPlanes = 3;       // bf16 numbers that hold a low-rank value of bf16 operands
constexpr int kRowTile = 16;        // rows of a workgroup of the low-rank sums,
constexpr int kWideRows = 64;       // and of their form for many bf16 rows,
constexpr int kFewRows = 128;       // which more rows than this take
constexpr int kMaxLowSplits = 32;   // parts of such a sum
constexpr int kLowBlocks = 512;     // workgroups that they are split up for
constexpr int64_t kOuterBytes = 64LL << 20;  // most memory for the parts of an adapter's gradient

// Ranks are padded to whole steps of the matrix instructions.
inline int64_t rank_pad(int rank) { return round_up(rank, 32); }

// What a handle was created for and the workspaces' sizes in bytes.
struct Capacity {
    int max_rows, max_dim, max_out, max_rank, max_adapters, dtype;
    bool train;
    int64_t hpack;    // hidden states in padded rows
    int64_t wpack;    // a piece of the weights in padded rows
    int64_t u, du;    // the rows' low-rank values
    int64_t parts;    // float32 parts of u, du, dA or dB, one after the other
    int64_t order;    // rows sorted by adapter, and where each one's begin
    int64_t at;       // A transposed
    int64_t dpack;    // a piece of dout in padded rows
    int64_t dhidden;  // float32 parts of the hidden states' gradient
};

inline void size_workspace(Capacity& c) {
    const int64_t rows = c.max_rows, es = elem_size(c.dtype), dim = round_up(c.max_dim, head::kPadK);
    const int64_t out = round_up(c.max_out, kTileM);
    c.hpack = es * rows * dim;
    c.wpack = es * dim * std::min(out, std::max<int64_t>(kTileM, ((64LL << 20) / (2 * dim)) / kTileM * kTileM));
    const int64_t upad = rank_pad(c.max_rank);
    c.u = c.max_adapters ? (c.dtype == GE_DTYPE_F32 ? 4 : 2 * kLowPlanes) * rows * upad : 0;
    // no call has more parts than fill the card, or than this many
    c.parts = c.max_adapters ? 4 * upad * std::min(kMaxLowSplits * rows, kWideRows * std::max<int64_t>(kLowBlocks, (rows + kRowTile - 1) / kRowTile)) : 0;
    c.du = c.order = c.at = c.dpack = c.dhidden = 0;
    if (!c.train) return;
    c.dpack = es * rows * std::min(out, std::max<int64_t>(kTileM, (256LL << 20) / (es * rows) / kTileM * kTileM));
    const int64_t tiles = (rows + 255) / 256 * ((dim + 255) / 256);
    c.dhidden = 4 * std::min<int64_t>(256 * 256 * std::max<int64_t>(tiles, 1024),
                                      std::min<int64_t>(head::kMaxSplits, (out + 63) / 64) * rows * round_up(c.max_dim, 4));
    if (!c.max_adapters) return;
    c.du = c.u;
    // a small call's parts, and as many of a large one's as fit
    const int64_t least = 4LL * c.max_adapters * c.max_rank * std::max(c.max_dim, c.max_out);
    c.parts = std::max(c.parts, std::min(kOuterBytes, kMaxLowSplits * least));
    c.order = 4 * (rows + c.max_adapters + 1);
    c.at = es * c.max_adapters * static_cast<int64_t>(c.max_dim) * c.max_rank;
}

inline int check_create(int max_rows, int max_dim, int max_out, int max_rank, int max_adapters, int dtype, char* msg, size_t n) {
    if (max_rows < 1 || max_dim < 1 || max_out < 1 || max_rank < 0 || max_adapters < 0 || (max_rank == 0) != (max_adapters == 0))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "max_rows=%d max_dim=%d max_out=%d max_rank=%d max_adapters=%d", max_rows, max_dim,
                         max_out, max_rank, max_adapters);
    if (!dtype_ok(dtype)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "dtype %d", dtype);
    if (max_dim > GE_PROJECT_MAX_DIM || max_out > (1 << 24) || max_rows > (1 << 22) || max_rank > GE_PROJECT_MAX_RANK ||
        max_adapters > GE_PROJECT_MAX_ADAPTERS)
        return plan_fail(msg, n, GE_ERR_CAPACITY, "max_rows %d / max_dim %d / max_out %d / max_rank %d / max_adapters %d above %d / %d / %d / %d / %d",
                         max_rows, max_dim, max_out, max_rank, max_adapters, 1 << 22, GE_PROJECT_MAX_DIM, 1 << 24, GE_PROJECT_MAX_RANK,
                         GE_PROJECT_MAX_ADAPTERS);
    return GE_OK;
}

// How a call runs.
struct Plan {
    bool pack_h, pack_w, pack_d;  // operands copied into padded rows first
    int64_t kpad;                 // packed rows' length
    int tile_m, tile_n;           // of the forward product
    int piece;                    // outputs of a launch
    int splits;                   // parts of the outputs' sum in dhidden
    int64_t parts;                // bytes for those of the low-rank sums
};

// Parts of a low-rank sum over k elements: enough workgroups, of a few steps a wave at least;
// a join costs 4.5 us.
inline int low_splits(int rows, int k, bool wide) {
    const int tile = wide ? kWideRows : kRowTile, least = wide ? 256 : 2048;
    const int tiles = (rows + tile - 1) / tile;
    return std::max(1, std::min(std::min(kLowBlocks / std::max(tiles, 1), kMaxLowSplits), k / least));
}

// Parts of an adapter's gradient, of `size` elements for all of them: enough workgroups
// of 256 columns, of 256 rows each if the rows are spread evenly.
inline int outer_splits(int rows, int adapters, int cols, int64_t size, int64_t bytes) {
    const int64_t blocks = (cols + 255) / 256 * static_cast<int64_t>(adapters);
    const int64_t most = std::min<int64_t>(bytes / (4 * size), 65535 / adapters);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kMaxLowSplits, kLowBlocks / blocks),
                                                                  std::min<int64_t>(most, rows / (256LL * adapters)))));
}

inline int check_project(const Capacity& c, const ge_project_args& x, bool backward, Plan& plan, char* msg, size_t n) {
    if (x.rows < 0 || x.dim < 1 || x.out_dim < 1 || x.adapters < 0)
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "rows %d, dim %d, out_dim %d, adapters %d", x.rows, x.dim, x.out_dim, x.adapters);
    if (x.adapters > 0 && x.rank < 1) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "rank %d", x.rank);
    if (x.rows > c.max_rows || x.dim > c.max_dim || x.out_dim > c.max_out || x.adapters > c.max_adapters ||
        (x.adapters > 0 && x.rank > c.max_rank))
        return plan_fail(msg, n, GE_ERR_CAPACITY, "rows %d / dim %d / out_dim %d / rank %d / adapters %d above capacity %d / %d / %d / %d / %d",
                         x.rows, x.dim, x.out_dim, x.rank, x.adapters, c.max_rows, c.max_dim, c.max_out, c.max_rank, c.max_adapters);
    if (backward && !c.train) return plan_fail(msg, n, GE_ERR_CAPACITY, "the handle was created without train");
    if (!backward && !dtype_ok(x.out_dtype)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "out_dtype %d", x.out_dtype);
    const size_t es = elem_size(c.dtype);
    if (x.rows > 0) {
        if (!x.hidden || !x.weight || (!backward && !x.out) || (backward && !x.dout))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "hidden, weight, out or dout is NULL");
        if (!stride_ok(x.hidden_stride, x.rows, x.dim) || !stride_ok(x.weight_stride, x.out_dim, x.dim) ||
            (!backward && !stride_ok(x.out_stride, x.rows, x.out_dim)) || (backward && !stride_ok(x.dout_stride, x.rows, x.out_dim)) ||
            (backward && x.dhidden && !stride_ok(x.dhidden_stride, x.rows, x.dim)))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "rows overlap: a stride below dim %d or out_dim %d", x.dim, x.out_dim);
        if (x.adapters > 0 && (!x.a || !x.b || !x.scale || !x.adapter))
            return plan_fail(msg, n, GE_ERR_INVALID_ARG, "a, b, scale or adapter is NULL");
    }
    if (backward && x.adapters == 0 && (x.da || x.db)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "da or db without adapters");
    if (!aligned_to(x.hidden, es) || !aligned_to(x.weight, es) || !aligned_to(x.a, es) || !aligned_to(x.b, es) || !aligned_to(x.scale, 4) ||
        !aligned_to(x.adapter, 4) || (!backward && !aligned_to(x.out, elem_size(x.out_dtype))) || !aligned_to(x.dout, es) ||
        !aligned_to(x.dhidden, es) || !aligned_to(x.da, es) || !aligned_to(x.db, es))
        return plan_fail(msg, n, GE_ERR_INVALID_ARG, "a tensor is not aligned to its elements");

    // As in the vocabulary loss: bf16 tiles are fetched 16 bytes a lane into LDS, other
    // rows are packed first; offsets in a tile have 31 bits.
    auto direct = [&](const void* p, int64_t stride, int rows, int dim) {
        if (rows > 1 && stride > head::kMaxStride) return false;
        return c.dtype == GE_DTYPE_F32 || (aligned_to(p, 16) && (rows <= 1 || stride % 8 == 0) && dim % 8 == 0);
    };
    plan.pack_h = !direct(x.hidden, x.hidden_stride, x.rows, x.dim);
    plan.pack_w = !direct(x.weight, x.weight_stride, x.out_dim, x.dim);
    plan.pack_d = backward && !direct(x.dout, x.dout_stride, x.rows, x.out_dim);
    plan.kpad = round_up(x.dim, head::kPadK);
    if (c.dtype == GE_DTYPE_F32) {
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
        // 64 rows, width 2,816, 262,144 outputs: 279 us in tiles of 64 rows, 351 in two of 32, for
        // which the weights pass LDS twice
        const bool small = x.rows <= head::kSmallRows;
        plan.tile_m = small ? head::kSmallTileM : kTileM;
        plan.tile_n = x.rows <= head::kSmallTileN ? head::kSmallTileN : small ? 64 : x.rows <= 128 ? 128 : 256;
    }
    const int64_t out_pad = round_up(x.out_dim, kTileM);
    const int64_t row_tiles = (std::max(x.rows, 1) + plan.tile_n - 1) / plan.tile_n;
    int64_t piece = std::min(out_pad, head::kMostTiles / row_tiles * plan.tile_m / kTileM * kTileM);
    if (plan.pack_w) piece = std::min(piece, c.wpack / (static_cast<int64_t>(es) * plan.kpad) / kTileM * kTileM);
    if (plan.pack_d)  // a handle for millions of rows has room for longer rows than a tile's offsets reach
        piece = std::min(std::min<int64_t>(piece, head::kMaxStride), c.dpack / (static_cast<int64_t>(es) * std::max(x.rows, 1)) / kTileM * kTileM);
    plan.piece = static_cast<int>(piece);
    plan.splits = 1;
    plan.parts = c.parts;
    if (backward) {
        // Parts of the sum over a piece, as in the loss's: rounds of tiles times the steps of one.
        const int64_t tile = c.dtype == GE_DTYPE_F32 ? kTile32 : 256, slots = c.dtype == GE_DTYPE_F32 ? 2 * kUnits : kUnits;
        const int64_t tiles = (x.rows + tile - 1) / tile * ((x.dim + tile - 1) / tile);
        const int64_t steps = (std::min<int64_t>(piece, x.out_dim) + 63) / 64;
        const int64_t most_bytes = 4 * std::max<int64_t>(x.rows, 1) * round_up(x.dim, 4);
        const int64_t fit = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(head::kMaxSplits, steps), c.dhidden / most_bytes));
        int64_t best = INT64_MAX;
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

// Rows of `width` bytes in memory, `stride` >= width bytes apart. 128 bits: strides and rows that
// check_project takes multiply to more than 63.
struct Memory {
    const char* what;
    __int128 at, stride, width;
    int64_t rows;
};

// Whether two share a byte. Columns of one buffer share none, though their ranges do.
inline bool share(const Memory& a, const Memory& b) {
    if (a.rows > b.rows) return share(b, a);
    if (a.rows < 1 || a.width < 1 || b.width < 1) return false;
    if (a.at >= b.at + (b.rows - 1) * b.stride + b.width || b.at >= a.at + (a.rows - 1) * a.stride + a.width) return false;
    if (a.rows > 1 && a.stride == b.stride) {
        // b begins `first` rows and `right` bytes behind a: its row j lies beside a's rows first + j and, on the right, first + j + 1
        const __int128 off = b.at - a.at, first = off >= 0 ? off / a.stride : -((a.stride - 1 - off) / a.stride), right = off - first * a.stride;
        auto meet = [&](__int128 by) { return by > -b.rows && by < a.rows; };
        return (right < a.width && meet(first)) || (right + b.width > a.stride && meet(first + 1));
    }
    for (int64_t r = 0; r < a.rows; ++r) {
        const __int128 from = a.at + r * a.stride;
        // the first of b's rows that ends behind it
        const __int128 n = from < b.at + b.width ? 0 : (from - b.at - b.width) / b.stride + 1;
        if (n < b.rows && b.at + n * b.stride < from + a.width) return true;
    }
    return false;
}

// What a call writes lies apart from what it reads and from what else it writes. For a call that
// check_project has taken.
inline int check_memory(const Capacity& c, const ge_project_args& x, bool backward, char* msg, size_t n) {
    const int64_t es = elem_size(c.dtype), k = x.adapters, rank = k ? x.rank : 0;
    auto memory = [&](const char* what, const void* p, int64_t rows, __int128 width, int64_t stride, int64_t size) {
        return Memory{what, static_cast<__int128>(reinterpret_cast<uintptr_t>(p)), static_cast<__int128>(stride) * size, width * size, p ? rows : 0};
    };
    auto flat = [&](const char* what, const void* p, __int128 count, int64_t size) { return memory(what, p, 1, count, 0, size); };
    const __int128 a_size = static_cast<__int128>(k) * rank * x.dim, b_size = static_cast<__int128>(k) * rank * x.out_dim;
    const bool any = x.rows > 0;  // nothing is read without rows
    const Memory reads[] = {
        memory("hidden", x.hidden, x.rows, x.dim, x.hidden_stride, es),
        memory("weight", x.weight, any ? x.out_dim : 0, x.dim, x.weight_stride, es),
        memory("dout", x.dout, backward ? x.rows : 0, x.out_dim, x.dout_stride, es),
        flat("a", any ? x.a : nullptr, a_size, es),
        flat("b", any ? x.b : nullptr, b_size, es),
        flat("scale", any ? x.scale : nullptr, k, 4),
        flat("adapter", k ? x.adapter : nullptr, x.rows, 4),
    };
    const Memory writes[] = {
        memory("out", x.out, backward ? 0 : x.rows, x.out_dim, x.out_stride, elem_size(x.out_dtype)),
        memory("dhidden", x.dhidden, backward ? x.rows : 0, x.dim, x.dhidden_stride, es),
        flat("da", backward ? x.da : nullptr, a_size, es),
        flat("db", backward ? x.db : nullptr, b_size, es),
    };
    for (const Memory& w : writes) {
        for (const Memory& r : reads)
            if (share(w, r)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "%s overlaps %s", w.what, r.what);
        for (const Memory& v : writes)
            if (&v < &w && share(w, v)) return plan_fail(msg, n, GE_ERR_INVALID_ARG, "%s overlaps %s", w.what, v.what);
    }
    return GE_OK;
}

}  // namespace projection
}  // namespace ge

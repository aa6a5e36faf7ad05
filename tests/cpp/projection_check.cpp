// Host side of the projection (gemmaedge_amd/csrc/projection_validate.h) under the
// address and undefined-behaviour sanitizers: every refusal, and for random
// sizes that a call within a handle's capacity stays within its workspaces.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../../gemmaedge_amd/csrc/projection_validate.h"

using namespace ge::projection;
using ge::head::kPadK;

static int failures = 0;
#define CHECK(c)                                                         \
    do {                                                                 \
        if (!(c)) {                                                      \
            std::printf("line %d: %s (%s)\n", __LINE__, #c, msg);        \
            if (++failures > 20) std::exit(1);                           \
        }                                                                \
    } while (0)

static char msg[256];

static void* at(uintptr_t a) { return reinterpret_cast<void*>(a); }

static Capacity capacity(int rows, int dim, int out, int rank, int adapters, int dtype, bool train) {
    Capacity c{rows, dim, out, rank, adapters, dtype, train, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    size_workspace(c);
    return c;
}

static ge_project_args args() {
    ge_project_args x{};
    x.hidden = x.weight = x.a = x.b = at(4096);
    x.scale = static_cast<float*>(at(8192));
    x.adapter = static_cast<int32_t*>(at(8192));
    x.out = x.dhidden = x.da = x.db = at(1 << 20);
    x.dout = at(4096);
    x.hidden_stride = x.weight_stride = x.dhidden_stride = 64;
    x.out_stride = x.dout_stride = 1000;
    x.rows = 8;
    x.dim = 64;
    x.out_dim = 1000;
    x.rank = 8;
    x.adapters = 3;
    x.out_dtype = GE_DTYPE_F32;
    return x;
}

template <typename F>
static void refuses(int code, bool backward, F change) {
    const Capacity c = capacity(16, 64, 1000, 8, 4, GE_DTYPE_BF16, true);
    Plan p{};
    ge_project_args x = args();
    CHECK(check_project(c, x, backward, p, msg, sizeof(msg)) == GE_OK);
    change(x);
    CHECK(check_project(c, x, backward, p, msg, sizeof(msg)) == code);
}

static void refusals() {
    for (const bool back : {false, true}) {
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.rows = -1; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.dim = 0; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.out_dim = 0; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.adapters = -1; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.rank = 0; });
        refuses(GE_ERR_CAPACITY, back, [](auto& x) { x.rows = 17; });
        refuses(GE_ERR_CAPACITY, back, [](auto& x) { x.dim = 65; });
        refuses(GE_ERR_CAPACITY, back, [](auto& x) { x.out_dim = 1001; });
        refuses(GE_ERR_CAPACITY, back, [](auto& x) { x.rank = 9; });
        refuses(GE_ERR_CAPACITY, back, [](auto& x) { x.adapters = 5; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.hidden = nullptr; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.weight = nullptr; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.a = nullptr; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.b = nullptr; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.scale = nullptr; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.adapter = nullptr; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.hidden_stride = 63; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.weight_stride = 63; });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.hidden = at(4097); });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.b = at(4097); });
        refuses(GE_ERR_INVALID_ARG, back, [](auto& x) { x.scale = static_cast<float*>(at(4098)); });
    }
    refuses(GE_ERR_INVALID_ARG, false, [](auto& x) { x.out = nullptr; });
    refuses(GE_ERR_INVALID_ARG, false, [](auto& x) { x.out_dtype = 2; });
    refuses(GE_ERR_INVALID_ARG, false, [](auto& x) { x.out_stride = 999; });
    refuses(GE_ERR_INVALID_ARG, false, [](auto& x) { x.out = at(4098); });
    refuses(GE_ERR_INVALID_ARG, true, [](auto& x) { x.dout = nullptr; });
    refuses(GE_ERR_INVALID_ARG, true, [](auto& x) { x.dout_stride = 999; });
    refuses(GE_ERR_INVALID_ARG, true, [](auto& x) { x.dhidden_stride = 63; });
    refuses(GE_ERR_INVALID_ARG, true, [](auto& x) { x.adapters = 0; });
    refuses(GE_ERR_INVALID_ARG, true, [](auto& x) { x.db = at(4097); });
    Plan p{};
    const Capacity c = capacity(16, 64, 1000, 8, 4, GE_DTYPE_BF16, false);
    CHECK(check_project(c, args(), false, p, msg, sizeof(msg)) == GE_OK);
    CHECK(check_project(c, args(), true, p, msg, sizeof(msg)) == GE_ERR_CAPACITY);
}

// A call within the capacity stays within the workspaces, and its launches within their grids.
static void plans() {
    std::mt19937 rng(7);
    auto up_to = [&](int most) {
        const double x = std::uniform_real_distribution<double>(0.0, 1.0)(rng);
        return std::max(1, static_cast<int>(std::exp(x * std::log(static_cast<double>(most))) + 0.5));
    };
    for (int round = 0; round < 20000; ++round) {
        const int dtype = rng() % 2 ? GE_DTYPE_BF16 : GE_DTYPE_F32;
        const int64_t es = elem_size(dtype);
        const int rows = up_to(1 << 22), dim = up_to(65536), out = up_to(1 << 24), rank = up_to(256), adapters = up_to(65535);
        const Capacity c = capacity(rows, dim, out, rank, adapters, dtype, true);
        ge_project_args x = args();
        x.rows = round % 3 ? rows : up_to(rows);
        x.dim = round % 5 ? dim : up_to(dim);
        x.out_dim = round % 7 ? out : up_to(out);
        x.rank = up_to(rank);
        x.adapters = up_to(adapters);
        x.hidden_stride = x.weight_stride = x.dhidden_stride = x.dim + rng() % 2 * (rng() % 9);
        x.out_stride = x.dout_stride = static_cast<int64_t>(x.out_dim) + rng() % 9;
        if (rng() % 3 == 0) x.weight = x.dout = x.hidden = at(4096 + 2 * es);
        for (const bool back : {false, true}) {
            Plan p{};
            CHECK(check_project(c, x, back, p, msg, sizeof(msg)) == GE_OK);
            CHECK(p.piece >= kTileM && p.piece % kTileM == 0);
            const int64_t n = std::min(p.piece, x.out_dim);
            const int64_t tiles = (x.rows + p.tile_n - 1) / p.tile_n * ((n + p.tile_m - 1) / p.tile_m);
            CHECK(tiles <= ge::head::kMostTiles);
            if (p.pack_h) CHECK(es * x.rows * p.kpad <= c.hpack);
            if (p.pack_w) CHECK(es * n * p.kpad <= c.wpack);
            if (dtype == GE_DTYPE_BF16 && !p.pack_w) CHECK(x.weight_stride % 8 == 0 || x.out_dim == 1);
            CHECK(4 * x.rows * rank_pad(x.rank) <= c.u);
            for (const bool wide : {false, true})
                for (const int k : {x.dim, x.out_dim}) {
                    const int64_t parts = low_splits(x.rows, k, wide);
                    CHECK(parts >= 1 && (parts == 1 || 4 * parts * x.rows * rank_pad(x.rank) <= c.parts));
                }
            if (!back) continue;
            if (p.pack_d) CHECK(es * x.rows * round_up(n, kPadK) <= c.dpack && round_up(n, kPadK) <= ge::head::kMaxStride);
            CHECK(p.splits >= 1 && (p.splits == 1 || 4 * p.splits * x.rows * round_up(x.dim, 4) <= c.dhidden));
            CHECK(4LL * x.rows * round_up(x.dim, 4) <= c.dhidden);
            for (const int cols : {x.dim, x.out_dim}) {
                const int64_t size = static_cast<int64_t>(x.adapters) * x.rank * cols, parts = outer_splits(x.rows, x.adapters, cols, size, p.parts);
                CHECK(parts >= 1 && parts * x.adapters <= 65535 && (parts == 1 || 4 * parts * size <= c.parts));
            }
            CHECK(4LL * x.rows * rank_pad(x.rank) <= c.du);
            CHECK(4LL * (x.rows + x.adapters + 1) <= c.order);
            CHECK(es * x.adapters * x.dim * x.rank <= c.at);
        }
    }
}

int main() {
    refusals();
    plans();
    if (failures) return 1;
    std::printf("projection checks passed\n");
    return 0;
}

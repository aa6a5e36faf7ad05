// Host side of the answer head (gemmaedge_amd/csrc/head_validate.h) under the
// address and undefined-behaviour sanitizers: every refusal, and for random
// sizes that a call within a handle's capacity stays within its workspaces.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <random>

#include "../../gemmaedge_amd/csrc/head_validate.h"

using namespace ge::head;

static int failures = 0;
#define CHECK(c)                                                         \
    do {                                                                 \
        if (!(c)) {                                                      \
            std::printf("line %d: %s (%s)\n", __LINE__, #c, msg);        \
            if (++failures > 20) std::exit(1);                           \
        }                                                                \
    } while (0)

static char msg[256];

static Capacity capacity(int rows, int dim, int vocab, int dtype, bool train) {
    Capacity c{rows, dim, vocab, dtype, train, 0, 0, 0, 0, 0, 0, 0};
    size_workspace(c);
    return c;
}

static void* at(uintptr_t a) { return reinterpret_cast<void*>(a); }

static ge_norm_args norm_args() {
    ge_norm_args x{};
    x.x = x.weight = at(4096);
    x.y = x.dx = at(8192);
    x.dy = at(12288);
    x.mean = x.rstd = static_cast<float*>(at(16384));
    x.x_stride = x.y_stride = x.dy_stride = x.dx_stride = 64;
    x.rows = 8;
    x.dim = 64;
    x.weight_dtype = GE_DTYPE_F32;
    x.center = 1;
    x.eps = 1e-6f;
    return x;
}

static ge_loss_args loss_args() {
    ge_loss_args x{};
    x.hidden = x.weight = at(4096);
    x.targets = static_cast<int32_t*>(at(8192));
    x.loss = x.lse = static_cast<float*>(at(12288));
    x.grad = static_cast<float*>(at(16384));
    x.dhidden = x.dweight = at(32768);
    x.hidden_stride = x.weight_stride = x.dhidden_stride = x.dweight_stride = 64;
    x.rows = 8;
    x.dim = 64;
    x.vocab = 1000;
    return x;
}

template <typename F>
static int norm_with(F change, bool backward, bool train = true) {
    const Capacity c = capacity(16, 64, 1000, GE_DTYPE_BF16, train);
    ge_norm_args x = norm_args();
    change(x);
    return check_norm(c, x, backward, msg, sizeof(msg));
}
template <typename F>
static int loss_with(F change, bool backward, bool train = true) {
    const Capacity c = capacity(16, 64, 1000, GE_DTYPE_BF16, train);
    ge_loss_args x = loss_args();
    change(x);
    LossPlan plan{};
    return check_loss(c, x, backward, plan, msg, sizeof(msg));
}

static void refusals() {
    CHECK(check_create(0, 1, 1, 0, msg, sizeof(msg)) == GE_ERR_INVALID_ARG);
    CHECK(check_create(1, 0, 1, 0, msg, sizeof(msg)) == GE_ERR_INVALID_ARG);
    CHECK(check_create(1, 1, -1, 0, msg, sizeof(msg)) == GE_ERR_INVALID_ARG);
    CHECK(check_create(1, 1, 1, 2, msg, sizeof(msg)) == GE_ERR_INVALID_ARG);
    CHECK(check_create(1, GE_HEAD_MAX_DIM + 1, 1, 0, msg, sizeof(msg)) == GE_ERR_CAPACITY);
    CHECK(check_create(1, 1, (1 << 24) + 1, 0, msg, sizeof(msg)) == GE_ERR_CAPACITY);
    CHECK(check_create(16, 64, 1000, 1, msg, sizeof(msg)) == GE_OK);
    for (int back = 0; back < 2; ++back) {
        CHECK(norm_with([](ge_norm_args&) {}, back) == GE_OK);
        CHECK(norm_with([](ge_norm_args& x) { x.rows = 0; x.x = nullptr; x.rstd = nullptr; }, back) == GE_OK);
        CHECK(norm_with([](ge_norm_args& x) { x.center = 0; x.mean = nullptr; }, back) == GE_OK);
        CHECK(norm_with([](ge_norm_args& x) { x.rows = 1; x.x_stride = 0; }, back) == GE_OK);
        CHECK(norm_with([](ge_norm_args& x) { x.rows = -1; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.rows = 17; }, back) == GE_ERR_CAPACITY);
        CHECK(norm_with([](ge_norm_args& x) { x.dim = 0; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.dim = 65; }, back) == GE_ERR_CAPACITY);
        CHECK(norm_with([](ge_norm_args& x) { x.x_stride = 63; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.weight_dtype = 2; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.center = 2; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.x = nullptr; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.weight = nullptr; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.rstd = nullptr; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.mean = nullptr; }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.x = at(4097); }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.weight = at(4098); }, back) == GE_ERR_INVALID_ARG);
        CHECK(norm_with([](ge_norm_args& x) { x.rstd = static_cast<float*>(at(4098)); }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args&) {}, back) == GE_OK);
        CHECK(loss_with([](ge_loss_args& x) { x.rows = 0; x.hidden = nullptr; x.targets = nullptr; }, back) == GE_OK);
        CHECK(loss_with([](ge_loss_args& x) { x.rows = -1; }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.rows = 17; }, back) == GE_ERR_CAPACITY);
        CHECK(loss_with([](ge_loss_args& x) { x.vocab = 0; }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.vocab = 1001; }, back) == GE_ERR_CAPACITY);
        CHECK(loss_with([](ge_loss_args& x) { x.dim = 65; }, back) == GE_ERR_CAPACITY);
        CHECK(loss_with([](ge_loss_args& x) { x.softcap = std::numeric_limits<float>::infinity(); }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.softcap = std::nanf(""); }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.hidden = nullptr; }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.weight = nullptr; }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.targets = nullptr; }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.lse = nullptr; }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.hidden_stride = 63; }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.weight_stride = 63; }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.weight = at(4097); }, back) == GE_ERR_INVALID_ARG);
        CHECK(loss_with([](ge_loss_args& x) { x.targets = static_cast<int32_t*>(at(4098)); }, back) == GE_ERR_INVALID_ARG);
    }
    CHECK(norm_with([](ge_norm_args& x) { x.y = nullptr; }, false) == GE_ERR_INVALID_ARG);
    CHECK(norm_with([](ge_norm_args& x) { x.y_stride = 10; }, false) == GE_ERR_INVALID_ARG);
    CHECK(norm_with([](ge_norm_args& x) { x.eps = -1.f; }, false) == GE_ERR_INVALID_ARG);
    CHECK(norm_with([](ge_norm_args& x) { x.eps = std::nanf(""); }, false) == GE_ERR_INVALID_ARG);
    CHECK(norm_with([](ge_norm_args& x) { x.dy = nullptr; }, true) == GE_ERR_INVALID_ARG);
    CHECK(norm_with([](ge_norm_args& x) { x.dy_stride = 10; }, true) == GE_ERR_INVALID_ARG);
    CHECK(norm_with([](ge_norm_args& x) { x.dx_stride = 10; }, true) == GE_ERR_INVALID_ARG);
    CHECK(norm_with([](ge_norm_args& x) { x.dx = nullptr; }, true) == GE_OK);
    CHECK(norm_with([](ge_norm_args&) {}, true, false) == GE_ERR_CAPACITY);
    CHECK(loss_with([](ge_loss_args& x) { x.grad = nullptr; }, true) == GE_ERR_INVALID_ARG);
    CHECK(loss_with([](ge_loss_args& x) { x.dhidden_stride = 10; }, true) == GE_ERR_INVALID_ARG);
    CHECK(loss_with([](ge_loss_args& x) { x.dweight_stride = 10; }, true) == GE_ERR_INVALID_ARG);
    CHECK(loss_with([](ge_loss_args& x) { x.dweight = at(4097); }, true) == GE_ERR_INVALID_ARG);
    CHECK(loss_with([](ge_loss_args&) {}, true, false) == GE_ERR_CAPACITY);
    ge_adamw_params p{1e-3, 0.9, 0.999, 1e-8, 0.01, 1.0, 1, 0};
    CHECK(check_adamw_params(p, msg, sizeof(msg)) == GE_OK);
    for (int i = 0; i < 8; ++i) {
        ge_adamw_params q = p;
        if (i == 0) q.beta1 = 1.0;
        if (i == 1) q.beta2 = -0.1;
        if (i == 2) q.eps = -1.0;
        if (i == 3) q.lr = std::numeric_limits<double>::infinity();
        if (i == 4) q.weight_decay = std::nan("");
        if (i == 5) q.grad_scale = std::nan("");
        if (i == 6) q.step = 0;
        if (i == 7) q.beta1 = std::nan("");
        CHECK(check_adamw_params(q, msg, sizeof(msg)) == GE_ERR_INVALID_ARG);
    }
}

static int spread(std::mt19937& r, int hi) {
    const double u = std::uniform_real_distribution<double>(0.0, std::log(static_cast<double>(hi) + 0.999))(r);
    return std::max(1, std::min(hi, static_cast<int>(std::exp(u))));
}

// A call of any size within the handle's capacity fits its workspaces.
static void workspaces() {
    std::mt19937 r(11);
    for (int i = 0; i < 200000; ++i) {
        const int dtype = static_cast<int>(r() & 1);
        const Capacity c = capacity(spread(r, 40000), spread(r, GE_HEAD_MAX_DIM), spread(r, 1 << 24), dtype, true);
        ge_loss_args x = loss_args();
        x.rows = spread(r, c.max_rows);
        x.dim = spread(r, c.max_dim);
        x.vocab = spread(r, c.max_vocab);
        x.hidden_stride = x.dhidden_stride = x.dim + (r() & 1 ? 0 : static_cast<int>(r() % 100));
        x.weight_stride = x.dweight_stride = x.dim + (r() & 1 ? 0 : static_cast<int>(r() % 100));
        LossPlan p{};
        CHECK(check_loss(c, x, true, p, msg, sizeof(msg)) == GE_OK);
        const int64_t tiles = (x.vocab + p.tile_m - 1) / p.tile_m;
        CHECK(8 * tiles * x.rows <= c.stats);
        CHECK(8LL * x.rows <= c.row);
        if (p.pack_h) CHECK(2LL * p.planes * x.rows * p.kpad <= c.hpack);
        CHECK(p.pack_piece >= kTileM && p.pack_piece % kTileM == 0);
        CHECK(p.piece >= kTileM && p.piece % kTileM == 0 && p.piece <= p.pack_piece);
        if (p.pack_w) CHECK(2LL * p.planes * p.pack_piece * p.kpad <= c.wpack);
        CHECK(2LL * p.planes * p.rows_pad * p.piece <= c.dlogits);
        CHECK(p.rows_pad >= (x.rows + p.tile_n - 1) / p.tile_n * p.tile_n);
        const int64_t hld = (x.dim + 3) / 4 * 4;
        CHECK(p.splits >= 1 && 4LL * p.splits * x.rows * hld <= c.dhidden);
        // offsets within a tile stay in 31 bits
        CHECK(255LL * p.piece * 2 + 128 < (1LL << 31));
        CHECK(4LL * 2 * kNormParts * x.dim <= c.norm);
        if (failures) {
            std::printf("rows %d of %d, dim %d of %d, vocab %d of %d, dtype %d\n", x.rows, c.max_rows, x.dim, c.max_dim, x.vocab,
                        c.max_vocab, dtype);
            return;
        }
    }
}

int main() {
    refusals();
    workspaces();
    if (failures) return 1;
    std::printf("head checks passed\n");
    return 0;
}

// How the loss's calls are divided (gemmaedge_amd/csrc/head_validate.h), under the
// address and undefined-behaviour sanitizers: that the sizes of the tests of several
// pieces have several pieces, that what the kernels write fits the workspaces, and that
// a handle holds no more than its calls can use.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../../gemmaedge_amd/csrc/head_validate.h"

using namespace ge::head;

static int failures = 0;
static char msg[256];
#define CHECK(c)                                                  \
    do {                                                          \
        if (!(c)) {                                               \
            std::printf("line %d: %s (%s)\n", __LINE__, #c, msg); \
            if (++failures > 20) std::exit(1);                    \
        }                                                         \
    } while (0)

static Capacity capacity(int rows, int dim, int vocab, int dtype) {
    Capacity c{};
    c.max_rows = rows;
    c.max_dim = dim;
    c.max_vocab = vocab;
    c.dtype = dtype;
    c.train = true;
    size_workspace(c);
    return c;
}

static void* at(uintptr_t a) { return reinterpret_cast<void*>(a); }

static LossPlan plan_of(const Capacity& c, int rows, int dim, int vocab, int64_t weight_stride, uintptr_t weight = 4096) {
    ge_loss_args x{};
    x.hidden = x.dhidden = x.dweight = at(4096);
    x.weight = at(weight);
    x.targets = static_cast<int32_t*>(at(4096));
    x.loss = x.lse = static_cast<float*>(at(4096));
    x.grad = static_cast<float*>(at(4096));
    x.hidden_stride = x.dhidden_stride = x.dweight_stride = dim;
    x.weight_stride = weight_stride;
    x.rows = rows;
    x.dim = dim;
    x.vocab = vocab;
    LossPlan p{};
    CHECK(check_loss(c, x, true, p, msg, sizeof(msg)) == GE_OK);
    return p;
}

// What the kernels write and read of the logits' gradient and of its product with the weights.
static void fits(const Capacity& c, const LossPlan& p, int rows, int dim, int vocab) {
    const int64_t size = elem_size(c.dtype);
    CHECK(size * p.rows_pad * p.dz_ld <= c.dlogits);
    CHECK(p.dz_ld >= round_up(std::min(p.piece, vocab), p.tile_m) && p.rows_pad >= rows);
    // the last byte of a tile: 256 rows of bf16, 128 of float32, along the vocabulary, 64 across it
    CHECK((512 / size - 1) * p.dz_ld * size + 128 < 0x7ffffff0);
    CHECK(4LL * p.splits * rows * round_up(dim, 4) <= c.dhidden);
    // launches of less than 2^32 threads
    const int64_t row_tiles = (rows + p.tile_n - 1) / p.tile_n;
    CHECK(p.pack_piece >= kTileM && p.piece <= p.pack_piece);
    CHECK(row_tiles * ((std::min(p.pack_piece, vocab) + p.tile_m - 1) / p.tile_m) * 256 < (1LL << 32));
}

static void pieces() {
    struct Case {
        int rows, dim, vocab, dtype;
        int64_t weight_stride;
        uintptr_t weight;
        int pieces;
        bool packed;
    };
    const Case cases[] = {
        {4096, 64, 70001, GE_DTYPE_BF16, 64, 4096, 2, false},
        {2000, 128, 131075, GE_DTYPE_BF16, 128, 4096, 2, false},
        {4096, 64, 40001, GE_DTYPE_F32, 64, 4096, 2, false},
        {3000, 33, 100003, GE_DTYPE_F32, 33, 4096, 3, false},
        {5, 65536, 601, GE_DTYPE_F32, (1 << 21) + 8, 4096 + 12, 2, true},
    };
    for (const Case& k : cases) {
        const Capacity c = capacity(k.rows, k.dim, k.vocab, k.dtype);
        const LossPlan p = plan_of(c, k.rows, k.dim, k.vocab, k.weight_stride, k.weight);
        CHECK((k.vocab + p.piece - 1) / p.piece == k.pieces);
        CHECK(p.pack_w == k.packed);
        if (k.packed) CHECK((k.vocab + p.pack_piece - 1) / p.pack_piece > 1);
        if (k.dtype == GE_DTYPE_BF16) CHECK(p.tile_n == 256);
        fits(c, p, k.rows, k.dim, k.vocab);
    }
}

static int spread(std::mt19937& r, int hi) {
    const double u = std::uniform_real_distribution<double>(0.0, std::log(static_cast<double>(hi) + 0.999))(r);
    return std::max(1, std::min(hi, static_cast<int>(std::exp(u))));
}

// Handles of every size that can be created, and calls within them.
static void random_plans() {
    std::mt19937 r(5);
    for (int i = 0; i < 200000 && !failures; ++i) {
        const Capacity c = capacity(spread(r, 1 << 22), spread(r, GE_HEAD_MAX_DIM), spread(r, 1 << 24), static_cast<int>(r() & 1));
        const int rows = spread(r, c.max_rows), dim = spread(r, c.max_dim), vocab = spread(r, c.max_vocab);
        const LossPlan p = plan_of(c, rows, dim, vocab, dim + static_cast<int64_t>(r() % 9));
        fits(c, p, rows, dim, vocab);
        if (failures)
            std::printf("rows %d of %d, dim %d of %d, vocab %d of %d, dtype %d: rows of %lld\n", rows, c.max_rows, dim, c.max_dim, vocab,
                        c.max_vocab, c.dtype, static_cast<long long>(p.dz_ld));
    }
    // few rows of a handle for very many, and the largest vocabulary
    for (int dtype = 0; dtype < 2; ++dtype)
        for (int rows : {1, 200, 256, 257, 512}) {
            const Capacity c = capacity(1 << 22, 8, 1 << 24, dtype);
            fits(c, plan_of(c, rows, 8, 1 << 24, 8), rows, 8, 1 << 24);
        }
}

// The parts of the hidden states' gradient take what the handle's calls can use, and their number does not depend on it.
static void parts() {
    CHECK(capacity(16, 64, 1, GE_DTYPE_BF16).dhidden == 4LL * 4 * 16 * 64);
    CHECK(capacity(16, 64, 1000, GE_DTYPE_F32).dhidden == 4LL * 16 * 16 * 64);
    std::mt19937 r(6);
    for (int i = 0; i < 100000 && !failures; ++i) {
        Capacity c = capacity(spread(r, 1 << 22), spread(r, GE_HEAD_MAX_DIM), spread(r, 1 << 24), static_cast<int>(r() & 1));
        const int rows = spread(r, c.max_rows), dim = spread(r, c.max_dim), vocab = spread(r, c.max_vocab);
        CHECK(c.dhidden <= 4LL * 32 * c.max_rows * round_up(c.max_dim, 4));
        const int splits = plan_of(c, rows, dim, vocab, dim).splits;
        c.dhidden = 4LL * 256 * 256 * std::max<int64_t>((c.max_rows + 255LL) / 256 * ((c.max_dim + 255) / 256), 1024);
        CHECK(plan_of(c, rows, dim, vocab, dim).splits == splits);
    }
}

int main() {
    pieces();
    random_plans();
    parts();
    if (failures) return 1;
    std::printf("head plans passed\n");
    return 0;
}

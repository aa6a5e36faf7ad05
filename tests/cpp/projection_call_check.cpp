// Host side of the projection's calls (gemmaedge_amd/csrc/projection_validate.h) under the
// address and undefined-behaviour sanitizers, at the sizes where a plan can go wrong.
#include <cstdio>
#include <cstdlib>
#include <ctime>
#include <random>

#include "../../gemmaedge_amd/csrc/projection_validate.h"

using namespace ge::projection;

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

static Capacity capacity(int rows, int dim, int out, int rank, int adapters, int dtype) {
    Capacity c{};
    c.max_rows = rows;
    c.max_dim = dim;
    c.max_out = out;
    c.max_rank = rank;
    c.max_adapters = adapters;
    c.dtype = dtype;
    c.train = true;
    size_workspace(c);
    return c;
}

// Calls without rows, whose tensors may have no address or any: outputs of every width, both types.
static void no_rows() {
    for (const int dtype : {GE_DTYPE_BF16, GE_DTYPE_F32})
        for (int out = 1; out <= 1100; out += out < 40 ? 1 : 53)
            for (const int dim : {1, 7, 64, 65})
                for (const int adapters : {0, 3})
                    for (const uintptr_t p : {uintptr_t{0}, uintptr_t{4096}, uintptr_t{4100}}) {
                        const Capacity c = capacity(5, 65, 1100, 8, 3, dtype);
                        ge_project_args x{};
                        x.hidden = x.weight = x.dout = x.a = x.b = at(p);
                        x.out = x.dhidden = at(p);
                        x.dim = dim;
                        x.out_dim = out;
                        x.rank = 8;
                        x.adapters = adapters;
                        x.out_dtype = GE_DTYPE_F32;
                        x.hidden_stride = x.weight_stride = x.dhidden_stride = dim;
                        x.out_stride = x.dout_stride = out;
                        for (const bool back : {false, true}) {
                            Plan plan{};
                            CHECK(check_project(c, x, back, plan, msg, sizeof(msg)) == GE_OK);
                            CHECK(plan.piece >= kTileM && plan.splits >= 1);
                        }
                    }
}

// share() against every pair of rows.
static void shared_bytes() {
    std::mt19937 rng(3);
    for (int round = 0; round < 200000; ++round) {
        Memory m[2];
        for (Memory& x : m) {
            x.width = rng() % 6;
            x.stride = x.width + rng() % 12;
            x.rows = rng() % 6;
            x.at = 1000 + rng() % 60;
        }
        if (rng() % 2) m[1].stride = m[0].stride = std::max(m[0].stride, m[1].stride);
        bool want = false;
        for (int64_t i = 0; i < m[0].rows; ++i)
            for (int64_t j = 0; j < m[1].rows; ++j) {
                const __int128 a = m[0].at + i * m[0].stride, b = m[1].at + j * m[1].stride;
                want |= m[0].width > 0 && m[1].width > 0 && a < b + m[1].width && b < a + m[0].width;
            }
        CHECK(share(m[0], m[1]) == want && share(m[1], m[0]) == want);
    }
    // columns of one buffer with many rows, as quickly as others
    const Memory left{"", 4096, 256, 128, 1 << 22}, right{"", 4096 + 128, 256, 128, 1 << 22};
    const clock_t began = clock();
    for (int i = 0; i < 1000; ++i) CHECK(!share(left, right) && !share(right, left));
    CHECK(clock() - began < CLOCKS_PER_SEC);
    // the largest that check_project takes
    const Memory far{"", 1, __int128{4} << 40, 1 << 18, 1 << 24}, one{"", (__int128{4} << 63) + 1, 4, 4, 1};
    CHECK(share(far, one) && share(one, far));
}

// Calls whose outputs lie apart from all else, and the same with one output moved.
static void apart() {
    constexpr int kRows = 6, kDim = 16, kOut = 40, kRank = 4, kAdapters = 3;
    const Capacity c = capacity(kRows, kDim, kOut, kRank, kAdapters, GE_DTYPE_BF16);
    auto good = [&] {
        ge_project_args x{};
        uintptr_t next = 1 << 20;
        auto place = [&](int64_t bytes) { return at((next += 65536) - bytes); };
        x.rows = kRows;
        x.dim = kDim;
        x.out_dim = kOut;
        x.rank = kRank;
        x.adapters = kAdapters;
        x.out_dtype = GE_DTYPE_F32;
        x.hidden_stride = x.weight_stride = x.dhidden_stride = kDim;
        x.out_stride = x.dout_stride = kOut;
        x.hidden = place(2 * kRows * kDim);  // each ends where the next 64 KiB begin
        x.weight = place(2 * kOut * kDim);
        x.dout = place(2 * kRows * kOut);
        x.a = place(2 * kAdapters * kRank * kDim);
        x.b = place(2 * kAdapters * kRank * kOut);
        x.scale = static_cast<float*>(place(4 * kAdapters));
        x.adapter = static_cast<int32_t*>(place(4 * kRows));
        x.out = place(4 * kRows * kOut);
        x.dhidden = place(2 * kRows * kDim);
        x.da = place(2 * kAdapters * kRank * kDim);
        x.db = place(2 * kAdapters * kRank * kOut);
        return x;
    };
    auto check = [&](bool back, int want, auto change) {
        ge_project_args x = good();
        change(x);
        Plan plan{};
        CHECK(check_project(c, x, back, plan, msg, sizeof(msg)) == GE_OK);
        msg[0] = 0;
        CHECK(check_memory(c, x, back, msg, sizeof(msg)) == want);
    };
    auto behind = [](const void* p, int64_t bytes) { return static_cast<char*>(const_cast<void*>(p)) + bytes; };
    for (const bool back : {false, true}) check(back, GE_OK, [](auto&) {});
    // an output over the last bytes of each input, and right behind it
#define AT_END(back, output, input, bytes)                                                                  \
    do {                                                                                                    \
        check(back, GE_ERR_INVALID_ARG, [&](auto& x) { x.output = behind(x.input, (bytes) - 4); });         \
        check(back, GE_OK, [&](auto& x) { x.output = behind(x.input, bytes); });                            \
    } while (0)
#define AT_ENDS(back, output)                                                                               \
    do {                                                                                                    \
        AT_END(back, output, hidden, 2 * kRows * kDim);                                                     \
        AT_END(back, output, weight, 2 * kOut * kDim);                                                      \
        AT_END(back, output, a, 2 * kAdapters * kRank * kDim);                                              \
        AT_END(back, output, b, 2 * kAdapters * kRank * kOut);                                              \
        AT_END(back, output, scale, 4 * kAdapters);                                                         \
        AT_END(back, output, adapter, 4 * kRows);                                                           \
    } while (0)
    AT_ENDS(false, out);
    AT_ENDS(true, dhidden);
    AT_ENDS(true, da);
    AT_ENDS(true, db);
    AT_END(true, dhidden, dout, 2 * kRows * kOut);
    AT_END(true, da, dout, 2 * kRows * kOut);
    AT_END(true, db, dout, 2 * kRows * kOut);
    AT_END(true, da, dhidden, 2 * kRows * kDim);
    AT_END(true, db, da, 2 * kAdapters * kRank * kDim);
    // what a call does not use may lie anywhere
    check(false, GE_OK, [&](auto& x) { x.dout = x.out; x.dhidden = x.da = x.db = const_cast<void*>(x.hidden); });
    check(true, GE_OK, [&](auto& x) { x.out = const_cast<void*>(x.hidden); });
    check(false, GE_OK, [&](auto& x) { x.adapters = 0; x.out = const_cast<void*>(x.b); });
    check(true, GE_OK, [&](auto& x) { x.rows = 0; x.dhidden = const_cast<void*>(x.weight); x.da = behind(x.hidden, 0); });
    check(true, GE_OK, [&](auto& x) { x.dhidden = x.da = nullptr; });
    // columns of one buffer, and the same one element further
    for (const int off : {kOut, kOut - 1})
        check(true, off == kOut ? GE_OK : GE_ERR_INVALID_ARG, [&](auto& x) {
            x.dhidden = behind(x.dout, 2 * off);
            x.dout_stride = x.dhidden_stride = 100;
        });
    // one row: strides mean nothing
    check(true, GE_OK, [&](auto& x) { x.rows = 1; x.hidden_stride = 0; x.dhidden = behind(x.hidden, 2 * kDim); });
}

int main() {
    no_rows();
    shared_bytes();
    apart();
    if (failures) return 1;
    std::printf("projection call checks passed\n");
    return 0;
}

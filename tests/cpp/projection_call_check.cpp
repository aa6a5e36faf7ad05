// Host side of the projection's calls (gemmaedge_amd/csrc/projection_validate.h) under the
// address and undefined-behaviour sanitizers, at the sizes where a plan can go wrong.
#include <cstdio>
#include <cstdlib>
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

int main() {
    no_rows();
    if (failures) return 1;
    std::printf("projection call checks passed\n");
    return 0;
}

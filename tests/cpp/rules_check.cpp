// Host side of the rules (gemmaedge_amd/csrc/rules_validate.h) under the address and
// undefined-behaviour sanitizers: the largest sizes and strides that a call may have.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "../../gemmaedge_amd/csrc/rules_validate.h"

using namespace ge::rules;

static int failures = 0;
#define CHECK(c)                                                         \
    do {                                                                 \
        if (!(c)) {                                                      \
            std::printf("line %d: %s (%s)\n", __LINE__, #c, msg);        \
            if (++failures > 20) std::exit(1);                           \
        }                                                                \
    } while (0)

static char msg[256];

static ge_rule_args args(uintptr_t logits, uintptr_t out) {
    ge_rule_args x{};
    x.logits = reinterpret_cast<const void*>(logits);
    x.out = reinterpret_cast<void*>(out);
    x.dtype = GE_DTYPE_BF16;
    x.out_dtype = GE_DTYPE_F32;
    x.rows = 1 << 24;
    x.vocab = 100;
    x.row_stride = x.out_stride = 100;
    x.params = ge_rule_params{0.f, 1.f, 0.f, 0.f};
    return x;
}

int main() {
    constexpr uintptr_t kFar = uintptr_t{1} << 50;
    // The rows of either side 2^40 elements apart, beyond what 63 bits hold; the other in front of them or among them.
    for (const int64_t stride : {int64_t{100}, int64_t{1} << 36, int64_t{1} << 39, int64_t{1} << 40}) {
        ge_rule_args x = args(kFar, 4096);
        x.row_stride = stride;
        CHECK(check_rules(x, msg, sizeof(msg)) == GE_OK);
        x = args(4096, kFar);
        x.out_stride = stride;
        CHECK(check_rules(x, msg, sizeof(msg)) == GE_OK);
        const int among = stride > 100 ? GE_ERR_INVALID_ARG : GE_OK;
        x = args(4096, kFar);
        x.row_stride = stride;
        CHECK(check_rules(x, msg, sizeof(msg)) == among);
        x = args(kFar, 4096);
        x.out_stride = stride;
        CHECK(check_rules(x, msg, sizeof(msg)) == among);
    }
    // A byte more or less than the rows take.
    const uintptr_t rows = 4096 + 2 * ((uintptr_t{1} << 24) * 100);
    CHECK(check_rules(args(4096, rows), msg, sizeof(msg)) == GE_OK);
    CHECK(check_rules(args(4096, rows - 4), msg, sizeof(msg)) == GE_ERR_INVALID_ARG);
    // At the end of the address space, and all of it.
    ge_rule_args x = args(UINTPTR_MAX - 511, 4096);
    x.rows = 1;
    x.vocab = 256;
    CHECK(check_rules(x, msg, sizeof(msg)) == GE_OK);
    x.vocab = kMostVocab;
    x.row_stride = x.out_stride = int64_t{1} << 40;
    x.rows = kMostRows;
    CHECK(check_rules(x, msg, sizeof(msg)) == GE_ERR_INVALID_ARG);
    // In place: as far apart as may be.
    x = args(4096, 4096);
    x.out_dtype = x.dtype;
    x.row_stride = x.out_stride = int64_t{1} << 40;
    CHECK(check_rules(x, msg, sizeof(msg)) == GE_OK);
    x.out_stride = x.row_stride + 1;
    CHECK(check_rules(x, msg, sizeof(msg)) == GE_ERR_INVALID_ARG);
    if (failures) return 1;
    std::printf("rules checks passed\n");
    return 0;
}

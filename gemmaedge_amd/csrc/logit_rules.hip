// Penalties, biases and masks on rows of logits (include/gemmaedge_rules.h).
//
// A workgroup takes a piece of a row's vocabulary and counts in LDS which of the
// row's history falls into it: a word a token, the low 31 bits its number behind
// the prompt, the highest bit that the prompt has it (integers, so the order of
// the additions does not matter). Every workgroup of a row reads the whole
// history, which the caches answer; nothing is sorted and no memory but LDS is
// needed. Biases go the same way: a word a token with the number of its last
// entry. Then the piece's logits pass once, 8 a lane. In place without a softcap
// the logits that nothing applies to are neither read nor written, and where
// none of 8 is allowed they are written without being read.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "ge_math.h"
#include "head_internal.h"
#include "rules_validate.h"

namespace ge {
namespace rules {
namespace {

using head::from_f32;
using head::to_f32;

constexpr int kUnit = 8;             // neighbouring tokens of a lane
constexpr uint32_t kPrompt = 1u << 31;

template <typename T>
struct Unit {
    T v[kUnit];
};
// The unit at p, of which n tokens are the row's.
template <typename T>
__device__ __forceinline__ Unit<T> load_unit(const T* p, int n) {
    Unit<T> u{};
    if (n >= kUnit) {
        __builtin_memcpy(&u, p, sizeof(u));
    } else {
#pragma unroll
        for (int e = 0; e < kUnit; ++e)
            if (e < n) u.v[e] = p[e];
    }
    return u;
}
template <typename T>
__device__ __forceinline__ void store_unit(T* p, int n, const float (&x)[kUnit]) {
    Unit<T> u;
#pragma unroll
    for (int e = 0; e < kUnit; ++e) u.v[e] = from_f32<T>(x[e]);
    if (n >= kUnit) {
        __builtin_memcpy(p, &u, sizeof(u));
    } else {
#pragma unroll
        for (int e = 0; e < kUnit; ++e)
            if (e < n) p[e] = u.v[e];
    }
}

// f(i, ids[i]) for the i < n that are this thread's, four neighbours
// a load and four loads in flight.
template <int kThreads, typename F>
__device__ __forceinline__ void for_list(const int32_t* ids, int n, F f) {
    struct Four {
        int32_t v[4];
    };
    constexpr int kStep = 4 * kThreads;
    const int64_t whole = n & ~3;
    for (int64_t i = threadIdx.x * 4; i < whole; i += 4 * kStep) {
        Four q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (whole - i > k * kStep) __builtin_memcpy(&q[k], ids + i + k * kStep, sizeof(Four));
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (whole - i > k * kStep) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f(static_cast<int>(i) + k * kStep + e, q[k].v[e]);
            }
    }
    const int rest = (n & ~3) + static_cast<int>(threadIdx.x);
    if (rest < n && threadIdx.x < 3) f(rest, ids[rest]);
}

template <typename T, typename O, bool kBias, int kThreads, int kUnits>
__global__ __launch_bounds__(kThreads) void rules_kernel(ge_rule_args x, int first_row, int pieces) {
    constexpr int kPiece = kThreads * kUnits * kUnit;
    __shared__ __align__(16) uint32_t words[kPiece];
    __shared__ __align__(16) int32_t last[kBias ? kPiece : 4];
    const int64_t row = first_row + blockIdx.x / pieces;
    const int piece = blockIdx.x % pieces;
    const int t0 = piece * kPiece;                     // the piece's first token
    const int length = min(kPiece, x.vocab - t0);
    const ge_rule_params p = x.row_params ? x.row_params[row] : x.params;
    const T* const in = static_cast<const T*>(x.logits) + row * x.row_stride + t0;
    O* const out = static_cast<O*>(x.out) + row * x.out_stride + t0;
    const bool dense = static_cast<const void*>(x.logits) != x.out || p.softcap > 0.0f;

    const uint32_t* mask = x.mask;
    if (mask) {
        const int m = x.mask_rows ? x.mask_rows[row] : static_cast<int>(row);
        mask = m >= 0 && m < x.masks ? mask + m * x.mask_stride : nullptr;
    }
    Unit<T> raw[kUnits];
    if (dense) {
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const int at = (j * kThreads + threadIdx.x) * kUnit;
            raw[j] = load_unit(in + at, length - at);
        }
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int at = (j * kThreads + threadIdx.x) * kUnit;
#pragma unroll
        for (int e = 0; e < kUnit; e += 4) {
            *reinterpret_cast<uint4*>(&words[at + e]) = make_uint4(0, 0, 0, 0);
            if (kBias) *reinterpret_cast<uint4*>(&last[at + e]) = make_uint4(0, 0, 0, 0);
        }
    }
    __syncthreads();

    bool any = false;
    const int prompt = x.prompt_len ? x.prompt_len[row] : 0;
    auto count = [&](int id, bool behind) {
        const uint32_t at = static_cast<uint32_t>(id) - static_cast<uint32_t>(t0);
        if (at >= static_cast<uint32_t>(length)) return;
        any = true;
        if (behind)
            atomicAdd(&words[at], 1u);
        else
            atomicOr(&words[at], kPrompt);
    };
    if (x.history) {
        const int from = x.history_offsets[row], n = x.history_offsets[row + 1] - from;
        for_list<kThreads>(x.history + from, n, [&](int i, int id) { count(id, i >= prompt); });
    } else if (x.ring) {
        const int len = x.ring_len[row], cap = x.ring_capacity;
        for_list<kThreads>(x.ring + row * cap, min(len, cap), [&](int i, int id) {
            // the last of the appended ids that went to place i
            const int number = len <= cap ? i : i + (len - 1 - i) / cap * cap;
            count(id, number >= prompt);
        });
    }
    int bias_from = 0;
    if (kBias) {
        bias_from = x.bias_offsets[row];
        for_list<kThreads>(x.bias_ids + bias_from, x.bias_offsets[row + 1] - bias_from, [&](int i, int id) {
            const uint32_t at = static_cast<uint32_t>(id) - static_cast<uint32_t>(t0);
            if (at >= static_cast<uint32_t>(length)) return;
            any = true;
            atomicMax(&last[at], i + 1);
        });
    }
    const bool touched = __syncthreads_or(any);  // some word is not 0
    if (x.flags_out && piece == 0) {
        bool allowed = !mask;
        if (mask) {
            const int whole = x.vocab / 32;
#pragma unroll 4
            for (int i = threadIdx.x; i < whole; i += kThreads) allowed |= mask[i] != 0;
            if (threadIdx.x == 0 && x.vocab % 32) allowed |= (mask[whole] & ((1u << (x.vocab % 32)) - 1)) != 0;
        }
        allowed = __syncthreads_or(allowed);
        if (threadIdx.x == 0) x.flags_out[row] = allowed ? 0 : GE_RULE_EMPTY;
    }
    if (!dense && !touched && !mask) return;

#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int at = (j * kThreads + threadIdx.x) * kUnit;
        const int n = length - at;  // tokens of the unit that are the row's
        if (n <= 0) continue;
        const uint32_t ok = mask ? mask[(t0 + at) >> 5] >> (at & 31) & 0xffu : 0xffu;
        uint32_t w[kUnit] = {}, b[kUnit] = {};
        bool some = false;
        if (touched) {
#pragma unroll
            for (int e = 0; e < kUnit; ++e) {
                w[e] = words[at + e];
                if (kBias) b[e] = last[at + e];
                some |= (w[e] | b[e]) != 0;
            }
        }
        float v[kUnit];
        if (!dense) {
            if (!some && ok == 0xffu) continue;
            if (ok != 0)
                raw[j] = load_unit(in + at, n);
            else
                raw[j] = Unit<T>{};
        }
#pragma unroll
        for (int e = 0; e < kUnit; ++e) v[e] = softcap(to_f32(raw[j].v[e]), p.softcap);
        if (some) {
#pragma unroll
            for (int e = 0; e < kUnit; ++e) {
                const float c = static_cast<float>(w[e] & ~kPrompt);
                if (w[e] != 0) v[e] = penalize(v[e], p.repetition_penalty);
                if (c > 0.0f) v[e] = v[e] - p.frequency_penalty * c - p.presence_penalty;
                if (kBias && b[e] != 0) v[e] += x.bias_values[bias_from + b[e] - 1];
            }
        }
#pragma unroll
        for (int e = 0; e < kUnit; ++e)
            if (!(ok >> e & 1)) v[e] = -__builtin_inff();
        store_unit(out + at, n, v);
    }
}

template <typename T, typename O, bool kBias>
void launch(const ge_rule_args& x, hipStream_t st) {
    auto run = [&](auto threads, auto units) {
        constexpr int kThreads = decltype(threads)::value, kUnits = decltype(units)::value;
        constexpr int kPiece = kThreads * kUnits * kUnit;
        const int pieces = (x.vocab + kPiece - 1) / kPiece;
        const int most = (1 << 22) / pieces;  // rows of a launch, of less than 2^32 threads
        for (int r = 0; r < x.rows; r += most)
            rules_kernel<T, O, kBias, kThreads, kUnits>
                <<<static_cast<unsigned>(std::min(most, x.rows - r)) * pieces, kThreads, 0, st>>>(x, r, pieces);
    };
    if (static_cast<int64_t>(x.rows) * ((x.vocab + 8191) / 8192) >= 512)
        run(std::integral_constant<int, 512>{}, std::integral_constant<int, 2>{});
    else
        run(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
}

}  // namespace
}  // namespace rules
}  // namespace ge

extern "C" int ge_apply_rules(void* stream, const ge_rule_args* args) {
    using namespace ge::rules;
    char msg[256] = "";
    if (!args) return ge::report(GE_ERR_INVALID_ARG, "args is NULL");
    const ge_rule_args& x = *args;
    if (const int rc = check_rules(x, msg, sizeof(msg))) return ge::report(rc, msg);
    if (x.rows == 0) return GE_OK;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto by_out = [&](auto t, auto bias) {
        using T = decltype(t);
        if (x.out_dtype == GE_DTYPE_F32)
            launch<T, float, decltype(bias)::value>(x, st);
        else
            launch<T, uint16_t, decltype(bias)::value>(x, st);
    };
    auto by_bias = [&](auto t) {
        if (x.bias_ids)
            by_out(t, std::integral_constant<bool, true>{});
        else
            by_out(t, std::integral_constant<bool, false>{});
    };
    if (x.dtype == GE_DTYPE_F32)
        by_bias(float{});
    else
        by_bias(uint16_t{});
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return GE_OK;
    ge::plan_fail(msg, sizeof(msg), 0, "launch (rules): %s", hipGetErrorString(e));
    return ge::report(GE_ERR_DEVICE, msg);
}

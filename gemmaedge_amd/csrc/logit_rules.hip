// Penalties, biases and masks on rows of logits (include/gemmaedge_rules.h).
//
// Two kinds of work that need each other only at single tokens:
//
//   stream  every token of a piece of a row: softcap, mask, conversion, 8 tokens a
//           lane. In place without a softcap only tokens that are not allowed are
//           written, and nothing is read but the mask.
//   single  the tokens of a row's history and biases: a workgroup (or several, each
//           for a slice of the vocabulary) counts them in LDS and gives each its
//           final value, from the logit on.
//
// Into another memory the single tokens come in a second launch, over what the first has
// streamed. In place without a softcap the two touch different tokens and share a
// launch. Rows that are capped in place need both at once (merged): a rounded cap is no
// logit to go on from.
//
// Counting is by integers, so the order of the additions does not matter. Where a word for
// each token of a slice fits LDS the words are it; else a hash table takes up to kMostHashed
// ids of whatever vocabulary, and longer lists are read again for each piece of the slice.
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
// and where either side is float32: a wave's 16-byte accesses then lie together
template <typename T, typename O>
constexpr int kStreamUnit = sizeof(T) == 2 && sizeof(O) == 2 ? kUnit : 4;
constexpr uint32_t kPrompt = 1u << 31;

template <typename T, int kN>
struct Unit {
    T v[kN];
};
// The unit at p, of which n tokens are the row's.
template <int kN, typename T>
__device__ __forceinline__ Unit<T, kN> load_unit(const T* p, int n) {
    Unit<T, kN> u{};
    if (n >= kN) {
        __builtin_memcpy(&u, p, sizeof(u));
    } else {
#pragma unroll
        for (int e = 0; e < kN; ++e)
            if (e < n) u.v[e] = p[e];
    }
    return u;
}
template <typename T, int kN>
__device__ __forceinline__ void store_unit(T* p, int n, const float (&x)[kN]) {
    Unit<T, kN> u;
#pragma unroll
    for (int e = 0; e < kN; ++e) u.v[e] = from_f32<T>(x[e]);
    if (n >= kN) {
        __builtin_memcpy(p, &u, sizeof(u));
    } else {
#pragma unroll
        for (int e = 0; e < kN; ++e)
            if (e < n) p[e] = u.v[e];
    }
}

// f(i, ids[i]) for the i < n that are this thread's, four neighbours a load and four
// loads in flight.
template <int kThreads, typename F>
__device__ __forceinline__ void for_list(const int32_t* ids, int n, F f) {
    struct Four {
        int32_t v[4];
    };
    constexpr int kStep = 4 * kThreads, kLoads = 4;
    const int64_t whole = n & ~3;
    for (int64_t i = threadIdx.x * 4; i < whole; i += kLoads * kStep) {
        Four q[kLoads];
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
            if (whole - i > k * kStep) __builtin_memcpy(&q[k], ids + i + k * kStep, sizeof(Four));
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
            if (whole - i > k * kStep) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f(static_cast<int>(i) + k * kStep + e, q[k].v[e]);
            }
    }
    if (threadIdx.x < (n & 3)) f((n & ~3) + static_cast<int>(threadIdx.x), ids[(n & ~3) + threadIdx.x]);
}

// ---- what a row asks for ----------------------------------------------------------

__device__ __forceinline__ ge_rule_params row_rules(const ge_rule_args& x, int64_t row) { return x.row_params ? x.row_params[row] : x.params; }

// The row's mask, or NULL.
__device__ __forceinline__ const uint32_t* row_mask(const ge_rule_args& x, int64_t row) {
    if (!x.mask) return nullptr;
    const int m = x.mask_rows ? x.mask_rows[row] : static_cast<int>(row);
    return m >= 0 && m < x.masks ? x.mask + m * x.mask_stride : nullptr;
}
__device__ __forceinline__ bool allows(const uint32_t* mask, int token) { return !mask || (mask[token >> 5] >> (token & 31) & 1); }

// The row's history and biases.
struct Lists {
    const int32_t* ids;
    int n;
    int prompt;
    int turn, older, newer;  // of a ring: places before `turn` hold ids whose numbers are `newer` above their places, the others `older`
    const int32_t* bias_ids;
    const float* bias_values;
    int biases;
    __device__ __forceinline__ Lists(const ge_rule_args& x, int64_t row) {
        ids = nullptr;
        n = turn = older = newer = biases = 0;
        prompt = x.prompt_len ? x.prompt_len[row] : 0;
        if (x.history) {
            const int from = x.history_offsets[row];
            ids = x.history + from;
            n = max(0, x.history_offsets[row + 1] - from);
        } else if (x.ring) {
            ids = x.ring + row * x.ring_capacity;
            const int appended = max(0, x.ring_len[row]);
            n = min(appended, x.ring_capacity);
            if (appended > x.ring_capacity) {
                turn = appended % x.ring_capacity;
                newer = appended - turn;
                older = newer - x.ring_capacity;
            }
        }
        if (x.bias_ids) {
            const int from = x.bias_offsets[row];
            bias_ids = x.bias_ids + from;
            bias_values = x.bias_values + from;
            biases = max(0, x.bias_offsets[row + 1] - from);
        }
    }
    // Whether id i lies behind the prompt, by its number among all that were appended.
    __device__ __forceinline__ bool behind(int i) const { return i + (i < turn ? newer : older) >= prompt; }
};

// A token's count in a word: its number behind the prompt, and kPrompt if the prompt has it.
__device__ __forceinline__ void count(uint32_t* word, bool behind) {
    if (behind)
        atomicAdd(word, 1u);
    else
        atomicOr(word, kPrompt);
}

// A capped logit's final value, the mask apart. `bias`: 1 + the number of its entry, 0: none.
__device__ __forceinline__ float penalised(float v, const ge_rule_params& p, uint32_t word, int bias, const float* bias_values) {
    const float c = static_cast<float>(word & ~kPrompt);
    if (word != 0) v = penalize(v, p.repetition_penalty);
    if (c > 0.0f) v = v - p.frequency_penalty * c - p.presence_penalty;
    if (bias != 0) v += bias_values[bias - 1];
    return v;
}

// Softcaps of bf16 logits: a logit has 16 bits, and those from 2^-kLow to 2^kHigh (and their
// negatives, whose caps are the negatives) are looked up in a table that a workgroup
// makes: 2 to 5 evaluations a thread instead of one for each of its logits. The entries are
// softcap() itself, and so are the values of logits that the table does not hold.
constexpr int kLow = 10, kHigh = 8;
constexpr int kFirst = (127 - kLow) << 7, kTable = (kLow + kHigh) << 7;

template <typename T>
struct Softcaps {
    static constexpr int kSize = sizeof(T) == 2 ? kTable : 1;
    float* table;
    float cap;
    template <int kThreads>
    __device__ __forceinline__ void fill() const {
        if constexpr (sizeof(T) == 2) {
            if (cap > 0.0f)
                for (int i = threadIdx.x; i < kTable; i += kThreads) table[i] = softcap(bf16_to_f32(static_cast<uint16_t>(kFirst + i)), cap);
        }
    }
    __device__ __forceinline__ float operator()(T raw) const {
        const float l = to_f32(raw);
        if (!(cap > 0.0f)) return l;
        if constexpr (sizeof(T) == 2) {
            const uint32_t i = (raw & 0x7fffu) - kFirst;
            if (i < static_cast<uint32_t>(kTable)) return __builtin_copysignf(table[i], l);
        }
        return softcap(l, cap);
    }
};

constexpr int kStreamThreads = 512;

// ---- streamed tokens ----------------------------------------------------------------

// The mask's bits of a unit at token t.
template <int kN>
__device__ __forceinline__ uint32_t unit_mask(const uint32_t* mask, int t, int n) {
    constexpr uint32_t kAll = (1u << kN) - 1;
    return mask && n > 0 ? mask[t >> 5] >> (t & 31) & kAll : kAll;
}

// Bound by memory: 512 rows of 262,144 bf16 logits, capped and masked, into float32 212 us, 3.8 TB/s read and
// written (4.9 is what a copy reaches); without the table of softcaps their evaluation
// bounds it. Two units a thread from 2^24 tokens on: more loads in flight, while fewer
// tokens make more workgroups of one.
//
// Every token of the rows from `first_row` on, in pieces of kUnits units a thread, `pieces` to a row, of
// which a workgroup takes every `step`-th from `item` on: it makes the table once, and a
// piece's loads are in flight while the one before is worked on.
template <typename T, typename O, int kUnits>
__device__ __forceinline__ void stream(const ge_rule_args& x, int first_row, unsigned item, unsigned items, unsigned step, int pieces, float* table) {
    constexpr int kN = kStreamUnit<T, O>, kPiece = kStreamThreads * kUnits * kN;
    struct Piece {
        int64_t row;
        int t0;
        float cap;
        Unit<T, kN> raw[kUnits];
        uint32_t ok[kUnits];
    } next;
    auto load = [&](unsigned i) {
        next.row = first_row + static_cast<int64_t>(i / pieces);
        next.t0 = static_cast<int>(i % pieces) * kPiece;
        next.cap = row_rules(x, next.row).softcap;
        const T* const in = static_cast<const T*>(x.logits) + next.row * x.row_stride;
        const uint32_t* const mask = row_mask(x, next.row);
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const int t = next.t0 + (j * kStreamThreads + threadIdx.x) * kN;
            next.raw[j] = load_unit<kN>(in + t, x.vocab - t);
            next.ok[j] = unit_mask<kN>(mask, t, x.vocab - t);
        }
    };
    float filled = 0.0f;
    load(item);
    for (; item < items; item += step) {
        const Piece now = next;
        const Softcaps<T> capped{table, now.cap};
        if (now.cap > 0.0f && now.cap != filled) {
            __syncthreads();
            capped.template fill<kStreamThreads>();
            __syncthreads();
            filled = now.cap;
        }
        if (item + step < items) load(item + step);
        O* const out = static_cast<O*>(x.out) + now.row * x.out_stride;
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const int t = now.t0 + (j * kStreamThreads + threadIdx.x) * kN, n = x.vocab - t;
            if (n <= 0) continue;
            float v[kN];
#pragma unroll
            for (int e = 0; e < kN; ++e) {
                v[e] = capped(now.raw[j].v[e]);
                if (!(now.ok[j] >> e & 1)) v[e] = -__builtin_inff();
            }
            store_unit(out + t, n, v);
        }
    }
}

// ---- single tokens --------------------------------------------------------------------

constexpr int kSingleThreads = 1024;
constexpr int kSlots = 6900;        // of the hash table: two workgroups share a compute unit's LDS
constexpr int kMostHashed = 5000;
constexpr int kDirect = 8192;       // tokens of a piece that is counted by a word each
struct SingleLds {
    union {
        struct {
            int32_t key[kSlots];      // token, -1: free
            uint32_t word[kSlots];
            uint16_t bias[kSlots];    // 1 + the number of the last entry
            uint16_t used[kMostHashed];
            int n_used;
        } hash;
        struct {
            uint32_t word[kDirect];
            int32_t bias[kDirect];
            float table[kTable];      // of rows that are capped in place
        } direct;
    };
};
static_assert(sizeof(SingleLds) <= 80 * 1024 && kSlots % 4 == 0);

__device__ __forceinline__ void clear(void* p, int bytes) {  // a multiple of 16
    for (int i = threadIdx.x; i < bytes / 16; i += kSingleThreads) static_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
}

// Counts the lists' tokens in [t0, t0 + length), at most kDirect of them.
__device__ __forceinline__ void count_direct(const Lists& lists, int t0, int length, SingleLds& lds) {
    auto& d = lds.direct;
    __syncthreads();
    const int bytes = (length + kUnit - 1) / kUnit * kUnit * 4;  // whole units, which are read whole
    clear(d.word, bytes);
    if (lists.biases) clear(d.bias, bytes);
    __syncthreads();
    for_list<kSingleThreads>(lists.ids, lists.n, [&](int i, int id) {
        if (id >= t0 && id - t0 < length) count(&d.word[id - t0], lists.behind(i));
    });
    for_list<kSingleThreads>(lists.bias_ids, lists.biases, [&](int i, int id) {
        if (id >= t0 && id - t0 < length) atomicMax(&d.bias[id - t0], i + 1);
    });
    __syncthreads();
}

// The tokens of the row's lists that lie in [t0, end). Bound by latency (the list, its atomics in LDS,
// the mask's word and the logit, one after the other), with long lists by LDS atomics on the
// same word where a few tokens make up much of a list: 512 rows with up to 2,000 ids 37 us, 9 rows
// with up to 60,000, of which one token is 7 %, 14 us, one row with 700 ids in place 7 us.
template <typename T, typename O>
__device__ __forceinline__ void single(const ge_rule_args& x, int64_t row, int t0, int end, SingleLds& lds) {
    const Lists lists(x, row);
    const int64_t all = static_cast<int64_t>(lists.n) + lists.biases;  // each up to 2^31 - 1
    if (all == 0) return;
    const ge_rule_params p = row_rules(x, row);
    const uint32_t* const mask = row_mask(x, row);
    const T* const in = static_cast<const T*>(x.logits) + row * x.row_stride;
    O* const out = static_cast<O*>(x.out) + row * x.out_stride;
    auto finish = [&](int token, T raw, uint32_t word, int bias) {
        out[token] = from_f32<O>(penalised(softcap(to_f32(raw), p.softcap), p, word, bias, lists.bias_values));
    };
    if (end - t0 <= kDirect || all > kMostHashed) {
        const auto& d = lds.direct;
        for (int first = t0; first < end; first += kDirect) {
            const int length = min(kDirect, end - first);
            count_direct(lists, first, length, lds);
            constexpr int kEach = 4;  // tokens of a thread at a time
            for (int i0 = threadIdx.x; i0 < length; i0 += kEach * kSingleThreads) {
                uint32_t word[kEach];
                int bias[kEach];
                T raw[kEach];
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    const int i = i0 + k * kSingleThreads;
                    word[k] = i < length ? d.word[i] : 0;
                    bias[k] = i < length && lists.biases ? d.bias[i] : 0;
                    if ((word[k] != 0 || bias[k] != 0) && !allows(mask, first + i)) word[k] = bias[k] = 0;
                    if (word[k] != 0 || bias[k] != 0) raw[k] = in[first + i];
                }
#pragma unroll
                for (int k = 0; k < kEach; ++k)
                    if (word[k] != 0 || bias[k] != 0) finish(first + i0 + k * kSingleThreads, raw[k], word[k], bias[k]);
            }
        }
        return;
    }
    auto& h = lds.hash;
    for (int i = threadIdx.x; i < kSlots / 4; i += kSingleThreads) reinterpret_cast<int4*>(h.key)[i] = make_int4(-1, -1, -1, -1);
    clear(h.word, kSlots * 4);
    if (lists.biases)
        for (int i = threadIdx.x; i < kSlots / 2; i += kSingleThreads) reinterpret_cast<uint32_t*>(h.bias)[i] = 0;
    if (threadIdx.x == 0) h.n_used = 0;
    __syncthreads();
    // Free slots remain, so the search ends.
    auto slot_of = [&](int token) {
        int s = static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(token) * 0x9e3779b1u) * kSlots >> 32);
        for (;;) {
            int key = h.key[s];
            if (key == -1) key = atomicCAS(&h.key[s], -1, token);
            if (key == -1 || key == token) return s;
            s = s + 1 == kSlots ? 0 : s + 1;
        }
    };
    for_list<kSingleThreads>(lists.ids, lists.n, [&](int i, int id) {
        if (id >= t0 && id < end) count(&h.word[slot_of(id)], lists.behind(i));
    });
    for_list<kSingleThreads>(lists.bias_ids, lists.biases, [&](int i, int id) {
        if (id < t0 || id >= end) return;
        // the larger of two 16-bit numbers, of which a word holds two
        const int s = slot_of(id);
        uint32_t* const word = reinterpret_cast<uint32_t*>(h.bias) + (s >> 1);
        const int shift = (s & 1) * 16;
        uint32_t old = *word;
        while (static_cast<int>(old >> shift & 0xffffu) < i + 1) {
            const uint32_t seen = atomicCAS(word, old, (old & ~(0xffffu << shift)) | static_cast<uint32_t>(i + 1) << shift);
            if (seen == old) break;
            old = seen;
        }
    });
    __syncthreads();
    // The slots in use, close together: a token costs as much as a wave of them.
    for (int first = 0; first < kSlots; first += kSingleThreads) {
        const int s = first + threadIdx.x;
        const bool mine = s < kSlots && h.key[s] >= 0;
        const uint64_t in_use = __ballot(mine);
        int base = 0;
        if ((threadIdx.x & 63) == 0 && in_use) base = atomicAdd(&h.n_used, __popcll(in_use));
        base = __shfl(base, 0);
        if (mine) h.used[base + __popcll(in_use & ((1ull << (threadIdx.x & 63)) - 1))] = static_cast<uint16_t>(s);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < h.n_used; i += kSingleThreads) {
        const int s = h.used[i], token = h.key[s];
        if (allows(mask, token)) finish(token, in[token], h.word[s], lists.biases ? h.bias[s] : 0);
    }
}

// A piece of kDirect tokens of a row that is capped in place: its words are counted first, then
// every token passes. The logits' loads are in flight while the lists are counted.
template <typename T>
__device__ __forceinline__ void merged(const ge_rule_args& x, int64_t row, int t0, SingleLds& lds) {
    constexpr int kUnits = kDirect / (kSingleThreads * kUnit);
    auto& d = lds.direct;
    const ge_rule_params p = row_rules(x, row);
    const int length = min(kDirect, x.vocab - t0);
    T* const logits = static_cast<T*>(x.out) + row * x.out_stride + t0;
    const uint32_t* const mask = row_mask(x, row);
    Unit<T, kUnit> raw[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int at = (j * kSingleThreads + threadIdx.x) * kUnit;
        raw[j] = load_unit<kUnit>(logits + at, length - at);
    }
    const Lists lists(x, row);
    const Softcaps<T> capped{d.table, p.softcap};
    capped.template fill<kSingleThreads>();
    count_direct(lists, t0, length, lds);
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int at = (j * kSingleThreads + threadIdx.x) * kUnit, n = length - at;
        if (n <= 0) continue;
        const uint32_t ok = unit_mask<kUnit>(mask, t0 + at, n);
        float v[kUnit];
#pragma unroll
        for (int e = 0; e < kUnit; ++e) {
            v[e] = capped(raw[j].v[e]);
            const uint32_t word = d.word[at + e];
            const int bias = lists.biases ? d.bias[at + e] : 0;
            if (word != 0 || bias != 0) v[e] = penalised(v[e], p, word, bias, lists.bias_values);
            if (!(ok >> e & 1)) v[e] = -__builtin_inff();
        }
        store_unit(logits + at, n, v);
    }
}

// What is not allowed of kUnits units a thread from t0 on: reads the mask, and writes what it leaves out.
// 64 rows of 262,144 tokens with grammars that allow few of them, and histories of 300 ids
// beside: 16.3 us, 6 of which are the bytes; the rest is the lists' latency.
template <typename T, int kUnits>
__device__ __forceinline__ void forbid(const ge_rule_args& x, int64_t row, int t0) {
    T* const out = static_cast<T*>(x.out) + row * x.out_stride;
    const uint32_t* const mask = row_mask(x, row);
    if (!mask) return;
    const float inf = __builtin_inff();
    const float none[kUnit] = {-inf, -inf, -inf, -inf, -inf, -inf, -inf, -inf};
    uint32_t ok[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int t = t0 + (j * kSingleThreads + threadIdx.x) * kUnit;
        ok[j] = unit_mask<kUnit>(mask, t, x.vocab - t);
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int t = t0 + (j * kSingleThreads + threadIdx.x) * kUnit, n = x.vocab - t;
        if (ok[j] == 0) {
            store_unit(out + t, n, none);
        } else if (ok[j] != 0xffu) {
#pragma unroll
            for (int e = 0; e < kUnit; ++e)
                if (e < n && !(ok[j] >> e & 1)) out[t + e] = from_f32<T>(-inf);
        }
    }
}

// ---- flags ------------------------------------------------------------------------------

template <int kThreads>
__device__ __forceinline__ void flag(const ge_rule_args& x, int64_t row) {
    const uint32_t* const mask = row_mask(x, row);
    bool allowed = !mask;
    if (mask) {
        const int whole = x.vocab / 32;
        for_list<kThreads>(reinterpret_cast<const int32_t*>(mask), whole, [&](int, int w) { allowed |= w != 0; });
        if (threadIdx.x == 0 && x.vocab % 32) allowed |= (mask[whole] & ((1u << (x.vocab % 32)) - 1)) != 0;
    }
    allowed = __syncthreads_or(allowed);
    if (threadIdx.x == 0) x.flags_out[row] = allowed ? 0 : GE_RULE_EMPTY;
}

// ---- launches -----------------------------------------------------------------------------

// What the blocks of a launch do, in this order: `singles` of them a slice of `slice` tokens each,
// `slices` to a row, `streams` a piece each, `pieces` to a row, and one a row for the flags.
struct Blocks {
    int first_row;
    int slice, slices;
    unsigned singles;
    int pieces;
    unsigned items;    // pieces of all rows, if `streams` blocks share them
    unsigned streams;
};

template <typename T, typename O, int kUnits>
__global__ __launch_bounds__(kStreamThreads) void stream_kernel(ge_rule_args x, Blocks b) {
    __shared__ float table[Softcaps<T>::kSize];
    const unsigned block = blockIdx.x;
    if (block >= b.streams) return flag<kStreamThreads>(x, b.first_row + static_cast<int64_t>(block - b.streams));
    stream<T, O, kUnits>(x, b.first_row, block, b.items, b.streams, b.pieces, table);
}

template <typename T, typename O>
__global__ __launch_bounds__(kSingleThreads, 8) void single_kernel(ge_rule_args x, Blocks b) {
    __shared__ __align__(16) SingleLds lds;
    const int t0 = static_cast<int>(blockIdx.x % b.slices) * b.slice;
    single<T, O>(x, b.first_row + static_cast<int64_t>(blockIdx.x / b.slices), t0, min(x.vocab, t0 + b.slice), lds);
}

constexpr int kForbidUnits = 4;   // units a thread
constexpr int kForbidPiece = kForbidUnits * kSingleThreads * kUnit;
template <typename T>
__global__ __launch_bounds__(kSingleThreads, 8) void in_place_kernel(ge_rule_args x, Blocks b) {
    __shared__ __align__(16) SingleLds lds;
    unsigned block = blockIdx.x;
    if (block < b.singles) {
        const int64_t row = b.first_row + static_cast<int64_t>(block / b.slices);
        const int t0 = static_cast<int>(block % b.slices) * b.slice;
        if (!(row_rules(x, row).softcap > 0.0f)) single<T, T>(x, row, t0, min(x.vocab, t0 + b.slice), lds);
        return;
    }
    block -= b.singles;
    if (block >= b.streams) return flag<kSingleThreads>(x, b.first_row + static_cast<int64_t>(block - b.streams));
    const int64_t row = b.first_row + static_cast<int64_t>(block / b.pieces);
    const int t0 = static_cast<int>(block % b.pieces) * kForbidPiece;
    if (!(row_rules(x, row).softcap > 0.0f)) return forbid<T, kForbidUnits>(x, row, t0);
    for (int t = t0; t < min(x.vocab, t0 + kForbidPiece); t += kDirect) merged<T>(x, row, t, lds);
}

// launch(first row, rows) for at most `most` rows at a time.
template <typename F>
void for_rows(int rows, int64_t most, F launch) {
    for (int r = 0; r < rows; r += static_cast<int>(most)) launch(r, static_cast<int>(std::min<int64_t>(most, rows - r)));
}

constexpr unsigned kStreamBlocks = 1024;   // that run at a time, 4 on each compute unit
constexpr int64_t kMostBlocks = 1 << 21;  // of a launch: less than 2^32 threads

// Slices of the vocabulary: a workgroup for each compute unit where rows are few, of kDirect tokens if that is
// enough (64 rows, 262,144 tokens, in place: with 4,000 ids each 13.0 us, with two workgroups
// 15.0, which clear and search two tables for the same list; with 20,000 ids 63 against 51).
Blocks single_blocks(const ge_rule_args& x) {
    Blocks b{};
    b.slices = std::max(1, std::min((x.vocab + kDirect - 1) / kDirect, std::min(64, 256 / x.rows)));
    b.slice = (x.vocab + b.slices - 1) / b.slices;
    return b;
}

template <typename T, typename O>
void launch(const ge_rule_args& x, hipStream_t st) {
    const bool lists = x.history || x.ring || x.bias_ids;
    const bool some_capped = x.row_params || x.params.softcap > 0.f, some_not = x.row_params || !(x.params.softcap > 0.f);
    Blocks b = single_blocks(x);
    if constexpr (std::is_same<T, O>::value) {
        if (in_place(x)) {
            b.pieces = (x.vocab + kForbidPiece - 1) / kForbidPiece;
            for_rows(x.rows, kMostBlocks / (b.pieces + b.slices + 1), [&](int r, int n) {
                b.first_row = r;
                b.singles = some_not && lists ? static_cast<unsigned>(n) * b.slices : 0;
                b.streams = some_capped || x.mask ? static_cast<unsigned>(n) * b.pieces : 0;
                const unsigned all = b.singles + b.streams + (x.flags_out ? n : 0);
                if (all) in_place_kernel<T><<<all, kSingleThreads, 0, st>>>(x, b);
            });
            return;
        }
    }
    auto streams = [&](auto units) {
        constexpr int kUnits = decltype(units)::value;
        constexpr int kPiece = kStreamThreads * kUnits * kStreamUnit<T, O>;
        b.pieces = (x.vocab + kPiece - 1) / kPiece;
        for_rows(x.rows, kMostBlocks / (b.pieces + 1), [&](int r, int n) {
            b.first_row = r;
            b.items = static_cast<unsigned>(n) * b.pieces;
            b.streams = std::min(b.items, kStreamBlocks);
            stream_kernel<T, O, kUnits><<<b.streams + (x.flags_out ? n : 0), kStreamThreads, 0, st>>>(x, b);
        });
    };
    if (static_cast<int64_t>(x.rows) * x.vocab >= (int64_t{1} << 24))
        streams(std::integral_constant<int, 2>{});
    else
        streams(std::integral_constant<int, 1>{});
    if (lists)
        for_rows(x.rows, kMostBlocks / b.slices, [&](int r, int n) {
            b.first_row = r;
            single_kernel<T, O><<<static_cast<unsigned>(n) * b.slices, kSingleThreads, 0, st>>>(x, b);
        });
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
    auto by_out = [&](auto t) {
        using T = decltype(t);
        if (x.out_dtype == GE_DTYPE_F32)
            launch<T, float>(x, st);
        else
            launch<T, uint16_t>(x, st);
    };
    if (x.dtype == GE_DTYPE_F32)
        by_out(float{});
    else
        by_out(uint16_t{});
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return GE_OK;
    ge::plan_fail(msg, sizeof(msg), 0, "launch (rules): %s", hipGetErrorString(e));
    return ge::report(GE_ERR_DEVICE, msg);
}

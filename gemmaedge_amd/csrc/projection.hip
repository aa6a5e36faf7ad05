// A projection shared by all rows with a low-rank adapter for each row's request
// (include/gemmaedge_projection.h), on the matrix products of head_gemm.h and
// head_gemm32.h.
//
// Forward: u = scale A h of every row first; then the large product, whose
// epilogue adds B u to the accumulators while they are still in registers: for
// each adapter that the wave's rows have, in turn, the other rows' u count as
// zeros. An adapter's rows of B are read once by each tile that needs them, and
// rows of different requests need no sorting.
//
// Backward: dhidden = weight^T dout by the same product across the weights, with A^T
// du added by the same epilogue (A is transposed first, which is small); du = scale
// B^T dout and u as low-rank sums over all channels; dA and dB as sums over each
// adapter's rows, which a launch lists in order.
//
// The large product bounds a call: with one row its weights' bytes (1.48 GB in 245 us, 6.0
// TB/s), with many the matrix cores (4,096 rows, width 2,816, 262,144 outputs, 9 adapters of rank 32:
// 5.3 ms, 1,150 TFLOP/s; 4.8 of them without adapters). Adapters inside it save the outputs' second
// pass; what they cost is their rows' bytes and the epilogue's time, in which nothing is loaded
// for the next tile: 8,192 rows, 2,816 to 11,264, 5 adapters of rank 64, 540 us, 436 without.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstring>
#include <new>
#include <type_traits>

#include "head_tiles.h"
#include "projection_validate.h"

namespace ge {
namespace projection {
namespace {

using head::bf16x8;
using head::epi_row;
using head::f32x4;
using head::from_f32;
using head::GemmArgs;
using head::Operand;
using head::s16x4;
using head::TilePlace;
using head::to_bf16;
using head::to_f32;
using head::u32x4;

struct Buffers {
    void* hpack;
    void* wpack;
    void* u;
    void* du;
    float* parts;
    int32_t* order;
    void* at;
    void* dpack;
    float* dhidden;
};

// ---- low-rank values ------------------------------------------------------------
//
// The rows' u and du, `pad` (rank_pad) values each, zeros behind the rank: float32
// rows, or bf16 in three planes, of which each has the next 8 bits, cut off: together
// the float32 value itself, for magnitudes from 2^-102 on. Two planes would leave 2^-17
// of it out, which float32 outputs show, and which turns one rounding to bf16 in some hundreds.
//
// The planes of a value have its sign and none is zero unless it is, so that times an
// infinity they are one infinity: a plane of which nothing is left shares the one before. (The
// smallest normal number there instead would show: the matrix instructions cut sums off downwards.)
// All planes of an infinity are that infinity, since what it leaves would be NaN.
template <typename T>
struct Low {
    T* p;
    int64_t plane;  // elements from a plane to the next (bf16)
    int pad;
};
template <typename T>
__device__ __forceinline__ void low_store(const Low<T>& u, int64_t row, int r, float x) {
    T* const to = u.p + row * u.pad + r;
    if constexpr (sizeof(T) == 4) {
        *to = x;
    } else {
        static_assert(kLowPlanes == 3);
        auto top = [](float v) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xffff0000u); };
        float hi = top(x), mid = top(x - hi), lo = x - hi - mid;
        if (mid == 0.f) {
            hi = x * 0.5f;
            mid = lo = x * 0.25f;
        } else if (lo == 0.f) {
            mid = lo = mid * 0.5f;
        }
        if (!(__builtin_fabsf(x) < __builtin_inff())) hi = mid = lo = x;
        to[0] = to_bf16(hi);
        to[u.plane] = to_bf16(mid);
        to[2 * u.plane] = to_bf16(lo);
    }
}

// At most 2^31 - 16 bytes from p on, `left` of which are the operand's.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* p, int64_t left) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(max(int64_t{0}, min(left, int64_t{0x7ffffff0}))),
                                             0x00027000);
}
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t rs, uint32_t at) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, static_cast<int>(at), 0, 0));
}
// The first n of a lane's elements of type T (8 or 4): what the others' bits are cut off by.
template <typename T>
__device__ __forceinline__ u32x4 mask_below(int n) {
    u32x4 m;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        m[q] = sizeof(T) == 4 ? (q < n ? 0xffffffffu : 0u) : 2 * q + 1 < n ? 0xffffffffu : 2 * q < n ? 0xffffu : 0u;
    return m;
}
// The hardware checks bounds four bytes at a time and reads a zero for the last of an odd number
// of bf16 elements: `last`, read by itself, as element e of a lane's 8, to be added to that.
__device__ __forceinline__ u32x4 at_element(int e, uint16_t last) {
    u32x4 v;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = e >> 1 == q ? static_cast<uint32_t>(last) << 16 * (e & 1) : 0u;
    return v;
}

// Adapters' rows along the rank, one for each row of the large product's M side.
template <typename T>
struct Adapters {
    const T* table;       // [adapters][m][rank]
    int64_t m;
    int rank, adapters;   // adapters 0: none
    const int32_t* ids;   // [rows]
    Low<T> u;
};

// Column j's accumulators stay where they are until here: see the products' kernel, whose
// large tiles have no registers to read them all into. They are not written again:
// with other values in them the compiler moves some between the product's steps,
// whose instructions it knows nothing of.
template <int kMt, int kNt>
__device__ __forceinline__ void hold(f32x4 (&acc)[kMt][kNt], int j) {
    if constexpr (kMt * kNt >= 32) {
#pragma unroll
        for (int t = 0; t < kMt; ++t) asm volatile("" : "+a"(acc[t][j]));
    }
}

// Ranks of a chunk, which is a fragment of an adapter's rows.
template <typename T>
constexpr int kChunk = sizeof(T) == 2 ? 32 : 16;

template <typename T>
using Frag = typename std::conditional<sizeof(T) == 2, bf16x8, f32x4>::type;

// An adapter's rows of a wave for the chunk of ranks from r0 on, as the matrix instructions take them.
template <bool kAAlong, typename T, int kMt>
__device__ __forceinline__ void load_table(const Adapters<T>& x, int64_t m0, int adapter, int r0, int lane, Frag<T> (&f)[kMt]) {
    const int i = lane & 15, r = r0 + (kChunk<T> / 4) * (lane >> 4), left = x.rank - r;
    // Rows past the last are another adapter's, or nothing: outputs that nobody reads.
    const T* const end = x.table + x.adapters * x.m * x.rank;
    const T* const p = x.table + (adapter * x.m + m0) * x.rank;
    const auto rs = resource(p, (end - p) * static_cast<int64_t>(sizeof(T)));
    u32x4 v[kMt];
#pragma unroll
    for (int t = 0; t < kMt; ++t) {
        const int row = kAAlong ? epi_row(t, i) : t * 16 + i;
        v[t] = load16(rs, left > 0 ? static_cast<uint32_t>(row * x.rank + r) * sizeof(T) : 0x80000000u);
    }
    if (x.rank % (kChunk<T> / 4)) {  // a row ends within a lane's elements
        const u32x4 below = mask_below<T>(left);
        u32x4 tail{0, 0, 0, 0};
        int last_row = -1;
        if constexpr (sizeof(T) == 2) {
            if ((x.rank & 1) && adapter == x.adapters - 1) {
                last_row = static_cast<int>(min(x.m - 1 - m0, int64_t{INT_MAX}));
                tail = at_element(left - 1, end[-1]);
            }
        }
#pragma unroll
        for (int t = 0; t < kMt; ++t) {
            v[t] &= below;
            if constexpr (sizeof(T) == 2) {
                const int row = kAAlong ? epi_row(t, i) : t * 16 + i;
#pragma unroll
                for (int q = 0; q < 4; ++q) v[t][q] |= row == last_row ? tail[q] : 0u;
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kMt; ++t) f[t] = __builtin_bit_cast(Frag<T>, v[t]);
}

// The row's own values for the same ranks, zeros without an adapter; bf16: all planes.
template <typename T>
struct RowValues {
    static constexpr int kPlanes = sizeof(T) == 2 ? kLowPlanes : 1;
    u32x4 v[kPlanes];
};
template <typename T>
__device__ __forceinline__ RowValues<T> load_values(const Adapters<T>& x, int id, int64_t n, int r0, int lane) {
    RowValues<T> u;
    const T* const p = x.u.p + n * x.u.pad + r0 + (kChunk<T> / 4) * (lane >> 4);
#pragma unroll
    for (int i = 0; i < RowValues<T>::kPlanes; ++i) {
        u.v[i] = u32x4{0, 0, 0, 0};
        if (id >= 0) u.v[i] = *reinterpret_cast<const u32x4*>(p + i * x.u.plane);
    }
    return u;
}

// acc += table u for the lanes whose row is this adapter's. Products with the rows that are not its
// own are left out, not added as zeros: an infinity in one request's adapter stays there.
template <typename T>
__device__ __forceinline__ void add_product(const Frag<T>& f, const RowValues<T>& u, bool mine, f32x4& acc) {
    f32x4 y{0.f, 0.f, 0.f, 0.f};
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int p = kLowPlanes - 1; p >= 0; --p) y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, u.v[p]), y, 0, 0, 0);
    } else {
        const f32x4 fu = __builtin_bit_cast(f32x4, u.v[0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) y = __builtin_amdgcn_mfma_f32_16x16x4f32(f[e], fu[e], y, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += mine ? y[e] : 0.f;
}

// Adds table[k] u to the accumulators, whose column j has row n0 + 16 j in lanes i, i + 16, ... (n0: of
// lane i), of adapter k = id[j], and whose first row along M is m0.
//
// Short tiles, whose columns are rows of many requests: one adapter after the other over all
// columns, its rows loaded once (64 rows, 22 adapters of rank 16, width 2,816, 262,144 outputs: 352
// us, 279 of them without adapters; column by column 372 us; two adapters' rows in flight
// together take registers and with them workgroups of a compute unit, which hide more: 384 us).
template <bool kAAlong, typename T, int kMt, int kNt>
__device__ __forceinline__ void add_adapters(const Adapters<T>& x, const int (&id)[kNt], int64_t m0, int64_t n0, int lane, f32x4 (&acc)[kMt][kNt]) {
    if (!x.adapters) return;
    for (int r0 = 0; r0 < x.rank; r0 += kChunk<T>) {
        RowValues<T> u[kNt];
        uint64_t left[kNt];
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            u[j] = load_values(x, id[j], n0 + j * 16, r0, lane);
            left[j] = __ballot(id[j] >= 0);
        }
        for (;;) {
            int k = -1;
            Frag<T> f[kMt];
#pragma unroll
            for (int j = 0; j < kNt; ++j)
                if (k < 0 && left[j]) k = __builtin_amdgcn_readlane(id[j], __builtin_ctzll(left[j]));
            if (k >= 0) {
#pragma unroll
                for (int j = 0; j < kNt; ++j) left[j] &= ~__ballot(id[j] == k);
                load_table<kAAlong>(x, m0, k, r0, lane, f);
            }
            if (k < 0) break;
            // Columns without this adapter add nothing: that is cheaper than branches around them.
#pragma unroll
            for (int j = 0; j < kNt; ++j) {
#pragma unroll
                for (int t = 0; t < kMt; ++t) add_product<T>(f[t], u[j], id[j] == k && k >= 0, acc[t][j]);
            }
        }
    }
}

// Tall tiles, whose accumulators are read once and not written again: column by column, a row's values on
// their way a column ahead, two chunks of the adapter's rows kept while the columns that follow
// have the same adapter.
template <bool kAAlong, typename T, int kMt, int kNt>
struct AdapterSum {
    static constexpr int kKept = 2;
    const Adapters<T>& x;
    const int (&id)[kNt];
    int64_t m0, n0;
    int lane;
    RowValues<T> next[kKept];
    Frag<T> f[kKept][kMt];
    int kept = -1;
    __device__ __forceinline__ AdapterSum(const Adapters<T>& a, const int (&ids)[kNt], int64_t m, int64_t n, int l)
        : x(a), id(ids), m0(m), n0(n), lane(l) {
        if (x.adapters) values(0, 0, next);
    }
    __device__ __forceinline__ void values(int j, int r0, RowValues<T> (&u)[kKept]) const {
#pragma unroll
        for (int c = 0; c < kKept; ++c)
            if (r0 + c * kChunk<T> < x.rank) u[c] = load_values(x, id[j], n0 + j * 16, r0 + c * kChunk<T>, lane);
    }
    __device__ __forceinline__ void add(int j, f32x4 (&acc)[kMt]) {
        constexpr int kStep = kKept * kChunk<T>;
        if (!x.adapters) return;
        RowValues<T> u[kKept];
#pragma unroll
        for (int c = 0; c < kKept; ++c) u[c] = next[c];
        if (j + 1 < kNt) values(j + 1, 0, next);
        uint64_t left = __ballot(id[j] >= 0);
        while (left) {
            const int k = __builtin_amdgcn_readlane(id[j], __builtin_ctzll(left));
            left &= ~__ballot(id[j] == k);
            for (int r0 = 0; r0 < x.rank; r0 += kStep) {
                if (x.rank > kStep) values(j, r0, u);
                if (k != kept || x.rank > kStep) {
#pragma unroll
                    for (int c = 0; c < kKept; ++c)
                        if (r0 + c * kChunk<T> < x.rank) load_table<kAAlong>(x, m0, k, r0 + c * kChunk<T>, lane, f[c]);
                    kept = k;
                }
#pragma unroll
                for (int c = 0; c < kKept; ++c)
                    if (r0 + c * kChunk<T> < x.rank) {
#pragma unroll
                        for (int t = 0; t < kMt; ++t) add_product<T>(f[c][t], u[c], id[j] == k, acc[t]);
                    }
            }
        }
    }
};
template <int kMt, int kNt>
constexpr bool kTall = kMt * kNt >= 32;

// Nothing by columns: short tiles have it all by then.
struct NoSum {
    template <typename... Args>
    __device__ __forceinline__ explicit NoSum(const Args&...) {}
};
template <bool kAAlong, typename T, int kMt, int kNt>
using ColumnSum = typename std::conditional<kTall<kMt, kNt>, AdapterSum<kAAlong, T, kMt, kNt>, NoSum>::type;

// The adapters of a lane's rows, -1: none.
template <int kNt>
__device__ __forceinline__ void load_ids(const int32_t* ids, int adapters, int64_t n_first, int rows, int (&id)[kNt]) {
#pragma unroll
    for (int j = 0; j < kNt; ++j) {
        id[j] = -1;
        if (adapters && n_first + j * 16 < rows) id[j] = ids[n_first + j * 16];
        if (id[j] >= adapters) id[j] = -1;
    }
}

template <typename O, int kCount>
__device__ __forceinline__ void store_out(O* o, const float (&x)[kCount], int n) {
    struct Vec {
        O v[kCount];
    } q;
#pragma unroll
    for (int e = 0; e < kCount; ++e) q.v[e] = from_f32<O>(x[e]);
    if (n >= kCount) {
        __builtin_memcpy(o, &q, sizeof(q));
    } else {
#pragma unroll
        for (int e = 0; e < kCount; ++e)
            if (e < n) o[e] = q.v[e];
    }
}

// The projection's outputs: a lane has 8 neighbours of a row in every two tiles.
template <typename T, typename O>
struct OutEpi {
    Adapters<T> low;
    int rows, m;   // m: outputs from the product's first row on
    int v0;        // number of that row
    O* out;        // of row 0 and output v0
    int64_t ld;

    template <int kNt>
    struct State {
        int id[kNt];
    };
    template <int kWm, int kNt>
    __device__ __forceinline__ State<kNt> prepare(int, int col0, int lane) const {
        State<kNt> s;
        load_ids(low.ids, low.adapters, col0 + (lane & 15), rows, s.id);
        return s;
    }
    template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, int kMt, int kNt>
    __device__ __forceinline__ void finish(f32x4 (&acc)[kMt][kNt], const State<kNt>& s, int m0, int n0, TilePlace, int wm, int wn, int lane,
                                           float2*) const {
        constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
        const int row0 = m0 + wm * kWm, col0 = n0 + wn * kWn;
        if (row0 >= m) return;
        if constexpr (!kTall<kMt, kNt>) add_adapters<kAAlong>(low, s.id, v0 + row0, col0 + (lane & 15), lane, acc);
        ColumnSum<kAAlong, T, kMt, kNt> sum(low, s.id, v0 + row0, col0 + (lane & 15), lane);
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            hold(acc, j);
            const int n = col0 + j * 16 + (lane & 15);
            f32x4 y[kMt];
#pragma unroll
            for (int i = 0; i < kMt; ++i) y[i] = acc[i][j];
            if constexpr (kTall<kMt, kNt>) sum.add(j, y);
            if (n >= rows) continue;
            const int v = row0 + (lane >> 4) * 8;
            O* const o = out + n * ld + v;
#pragma unroll
            for (int i = 0; i < kMt; i += 2) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = y[i + (e >> 2)][e & 3];
                if (v + i * 16 < m) store_out(o + i * 16, x, m - v - i * 16);
            }
        }
    }
};

// dhidden of a piece of the outputs and part of it: rounded into the result if that is
// all of the sum, else in float32, added to what earlier pieces left.
template <typename T, bool kDirect>
struct HiddenEpi {
    Adapters<T> low;  // of the first part of the first piece
    int rows, dim;
    typename std::conditional<kDirect, T, float>::type* out;  // [splits][rows][ld]
    int64_t ld, split;
    bool add;

    template <int kNt>
    struct State {
        int id[kNt];
    };
    template <int kWm, int kNt>
    __device__ __forceinline__ State<kNt> prepare(int, int col0, int lane) const {
        State<kNt> s;
        load_ids(low.ids, low.adapters, col0 + (lane & 15), rows, s.id);
        return s;
    }
    template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, int kMt, int kNt>
    __device__ __forceinline__ void finish(f32x4 (&acc)[kMt][kNt], const State<kNt>& s, int m0, int n0, TilePlace place, int wm, int wn,
                                           int lane, float2*) const {
        constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
        const int row0 = m0 + wm * kWm, col0 = n0 + wn * kWn;
        if (row0 >= dim) return;
        if constexpr (!kTall<kMt, kNt>) {
            if (place.split == 0) add_adapters<kAAlong>(low, s.id, row0, col0 + (lane & 15), lane, acc);
        }
        ColumnSum<kAAlong, T, kMt, kNt> sum(low, s.id, row0, col0 + (lane & 15), lane);
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            hold(acc, j);
            const int64_t n = col0 + j * 16 + (lane & 15);
            f32x4 y[kMt];
#pragma unroll
            for (int i = 0; i < kMt; ++i) y[i] = acc[i][j];
            if constexpr (kTall<kMt, kNt>) {
                if (place.split == 0) sum.add(j, y);
            }
            if (n >= rows) continue;
            const int d0 = row0 + 4 * (lane >> 4);
#pragma unroll
            for (int i = 0; i < kMt; ++i) {
                const int d = d0 + i * 16;
                if constexpr (kDirect) {
                    const float x[4] = {y[i][0], y[i][1], y[i][2], y[i][3]};
                    if (d < dim) store_out(out + n * ld + d, x, dim - d);
                } else {  // ld is a multiple of 4 above dim
                    f32x4* const o = reinterpret_cast<f32x4*>(out + place.split * split + n * ld + d);
                    if (d < dim) *o = add ? *o + y[i] : y[i];
                }
            }
        }
    }
};

// The parts of dhidden in order, rounded once: 4 channels a thread (ld is a multiple of 4 above dim).
// Bound by memory: 8,192 rows of 2,816 channels in 2 parts 39 us, 5.9 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void hidden_sum_kernel(const float* parts, int64_t ld, int64_t split, int splits, unsigned rows, int dim, T* out,
                                                         int64_t out_ld) {
    const int d = (blockIdx.x * blockDim.x + threadIdx.x) * 4;
    const int64_t r = blockIdx.y * blockDim.y + threadIdx.y;
    if (r >= rows || d >= dim) return;
    f32x4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < splits; ++i) sum += *reinterpret_cast<const f32x4*>(parts + i * split + r * ld + d);
    const float x[4] = {sum[0], sum[1], sum[2], sum[3]};
    store_out(out + r * out_ld + d, x, dim - d);
}

// ---- sums of a row's channels with each rank -------------------------------------
//
// y[n][r] = scale[k] * sum over c of x[n][c] * table[k](r, c), k the row's adapter.
// kAlong: the table is [adapters][rank][cols] (u from A); else [adapters][cols][rank]
// (du from B), and its tiles are transposed on their way from LDS, like those of
// the large product. A workgroup takes a tile of rows and one of the adapters they have (at most as
// many as rows: a grid's y), and a part of the sum.
template <typename T>
struct SumArgs {
    const T* x;
    int64_t ld;
    int rows, cols;
    const T* table;
    const float* scale;
    const int32_t* ids;
    int adapters, rank;
    Low<T> y;
    float* parts;   // [splits][rows][pad], or NULL: the only part
    int splits, steps_per_split;
    // Many rows: the rows that have adapters, sorted by them, and their number; or NULL: all rows. Rows
    // that are not listed get no values, and nobody reads any.
    const int32_t* order;
    const int32_t* listed;
};

// The slot-th of the adapters that a wave's lanes have; INT_MAX: they have fewer.
__device__ __forceinline__ int slot_adapter(int id, int slot) {
    uint64_t left = __ballot(id >= 0);
    for (; left; --slot) {
        const int k = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        if (slot == 0) return k;
        left &= ~__ballot(id == k);
    }
    return INT_MAX;
}

template <typename T>
__device__ __forceinline__ int row_adapter(const SumArgs<T>& s, int n) {
    const int id = n < s.rows ? s.ids[n] : -1;
    return id < s.adapters ? id : -1;
}

// A row's sum with rank r: into its part, or as the value itself. `who`: the row's adapter.
template <typename T>
__device__ __forceinline__ void low_result(const SumArgs<T>& s, int split, int64_t n, int r, float x, int who) {
    const bool there = who >= 0 && r < s.rank;
    if (s.parts)
        s.parts[(static_cast<int64_t>(split) * s.rows + n) * s.y.pad + r] = there ? x : 0.f;
    else
        low_store(s.y, n, r, there ? x * s.scale[who] : 0.f);  // zeros behind the rank whatever the scale is
}

// The first `left` of 8 elements at p (any address), zeros behind them.
__device__ __forceinline__ u32x4 load_row8(const uint16_t* p, int left) {
    u32x4 raw{0, 0, 0, 0};
    if (left >= 8) {
        __builtin_memcpy(&raw, p, 16);
    } else if (left > 0) {
        struct {
            uint16_t v[8];
        } q{};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) q.v[e] = p[e];
        raw = __builtin_bit_cast(u32x4, q);
    }
    return raw;
}

// A tile of bf16 columns in LDS, rows `ld` elements apart: 16 columns from `col` on of 32 rows,
// transposed into a fragment.
__device__ __forceinline__ bf16x8 frag_across(uint16_t* tile, int ld, int col, int lane) {
    typedef __attribute__((address_space(3))) s16x4* lds4;
    const int i = lane & 15, g = lane >> 4;
    uint16_t* const p = tile + (8 * g + (i >> 2)) * ld + col + (i & 3) * 4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * ld));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Few rows, or float32: a workgroup has 16 rows, and its waves take every kSumWaves-th step of 32 channels,
// kBatch of them at a time, whose loads are in flight together. Bound by their latency: 64
// rows of 2,816 channels with 22 adapters of rank 16: 9.5 us (18 us a step at a time with four waves).
constexpr int kSumStep = 32;
constexpr int kSumWaves = 8;

template <typename T, bool kAlong, int kR>
__global__ __launch_bounds__(64 * kSumWaves) void low_sum_kernel(SumArgs<T> s) {
    constexpr int kRanks = kR * 16, kBatch = kR == 4 ? 2 : 4;
    __shared__ __align__(16) float red[kSumWaves][kRanks][17];
    constexpr int kRow = kRanks + 8;  // bf16 elements of a transposed tile's row in LDS
    constexpr bool kTiled = !kAlong && sizeof(T) == 2;
    __shared__ __align__(16) uint16_t tiles[kTiled ? kSumWaves * kBatch * kSumStep * kRow : 8];
    __shared__ int owner[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * kRowTile;
    const int id = row_adapter(s, n0 + i);
    const int k = slot_adapter(id, blockIdx.y);
    // Rows without an adapter have zeros; the first slot writes them.
    if (k == INT_MAX && blockIdx.y != 0) return;
    const int split = blockIdx.z % s.splits, r0 = blockIdx.z / s.splits * kRanks;
    f32x4 acc[kR];
#pragma unroll
    for (int t = 0; t < kR; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (k != INT_MAX && r0 < s.rank) {
        const T* const xr = s.x + min(n0 + i, s.rows - 1) * s.ld;
        const T* const table = s.table + k * (static_cast<int64_t>(s.rank) * s.cols);
        const T* const end = s.table + s.adapters * (static_cast<int64_t>(s.rank) * s.cols);
        const bool odd = (s.rank & 1) && k == s.adapters - 1;
        const int first = split * s.steps_per_split;
        const int last = min((s.cols + kSumStep - 1) / kSumStep, first + s.steps_per_split);
        for (int step = first + wave; step < last; step += kSumWaves * kBatch) {
            if constexpr (sizeof(T) == 2) {
                uint16_t* const my = tiles + (kTiled ? wave * kBatch * kSumStep * kRow : 0);
                u32x4 fx[kBatch], fw[kBatch][kR];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                    const int at = step + b * kSumWaves, c0 = at * kSumStep, c = c0 + 8 * g;
                    const int left = at < last ? s.cols - c : 0;
                    fx[b] = load_row8(xr + c, left);
                    if constexpr (kAlong) {
#pragma unroll
                        for (int t = 0; t < kR; ++t)  // ranks past the last: outputs that nobody reads
                            fw[b][t] = load_row8(table + static_cast<int64_t>(min(r0 + t * 16 + i, s.rank - 1)) * s.cols + c, left);
                    } else {
                        // 32 channels of the ranks, 8 a lane; columns past the rank belong to the next
                        // channel and to outputs that nobody reads.
                        const uint16_t* const p = table + static_cast<int64_t>(c0) * s.rank;
                        const auto rs = resource(p, (end - p) * 2);
                        const int rows = at < last ? s.cols - c0 : 0;
                        constexpr int kPerRow = kRanks / 8;
#pragma unroll
                        for (int q = 0; q < kR; ++q) {
                            const int unit = q * 64 + lane, row = unit / kPerRow, col = unit % kPerRow * 8;
                            fw[b][q] = load16(rs, row < rows && r0 + col < s.rank ? static_cast<uint32_t>(row * s.rank + r0 + col) * 2 : 0x80000000u);
                            if (odd && row == rows - 1) fw[b][q] |= at_element(s.rank - 1 - r0 - col, end[-1]);
                        }
                    }
                }
                if constexpr (!kAlong) {
                    constexpr int kPerRow = kRanks / 8;
#pragma unroll
                    for (int b = 0; b < kBatch; ++b)
#pragma unroll
                        for (int q = 0; q < kR; ++q) {
                            const int unit = q * 64 + lane, row = unit / kPerRow, col = unit % kPerRow * 8;
                            *reinterpret_cast<u32x4*>(my + (b * kSumStep + row) * kRow + col) = fw[b][q];
                        }
                    __builtin_amdgcn_wave_barrier();
                }
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
#pragma unroll
                    for (int t = 0; t < kR; ++t) {
                        bf16x8 w;
                        if constexpr (kAlong)
                            w = __builtin_bit_cast(bf16x8, fw[b][t]);
                        else
                            w = frag_across(my + b * kSumStep * kRow, kRow, t * 16, lane);
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, __builtin_bit_cast(bf16x8, fx[b]), acc[t], 0, 0, 0);
                    }
                __builtin_amdgcn_wave_barrier();
            } else {
                f32x4 fx[kBatch][2], fw[kBatch][2][kR];
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at = step + b * kSumWaves, c = at * kSumStep + h * 16 + 4 * g;
                        const bool there = at < last;
                        const f32x4 none{0.f, 0.f, 0.f, 0.f};
                        fx[b][h] = none;
                        if (there && c + 4 <= s.cols) {
                            __builtin_memcpy(&fx[b][h], xr + c, 16);
                        } else if (there) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (c + e < s.cols) fx[b][h][e] = xr[c + e];
                        }
#pragma unroll
                        for (int t = 0; t < kR; ++t) {
                            const int r = min(r0 + t * 16 + i, s.rank - 1);
                            fw[b][h][t] = none;
                            if constexpr (kAlong) {
                                const T* const p = table + static_cast<int64_t>(r) * s.cols + c;
                                if (there && c + 4 <= s.cols) {
                                    __builtin_memcpy(&fw[b][h][t], p, 16);
                                } else if (there) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        if (c + e < s.cols) fw[b][h][t][e] = p[e];
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (there && c + e < s.cols) fw[b][h][t][e] = table[static_cast<int64_t>(c + e) * s.rank + r];
                            }
                        }
                    }
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int t = 0; t < kR; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(fw[b][h][t][e], fx[b][h][e], acc[t], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kR; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][t * 16 + 4 * g + e][i] = acc[t][e];
    if (threadIdx.x < 16) owner[threadIdx.x] = id;
    __syncthreads();
    for (int at = threadIdx.x; at < kRanks * kRowTile; at += 64 * kSumWaves) {
        const int c = at / kRanks, r = at % kRanks;
        const int who = owner[c];  // this workgroup's adapter, or none and this is the first
        if (n0 + c >= s.rows || r0 + r >= s.y.pad || !(who == k || (who < 0 && blockIdx.y == 0))) continue;
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kSumWaves; ++w) x += red[w][r][c];
        low_result(s, split, n0 + c, r0 + r, x, who);
    }
}

// Many bf16 rows: a workgroup has 64, 16 a wave, which share the table's tiles of 64 channels in two
// LDS buffers in turn; the next tile and the next rows' channels are on their way meanwhile. Rows
// are read again for each of the adapters that 64 of them have: sorted, that is mostly one
// (1,021 rows in runs of 25, 32,003 outputs, rank 8: 45 us, as they come 66 us; 8,192 rows, rank 64: 90 us
// over 11,264 outputs, 25 over 2,816 channels). Bound by the loads' latency: two steps in flight.
constexpr int kWideRows = 64, kWideStep = 64;

template <bool kAlong, int kR>
__global__ __launch_bounds__(256) void low_wide_kernel(SumArgs<uint16_t> s) {
    constexpr int kRanks = kR * 16;
    constexpr int kRow = (kAlong ? kWideStep : kRanks) + 8, kRowsOf = kAlong ? kRanks : kWideStep;
    constexpr int kUnits = kRanks * kWideStep / 8, kPer = (kUnits + 255) / 256;
    __shared__ __align__(16) uint16_t tiles[2][kRowsOf * kRow];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    int all_rows = blockIdx.x * kWideRows + lane;  // a row of a lane, -1: none
    if (s.order) all_rows = all_rows < *s.listed ? s.order[all_rows] : -1;
    const int all_ids = all_rows >= 0 ? row_adapter(s, all_rows) : -1;
    const int n = __shfl(all_rows, wave * 16 + i);
    const int k = slot_adapter(all_ids, blockIdx.y);
    if (k == INT_MAX && blockIdx.y != 0) return;
    const int split = blockIdx.z % s.splits, r0 = blockIdx.z / s.splits * kRanks;
    const int who = __shfl(all_ids, wave * 16 + i);
    f32x4 acc[kR];
#pragma unroll
    for (int t = 0; t < kR; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (k != INT_MAX && r0 < s.rank) {
        const uint16_t* const xr = s.x + max(0, min(n, s.rows - 1)) * s.ld;
        const uint16_t* const table = s.table + k * (static_cast<int64_t>(s.rank) * s.cols);
        const uint16_t* const end = s.table + s.adapters * (static_cast<int64_t>(s.rank) * s.cols);
        const bool odd = (s.rank & 1) && k == s.adapters - 1;
        const int first = split * s.steps_per_split;
        const int last = min((s.cols + kWideStep - 1) / kWideStep, first + s.steps_per_split);
        u32x4 fx[2], next[2], w[kPer];
        auto load = [&](int step) {
            const int c0 = step * kWideStep;
#pragma unroll
            for (int h = 0; h < 2; ++h) next[h] = load_row8(xr + c0 + h * 32 + 8 * g, s.cols - (c0 + h * 32 + 8 * g));
            const uint16_t* const p = table + static_cast<int64_t>(c0) * s.rank;
            const auto rs = resource(p, (end - p) * 2);
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                const int unit = q * 256 + threadIdx.x;
                if (unit >= kUnits) break;
                if constexpr (kAlong) {
                    const int row = unit / (kWideStep / 8), c = c0 + unit % (kWideStep / 8) * 8;
                    w[q] = load_row8(table + static_cast<int64_t>(min(r0 + row, s.rank - 1)) * s.cols + c, s.cols - c);
                } else {
                    const int row = unit / (kRanks / 8), col = unit % (kRanks / 8) * 8;
                    w[q] = load16(rs, row < s.cols - c0 && r0 + col < s.rank ? static_cast<uint32_t>(row * s.rank + r0 + col) * 2 : 0x80000000u);
                    if (odd && c0 + row == s.cols - 1) w[q] |= at_element(s.rank - 1 - r0 - col, end[-1]);
                }
            }
        };
        if (first < last) load(first);
        for (int step = first; step < last; ++step) {
            uint16_t* const tile = tiles[(step - first) & 1];
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                const int unit = q * 256 + threadIdx.x;
                if (unit >= kUnits) break;
                constexpr int kPerRow = (kAlong ? kWideStep : kRanks) / 8;
                *reinterpret_cast<u32x4*>(tile + unit / kPerRow * kRow + unit % kPerRow * 8) = w[q];
            }
            fx[0] = next[0];
            fx[1] = next[1];
            __syncthreads();  // a buffer is written again two steps on, behind the next barrier
            if (step + 1 < last) load(step + 1);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < kR; ++t) {
                    bf16x8 f;
                    if constexpr (kAlong)
                        f = *reinterpret_cast<const bf16x8*>(tile + (t * 16 + i) * kRow + h * 32 + 8 * g);
                    else
                        f = frag_across(tile + h * 32 * kRow, kRow, t * 16, lane);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, fx[h]), acc[t], 0, 0, 0);
                }
        }
    }
    if (n < 0 || n >= s.rows || !(who == k || (who < 0 && blockIdx.y == 0))) return;
#pragma unroll
    for (int t = 0; t < kR; ++t) {
        const int r = r0 + t * 16 + 4 * g;
        if (r >= s.y.pad) continue;
        if (s.parts) {  // 4 neighbours; the padding is a multiple of 32
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = who >= 0 && r + e < s.rank ? acc[t][e] : 0.f;
            *reinterpret_cast<f32x4*>(s.parts + (static_cast<int64_t>(split) * s.rows + n) * s.y.pad + r) = x;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) low_result(s, split, n, r + e, acc[t][e], who);
        }
    }
}

// The parts in order, times the row's scale. Latency: 5 us.
template <typename T>
__global__ __launch_bounds__(256) void low_join_kernel(SumArgs<T> s) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, all = static_cast<int64_t>(s.rows) * s.y.pad;
    if (at >= all) return;
    const int64_t n = at / s.y.pad;
    const int r = static_cast<int>(at % s.y.pad);
    float x = 0.f;
    if (r < s.rank) {
#pragma unroll 8
        for (int i = 0; i < s.splits; ++i) x += s.parts[i * all + at];
    }
    const int id = row_adapter(s, static_cast<int>(n));
    low_store(s.y, n, r, id >= 0 && r < s.rank ? x * s.scale[id] : 0.f);
}

// ---- an adapter's rows -------------------------------------------------------------
//
// begin[k] .. begin[k + 1] of `order` are the rows of adapter k, in their order: a workgroup per
// adapter counts the rows of those before it and lists its own, so that no workgroup waits
// for another. Bound by the barriers of its steps: 8,192 rows and 5 adapters 9 us.
__global__ __launch_bounds__(1024) void order_kernel(const int32_t* ids, int rows, int adapters, int32_t* begin, int32_t* order) {
    __shared__ int sums[16];
    const int k = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0;
    for (int n = threadIdx.x; n < rows; n += 1024) before += ids[n] >= 0 && ids[n] < k;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
    if (lane == 0) sums[wave] = before;
    __syncthreads();
    int at = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) at += sums[w];
    __syncthreads();
    if (threadIdx.x == 0) begin[k] = at;
    for (int base = 0; base < rows; base += 1024) {
        const int n = base + threadIdx.x;
        const bool mine = n < rows && ids[n] == k;
        const uint64_t all = __ballot(mine);
        if (lane == 0) sums[wave] = __popcll(all);
        __syncthreads();
        int to = at;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            if (w < wave) to += sums[w];
            at += sums[w];
        }
        if (mine) order[to + __popcll(all & ((1ull << lane) - 1))] = n;
        __syncthreads();
    }
    if (k == adapters - 1 && threadIdx.x == 0) begin[adapters] = at;
}

// ---- sums over an adapter's rows ----------------------------------------------------
//
// g[k](r, c) = sum over the rows n of adapter k of x[n][c] * y[n][r], stored as
// [adapters][cols][rank] (kRanksLast: dB, of dout and u) or [adapters][rank][cols] (dA, of
// hidden and du). bf16 operands are both across the sum: they go through LDS, transposed on
// their way to the registers. A wave takes 64 columns; the matrix instructions' M side,
// of which a lane has 4 neighbours, is the side that lies together in memory. An adapter's
// rows are divided where the columns do not fill the card, and the parts joined in order.
// 8,192 rows, 5 adapters of rank 64: dB, of 11,264 columns, 79 us (185 MB of dout, 2.3 TB/s) and 10 for
// the join, dA, of 2,816, 34 and 8: bound by the steps' latency, with 440 and 330 workgroups, two
// to a compute unit. Steps of 64 rows: the same with one buffer for y and two barriers a
// step, 20 us more with two buffers, whose 92 KiB of LDS leave room for one workgroup.
template <typename T>
struct OuterArgs {
    const T* x;
    int64_t ld;
    int cols, rank;
    Low<T> y;
    const int32_t* begin;
    const int32_t* order;
    T* out;
    float* parts;  // [splits], each of the output's size, or NULL
    int splits;
    int64_t size;  // of all adapters
};

constexpr int kOuterCols = 64;  // of a wave
constexpr int kOuterRows = 32;  // of a step (bf16)

template <typename T, bool kRanksLast, int kR>
__global__ __launch_bounds__(256) void outer_kernel(OuterArgs<T> s) {
    constexpr int kRanks = kR * 16, kC = kOuterCols / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int k = blockIdx.z / s.splits, split = blockIdx.z % s.splits, r0 = blockIdx.y * kRanks;
    const int c0 = (blockIdx.x * 4 + wave) * kOuterCols;
    const int begin = s.begin[k], mine = s.begin[k + 1] - begin;
    // this part's rows, whole steps of them
    const int steps = (mine + kOuterRows - 1) / kOuterRows, each = (steps + s.splits - 1) / s.splits * kOuterRows;
    const int from = min(mine, split * each), count = min(mine, from + each) - from;
    const int32_t* const rows = s.order + begin + from;
    f32x4 acc[kC][kR];
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int r = 0; r < kR; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (sizeof(T) == 2) {
        // A wave's columns are its own, the ranks the workgroup's, in two buffers in turn. The next
        // step's loads are in flight while this one is multiplied, and the rows' numbers a step ahead of them.
        constexpr int kXRow = kOuterCols + 8, kYRow = kRanks + 8;
        constexpr int kX = kOuterRows / 8, kYUnits = kLowPlanes * kOuterRows * kRanks / 8, kY = (kYUnits + 255) / 256;
        __shared__ __align__(16) uint16_t xs[4][kOuterRows * kXRow];
        __shared__ __align__(16) uint16_t ys[2][kLowPlanes * kOuterRows * kYRow];
        u32x4 x[kX], y[kY];
        int xn[kX], yn[kY];
        const int c = c0 + (lane & 7) * 8;
        auto y_row = [&](int q) { return (q * 256 + static_cast<int>(threadIdx.x)) / (kRanks / 8) % kOuterRows; };
        auto number = [&](int n0) {
#pragma unroll
            for (int q = 0; q < kX; ++q) {
                const int at = n0 + q * 8 + (lane >> 3);
                xn[q] = at < count ? rows[at] : -1;
            }
#pragma unroll
            for (int q = 0; q < kY; ++q) {
                const int at = n0 + y_row(q);
                yn[q] = at < count ? rows[at] : -1;
            }
        };
        auto load = [&]() {
#pragma unroll
            for (int q = 0; q < kX; ++q) x[q] = load_row8(s.x + xn[q] * s.ld + c, xn[q] >= 0 ? s.cols - c : 0);
#pragma unroll
            for (int q = 0; q < kY; ++q) {
                const int at = q * 256 + threadIdx.x, plane = at / (kOuterRows * kRanks / 8), col = r0 + at % (kRanks / 8) * 8;
                y[q] = u32x4{0, 0, 0, 0};
                if (yn[q] >= 0 && at < kYUnits && col < s.y.pad)
                    y[q] = *reinterpret_cast<const u32x4*>(s.y.p + plane * s.y.plane + static_cast<int64_t>(yn[q]) * s.y.pad + col);
            }
        };
        number(0);
        load();
        number(kOuterRows);
        for (int n0 = 0, turn = 0; n0 < count; n0 += kOuterRows, turn ^= 1) {
            uint16_t* const xt = xs[wave];
            uint16_t* const yt = ys[turn];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < kX; ++q) *reinterpret_cast<u32x4*>(xt + (q * 8 + (lane >> 3)) * kXRow + (lane & 7) * 8) = x[q];
#pragma unroll
            for (int q = 0; q < kY; ++q) {
                const int at = q * 256 + threadIdx.x, plane = at / (kOuterRows * kRanks / 8), col = at % (kRanks / 8) * 8;
                if (at < kYUnits) *reinterpret_cast<u32x4*>(yt + (plane * kOuterRows + y_row(q)) * kYRow + col) = y[q];
            }
            __syncthreads();
            if (n0 + kOuterRows < count) {
                load();
                number(n0 + 2 * kOuterRows);
            }
#pragma unroll
            for (int h = 0; h < kOuterRows / 32; ++h) {
                bf16x8 fy[kLowPlanes][kR];
#pragma unroll
                for (int p = 0; p < kLowPlanes; ++p)
#pragma unroll
                    for (int r = 0; r < kR; ++r) fy[p][r] = frag_across(yt + (p * kOuterRows + h * 32) * kYRow, kYRow, r * 16, lane);
#pragma unroll
                for (int t = 0; t < kC; ++t) {
                    const bf16x8 fx = frag_across(xt + h * 32 * kXRow, kXRow, t * 16, lane);
#pragma unroll
                    for (int p = kLowPlanes - 1; p >= 0; --p)
#pragma unroll
                        for (int r = 0; r < kR; ++r)
                            acc[t][r] = kRanksLast ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(fy[p][r], fx, acc[t][r], 0, 0, 0)
                                                   : __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx, fy[p][r], acc[t][r], 0, 0, 0);
                }
            }
        }
    } else {
        constexpr int kDeep = kR == 4 ? 4 : 8;  // groups of 4 rows whose loads are in flight together
        for (int n0 = 0; n0 < count; n0 += 4 * kDeep) {
            float fx[kDeep][kC], fy[kDeep][kR];
            int64_t n[kDeep];
#pragma unroll
            for (int b = 0; b < kDeep; ++b) n[b] = rows[min(n0 + 4 * b + g, count - 1)];
#pragma unroll
            for (int b = 0; b < kDeep; ++b) {
                const bool there = n0 + 4 * b + g < count;
#pragma unroll
                for (int t = 0; t < kC; ++t) {
                    const int col = c0 + t * 16 + i;
                    fx[b][t] = there && col < s.cols ? s.x[n[b] * s.ld + col] : 0.f;
                }
#pragma unroll
                for (int r = 0; r < kR; ++r) {
                    const int at = r0 + r * 16 + i;
                    fy[b][r] = there && at < s.y.pad ? s.y.p[n[b] * s.y.pad + at] : 0.f;
                }
            }
#pragma unroll
            for (int b = 0; b < kDeep; ++b)
#pragma unroll
                for (int t = 0; t < kC; ++t)
#pragma unroll
                    for (int r = 0; r < kR; ++r)
                        acc[t][r] = kRanksLast ? __builtin_amdgcn_mfma_f32_16x16x4f32(fy[b][r], fx[b][t], acc[t][r], 0, 0, 0)
                                               : __builtin_amdgcn_mfma_f32_16x16x4f32(fx[b][t], fy[b][r], acc[t][r], 0, 0, 0);
        }
    }
    const int64_t base = static_cast<int64_t>(k) * s.cols * s.rank;
#pragma unroll
    for (int t = 0; t < kC; ++t)
#pragma unroll
        for (int r = 0; r < kR; ++r) {
            const float x[4] = {acc[t][r][0], acc[t][r][1], acc[t][r][2], acc[t][r][3]};
            const int col = c0 + t * 16 + (kRanksLast ? i : 4 * g), rank = r0 + r * 16 + (kRanksLast ? 4 * g : i);
            if (col >= s.cols || rank >= s.rank) continue;
            const int64_t at = base + (kRanksLast ? static_cast<int64_t>(col) * s.rank + rank : static_cast<int64_t>(rank) * s.cols + col);
            const int n = kRanksLast ? s.rank - rank : s.cols - col;
            if (s.parts)
                store_out(s.parts + split * s.size + at, x, n);
            else
                store_out(s.out + at, x, n);
        }
}

// An adapter's gradient from its parts, in their order.
template <typename T>
__global__ __launch_bounds__(256) void outer_join_kernel(OuterArgs<T> s) {
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (at >= s.size) return;
    const int n = static_cast<int>(min(s.size - at, int64_t{4}));
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < s.splits; ++i) {
        const float* const p = s.parts + i * s.size + at;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += e < n ? p[e] : 0.f;
    }
    store_out(s.out + at, x, n);
}

// A of the adapters that have rows, transposed: [adapters][dim][rank], 8 ranks a thread. Latency: 3 to 6 us.
template <typename T>
__global__ __launch_bounds__(256) void transpose_kernel(const T* a, int rank, int dim, const int32_t* begin, T* to) {
    const int k = blockIdx.z;
    if (begin[k] == begin[k + 1]) return;
    const int d = blockIdx.x * 256 + threadIdx.x, r0 = blockIdx.y * 8;
    if (d >= dim) return;
    const T* const p = a + (static_cast<int64_t>(k) * rank + r0) * dim + d;
    T* const q = to + (static_cast<int64_t>(k) * dim + d) * rank + r0;
    T v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = r0 + r < rank ? p[static_cast<int64_t>(r) * dim] : T(0);
    if (r0 + 8 <= rank) {
        __builtin_memcpy(q, v, sizeof(v));
    } else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r0 + r < rank) q[r] = v[r];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void zero_kernel(T* p, int64_t n) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at < n) p[at] = T(0);
}
template <typename T>
void zero(T* p, int64_t n, hipStream_t st) {
    constexpr int64_t kMost = int64_t{256} << 22;
    for (int64_t at = 0; at < n; at += kMost) zero_kernel<T><<<static_cast<unsigned>((std::min(n - at, kMost) + 255) / 256), 256, 0, st>>>(p + at, std::min(n - at, kMost));
}

// f(rank tiles of a workgroup)
template <typename F>
void by_rank(int rank, F f) {
    if (rank <= 16)
        f(std::integral_constant<int, 1>{});
    else if (rank <= 32)
        f(std::integral_constant<int, 2>{});
    else
        f(std::integral_constant<int, 4>{});
}

template <typename T>
struct Call {
    const ge_project_args& x;
    const Plan& plan;
    const Buffers& b;
    hipStream_t st;

    int64_t hidden_ld() const { return x.rows > 1 ? x.hidden_stride : x.dim; }
    int64_t dout_ld() const { return x.rows > 1 ? x.dout_stride : x.out_dim; }
    Operand rows(const void* p, int64_t ld, int64_t n, int dim, bool packed, int64_t kpad, void* to) const {
        return packed ? head::packed_rows(static_cast<const T*>(p), ld, n, dim, kpad, to, st) : Operand{p, ld, (n - 1) * ld + dim};
    }
    Operand weights(int v0, int n) const {
        const int64_t ld = x.out_dim > 1 ? x.weight_stride : x.dim;
        return rows(static_cast<const T*>(x.weight) + v0 * ld, ld, n, x.dim, plan.pack_w, plan.kpad, b.wpack);
    }
    template <int kBm, int kBn, int kWm, int kWn, bool kA, bool kB, typename Epi>
    void run(const Operand& a, const Operand& bb, int64_t k, int m, int n, int splits, int group, const Epi& e) const {
        head::run_tiles<T, kBm, kBn, kWm, kWn, kA, kB>(a, bb, k, m, n, splits, group, e, st);
    }
    Low<T> low(void* p) const {
        const int pad = static_cast<int>(rank_pad(x.rank));
        return Low<T>{static_cast<T*>(p), static_cast<int64_t>(x.rows) * pad, pad};
    }
    Adapters<T> adapters(const void* table, int64_t m, void* u) const {
        if (x.adapters == 0) return Adapters<T>{};
        return Adapters<T>{static_cast<const T*>(table), m, x.rank, x.adapters, x.adapter, low(u)};
    }
    template <bool kAlong>
    void low_sum(const void* in, int64_t ld, int cols, const void* table, void* to, bool sorted) const {
        const bool wide = sizeof(T) == 2 && x.rows > kFewRows;
        const int tile = wide ? kWideRows : kRowTile, step = wide ? kWideStep : kSumStep;
        const int splits = low_splits(x.rows, cols, wide);
        SumArgs<T> s{static_cast<const T*>(in), ld, x.rows, cols, static_cast<const T*>(table), x.scale, x.adapter, x.adapters, x.rank,
                     low(to), splits > 1 ? b.parts : nullptr, splits, 0, nullptr, nullptr};
        if (sorted && wide) {
            s.order = b.order + x.adapters + 1;
            s.listed = b.order + x.adapters;
        }
        s.steps_per_split = ((cols + step - 1) / step + splits - 1) / splits;
        by_rank(x.rank, [&](auto r) {
            constexpr int kR = decltype(r)::value;
            // the padding's zeros too, or the join adds them
            const int ranks = ((splits > 1 ? x.rank : s.y.pad) + kR * 16 - 1) / (kR * 16);
            const dim3 grid((x.rows + tile - 1) / tile, std::min(tile, x.adapters), splits * ranks);
            if constexpr (sizeof(T) == 2) {
                if (wide) {
                    low_wide_kernel<kAlong, kR><<<grid, 256, 0, st>>>(s);
                    return;
                }
            }
            low_sum_kernel<T, kAlong, kR><<<grid, 64 * kSumWaves, 0, st>>>(s);
        });
        if (splits > 1) low_join_kernel<T><<<static_cast<unsigned>((static_cast<int64_t>(x.rows) * s.y.pad + 255) / 256), 256, 0, st>>>(s);
    }
    template <bool kRanksLast>
    void outer(const void* in, int64_t ld, int cols, void* y, void* out) const {
        const int64_t size = static_cast<int64_t>(x.adapters) * cols * x.rank;
        const int splits = outer_splits(x.rows, x.adapters, cols, size, plan.parts);
        OuterArgs<T> s{static_cast<const T*>(in), ld, cols, x.rank, low(y), b.order, b.order + x.adapters + 1, static_cast<T*>(out),
                       splits > 1 ? b.parts : nullptr, splits, size};
        by_rank(x.rank, [&](auto r) {
            constexpr int kR = decltype(r)::value;
            outer_kernel<T, kRanksLast, kR><<<dim3((cols + 4 * kOuterCols - 1) / (4 * kOuterCols), (x.rank + kR * 16 - 1) / (kR * 16), x.adapters * splits),
                                              256, 0, st>>>(s);
        });
        if (splits > 1) outer_join_kernel<T><<<static_cast<unsigned>(((size + 3) / 4 + 255) / 256), 256, 0, st>>>(s);
    }
    template <typename Epi>
    void product(const Operand& w, const Operand& h, int n, const Epi& e) const {
        const int64_t k = plan.pack_w && plan.pack_h ? plan.kpad : x.dim;
        if constexpr (sizeof(T) == 4) {
            if (plan.tile_n == 32)
                run<128, 32, 4, 1, true, true>(w, h, k, n, x.rows, 1, 8, e);
            else if (plan.tile_n == 64)
                run<128, 64, 2, 2, true, true>(w, h, k, n, x.rows, 1, 8, e);
            else if (plan.tile_n == 96)
                run<128, 96, 2, 2, true, true>(w, h, k, n, x.rows, 1, 8, e);
            else
                run<128, 128, 2, 2, true, true>(w, h, k, n, x.rows, 1, 8, e);
        } else if (plan.tile_n == head::kSmallTileN) {
            run<head::kSmallTileM, head::kSmallTileN, 4, 1, true, true>(w, h, k, n, x.rows, 1, 4, e);
        } else if (plan.tile_n == 64) {
            run<head::kSmallTileM, 64, 4, 1, true, true>(w, h, k, n, x.rows, 1, 4, e);
        } else if (plan.tile_n == 128) {
            run<256, 128, 2, 2, true, true>(w, h, k, n, x.rows, 1, 6, e);
        } else {
            run<256, 256, 2, 2, true, true>(w, h, k, n, x.rows, 1, 6, e);
        }
    }
    template <typename O>
    void forward() const {
        if (x.adapters) low_sum<true>(x.hidden, hidden_ld(), x.dim, x.a, b.u, false);
        const Operand h = rows(x.hidden, hidden_ld(), x.rows, x.dim, plan.pack_h, plan.kpad, b.hpack);
        const int64_t ld = x.rows > 1 ? x.out_stride : x.out_dim;
        for (int v0 = 0; v0 < x.out_dim; v0 += plan.piece) {
            const int n = std::min(plan.piece, x.out_dim - v0);
            const OutEpi<T, O> e{adapters(x.b, x.out_dim, b.u), x.rows, n, v0, static_cast<O*>(x.out) + v0, ld};
            product(weights(v0, n), h, n, e);
        }
    }
    template <typename Epi>
    void hidden(const Operand& w, const Operand& d, int n, const Epi& e) const {
        constexpr int kTile = sizeof(T) == 4 ? 128 : 256;
        if (sizeof(T) == 2 && x.rows <= 128)
            run<kTile, 128, 2, 2, false, true>(w, d, n, x.dim, x.rows, plan.splits, 6, e);
        else
            run<kTile, kTile, 2, 2, false, true>(w, d, n, x.dim, x.rows, plan.splits, 6, e);
    }
    void backward() const {
        const bool low_rank = x.adapters > 0;
        if (low_rank) order_kernel<<<x.adapters, 1024, 0, st>>>(x.adapter, x.rows, x.adapters, b.order, b.order + x.adapters + 1);
        if (low_rank && (x.dhidden || x.da)) low_sum<false>(x.dout, dout_ld(), x.out_dim, x.b, b.du, true);
        if (x.dhidden) {
            if (low_rank)
                transpose_kernel<T><<<dim3((x.dim + 255) / 256, (x.rank + 7) / 8, x.adapters), 256, 0, st>>>(
                    static_cast<const T*>(x.a), x.rank, x.dim, b.order, static_cast<T*>(b.at));
            T* const dh = static_cast<T*>(x.dhidden);
            const int64_t dh_ld = x.rows > 1 ? x.dhidden_stride : x.dim;
            const int64_t hld = (x.dim + 3) / 4 * 4;
            const bool direct = plan.splits == 1 && plan.piece >= x.out_dim;
            for (int v0 = 0; v0 < x.out_dim; v0 += plan.piece) {
                const int n = std::min(plan.piece, x.out_dim - v0);
                const int64_t npad = head::round_up(n, head::kPadK);
                const Operand w = weights(v0, n);
                const Operand d = rows(static_cast<const T*>(x.dout) + v0, dout_ld(), x.rows, n, plan.pack_d, npad, b.dpack);
                const Adapters<T> low = v0 == 0 ? adapters(b.at, x.dim, b.du) : Adapters<T>{};
                if (direct)
                    hidden(w, d, n, HiddenEpi<T, true>{low, x.rows, x.dim, dh, dh_ld, 0, false});
                else
                    hidden(w, d, n, HiddenEpi<T, false>{low, x.rows, x.dim, b.dhidden, hld, x.rows * hld, v0 > 0});
            }
            if (!direct)
                head::for_units(x.rows, 2 * hld, [&](int64_t r, unsigned n, dim3 grid, dim3 block) {
                    hidden_sum_kernel<T><<<grid, block, 0, st>>>(b.dhidden + r * hld, hld, x.rows * hld, plan.splits, n, x.dim, dh + r * dh_ld, dh_ld);
                });
        }
        if (x.da) outer<false>(x.hidden, hidden_ld(), x.dim, b.du, x.da);
        if (x.db) {
            low_sum<true>(x.hidden, hidden_ld(), x.dim, x.a, b.u, true);
            outer<true>(x.dout, dout_ld(), x.out_dim, b.u, x.db);
        }
    }
    void no_rows() const {  // the adapters' gradients are zeros
        const int64_t n = static_cast<int64_t>(x.adapters) * x.rank;
        if (x.da) zero(static_cast<T*>(x.da), n * x.dim, st);
        if (x.db) zero(static_cast<T*>(x.db), n * x.out_dim, st);
    }
};

template <typename T>
void launch(const ge_project_args& x, const Plan& plan, const Buffers& b, bool backward, hipStream_t st) {
    const Call<T> call{x, plan, b, st};
    if (backward && x.rows == 0)
        call.no_rows();
    else if (backward)
        call.backward();
    else if (x.rows == 0)
        return;
    else if (x.out_dtype == GE_DTYPE_F32)
        call.template forward<float>();
    else
        call.template forward<uint16_t>();
}

int hip_error(hipError_t e, const char* what) {
    (void)hipGetLastError();  // reported here: the next launch's check shall not find it
    char msg[256];
    plan_fail(msg, sizeof(msg), 0, "%s: %s", what, hipGetErrorString(e));
    return report(GE_ERR_DEVICE, msg);
}

// Switches the calling thread to `device` for the lifetime of the object.
struct OnDevice {
    int prev = -1;
    bool ok = true;
    explicit OnDevice(int device) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != device) ok = hipSetDevice(device) == hipSuccess;
    }
    ~OnDevice() {
        int cur = -1;
        if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
    }
};

}  // namespace
}  // namespace projection
}  // namespace ge

struct ge_projection {
    int device;
    ge::projection::Capacity cap;
    ge::projection::Buffers buf;
};

extern "C" {

int ge_projection_create(int device, int max_rows, int max_dim, int max_out, int max_rank, int max_adapters, int dtype, int train,
                         ge_projection** out) {
    using namespace ge::projection;
    char msg[256] = "";
    if (!out) return ge::report(GE_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (const int rc = check_create(max_rows, max_dim, max_out, max_rank, max_adapters, dtype, msg, sizeof(msg))) return ge::report(rc, msg);
    int n = 0;
    hipDeviceProp_t prop;
    if (hipGetDeviceCount(&n) != hipSuccess || device < 0 || device >= n || hipGetDeviceProperties(&prop, device) != hipSuccess ||
        std::strncmp(prop.gcnArchName, "gfx950", 6) != 0) {
        ge::plan_fail(msg, sizeof(msg), 0, "device %d is not a gfx950 device (%d devices)", device, n);
        return ge::report(GE_ERR_NO_DEVICE, msg);
    }
    OnDevice guard(device);
    if (!guard.ok) return ge::report(GE_ERR_DEVICE, "hipSetDevice failed");
    ge_projection* h = new (std::nothrow) ge_projection{};
    if (!h) return ge::report(GE_ERR_DEVICE, "out of host memory");
    h->device = device;
    Capacity& c = h->cap;
    c = Capacity{max_rows, max_dim, max_out, max_rank, max_adapters, dtype, train != 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    size_workspace(c);
    hipError_t e = hipSuccess;
    auto alloc = [&](auto*& p, int64_t bytes) {
        if (e == hipSuccess && bytes > 0) e = hipMalloc(reinterpret_cast<void**>(&p), static_cast<size_t>(bytes));
    };
    Buffers& b = h->buf;
    alloc(b.hpack, c.hpack);
    alloc(b.wpack, c.wpack);
    alloc(b.u, c.u);
    alloc(b.du, c.du);
    alloc(b.parts, c.parts);
    alloc(b.order, c.order);
    alloc(b.at, c.at);
    alloc(b.dpack, c.dpack);
    alloc(b.dhidden, c.dhidden);
    if (e != hipSuccess) {
        ge_projection_destroy(h);
        return hip_error(e, "ge_projection_create");
    }
    *out = h;
    return GE_OK;
}

void ge_projection_destroy(ge_projection* h) {
    if (!h) return;
    ge::projection::OnDevice guard(h->device);
    const ge::projection::Buffers& b = h->buf;
    for (void* p : {b.hpack, b.wpack, b.u, b.du, static_cast<void*>(b.parts), static_cast<void*>(b.order), b.at, b.dpack,
                    static_cast<void*>(b.dhidden)})
        (void)hipFree(p);
    delete h;
}

static int project_call(ge_projection* h, void* stream, const ge_project_args* args, bool backward) {
    using namespace ge::projection;
    char msg[256] = "";
    if (!h || !args) return ge::report(GE_ERR_INVALID_ARG, "projection or args is NULL");
    Plan plan{};
    if (const int rc = check_project(h->cap, *args, backward, plan, msg, sizeof(msg))) return ge::report(rc, msg);
    if (const int rc = check_memory(h->cap, *args, backward, msg, sizeof(msg))) return ge::report(rc, msg);
    OnDevice guard(h->device);
    if (!guard.ok) return ge::report(GE_ERR_DEVICE, "hipSetDevice failed");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (h->cap.dtype == GE_DTYPE_F32)
        launch<float>(*args, plan, h->buf, backward, st);
    else
        launch<uint16_t>(*args, plan, h->buf, backward, st);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GE_OK : hip_error(e, "launch (projection)");
}

int ge_project(ge_projection* h, void* stream, const ge_project_args* args) { return project_call(h, stream, args, false); }
int ge_project_backward(ge_projection* h, void* stream, const ge_project_args* args) { return project_call(h, stream, args, true); }

}  // extern "C"

// The norm over a row's channels and its gradients (include/gemmaedge_head.h).
//
// A row's channels stay in the registers of the threads that share it, 8
// neighbouring ones a vector, so x and dy are read once: the sum and then the
// sum of squared differences from the mean are taken of the registers (one pass
// of sum and sum of squares would lose the variance of channels whose offset is
// large against their spread). Rows of up to 1,024 channels belong to a group of
// 8 to 64 lanes, whose sums need no barrier; longer ones to a whole workgroup.
// A workgroup takes several rows, one after another, and has the next one's
// loads in flight while it works on a row; the weights are read once.
//
// Backward: dx needs two sums over the row, of a = dy w and of a xhat, taken
// together. The weights' gradients are sums over the rows of one channel each:
// a thread adds up its channels over its rows in registers, and a second launch
// adds the workgroups' parts in one fixed order, so the result does not depend
// on the order in which workgroups run.
//
// Both passes are bound by memory. 16,384 rows of 2,816 bf16 channels: forward
// 39 us (4.7 TB/s), backward 65 us (4.3 TB/s) + 4 us for the second launch; a large
// copy moves 4.8 TB/s. Two or three rows ahead, or more workgroups, are no faster.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "head_internal.h"

namespace ge {
namespace head {
namespace {

// Channels of a vector: 16 bytes, so that neighbouring lanes' loads are neighbours.
template <typename T>
constexpr int vec_of = 16 / sizeof(T);
constexpr int kNormThreads = 512;    // most threads of a workgroup
constexpr int kGroupDim = 1024;      // longest row of a lane group
constexpr int kRegisterDim = 8192;   // longest row that stays in registers

template <typename T, int kVec>
struct Vec {
    T v[kVec];
};

// kVec channels of a row of `dim` from i on, zeros behind its end. Rows need no
// alignment beyond their elements': the loads are 16 bytes wide at any address.
template <int kVec, typename T>
__device__ __forceinline__ Vec<T, kVec> load_vec(const T* row, int i, int dim) {
    Vec<T, kVec> r;
    if (i + kVec <= dim) {
        __builtin_memcpy(&r, row + i, sizeof(r));
    } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) r.v[e] = i + e < dim ? row[i + e] : T(0);
    }
    return r;
}
template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T* row, int i, int dim, const float (&x)[kVec]) {
    Vec<T, kVec> r;
#pragma unroll
    for (int e = 0; e < kVec; ++e) r.v[e] = from_f32<T>(x[e]);
    if (i + kVec <= dim) {
        __builtin_memcpy(row + i, &r, sizeof(r));
    } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
            if (i + e < dim) row[i + e] = r.v[e];
    }
}

// How a row is read and written. kWhole: by buffer loads and stores of the row,
// whose bounds the hardware checks four bytes at a time; without branches the
// compiler knows how many are in flight, and the next row's loads are not waited
// for together with this row's stores. The row is then the same in the whole wave.
// kOdd: the same for rows of an odd number of bf16 channels, the last one apart.
// kBranches: rows of lane groups within a wave.
enum Mode { kBranches, kWhole, kOdd };

// A thread's channels of a row, the vectors at at[0], at[1], ..., and how it reads them.
template <Mode kMode, int kVec, int kVecs>
struct Place {
    int dim;
    int at[kVecs];
    int last_vec, last_off;  // kOdd: the thread's vector with the last channel, and the channel's bytes from the row
    __device__ __forceinline__ void init(int d, int lane, int lanes) {
        dim = d;
        last_vec = -1;
        last_off = 0x7ffffff0;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            at[j] = (j * lanes + lane) * kVec;
            if (kMode == kOdd && d - 1 - at[j] >= 0 && d - 1 - at[j] < kVec) {
                last_vec = j;
                last_off = (d - 1) * 2;
            }
        }
    }
    __device__ __forceinline__ bool is_last(int j, int e) const { return kMode == kOdd && j == last_vec && e == (dim - 1) % kVec; }
};

// A row's values in a thread.
template <typename T, Mode kMode, int kVec, int kVecs>
struct RowOf {
    Vec<T, kVec> v[kVecs];
    T last;
    __device__ __forceinline__ float get(const Place<kMode, kVec, kVecs>& p, int j, int e) const {
        return to_f32(p.is_last(j, e) ? last : v[j].v[e]);
    }
};

template <typename T, Mode kMode, int kVec, int kVecs>
__device__ __forceinline__ void load_row(const T* p, int64_t stride, int64_t r, int64_t rows, const Place<kMode, kVec, kVecs>& pl,
                                         RowOf<T, kMode, kVec, kVecs>& to) {
    if constexpr (kMode != kBranches) {
        constexpr int kSize = sizeof(T);
        T* const row = const_cast<T*>(p + r * stride);
        const int bytes = r < rows ? pl.dim * kSize : 0;
        __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(row, 0, kMode == kOdd && bytes ? bytes - kSize : bytes, 0x00027000);
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
            to.v[j] = __builtin_bit_cast(Vec<T, kVec>, __builtin_amdgcn_raw_buffer_load_b128(rs, pl.at[j] * kSize, 0, 0));
        if constexpr (kMode == kOdd) {
            rs = __builtin_amdgcn_make_buffer_rsrc(row, 0, bytes, 0x00027000);
            to.last = __builtin_amdgcn_raw_buffer_load_b16(rs, pl.last_off, 0, 0);
        }
    } else if (r < rows) {
#pragma unroll
        for (int j = 0; j < kVecs; ++j) to.v[j] = load_vec<kVec>(p + r * stride, pl.at[j], pl.dim);
    }
}
template <Mode kMode, int kVec, int kVecs, typename T>
__device__ __forceinline__ void store_row(T* p, int64_t stride, int64_t r, const Place<kMode, kVec, kVecs>& pl, const float (&x)[kVecs][kVec]) {
    if constexpr (kMode != kBranches) {
        constexpr int kSize = sizeof(T);
        T* const row = p + r * stride;
        const int bytes = pl.dim * kSize;
        __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(row, 0, kMode == kOdd ? bytes - kSize : bytes, 0x00027000);
        using Words = decltype(__builtin_amdgcn_raw_buffer_load_b128(rs, 0, 0, 0));
        T last = T(0);
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            Vec<T, kVec> v;
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                v.v[e] = from_f32<T>(x[j][e]);
                if (pl.is_last(j, e)) last = v.v[e];
            }
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(Words, v), rs, pl.at[j] * kSize, 0, 0);
        }
        if constexpr (kMode == kOdd) {
            rs = __builtin_amdgcn_make_buffer_rsrc(row, 0, bytes, 0x00027000);
            __builtin_amdgcn_raw_buffer_store_b16(last, rs, pl.last_off, 0, 0);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kVecs; ++j) store_vec(p + r * stride, pl.at[j], pl.dim, x[j]);
    }
}

// Sum over groups of kLanes lanes, the same in each of them. Steps within 16 lanes
// are modifiers of the addition, the others swap rows of lanes between registers:
// nothing passes LDS, whose six round trips a sum took longer than a row's loads.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
    auto dpp = [&](auto ctrl) {
        const int w = __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true);
        v += __builtin_bit_cast(float, w);
    };
    dpp(std::integral_constant<int, 0xB1>{});   // lane ^ 1
    dpp(std::integral_constant<int, 0x4E>{});   // lane ^ 2
    dpp(std::integral_constant<int, 0x141>{});  // mirrored in 8
    if (kLanes >= 16) dpp(std::integral_constant<int, 0x140>{});  // mirrored in 16
    if (kLanes >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const uint32_t a = r[0], b = r[1];
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    if (kLanes >= 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const uint32_t a = r[0], b = r[1];
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    return v;
}

// The threads of one row: kGroup lanes of a wave, or (0) the whole workgroup.
constexpr int kMostWaves = kNormThreads / 64;
template <int kGroup>
struct Team {
    int lane, slot, lanes, slots;
    float2* red;  // [2][kMostWaves]
    int turn = 0;
    __device__ __forceinline__ explicit Team(float2* lds) : red(lds) {
        lanes = kGroup ? kGroup : blockDim.x;
        lane = kGroup ? threadIdx.x % (kGroup ? kGroup : 1) : threadIdx.x;
        slot = kGroup ? threadIdx.x / (kGroup ? kGroup : 1) : 0;
        if (kGroup == 64) slot = __builtin_amdgcn_readfirstlane(slot);
        slots = kGroup ? blockDim.x / (kGroup ? kGroup : 1) : 1;
        if (!kGroup) {  // waves that are not there add nothing
            if (threadIdx.x < 2 * kMostWaves) red[threadIdx.x] = make_float2(0.f, 0.f);
            __syncthreads();
        }
    }
    // Sums of two values over the team, the same in every thread. Two buffers in
    // turn: a wave writes one again only after a barrier that every wave reaches
    // when it has read it.
    __device__ __forceinline__ float2 sum(float2 v) {
        v.x = lanes_sum<kGroup ? kGroup : 64>(v.x);
        v.y = lanes_sum<kGroup ? kGroup : 64>(v.y);
        if (kGroup) return v;
        float2* buf = red + turn * kMostWaves;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
        __syncthreads();
        float2 s = buf[0];
#pragma unroll
        for (int i = 1; i < kMostWaves; ++i) {
            s.x += buf[i].x;
            s.y += buf[i].y;
        }
        return s;
    }
};

template <typename T, typename W, int kGroup, int kVecs, Mode kMode>
__global__ __launch_bounds__(kNormThreads) void norm_kernel(ge_norm_args x) {
    __shared__ __align__(16) float2 red[2 * kMostWaves];
    constexpr int kVec = vec_of<T>;
    Team<kGroup> team(red);
    const int dim = x.dim;
    const float n = static_cast<float>(dim);
    float w[kVecs][kVec], b[kVecs][kVec];
    Place<kMode, kVec, kVecs> place;
    place.init(dim, team.lane, team.lanes);
    const int(&at)[kVecs] = place.at;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
        const Vec<W, kVec> vw = load_vec<kVec>(static_cast<const W*>(x.weight), at[j], dim);
        Vec<W, kVec> vb{};
        if (x.bias) vb = load_vec<kVec>(static_cast<const W*>(x.bias), at[j], dim);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            w[j][e] = to_f32(vw.v[e]);
            b[j][e] = to_f32(vb.v[e]);
        }
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * team.slots;
    int64_t r = static_cast<int64_t>(blockIdx.x) * team.slots + team.slot;
    if (r >= x.rows) return;  // a lane group of its own; a workgroup's first row is there
    const T* in = static_cast<const T*>(x.x);
    RowOf<T, kMode, kVec, kVecs> next;
    load_row(in, x.x_stride, r, x.rows, place, next);
    for (; r < x.rows; r += step) {
        float h[kVecs][kVec];
        float2 s{0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                h[j][e] = next.get(place, j, e);
                s.x += h[j][e];
            }
        load_row(in, x.x_stride, r + step, x.rows, place, next);
        const float mean = x.center ? team.sum(s).x / n : 0.f;
        float2 q{0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                h[j][e] -= mean;
                if (at[j] + e < dim) q.x = fmaf(h[j][e], h[j][e], q.x);
            }
        const float rstd = 1.0f / sqrtf(team.sum(q).x / n + x.eps);
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
#pragma unroll
            for (int e = 0; e < kVec; ++e) h[j][e] = fmaf(h[j][e] * rstd, w[j][e], b[j][e]);
        store_row(static_cast<T*>(x.y), x.y_stride, r, place, h);
        if (team.lane == 0) {
            x.rstd[r] = rstd;
            if (x.mean) x.mean[r] = mean;
        }
    }
}

// dx, and with kWeight a workgroup's part of the weights' gradients.
template <typename T, typename W, int kGroup, int kVecs, Mode kMode, bool kWeight>
__global__ __launch_bounds__(kNormThreads) void norm_backward_kernel(ge_norm_args x, float* parts) {
    __shared__ __align__(16) float2 red[2 * kMostWaves];
    constexpr int kVec = vec_of<T>;
    __shared__ float over[kWeight && kGroup ? kNormThreads * kVec : 1];
    Team<kGroup> team(red);
    const int dim = x.dim;
    const float inv = 1.0f / static_cast<float>(dim);
    float w[kVecs][kVec], sw[kVecs][kVec], sb[kVecs][kVec];
    Place<kMode, kVec, kVecs> place;
    place.init(dim, team.lane, team.lanes);
    const int(&at)[kVecs] = place.at;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
        const Vec<W, kVec> vw = load_vec<kVec>(static_cast<const W*>(x.weight), at[j], dim);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            w[j][e] = to_f32(vw.v[e]);
            sw[j][e] = sb[j][e] = 0.f;
        }
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * team.slots;
    int64_t r = static_cast<int64_t>(blockIdx.x) * team.slots + team.slot;
    const T* in = static_cast<const T*>(x.x);
    const T* dy = static_cast<const T*>(x.dy);
    struct Row {
        RowOf<T, kMode, kVec, kVecs> x, y;
        float mean, rstd;
    };
    Row next{};
    // A row's statistics by vector loads, which are waited for where they are used:
    // scalar ones would be waited for with the next sum's LDS, a memory's latency a row.
    int lane_zero;
    asm volatile("v_mov_b32 %0, 0" : "=v"(lane_zero));
    const float *mean_of = x.mean + lane_zero, *rstd_of = x.rstd + lane_zero;
    auto fetch = [&](int64_t row) __attribute__((always_inline)) {
        load_row(in, x.x_stride, row, x.rows, place, next.x);
        load_row(dy, x.dy_stride, row, x.rows, place, next.y);
        const int64_t last = min(row, static_cast<int64_t>(x.rows) - 1);
        next.mean = x.center ? mean_of[last] : 0.f;
        next.rstd = rstd_of[last];
    };
    fetch(r);
    for (; r < x.rows; r += step) {
        const float mean = next.mean, rstd = next.rstd;
        float h[kVecs][kVec], a[kVecs][kVec];
        float2 s{0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const float g = next.y.get(place, j, e);
                h[j][e] = (next.x.get(place, j, e) - mean) * rstd;
                a[j][e] = g * w[j][e];
                s.x += a[j][e];
                s.y = fmaf(a[j][e], h[j][e], s.y);
                if (kWeight) {
                    sw[j][e] = fmaf(g, h[j][e], sw[j][e]);
                    sb[j][e] += g;
                }
            }
        fetch(r + step);
        if (!x.dx) continue;
        s = team.sum(s);
        const float sa = x.center ? s.x * inv : 0.f, sx = s.y * inv;
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
#pragma unroll
            for (int e = 0; e < kVec; ++e) a[j][e] = rstd * (a[j][e] - sa - h[j][e] * sx);
        store_row(static_cast<T*>(x.dx), x.dx_stride, r, place, a);
    }
    if constexpr (kWeight) {
        float* p = parts + static_cast<int64_t>(blockIdx.x) * 2 * dim;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (!(k == 0 ? x.dweight : x.dbias)) continue;
#pragma unroll
            for (int j = 0; j < kVecs; ++j) {
                float* o = p + k * dim;
                const float(&v)[kVec] = k == 0 ? sw[j] : sb[j];
                if constexpr (kGroup == 0) {
                    store_vec<float>(o, at[j], dim, v);
                } else {  // the lane groups' sums first, in their order
                    __syncthreads();
#pragma unroll
                    for (int e = 0; e < kVec; ++e) over[e * kNormThreads + threadIdx.x] = v[e];
                    __syncthreads();
                    for (int c = threadIdx.x; c < kGroup * kVec; c += blockDim.x) {
                        const float* q = over + (c % kVec) * kNormThreads + c / kVec;
                        float sum = 0.f;
                        for (int i = 0; i < team.slots; ++i) sum += q[i * kGroup];
                        const int d = j * kGroup * kVec + c;
                        if (d < dim) o[d] = sum;
                    }
                }
            }
        }
    }
}

// The weights' gradients from `n` parts of 2 dim sums: 64 columns of a workgroup,
// 16 waves that take every 16th part.
template <typename W>
__global__ __launch_bounds__(1024) void norm_dw_sum_kernel(ge_norm_args x, const float* parts, int n, int first, int end) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = first + blockIdx.x * 64 + lane;
    const int64_t ld = 2 * static_cast<int64_t>(x.dim);
    float s = 0.f;
    if (c < end) {
#pragma unroll 8
        for (int i = wave; i < n; i += 16) s += parts[i * ld + c];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || c >= end) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][lane];
    if (c < x.dim)
        static_cast<W*>(x.dweight)[c] = from_f32<W>(s);
    else
        static_cast<W*>(x.dbias)[c - x.dim] = from_f32<W>(s);
}

// ---- rows too long for the registers: read again for each sum -------------------

constexpr int kLongThreads = 256;

__device__ __forceinline__ float long_sum(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kLongThreads / 64; ++i) s += red[i];
    return s;
}

template <typename T, typename W>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(ge_norm_args x) {
    __shared__ float red[kLongThreads / 64];
    const int64_t r = blockIdx.x;
    const T* in = static_cast<const T*>(x.x) + r * x.x_stride;
    T* out = static_cast<T*>(x.y) + r * x.y_stride;
    const W* w = static_cast<const W*>(x.weight);
    const W* b = static_cast<const W*>(x.bias);
    const float n = static_cast<float>(x.dim);
    float mean = 0.f;
    if (x.center) {
        float s = 0.f;
        for (int i = threadIdx.x; i < x.dim; i += kLongThreads) s += to_f32(in[i]);
        mean = long_sum(s, red) / n;
    }
    float q = 0.f;
    for (int i = threadIdx.x; i < x.dim; i += kLongThreads) {
        const float d = to_f32(in[i]) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(long_sum(q, red) / n + x.eps);
    for (int i = threadIdx.x; i < x.dim; i += kLongThreads) {
        const float h = (to_f32(in[i]) - mean) * rstd;
        out[i] = from_f32<T>(fmaf(h, to_f32(w[i]), b ? to_f32(b[i]) : 0.f));
    }
    if (threadIdx.x == 0) {
        x.rstd[r] = rstd;
        if (x.mean) x.mean[r] = mean;
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(kLongThreads) void norm_long_dx_kernel(ge_norm_args x) {
    __shared__ float red[kLongThreads / 64];
    const int64_t r = blockIdx.x;
    const T* in = static_cast<const T*>(x.x) + r * x.x_stride;
    const T* dy = static_cast<const T*>(x.dy) + r * x.dy_stride;
    T* dx = static_cast<T*>(x.dx) + r * x.dx_stride;
    const W* w = static_cast<const W*>(x.weight);
    const float inv = 1.0f / static_cast<float>(x.dim);
    const float mean = x.center ? x.mean[r] : 0.f, rstd = x.rstd[r];
    float sa = 0.f, sx = 0.f;
    for (int i = threadIdx.x; i < x.dim; i += kLongThreads) {
        const float a = to_f32(dy[i]) * to_f32(w[i]);
        sa += a;
        sx = fmaf(a, (to_f32(in[i]) - mean) * rstd, sx);
    }
    sx = long_sum(sx, red) * inv;
    sa = x.center ? long_sum(sa, red) * inv : 0.f;
    for (int i = threadIdx.x; i < x.dim; i += kLongThreads) {
        const float a = to_f32(dy[i]) * to_f32(w[i]);
        const float h = (to_f32(in[i]) - mean) * rstd;
        dx[i] = from_f32<T>(rstd * (a - sa - h * sx));
    }
}

// Rows part, part + parts, ... summed for each channel of a workgroup's 256.
template <typename T>
__global__ __launch_bounds__(kLongThreads) void norm_long_dw_kernel(ge_norm_args x, float* parts) {
    const int c = blockIdx.x * kLongThreads + threadIdx.x;
    if (c >= x.dim) return;
    const T* in = static_cast<const T*>(x.x) + c;
    const T* dy = static_cast<const T*>(x.dy) + c;
    float sw = 0.f, sb = 0.f;
    for (int64_t r = blockIdx.y; r < x.rows; r += gridDim.y) {
        const float mean = x.center ? x.mean[r] : 0.f;
        const float g = to_f32(dy[r * x.dy_stride]);
        sw = fmaf(g, (to_f32(in[r * x.x_stride]) - mean) * x.rstd[r], sw);
        sb += g;
    }
    float* p = parts + static_cast<int64_t>(blockIdx.y) * 2 * x.dim;
    p[c] = sw;
    p[x.dim + c] = sb;
}

// How a call's rows are dealt out: lanes of a row (0: the workgroup), vectors of
// a lane, threads of a workgroup, rows of a workgroup at a time.
struct NormPlan {
    int group, vecs, threads, slots;
};
NormPlan norm_plan(int dim, int vec) {
    const int vectors = (dim + vec - 1) / vec;
    NormPlan p{0, 1, 0, 1};
    if (dim <= kGroupDim) {
        while (p.vecs * 64 < vectors) p.vecs *= 2;
        p.group = 8;
        while (p.group * p.vecs < vectors) p.group *= 2;
        p.threads = kNormThreads;
        p.slots = p.threads / p.group;
        return p;
    }
    while (p.vecs * kNormThreads < vectors) p.vecs *= 2;
    p.threads = ((vectors + p.vecs - 1) / p.vecs + 63) / 64 * 64;
    return p;
}

// Calls f with the plan's group and vectors and the rows' mode as constants.
template <typename T, typename F>
void with_plan(const NormPlan& p, int dim, F f) {
    using std::integral_constant;
    constexpr integral_constant<Mode, kBranches> branches{};
    constexpr integral_constant<int, 1> one{};
    if (p.group == 8) return f(integral_constant<int, 8>{}, one, branches);
    if (p.group == 16) return f(integral_constant<int, 16>{}, one, branches);
    if (p.group == 32) return f(integral_constant<int, 32>{}, one, branches);
    auto by_vecs = [&](auto group, auto mode) {
        if (p.vecs == 1) return f(group, one, mode);
        if (sizeof(T) == 2 || p.vecs == 2) return f(group, integral_constant<int, 2>{}, mode);
        if constexpr (sizeof(T) == 4) f(group, integral_constant<int, 4>{}, mode);
    };
    auto by_group = [&](auto mode) {
        if (p.group == 64) return by_vecs(integral_constant<int, 64>{}, mode);
        by_vecs(integral_constant<int, 0>{}, mode);
    };
    if constexpr (sizeof(T) == 2) {
        if (dim % 2 != 0) return by_group(integral_constant<Mode, kOdd>{});
    }
    by_group(integral_constant<Mode, kWhole>{});
}

template <typename T, typename W>
void norm_forward(const ge_norm_args& x, hipStream_t st) {
    if (x.dim > kRegisterDim) {
        norm_long_kernel<T, W><<<x.rows, kLongThreads, 0, st>>>(x);
        return;
    }
    const NormPlan p = norm_plan(x.dim, vec_of<T>);
    const unsigned blocks = std::min((x.rows + p.slots - 1) / p.slots, kNormBlocks);
    with_plan<T>(p, x.dim, [&](auto group, auto vecs, auto mode) {
        norm_kernel<T, W, decltype(group)::value, decltype(vecs)::value, decltype(mode)::value><<<blocks, p.threads, 0, st>>>(x);
    });
}

template <typename T, typename W>
void norm_backward(const ge_norm_args& x, const Buffers& b, hipStream_t st) {
    const bool weight = x.dweight || x.dbias;
    int parts = 0;
    if (x.dim > kRegisterDim) {
        if (weight) {  // before dx, which may be written over dy
            parts = std::min(x.rows, kNormParts);
            if (parts > 0)
                norm_long_dw_kernel<T><<<dim3((x.dim + kLongThreads - 1) / kLongThreads, parts), kLongThreads, 0, st>>>(x, b.norm);
        }
        if (x.dx && x.rows > 0) norm_long_dx_kernel<T, W><<<x.rows, kLongThreads, 0, st>>>(x);
    } else if (x.rows > 0) {
        const NormPlan p = norm_plan(x.dim, vec_of<T>);
        parts = std::min((x.rows + p.slots - 1) / p.slots, kNormParts);
        with_plan<T>(p, x.dim, [&](auto group, auto vecs, auto mode) {
            constexpr int g = decltype(group)::value, v = decltype(vecs)::value;
            constexpr Mode m = decltype(mode)::value;
            if (weight)
                norm_backward_kernel<T, W, g, v, m, true><<<parts, p.threads, 0, st>>>(x, b.norm);
            else if (x.dx)
                norm_backward_kernel<T, W, g, v, m, false><<<parts, p.threads, 0, st>>>(x, b.norm);
        });
    }
    if (weight) {
        const int first = x.dweight ? 0 : x.dim, end = x.dbias ? 2 * x.dim : x.dim;
        norm_dw_sum_kernel<W><<<(end - first + 63) / 64, 1024, 0, st>>>(x, b.norm, parts, first, end);
    }
}

}  // namespace

hipError_t launch_norm(const ge_norm_args& x, int dtype, hipStream_t st) {
    if (x.rows == 0) return hipSuccess;
    const bool xf = dtype == GE_DTYPE_F32, wf = x.weight_dtype == GE_DTYPE_F32;
    if (xf && wf) norm_forward<float, float>(x, st);
    if (xf && !wf) norm_forward<float, uint16_t>(x, st);
    if (!xf && wf) norm_forward<uint16_t, float>(x, st);
    if (!xf && !wf) norm_forward<uint16_t, uint16_t>(x, st);
    return hipGetLastError();
}

hipError_t launch_norm_backward(const ge_norm_args& x, int dtype, const Buffers& b, hipStream_t st) {
    const bool xf = dtype == GE_DTYPE_F32, wf = x.weight_dtype == GE_DTYPE_F32;
    if (xf && wf) norm_backward<float, float>(x, b, st);
    if (xf && !wf) norm_backward<float, uint16_t>(x, b, st);
    if (!xf && wf) norm_backward<uint16_t, float>(x, b, st);
    if (!xf && !wf) norm_backward<uint16_t, uint16_t>(x, b, st);
    return hipGetLastError();
}

}  // namespace head
}  // namespace ge

// Products of float32 operands on the bf16 matrix cores (gfx950), for the
// vocabulary loss; tiles, epilogues and operand layouts as in head_gemm.h.
//
// x = hi + mid + lo, three bf16 numbers of 8 bits of mantissa each, holds all 24
// bits of a float32; of the nine products of two such sums the six above 2^-24 are
// taken, the small ones first. That is 6 matrix instructions for one, 400 TFLOP/s
// of the bf16 rate against 157 of the float32 matrix instructions.
//
// A tile's float32 elements go through registers, where they are split once, into
// three planes in LDS; a fragment of each plane then serves two to three products.
// (Planes written to memory by a launch before cost 3 bytes more an element than the
// operand has, and each fragment was read twice.) Two workgroups share a compute unit: one splits and
// waits while the other multiplies, so one stage of LDS is enough.
//
// 1,000 rows, width 1,000, vocabulary 50,257: 187 TFLOP/s of float32 products, 1.15
// PFLOP/s of the matrix cores; 300 rows, width 768: 140 with the rows that pad its
// tiles. Keeping the hidden states and the logits' gradient as planes in memory,
// which takes half of the splitting out, was no faster (1,000 rows: 3 % slower).
#pragma once

#include "head_gemm.h"

namespace ge {
namespace head {

constexpr int kStepK32 = 32;

// hi + mid + lo = x to 24 bits, of two numbers, the first in the low halves. A
// non-finite x keeps its value in hi; mid and lo are NaN, as is what it is part of.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        p[i] = to_bf16(x, y);
        x -= __builtin_bit_cast(float, p[i] << 16);
        y -= __builtin_bit_cast(float, p[i] & 0xffff0000u);
    }
}

// A tile along k has rows of 64 bytes; slot s (16 bytes) of row r is kept in slot
// s ^ slot32(r). Four rows fill the banks; see slot_along for the lanes that are
// answered together: 0, 2, 3, 1 by the bits that tell the rows of one place among
// the four apart.
template <bool kEpiRows>
__device__ __forceinline__ int slot32(int r) {
    const int g = (kEpiRows ? r >> 3 : r >> 2) & 3;
    return (g >> 1) | (((g ^ (g >> 1)) & 1) << 1);
}

// One operand's tile: `kRows` rows along k, or as many columns across k.
template <int kRows, bool kAlong, bool kEpiRows>
struct Tile32 {
    static_assert(kAlong || kRows == 128, "slots across k");
    static constexpr int kPerThread = kRows * kStepK32 / (256 * 4);  // 16-byte loads
    static constexpr int kPlane = kRows * kStepK32;                  // bf16 elements
    uint32_t voff[kPerThread];
    uint32_t at[kPerThread];  // bytes into a plane
    int kpos;                 // along k: first k of the lane's 4
    const char* base;
    int64_t left;
    int64_t step;
    u32x4 raw[kPerThread];

    __device__ __forceinline__ void init(const Operand& o, int row0, int first) {
        step = kAlong ? kStepK32 * 4 : kStepK32 * o.ld * 4;
        const int64_t skip = (kAlong ? static_cast<int64_t>(row0) * o.ld : row0) * 4 + step * first;
        base = static_cast<const char*>(o.p) + skip;
        left = o.end * 4 - skip;
        kpos = (threadIdx.x & 7) * 4;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            if (kAlong) {
                const int r = i * 32 + (threadIdx.x >> 3), c = threadIdx.x & 7;
                voff[i] = static_cast<uint32_t>(r * o.ld * 4) + c * 16;
                at[i] = r * 64 + ((c >> 1) ^ slot32<kEpiRows>(r)) * 16 + (c & 1) * 8;
            } else {
                const int u = i * 256 + threadIdx.x;
                const int r = u / (kRows / 4), c = u % (kRows / 4);
                voff[i] = static_cast<uint32_t>(r * o.ld * 4) + c * 16;
                at[i] = r * (kRows * 2) + ((c >> 1) ^ slot_across<kRows>(r)) * 16 + (c & 1) * 8;
            }
        }
    }
    // The loads of the step at `base`, of which `k_left` are before the sum's end.
    __device__ __forceinline__ void load(int k_left) {
        const int64_t n = left < 0 ? 0 : left > 0x7ffffff0 ? 0x7ffffff0 : left;
        __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, static_cast<int>(n), 0x00027000);
        // bounds are checked element by element
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) raw[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, static_cast<int>(voff[i]), 0, 0));
        base += step;
        left -= step;
        if (kAlong && k_left < kStepK32) {
#pragma unroll
            for (int i = 0; i < kPerThread; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) raw[i][e] = kpos + e < k_left ? raw[i][e] : 0u;
        }
    }
    __device__ __forceinline__ void split(uint16_t* planes) const {
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            uint32_t x[3], y[3];
            const f32x4 v = __builtin_bit_cast(f32x4, raw[i]);
            split3(v[0], v[1], x);
            split3(v[2], v[3], y);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<uint2*>(reinterpret_cast<char*>(planes + p * kPlane) + at[i]) = make_uint2(x[p], y[p]);
        }
    }
};

template <bool kEpiRows>
struct Frag32 {
    uint32_t at;
    __device__ __forceinline__ void init(int row0, int lane) {
        const int row = row0 + (kEpiRows ? epi_row(0, lane & 15) : lane & 15);
        at = row * 64 + ((lane >> 4) ^ slot32<kEpiRows>(row)) * 16;
    }
    __device__ __forceinline__ bf16x8 read(const uint16_t* lds, int f, int) const {
        const int rows = kEpiRows ? epi_row(f, 0) : f * 16;
        return *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(lds) + at + rows * 64);
    }
};

template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, bool kBAlong, typename Epi>
__global__ __launch_bounds__(256, 2) void gemm32_kernel(GemmArgs g, Epi epi) {
    static_assert(kWavesM * kWavesN == 4);
    constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
    constexpr int kMt = kWm / 16, kNt = kWn / 16;
    using TileA = Tile32<kBm, kAAlong, true>;
    using TileB = Tile32<kBn, kBAlong, false>;
    __shared__ __align__(1024) uint16_t lds[3 * (TileA::kPlane + TileB::kPlane)];
    uint16_t* const lds_b = lds + 3 * TileA::kPlane;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const TilePlace place = tile_place(g, blockIdx.x, gridDim.x);
    const int m0 = place.m * kBm, n0 = place.n * kBn;
    const int wm = wave % kWavesM, wn = wave / kWavesM;
    const int steps = (g.k + kStepK32 - 1) / kStepK32;
    const int first = place.split * g.steps_per_split;
    const int last = min(steps, first + g.steps_per_split);

    TileA ta;
    TileB tb;
    ta.init(g.a, m0, first);
    tb.init(g.b, n0, first);
    typename std::conditional<kAAlong, Frag32<true>, FragAcross<kBm, kMt>>::type fra;
    typename std::conditional<kBAlong, Frag32<false>, FragAcross<kBn, kNt>>::type frb;
    fra.init(wm * kWm, lane);
    frb.init(wn * kWn, lane);

    f32x4 acc[kMt][kNt];
#pragma unroll
    for (int i = 0; i < kMt; ++i)
#pragma unroll
        for (int j = 0; j < kNt; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    int k_left = g.k - first * kStepK32;
    if (first < last) {
        ta.load(k_left);
        tb.load(k_left);
    }
    for (int t = first; t < last; ++t) {
        ta.split(lds);
        tb.split(lds_b);
        __syncthreads();
        k_left -= kStepK32;
        if (t + 1 < last) {
            ta.load(k_left);
            tb.load(k_left);
        }
        bf16x8 fa[3][kMt], fb[3][kNt];
#pragma unroll
        for (int p = 2; p >= 0; --p) {
#pragma unroll
            for (int i = 0; i < kMt; ++i) fa[p][i] = fra.read(lds + p * TileA::kPlane, i, 0);
#pragma unroll
            for (int j = 0; j < kNt; ++j) fb[p][j] = frb.read(lds_b + p * TileB::kPlane, j, 0);
        }
        constexpr int kPairs[6][2] = {{1, 1}, {2, 0}, {0, 2}, {1, 0}, {0, 1}, {0, 0}};
#pragma unroll
        for (int s = 0; s < 6; ++s)
#pragma unroll
            for (int i = 0; i < kMt; ++i)
#pragma unroll
                for (int j = 0; j < kNt; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[kPairs[s][0]][i], fb[kPairs[s][1]][j], acc[i][j], 0, 0, 0);
        __syncthreads();
    }
    auto state = epi.template prepare<kWm, kNt>(m0 + wm * kWm, n0 + wn * kWn, lane);
    epi.template finish<kBm, kBn, kWavesM, kWavesN, kAAlong>(acc, state, m0, n0, place, wm, wn, lane, reinterpret_cast<float2*>(lds));
}

}  // namespace head
}  // namespace ge

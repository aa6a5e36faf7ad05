// Matrix products of the vocabulary loss on the matrix cores (gfx950): one
// tiled kernel whose operands may run along the product's axis or across it,
// with the epilogue a functor on the accumulators.
//
//   C[m, n] = sum over k of A(m, k) * B(n, k), operands in bf16, sums in f32.
//
// An operand "along k" is stored [rows][k] (a row of the weights, of the
// hidden states or of the logits' gradient); one "across k" is stored
// [k][columns] and is transposed on its way from LDS to the registers
// (ds_read_b64_tr_b16: 16 lanes give the addresses of 4 k-rows x 4 groups of 4
// columns and lane i gets column i's 4 values), so no transposed copy of the
// weights, the hidden states or the gradient is ever written.
//
// float32 operands arrive as three bf16 planes (x = hi + mid + lo, 24 bits of
// mantissa in all) and the product is the sum of the six plane pairs above
// 2^-24: the same loop with six times the steps ("segments"), about 400
// TFLOP/s at most against 157 of the f32 matrix instructions.
//
// Tiles go from memory to LDS without passing registers (buffer loads to LDS,
// 16 bytes a lane). The hardware's bounds check gives zeros beyond an operand's
// end, so ragged rows and a ragged last step need no code of their own; along
// k the columns beyond k are masked in the last step only.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ge {
namespace head {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kStepK = 64;        // k per step of the loop: 128-byte rows along k
constexpr int kMaxSegments = 6;

// One operand: planes of bf16 elements, `ld` elements from row to row, `end`
// elements readable from the start of a plane, `plane` elements between planes.
struct Operand {
    const uint16_t* p;
    int64_t ld;
    int64_t end;
    int64_t plane;
};

struct GemmArgs {
    Operand a, b;
    int k;               // length of the sum
    int segments;        // 1 (bf16) or 6 (float32 in three planes)
    int tiles_m, tiles_n;
    int splits;          // parts of the sum, each with an output of its own
    int steps_per_split; // steps of kStepK in a part
    int group_m;         // tiles along m that run together
};

// Plane pairs of the segments, the smallest products first.
__device__ __forceinline__ int seg_a(int s, int segments) { return segments == 1 ? 0 : (0x210100 >> (4 * (5 - s))) & 3; }
__device__ __forceinline__ int seg_b(int s, int segments) { return segments == 1 ? 0 : (0x012010 >> (4 * (5 - s))) & 3; }

// The resource words of a raw buffer of `bytes` bytes at `p`.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t bytes) {
    const int n = bytes < 0 ? 0 : bytes > 0x7ffffff0 ? 0x7ffffff0 : static_cast<int>(bytes);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, n, 0x00027000);
}

// 16-byte slot in which slot s of row r of a tile along k is kept: any 8
// consecutive lanes of a fragment read (rows i, or rows 4 a + j of `epi_row`)
// find 8 different slots, so a 128-byte row stride costs no bank conflict.
__device__ __forceinline__ int slot_along(int r) {
    return (r & 3) | ((((r >> 2) ^ (r >> 3) ^ (r >> 4) ^ (r >> 5)) & 1) << 2);
}
// The same for a tile across k, in units of 16 bytes: 4 consecutive k-rows (and
// those 8 further on) of one column group lie 32 bytes apart.
template <int kCols>
__device__ __forceinline__ int slot_across(int r) {
    return ((r & 3) | (kCols > 64 ? ((r >> 3) & 1) << 2 : 0)) << 1;
}

// Loads of one operand's tile: `kRows` rows along k, or as many columns across k.
template <int kRows, bool kAlong, int kWaves>
struct TileLoader {
    static constexpr int kInstr = kRows * kStepK * 2 / 1024;         // wave instructions of 1 KiB
    static constexpr int kPerWave = (kInstr + kWaves - 1) / kWaves;
    int voff[kPerWave];
    int kpos[kPerWave];    // along k: first k of the lane's 8 within a step
    const char* base;
    int64_t left;          // readable bytes from `base`
    int64_t step;          // bytes from one k step to the next
    int64_t plane;

    __device__ __forceinline__ void init(const Operand& o, int row0, int wave, int lane) {
        plane = o.plane * 2;
        if (kAlong) {
            base = reinterpret_cast<const char*>(o.p) + static_cast<int64_t>(row0) * o.ld * 2;
            left = (o.end - static_cast<int64_t>(row0) * o.ld) * 2;
            step = kStepK * 2;
        } else {
            base = reinterpret_cast<const char*>(o.p) + static_cast<int64_t>(row0) * 2;
            left = (o.end - row0) * 2;
            step = kStepK * o.ld * 2;
        }
#pragma unroll
        for (int i = 0; i < kPerWave; ++i) {
            const int at = wave + i * kWaves;
            if (kAlong) {
                const int r = at * 8 + (lane >> 3);
                const int s = (lane & 7) ^ slot_along(r);
                voff[i] = static_cast<int>(r * o.ld * 2) + s * 16;
                kpos[i] = s * 8;
            } else {
                constexpr int kUnits = kRows / 8;
                const int u = at * 64 + lane;
                const int r = u / kUnits;
                voff[i] = static_cast<int>(r * o.ld * 2) + ((u % kUnits) ^ slot_across<kRows>(r)) * 16;
                kpos[i] = 0;
            }
        }
    }
    // Loads the tile of k step `t`, plane `seg`, into `lds`; `k_left`: k beyond the step's first.
    __device__ __forceinline__ void load(uint16_t* lds, int t, int seg, int k_left, int wave) const {
        const int64_t off = step * t + plane * seg;
        __amdgpu_buffer_rsrc_t rs = buffer(base + off, left - step * t);
#pragma unroll
        for (int i = 0; i < kPerWave; ++i) {
            const int at = wave + i * kWaves;
            if (kInstr % kWaves == 0 || at < kInstr) {
                int v = voff[i];
                if (kAlong) v = kpos[i] < k_left ? v : static_cast<int>(0x80000000u);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void*)(lds + at * 512), 16, v, 0, 0, 0);
            }
        }
    }
};

// A fragment of 16 rows (or columns) x 32 k for the 16x16x32 product: lane l
// holds row l % 16, k = 8 * (l / 16) .. + 7.
__device__ __forceinline__ bf16x8 frag_along(const uint16_t* lds, int row, int kk, int lane) {
    const int s = (kk * 4 + (lane >> 4)) ^ slot_along(row);
    return *reinterpret_cast<const bf16x8*>(lds + row * kStepK + s * 8);
}
template <int kCols>
__device__ __forceinline__ bf16x8 frag_across(const uint16_t* lds, int col0, int kk, int lane) {
    const int i = lane & 15;
    const int r = kk * 32 + 8 * (lane >> 4) + (i >> 2);
    const int u = (col0 >> 3) + ((i & 3) >> 1);
    const uint16_t* p0 = lds + r * kCols + ((u ^ slot_across<kCols>(r)) * 8) + (i & 1) * 4;
    const uint16_t* p1 = lds + (r + 4) * kCols + ((u ^ slot_across<kCols>(r + 4)) * 8) + (i & 1) * 4;
    typedef __attribute__((address_space(3))) s16x4* lds4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p0);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p1);
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Tile of a workgroup: blocks go to the 8 XCDs in turn, so block b takes place
// (b % 8) * (blocks / 8) + b / 8 of an order in which groups of `group_m`
// tiles along m meet every tile along n before the next group: an XCD's L2
// then holds the group's slices while they are used.
struct TilePlace {
    int m, n, split;
};
__device__ __forceinline__ TilePlace tile_place(const GemmArgs& g, int block, int blocks) {
    int at = block;
    const int even = blocks & ~7;
    if (block < even) at = (block & 7) * (even >> 3) + (block >> 3);
    TilePlace p;
    const int tiles = g.tiles_m * g.tiles_n;
    p.split = at / tiles;
    at -= p.split * tiles;
    const int full = g.group_m * g.tiles_n;
    const int group = at / full;
    at -= group * full;
    const int m0 = group * g.group_m;
    const int gm = min(g.group_m, g.tiles_m - m0);
    p.m = m0 + at % gm;
    p.n = at / gm;
    return p;
}

// Which row of the tile the wave's accumulator row (tile mt of 16, row i) is:
// lane group i / 4 holds kWm / 4 neighbouring rows over all its tiles, so that
// an epilogue's lane has a contiguous run of m.
template <int kWm>
__device__ __forceinline__ int epi_row(int mt, int i) {
    return (i >> 2) * (kWm / 4) + mt * 4 + (i & 3);
}

// One workgroup's tile of kBm x kBn, kWavesM x kWavesN waves. Epi: see the callers;
// it gets acc[mt][nt], whose element j is row epi_row(mt, 4 * (lane / 16) + j)
// (A along k) or mt * 16 + 4 * (lane / 16) + j (across k) of the wave's rows and
// column nt * 16 + lane % 16 of its columns.
template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, bool kBAlong, typename Epi>
__global__ __launch_bounds__(64 * kWavesM * kWavesN) void gemm_kernel(GemmArgs g, Epi epi) {
    constexpr int kWaves = kWavesM * kWavesN;
    constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
    constexpr int kMt = kWm / 16, kNt = kWn / 16;
    __shared__ __align__(1024) uint16_t a0[kBm * kStepK];
    __shared__ __align__(1024) uint16_t b0[kBn * kStepK];
    __shared__ __align__(1024) uint16_t a1[kBm * kStepK];
    __shared__ __align__(1024) uint16_t b1[kBn * kStepK];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const TilePlace place = tile_place(g, blockIdx.x, gridDim.x);
    const int m0 = place.m * kBm, n0 = place.n * kBn;
    const int wm = wave % kWavesM, wn = wave / kWavesM;

    TileLoader<kBm, kAAlong, kWaves> la;
    TileLoader<kBn, kBAlong, kWaves> lb;
    la.init(g.a, m0, wave, lane);
    lb.init(g.b, n0, wave, lane);

    const int steps = (g.k + kStepK - 1) / kStepK;
    const int first = place.split * g.steps_per_split;
    const int last = min(steps, first + g.steps_per_split);
    const int total = max(0, last - first) * g.segments;

    f32x4 acc[kMt][kNt];
#pragma unroll
    for (int i = 0; i < kMt; ++i)
#pragma unroll
        for (int j = 0; j < kNt; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto load = [&](int t, uint16_t* a, uint16_t* b) {
        const int k = first + t / g.segments, s = t % g.segments;
        const int left = g.k - k * kStepK;
        la.load(a, k, seg_a(s, g.segments), left, wave);
        lb.load(b, k, seg_b(s, g.segments), left, wave);
    };
    auto compute = [&](const uint16_t* a, const uint16_t* b) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x8 fa[kMt], fb[kNt];
#pragma unroll
            for (int i = 0; i < kMt; ++i)
                fa[i] = kAAlong ? frag_along(a, wm * kWm + epi_row<kWm>(i, lane & 15), kk, lane)
                                : frag_across<kBm>(a, wm * kWm + i * 16, kk, lane);
#pragma unroll
            for (int j = 0; j < kNt; ++j)
                fb[j] = kBAlong ? frag_along(b, wn * kWn + j * 16 + (lane & 15), kk, lane)
                                : frag_across<kBn>(b, wn * kWn + j * 16, kk, lane);
#pragma unroll
            for (int i = 0; i < kMt; ++i)
#pragma unroll
                for (int j = 0; j < kNt; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
    };

    if (total > 0) load(0, a0, b0);
    for (int t = 0; t < total; t += 2) {
        __syncthreads();
        if (t + 1 < total) load(t + 1, a1, b1);
        compute(a0, b0);
        if (t + 1 < total) {
            __syncthreads();
            if (t + 2 < total) load(t + 2, a0, b0);
            compute(a1, b1);
        }
    }
    __syncthreads();
    epi.template finish<kBm, kBn, kWavesM, kWavesN, kAAlong>(acc, m0, n0, place, wm, wn, lane, wave, reinterpret_cast<char*>(a0));
}

}  // namespace head
}  // namespace ge

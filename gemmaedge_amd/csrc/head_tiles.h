// What the callers of the matrix products share: rows copied into padded ones,
// and a product's launch by the type of its operands.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "head_internal.h"

#include "head_gemm.h"
#include "head_gemm32.h"

namespace ge {
namespace head {

// Rows into rows that are `kpad` long (a multiple of 8), zeros behind `dim`: 8
// elements a thread, read at any address, written aligned.
template <typename T>
__device__ __forceinline__ void pack_unit(const T* in, int64_t ld, int64_t r, int d, int dim, int kpad, T* out) {
    struct Vec {
        T v[8];
    } x;
    if (d + 8 <= dim) {
        __builtin_memcpy(&x, in + r * ld + d, sizeof(x));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] = d + e < dim ? in[r * ld + d + e] : T(0);
    }
    __builtin_memcpy(__builtin_assume_aligned(out + r * kpad + d, 16), &x, sizeof(x));
}
template <typename T>
static __global__ __launch_bounds__(256) void pack_kernel(const T* in, int64_t ld, unsigned rows, int dim, int kpad, T* out) {
    const int d = (blockIdx.x * blockDim.x + threadIdx.x) * 8;
    const int64_t r = blockIdx.y * blockDim.y + threadIdx.y;
    if (d >= kpad || r >= rows) return;
    pack_unit(in, ld, r, d, dim, kpad, out);
}

// Launches over rows on a grid's y, of at most 65,535: one is left for another use.
template <typename F>
void for_rows(int64_t rows, F launch) {
    constexpr int64_t kMost = 65534;
    for (int64_t r = 0; r < rows; r += kMost) launch(r, static_cast<unsigned>(std::min(rows - r, kMost)));
}

// launch(first row, rows, grid, workgroup) for rows of `kpad`, 8 elements a thread.
template <typename F>
void for_units(int64_t rows, int64_t kpad, F launch) {
    const unsigned units = static_cast<unsigned>(kpad / 8);
    unsigned tx = 8;
    while (tx < units && tx < 256) tx *= 2;
    const unsigned ty = 256 / tx;
    for_rows(rows, [&](int64_t r, unsigned n) { launch(r, n, dim3((units + tx - 1) / tx, (n + ty - 1) / ty), dim3(tx, ty)); });
}

// `rows` rows of `dim` copied into rows of `kpad` at `to`.
template <typename T>
Operand packed_rows(const T* p, int64_t ld, int64_t rows, int dim, int64_t kpad, void* to, hipStream_t st) {
    T* const out = static_cast<T*>(to);
    for_units(rows, kpad, [&](int64_t r, unsigned n, dim3 grid, dim3 block) {
        pack_kernel<T><<<grid, block, 0, st>>>(p + r * ld, ld, n, dim, static_cast<int>(kpad), out + r * kpad);
    });
    return Operand{to, kpad, rows * kpad};
}

// One product of m x n outputs over k in `splits` parts, by tiles of kBm x kBn.
template <typename T, int kBm, int kBn, int kWm, int kWn, bool kA, bool kB, typename Epi>
void run_tiles(const Operand& a, const Operand& b, int64_t k, int m, int n, int splits, int group, const Epi& e, hipStream_t st) {
    constexpr int kStep = sizeof(T) == 4 ? kStepK32 : kStepK;
    GemmArgs g{};
    g.a = a;
    g.b = b;
    g.k = static_cast<int>(k);
    g.tiles_m = (m + kBm - 1) / kBm;
    g.tiles_n = (n + kBn - 1) / kBn;
    g.steps_per_split = ((g.k + kStep - 1) / kStep + splits - 1) / splits;
    g.splits = splits;
    g.group_m = group;
    const int64_t tiles = static_cast<int64_t>(g.tiles_m) * g.tiles_n * g.splits;
    if constexpr (sizeof(T) == 4)
        gemm32_kernel<kBm, kBn, kWm, kWn, kA, kB, Epi><<<static_cast<unsigned>(tiles), 256, 0, st>>>(g, e);
    else
        gemm_kernel<kBm, kBn, kWm, kWn, kA, kB, Epi><<<static_cast<unsigned>(tiles), 256, 0, st>>>(g, e);
}

}  // namespace head
}  // namespace ge

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
// Tiles go from memory to LDS without passing registers (buffer loads to LDS,
// 16 bytes a lane). The hardware's bounds check gives zeros beyond an operand's
// end, so ragged rows and a ragged last step need no code of their own; along k
// the columns beyond k are masked from the last step on.
//
// A workgroup is four waves, one a SIMD, with up to 128 x 128 of the output each:
// the accumulators are half of the registers, and a wave reads 16 fragments for 64
// products (8 waves of 128 x 64 read 24 for them and were 10 % slower). With one
// wave a SIMD nothing covers a stall, so everything but the products is spread
// between them in the order it is written. A ring of four stages of 32 k, with
// loads four steps ahead, came out slower than two stages of 64: twice the
// barriers, and half a cache line at a time of an operand along k.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

namespace ge {
namespace head {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kStepK = 64;        // k per step of the loop: 128-byte rows along k

// One operand: elements of its type, `ld` from row to row, `end` readable from the start.
struct Operand {
    const void* p;
    int64_t ld;
    int64_t end;
};

struct GemmArgs {
    Operand a, b;
    int k;               // length of the sum
    int tiles_m, tiles_n;
    int splits;          // parts of the sum, each with an output of its own
    int steps_per_split; // steps of the kernel's k in a part
    int group_m;         // tiles along m that run together
};

// Which of the wave's rows row i of its tile mt of 16 is, for an operand of the M
// side along k: lanes that hold rows 4 a .. 4 a + 3 of the accumulators get 8
// neighbouring rows in every pair of tiles, and the four of them 32.
__device__ __forceinline__ constexpr int epi_row(int mt, int i) {
    return (mt >> 1) * 32 + (i >> 2) * 8 + (mt & 1) * 4 + (i & 3);
}

// A tile along k keeps slot s (16 bytes) of row r in slot s ^ slot_along(r). LDS
// answers a 16-byte read for 16 lanes at a time, of each half wave the lanes 0-3,
// 12-15, 20-23, 24-27 and then the others; two rows fill its 64 banks. The 8 even
// and the 8 odd rows of such 16 lanes, told apart by bits 1 to 3 of the row (dealt
// out by epi_row: 1, 3 and 4), fall into 8 different slots: no conflicts are counted.
template <bool kEpiRows>
__device__ __forceinline__ int slot_along(int r) {
    return kEpiRows ? ((r >> 1) & 1) | (((r >> 3) & 3) << 1) : (r >> 1) & 7;
}
// The same for a tile across k, in units of 16 bytes: 4 consecutive k-rows (and
// those 8 further on) of one column group lie 32 bytes apart.
template <int kCols>
__device__ __forceinline__ int slot_across(int r) {
    return ((r & 3) | (kCols > 64 ? ((r >> 3) & 1) << 2 : 0)) << 1;
}

// Loads of one operand's tile: `kRows` rows along k (kEpiRows: the operand of the
// M side), or as many columns across k.
template <int kRows, bool kAlong, bool kEpiRows, int kWaves>
struct TileLoader {
    static_assert(kWaves == 4, "a wave's instructions are 32 rows apart and share their slots");
    static constexpr int kInstr = kRows * kStepK * 2 / 1024;         // wave instructions of 1 KiB
    static constexpr int kPerWave = (kInstr + kWaves - 1) / kWaves;
    uint32_t voff[kPerWave];
    int kpos;              // along k: first k of the lane's 8 within a step
    const char* base;      // of the step to load
    uint32_t left_lo;      // readable bytes from `base`
    int32_t left_hi;
    int64_t step;          // bytes from one k step to the next

    __device__ __forceinline__ void init(const Operand& o, int row0, int first, int wave, int lane) {
        step = kAlong ? kStepK * 2 : kStepK * o.ld * 2;
        const int64_t skip = (kAlong ? static_cast<int64_t>(row0) * o.ld : row0) * 2 + step * first;
        base = reinterpret_cast<const char*>(o.p) + skip;
        const int64_t left = o.end * 2 > skip ? o.end * 2 - skip : 0;
        left_lo = static_cast<uint32_t>(left);
        left_hi = static_cast<int32_t>(left >> 32);
        kpos = 0;
#pragma unroll
        for (int i = 0; i < kPerWave; ++i) {
            const int at = wave + i * kWaves;
            if (kAlong) {
                const int r = at * 8 + (lane >> 3);
                const int s = (lane & 7) ^ slot_along<kEpiRows>(r);
                voff[i] = static_cast<uint32_t>(r * o.ld * 2) + s * 16;
                if (i == 0) kpos = s * 8;
            } else {
                constexpr int kUnits = kRows / 8;
                const int u = at * 64 + lane;
                const int r = u / kUnits;
                voff[i] = static_cast<uint32_t>(r * o.ld * 2) + ((u % kUnits) ^ slot_across<kRows>(r)) * 16;
            }
        }
    }
    // The step's resource, nothing of it if `none`.
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(bool none) const {
        const uint32_t n = left_hi > 0 ? 0x7ffffff0u : min(left_lo, 0x7ffffff0u);
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, static_cast<int>(none ? 0u : n), 0x00027000);
    }
    __device__ __forceinline__ void advance() {
        base += step;
        const int64_t left = (static_cast<int64_t>(left_hi) << 32 | left_lo) - step;
        left_lo = static_cast<uint32_t>(left);
        left_hi = static_cast<int32_t>(left >> 32);
    }
    // From here on the k beyond `k_left` of a step read as zeros.
    __device__ __forceinline__ void mask(int k_left) {
        if (!kAlong) return;
#pragma unroll
        for (int i = 0; i < kPerWave; ++i) voff[i] = kpos < k_left ? voff[i] : 0x80000000u;
    }
    // Instruction i of the tile's loads into `lds`.
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint16_t* lds, int i, int wave) const {
        const int at = wave + i * kWaves;
        if (kInstr % kWaves == 0 || at < kInstr)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(lds + at * 512), 16,
                                                     static_cast<int>(voff[i]), 0, 0, 0);
    }
};

// Fragments of 16 rows (or columns) x 32 k for the 16x16x32 product: lane l
// holds row l % 16, k = 8 * (l / 16) .. + 7. The addresses of a wave's fragments
// differ from a few registers by constants only, which the reads carry.
//
// Along k: the slot of a fragment's row depends on the lane alone.
template <bool kEpiRows>
struct FragAlong {
    uint32_t at[2];  // by kk
    __device__ __forceinline__ void init(int row0, int lane) {
        const int row = row0 + (kEpiRows ? epi_row(0, lane & 15) : lane & 15);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) at[kk] = row * (kStepK * 2) + ((kk * 4 + (lane >> 4)) ^ slot_along<kEpiRows>(row)) * 16;
    }
    __device__ __forceinline__ bf16x8 read(const uint16_t* lds, int f, int kk) const {
        const int rows = kEpiRows ? epi_row(f, 0) : f * 16;
        return *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(lds) + at[kk] + rows * (kStepK * 2));
    }
};
template <int kCols, int kFrags>
struct FragAcross {
    uint32_t at[kFrags];
    __device__ __forceinline__ void init(int col0, int lane) {
        const int i = lane & 15;
        const int r = 8 * (lane >> 4) + (i >> 2);
#pragma unroll
        for (int f = 0; f < kFrags; ++f) {
            const int u = ((col0 + f * 16) >> 3) + ((i & 3) >> 1);
            at[f] = r * (kCols * 2) + (u ^ slot_across<kCols>(r)) * 16 + (i & 1) * 8;
        }
    }
    // The rows 4 and 32 further on keep their slots.
    __device__ __forceinline__ bf16x8 read(const uint16_t* lds, int f, int kk) const {
        typedef __attribute__((address_space(3))) s16x4* lds4;
        const char* p = reinterpret_cast<const char*>(lds) + at[f] + kk * 32 * kCols * 2;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * kCols * 2));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

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

// f(0) .. f(N - 1) with constants.
template <typename F, int... kI>
__device__ __forceinline__ void static_for(std::integer_sequence<int, kI...>, F f) {
    (f(std::integral_constant<int, kI>{}), ...);
}
template <int kN, typename F>
__device__ __forceinline__ void static_for(F f) {
    static_for(std::make_integer_sequence<int, kN>{}, f);
}

// One product. Large tiles fill the accumulation registers, and a product is
// written as an instruction on them: left to itself the compiler moves them about
// between steps. Between two products on the same registers lie at least 31 others.
template <bool kInPlace>
__device__ __forceinline__ void product(f32x4& c, bf16x8 a, bf16x8 b) {
    if constexpr (kInPlace)
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// One workgroup's tile of kBm x kBn, kWavesM x kWavesN waves. Epi: see the callers;
// it gets acc[mt][nt], whose element j is row epi_row(mt, 4 * (lane / 16) + j)
// (A along k) or mt * 16 + 4 * (lane / 16) + j (across k) of the wave's rows and
// column nt * 16 + lane % 16 of its columns. `prepare` loads what it needs of them.
template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, bool kBAlong, typename Epi>
__global__ __launch_bounds__(64 * kWavesM * kWavesN) void gemm_kernel(GemmArgs g, Epi epi) {
    constexpr int kWaves = kWavesM * kWavesN;
    constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
    constexpr int kMt = kWm / 16, kNt = kWn / 16;
    // A stage each, A's tile and then B's: the compiler tells the stages apart.
    constexpr int kStage = (kBm + kBn) * kStepK;
    __shared__ __align__(1024) uint16_t s0[kStage];
    __shared__ __align__(1024) uint16_t s1[kStage];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % kWavesM, wn = wave / kWavesM;
    using LoaderA = TileLoader<kBm, kAAlong, true, kWaves>;
    using LoaderB = TileLoader<kBn, kBAlong, false, kWaves>;
    LoaderA la;
    LoaderB lb;
    f32x4 acc[kMt][kNt];
    typename std::conditional<kAAlong, FragAlong<true>, FragAcross<kBm, kMt>>::type fra;
    typename std::conditional<kBAlong, FragAlong<false>, FragAcross<kBn, kNt>>::type frb;
    fra.init(wm * kWm, lane);
    frb.init(wn * kWn, lane);

    bf16x8 fa[2][kMt], fb[2][kNt];
    constexpr int kLoadsA = LoaderA::kPerWave, kLoadsB = LoaderB::kPerWave;
    constexpr int kProducts = kMt * kNt;
    constexpr bool kInPlace = kProducts >= 32;
    // Loads of steps past the end bring zeros, whose products change nothing.
    int load_left, k_left;
    __amdgpu_buffer_rsrc_t ra, rb;
    auto mask = [&]() __attribute__((always_inline)) {
        if (k_left < kStepK) {
            la.mask(k_left);
            lb.mask(k_left);
        }
    };
    auto tile_a = [&]() __attribute__((always_inline)) { ra = la.tile(load_left <= 0); };
    auto tile_b = [&]() __attribute__((always_inline)) { rb = lb.tile(load_left <= 0); };
    auto advance = [&]() __attribute__((always_inline)) {
        --load_left;
        la.advance();
        lb.advance();
        k_left -= kStepK;
    };
    auto load_all = [&](uint16_t* to) __attribute__((always_inline)) {
        mask();
        tile_a();
        tile_b();
#pragma unroll
        for (int i = 0; i < kLoadsA; ++i) la.load(ra, to, i, wave);
#pragma unroll
        for (int i = 0; i < kLoadsB; ++i) lb.load(rb, to + kBm * kStepK, i, wave);
        advance();
    };
    auto fetch = [&](int i, int kk, const uint16_t* from) __attribute__((always_inline)) {
        if (i < kNt)
            fb[kk][i] = frb.read(from + kBm * kStepK, i, kk);
        else if (i < kNt + kMt)
            fa[kk][i - kNt] = fra.read(from, i - kNt, kk);
    };
    // Every wave's loads have arrived and every wave's reads are done. The wait for
    // the loads stands here in words: a barrier does not make the compiler wait for
    // loads to LDS that the wave does not read.
    auto arrive = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // A step in two halves of 32 k. The fragments of a half are read while the half
    // before is multiplied, so the step's stage is free at its middle: in the second
    // half the loads of the step after next go there, and have a step to arrive.
    auto half = [&](auto which, uint16_t* stage, const uint16_t* from) __attribute__((always_inline)) {
        constexpr int kk = decltype(which)::value;
        constexpr int kItems = kMt + kNt;
        // products between two reads; in the first half they are done well before the barrier
        constexpr int kMost = kProducts * (kk == 0 ? 3 : 4) / 4;
        constexpr int kEvery = kMost / kItems > 0 ? kMost / kItems : 1;
        constexpr int kReads = (kItems * kEvery + kProducts - 1) / kProducts;
        constexpr int kLoads = kLoadsA + kLoadsB;
        static_for<kProducts>([&](auto at) __attribute__((always_inline)) {
            constexpr int n = decltype(at)::value;
            product<kInPlace>(acc[n / kNt][n % kNt], fa[kk][n / kNt], fb[kk][n % kNt]);
            if constexpr (n % kEvery == 0)
                static_for<kReads>([&](auto i) __attribute__((always_inline)) { fetch(n / kEvery * kReads + i, 1 - kk, from); });
            if constexpr (kk == 0) {
                if constexpr (n == kProducts / 4) mask();
                if constexpr (n == kProducts / 2) tile_a();
                if constexpr (n == kProducts * 3 / 4) tile_b();
            } else {
                constexpr int l0 = n * kLoads / kProducts, l1 = (n + 1) * kLoads / kProducts;
                static_for<l1 - l0>([&](auto i) __attribute__((always_inline)) {
                    constexpr int l = l0 + decltype(i)::value;
                    if constexpr (l < kLoadsA)
                        la.load(ra, stage, l, wave);
                    else
                        lb.load(rb, stage + kBm * kStepK, l - kLoadsA, wave);
                });
            }
        });
        if (kk == 1) advance();
    };
    constexpr std::integral_constant<int, 0> lower{};
    constexpr std::integral_constant<int, 1> upper{};
    auto step = [&](uint16_t* stage, const uint16_t* next) __attribute__((always_inline)) {
        half(lower, stage, stage);
        arrive();
        half(upper, stage, next);
    };
    const TilePlace place = tile_place(g, blockIdx.x, gridDim.x);
    const int m0 = place.m * kBm, n0 = place.n * kBn;
    const int first = place.split * g.steps_per_split;
    const int total = max(0, min((g.k + kStepK - 1) / kStepK, first + g.steps_per_split) - first);
    load_left = total;
    k_left = g.k - first * kStepK;
    la.init(g.a, m0, first, wave, lane);
    lb.init(g.b, n0, first, wave, lane);
    load_all(s0);
    load_all(s1);
#pragma unroll
    for (int i = 0; i < kMt; ++i)
#pragma unroll
        for (int j = 0; j < kNt; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // The first stage has arrived; a wave has at least this many loads of the second.
    constexpr int kSecond = LoaderA::kInstr / kWaves + LoaderB::kInstr / kWaves;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kSecond) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < kMt + kNt; ++i) fetch(i, 0, s0);
    // Steps in pairs: an odd one's partner multiplies zeros. One way out of the loop
    // keeps the accumulators where they are.
    for (int t = 0; t < total; t += 2) {
        step(s0, s1);
        step(s1, s0);
        // The compiler does not know when the products written as instructions are
        // done (16 cycles); what reads the accumulators comes behind the loop.
        if (kInPlace) asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
    }
    // Every wave is done with the stages, and nothing is on its way there any more.
    arrive();
    auto state = epi.template prepare<kWm, kNt>(m0 + wm * kWm, n0 + wn * kWn, lane);
    epi.template finish<kBm, kBn, kWavesM, kWavesN, kAAlong>(acc, state, m0, n0, place, wm, wn, lane, reinterpret_cast<float2*>(s0));
}

}  // namespace head
}  // namespace ge

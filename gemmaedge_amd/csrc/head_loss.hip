// Cross entropy over the vocabulary and its gradients without the logits
// (include/gemmaedge_head.h), on the matrix products of head_gemm.h and head_gemm32.h.
//
// Forward: a tile of vocabulary x rows of logits stays in the accumulators; its
// epilogue leaves, for each row, the tile's largest logit and the sum of
// exp(l - largest), and the target's logit where the tile has it. A second
// launch joins a row's tiles into lse and loss.
//
// Backward, for a piece of the vocabulary at a time: the logits again, whose
// epilogue makes dz = g (exp(l - lse) - [target]) (1 - (l / c)^2) and stores it
// for the piece; dhidden += dz . weights (the piece's sum in parts, each added
// to its own float32 array, joined at the end in a fixed order); dweight rows
// of the piece = dz^T . hidden. bf16 operands: dz is rounded once to bf16.
//
// The vocabulary is the tile's M side: a lane of the accumulators then holds 4
// logits of one row per 16 x 16 product, and, with the rows of a wave's tile
// dealt out by epi_row, 8 neighbours in every two products: sums over the
// vocabulary are mostly sums over a lane's own registers, and dz is stored in
// 16-byte pieces. The epilogues have one wave a SIMD and nothing to hide behind:
// no branch an element, the target's element apart, and with a softcap two
// exponentials and a reciprocal an element, which are most of their 8 us a tile.
//
// 4,096 rows, width 2,816, vocabulary 262,144 in bf16: forward 4.7 ms (1,300
// TFLOP/s), backward 14.3 ms: logits again 4.8 (1,250), dhidden 4.9 (1,240),
// dweight 4.5 (1,350); a plain product of this size by the library reaches 1,480.
// Bound by the matrix cores (53 to 66 % of their cycles at the 2.0 to 2.2 GHz that
// the card holds under them) and the loads that feed them. One row: the weights'
// bytes, 5.9 TB/s.
#include <hip/hip_runtime.h>

#include <limits>

#include "head_internal.h"

#include "head_gemm.h"
#include "head_gemm32.h"

namespace ge {
namespace head {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// How logits are capped. kSmall: bf16 operands and caps up to 64; kWide: larger caps, and float32 operands.
enum Cap { kNone, kSmall, kWide };

// softcap * tanh(z / softcap). bf16 operands, caps up to 64: tanh = 1 - 2 r with
// r = 1 / (exp(2 x) + 1) of the hardware's exp2 and reciprocal, 4e-7 of the cap off at
// most, far below what the operands' 8 bits leave of z. Above 64 that error would
// reach the logits, which may be small against the cap: below x = 1 / 4 a series, whose
// first term is z itself, so that it is 1e-6 of the logit off at most (1,021 rows, width
// 1,152, vocabulary 32,003: forward 84 us against 76, backward 284 against 272). float32
// operands: tanhf, and z itself where x^2 / 3 < u (x has lost bits there if 1 / cap is
// subnormal).
struct Softcap {
    float cap, inv, two;  // cap <= 0: none; two = 2 log2(e) / cap
    __device__ __forceinline__ float r(float z) const { return __builtin_amdgcn_rcpf(exp2_fast(z * two) + 1.0f); }
    __device__ __forceinline__ float small_logit(float z) const { return fmaf(r(z), -2.0f * cap, cap); }
    // `z` and its r
    __device__ __forceinline__ float wide_logit(float z, float r) const {
        const float x = z * inv, q = x * x;
        const float s = fmaf(fmaf(fmaf(62.0f / 2835.0f, q, -17.0f / 315.0f), q, 2.0f / 15.0f), q, -1.0f / 3.0f);
        return q < 0.0625f ? fmaf(z, s * q, z) : fmaf(r, -2.0f * cap, cap);
    }
    __device__ __forceinline__ float exact_logit(float z, float tanh) const { return fabsf(z * inv) < 0x1p-12f ? z : cap * tanh; }
    __device__ __forceinline__ bool small() const { return cap > 0.f && cap <= 64.f; }
    // exp(-2 cap) is a normal number: sums of exp(l - cap) need no largest logit.
    __device__ __forceinline__ bool bounded() const { return cap > 0.f && cap <= 40.f; }
};

// Where a row's target lies among a lane's logits of one column of tiles: element
// 4 i + q is acc[i][.][q], row epi_row(i, 4 * (lane / 16) + q) of the wave's `kWm`. -1: not here.
template <int kWm>
__device__ __forceinline__ int target_place(int target, int first_row, int lane) {
    const int off = target - first_row;
    return off >= 0 && off < kWm && ((off >> 3) & 3) == (lane >> 4) ? (off >> 5) * 8 + (off & 7) : -1;
}

// The targets of a lane's columns, counted from the product's first row; -1: no loss or not in its vocabulary.
template <int kNt>
__device__ __forceinline__ void load_targets(const int32_t* targets, int n_first, int rows, int v0, int vocab, int (&t)[kNt]) {
#pragma unroll
    for (int j = 0; j < kNt; ++j) t[j] = targets[min(n_first + j * 16, rows - 1)];
#pragma unroll
    for (int j = 0; j < kNt; ++j) t[j] = n_first + j * 16 < rows && t[j] >= v0 && t[j] - v0 < vocab ? t[j] - v0 : -1;
}

// Column j's accumulators stay where they are until here: the compiler otherwise reads all
// of a large tile's into registers first, which do not hold them.
template <int kMt, int kNt>
__device__ __forceinline__ void hold(f32x4 (&acc)[kMt][kNt], int j) {
    if constexpr (kMt * kNt >= 32) {
#pragma unroll
        for (int i = 0; i < kMt; ++i) asm volatile("" : "+a"(acc[i][j]));
    }
}

template <bool kFast>
struct StatsEpi {
    Softcap sc;
    int vocab;   // end of the vocabulary, counted from the product's first row
    int v0;      // number of the product's first row in the whole vocabulary
    int rows;
    const int32_t* targets;
    float* target_logit;
    float2* stats;   // [rows][ld]
    int ld, tile0;

    template <int kNt>
    struct State {
        int t[kNt];
    };
    template <int kWm, int kNt>
    __device__ __forceinline__ State<kNt> prepare(int, int col0, int lane) const {
        State<kNt> s;
        load_targets(targets, col0 + (lane & 15), rows, v0, vocab, s.t);
        return s;
    }
    template <Cap kCap>
    __device__ __forceinline__ float logit(float z) const {
        if (kCap == kNone) return z;
        if (!kFast) return sc.exact_logit(z, tanhf(z * sc.inv));
        return kCap == kSmall ? sc.small_logit(z) : sc.wide_logit(z, sc.r(z));
    }
    // The largest logit, the sum and the target's logit of the wave's columns.
    template <int kWm, Cap kCap, int kMt, int kNt>
    __device__ __forceinline__ void columns(f32x4 (&acc)[kMt][kNt], const int (&t)[kNt], int row0, int n_first, int lane,
                                            float2* part) const {
        const bool tail = row0 + kWm > vocab;
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            hold(acc, j);
            float l[4 * kMt];
#pragma unroll
            for (int e = 0; e < 4 * kMt; ++e) l[e] = logit<kCap>(acc[e >> 2][j][e & 3]);
            if (tail) {
#pragma unroll
                for (int e = 0; e < 4 * kMt; ++e)
                    l[e] = row0 + epi_row(e >> 2, 4 * (lane >> 4) + (e & 3)) >= vocab ? -__builtin_inff() : l[e];
            }
            const int at = target_place<kWm>(t[j], row0, lane);
            if (t[j] >= 0 && at >= 0) {
                float x = 0.f;
#pragma unroll
                for (int e = 0; e < 4 * kMt; ++e)
                    if (at == e) x = l[e];
                target_logit[n_first + j * 16] = x;
            }
            float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
            for (int e = 0; e < 4 * kMt; ++e) top = fmaxf(top, l[e]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // A wave whose rows all lie past the vocabulary has nothing to add.
            const float ref = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
            for (int e = 0; e < 4 * kMt; ++e) sum += exp2_fast((l[e] - ref) * kLog2e);  // the difference is exact where it counts
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (lane < 16) part[j * 16 + lane] = make_float2(top, sum);
        }
    }
    // The same for caps up to 40 within the vocabulary: the cap stands for the largest logit.
    template <int kWm, int kMt, int kNt>
    __device__ __forceinline__ void bounded_columns(f32x4 (&acc)[kMt][kNt], const int (&t)[kNt], int row0, int n_first, int lane,
                                                    float2* part) const {
        const float k = -2.0f * kLog2e * sc.cap;
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            hold(acc, j);
            const int at = target_place<kWm>(t[j], row0, lane);
            if (t[j] >= 0 && at >= 0) {
                float x = 0.f;
#pragma unroll
                for (int e = 0; e < 4 * kMt; ++e)
                    if (at == e) x = acc[e >> 2][j][e & 3];
                target_logit[n_first + j * 16] = sc.small_logit(x);
            }
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 4 * kMt; ++e) sum += exp2_fast(sc.r(acc[e >> 2][j][e & 3]) * k);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (lane < 16) part[j * 16 + lane] = make_float2(sc.cap, sum);
        }
    }
    template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, int kMt, int kNt>
    __device__ __forceinline__ void finish(f32x4 (&acc)[kMt][kNt], const State<kNt>& s, int m0, int n0, TilePlace place, int wm, int wn,
                                           int lane, float2* part) const {
        constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
        const int row0 = m0 + wm * kWm;
        const int n_first = n0 + wn * kWn + (lane & 15);
        float2* const to = part + wm * kBn + wn * kWn;
        if (!(sc.cap > 0.f))
            columns<kWm, kNone>(acc, s.t, row0, n_first, lane, to);
        else if (!kFast || !sc.small())
            columns<kWm, kWide>(acc, s.t, row0, n_first, lane, to);
        else if (!sc.bounded() || row0 + kWm > vocab)
            columns<kWm, kSmall>(acc, s.t, row0, n_first, lane, to);
        else
            bounded_columns<kWm>(acc, s.t, row0, n_first, lane, to);
        __syncthreads();
        for (int c = threadIdx.x; c < kBn; c += 64 * kWavesM * kWavesN) {
            const int n = n0 + c;
            if (n >= rows) continue;
            float top = part[c].x, sum = part[c].y;
#pragma unroll
            for (int i = 1; i < kWavesM; ++i) {
                const float2 p = part[i * kBn + c];
                const float m = fmaxf(top, p.x);
                const float ref = m == -__builtin_inff() ? 0.f : m;
                sum = sum * exp2_fast((top - ref) * kLog2e) + p.y * exp2_fast((p.x - ref) * kLog2e);
                top = m;
            }
            stats[static_cast<int64_t>(n) * ld + tile0 + place.m] = make_float2(top, sum);
        }
    }
};

// lse and loss of a row from its tiles' statistics: a workgroup per row.
__global__ __launch_bounds__(256) void join_kernel(const float2* stats, int ld, int tiles, int vocab, const int32_t* targets,
                                                   const float* target_logit, float* loss, float* lse) {
    __shared__ float2 red[4];
    const int64_t r = blockIdx.x;
    const float2* s = stats + r * ld;
    float top = -__builtin_inff(), sum = 0.f;
    auto add = [&](float2 p) {
        const float m = fmaxf(top, p.x);
        const float ref = m == -__builtin_inff() ? 0.f : m;
        sum = sum * exp2_fast((top - ref) * kLog2e) + p.y * exp2_fast((p.x - ref) * kLog2e);
        top = m;
    };
    for (int i = threadIdx.x; i < tiles; i += 256) add(s[i]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) add(make_float2(__shfl_xor(top, o), __shfl_xor(sum, o)));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(top, sum);
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < 4; ++i) add(red[i]);
    const float z = top + logf(sum);
    lse[r] = z;
    if (loss) {
        const int t = targets[r];
        loss[r] = t >= 0 && t < vocab ? z - target_logit[r] : 0.f;
    }
}

// The mantissa of the largest finite |grad| of the rows that carry a loss, 1 if there
// is none. The logits' gradient is held in units of it: where all rows weigh the
// same, as in a mean, the weight's own rounding to 8 bits would scale whole gradients.
template <int kThreads>
__device__ __forceinline__ void grad_unit(const float* grad, const int32_t* targets, int rows, int vocab, float* unit, int thread) {
    __shared__ float red[kThreads / 64];
    float m = 0.f;
#pragma unroll 4
    for (int r = thread; r < rows; r += kThreads) {
        const float g = fabsf(grad[r]);
        const int t = targets[r];
        if (t >= 0 && t < vocab && g < __builtin_inff()) m = fmaxf(m, g);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((thread & 63) == 0) red[thread >> 6] = m;
    __syncthreads();
    if (thread != 0) return;
    for (int i = 1; i < kThreads / 64; ++i) m = fmaxf(m, red[i]);
    const uint32_t bits = __builtin_bit_cast(uint32_t, m);
    *unit = m >= 0x1p-126f ? __builtin_bit_cast(float, (bits & 0x007fffffu) | 0x3f800000u) : 1.f;
}
__global__ __launch_bounds__(1024) void grad_unit_kernel(const float* grad, const int32_t* targets, int rows, int vocab, float* unit) {
    grad_unit<1024>(grad, targets, rows, vocab, unit, threadIdx.x);
}

template <typename T>
struct GradEpi {
    static constexpr bool kFast = sizeof(T) == 2;
    Softcap sc;
    int v0, rows, vocab_all;
    int piece;  // words of the vocabulary from v0 on in this product
    const int32_t* targets;
    const float* lse;
    const float* grad;
    const float* unit;
    T* out;  // [rows_pad][ld]
    int64_t ld;

    // (exp(l - lse) - one) (1 - (l / c)^2) g; fast: `lse` is log2(e) times (-lse, or with kSmall,
    // whose l is cap - 2 cap r, cap - lse), `g` with a cap four times g, since the slope is 4 (r - r^2).
    template <Cap kCap>
    __device__ __forceinline__ float dz(float z, float lse, float g, float one) const {
        if (kFast) {
            if (kCap == kNone) return (exp2_fast(fmaf(z, kLog2e, lse)) - one) * g;
            const float r = sc.r(z);
            const float e = kCap == kSmall ? fmaf(r, -2.0f * kLog2e * sc.cap, lse) : fmaf(sc.wide_logit(z, r), kLog2e, lse);
            return (exp2_fast(e) - one) * fmaf(-r, r, r) * g;
        }
        const float y = kCap == kNone ? 0.f : tanhf(z * sc.inv);
        const float l = kCap == kNone ? z : sc.exact_logit(z, y);
        return (exp2_fast((l - lse) * kLog2e) - one) * fmaf(-y, y, 1.0f) * g;
    }

    template <int kNt>
    struct State {
        int t[kNt];
        float lse[kNt], grad[kNt], unit;
    };
    template <int kWm, int kNt>
    __device__ __forceinline__ State<kNt> prepare(int, int col0, int lane) const {
        State<kNt> s;
        load_targets(targets, col0 + (lane & 15), rows, 0, vocab_all, s.t);
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            const int n = min(col0 + (lane & 15) + j * 16, rows - 1);
            s.lse[j] = lse[n];
            s.grad[j] = grad[n];
        }
        s.unit = *unit;
        return s;
    }
    template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, int kMt, int kNt>
    __device__ __forceinline__ void finish(f32x4 (&acc)[kMt][kNt], const State<kNt>& s, int m0, int n0, TilePlace place, int wm, int wn,
                                           int lane, float2* part) const {
        constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
        const int row0 = m0 + wm * kWm;
        const int n_first = n0 + wn * kWn + (lane & 15);
        float ls[kNt], gr[kNt];
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            ls[j] = s.lse[j];
            gr[j] = s.grad[j] / s.unit;
            if (kFast) {
                ls[j] = sc.small() ? (sc.cap - ls[j]) * kLog2e : -ls[j] * kLog2e;
                if (sc.cap > 0.f) gr[j] *= 4.0f;
            }
        }
        if (!(sc.cap > 0.f))
            store<kWm, kNone>(acc, row0, n_first, lane, s.t, ls, gr);
        else if (kFast && sc.small())
            store<kWm, kSmall>(acc, row0, n_first, lane, s.t, ls, gr);
        else
            store<kWm, kWide>(acc, row0, n_first, lane, s.t, ls, gr);
    }
    template <int kWm, Cap kCap, int kMt, int kNt>
    __device__ __forceinline__ void store(f32x4 (&acc)[kMt][kNt], int row0, int n_first, int lane, const int (&t)[kNt],
                                          const float (&ls)[kNt], const float (&gr)[kNt]) const {
        // Words past the vocabulary have logits of 0, and exp(-lse) may be infinite: the
        // product over the words, which reads up to 7 of them, gets zeros instead.
        const bool tail = row0 + kWm > piece;
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            float d[kMt * 4];
#pragma unroll
            for (int e = 0; e < kMt * 4; ++e) d[e] = dz<kCap>(acc[e >> 2][j][e & 3], ls[j], gr[j], 0.f);
            const int at = t[j] < v0 ? -1 : target_place<kWm>(t[j] - v0, row0, lane);
            if (at >= 0) {
                float z = 0.f;
#pragma unroll
                for (int e = 0; e < kMt * 4; ++e)
                    if (at == e) z = acc[e >> 2][j][e & 3];
                const float x = dz<kCap>(z, ls[j], gr[j], 1.0f);
#pragma unroll
                for (int e = 0; e < kMt * 4; ++e)
                    if (at == e) d[e] = x;
            }
            if (tail) {
#pragma unroll
                for (int e = 0; e < kMt * 4; ++e) d[e] = row0 + epi_row(e >> 2, 4 * (lane >> 4) + (e & 3)) < piece ? d[e] : 0.f;
            }
            T* o = out + static_cast<int64_t>(n_first + j * 16) * ld + row0 + (lane >> 4) * 8;
#pragma unroll
            for (int i = 0; i < kMt; i += 2) {
                constexpr int kWords = 2 * sizeof(T);
                uint32_t pack[kWords];
#pragma unroll
                for (int q = 0; q < kWords; ++q) {
                    if constexpr (sizeof(T) == 2)
                        pack[q] = to_bf16(d[i * 4 + 2 * q], d[i * 4 + 2 * q + 1]);
                    else
                        pack[q] = __builtin_bit_cast(uint32_t, d[i * 4 + q]);
                    if (t[j] < 0) pack[q] = 0;  // no loss: nothing, not NaN either
                }
#pragma unroll
                for (int q = 0; q < kWords; q += 4)
                    *reinterpret_cast<u32x4*>(o + i * 16 + q * 4 / sizeof(T)) = u32x4{pack[q], pack[q + 1], pack[q + 2], pack[q + 3]};
            }
        }
    }
};

// dhidden of a piece and part of it: float32, added to what earlier pieces left.
struct HiddenEpi {
    float* out;  // [splits][rows][ld]
    int64_t ld, split;
    int dim, rows;
    bool add;

    struct State {};
    template <int kWm, int kNt>
    __device__ __forceinline__ State prepare(int, int, int) const { return {}; }
    template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, int kMt, int kNt>
    __device__ __forceinline__ void finish(f32x4 (&acc)[kMt][kNt], const State& s, int m0, int n0, TilePlace place, int wm, int wn,
                                           int lane, float2* part) const {
        constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            const int n = n0 + wn * kWn + j * 16 + (lane & 15);
            if (n >= rows) continue;
            float* o = out + place.split * split + n * ld;
            const int d0 = m0 + wm * kWm + 4 * (lane >> 4);
            f32x4 sum[kMt];
#pragma unroll
            for (int i = 0; i < kMt; ++i) {  // ld is a multiple of 4 above dim
                sum[i] = acc[i][j];
                if (add && d0 + i * 16 < dim) sum[i] += *reinterpret_cast<const f32x4*>(o + d0 + i * 16);
            }
#pragma unroll
            for (int i = 0; i < kMt; ++i)
                if (d0 + i * 16 < dim) *reinterpret_cast<f32x4*>(o + d0 + i * 16) = sum[i];
        }
    }
};

template <typename T>
struct WeightEpi {
    T* out;  // the piece's first row of dweight
    int64_t ld;
    int dim, vocab;
    bool vec;  // rows take 4-element stores
    const float* unit;

    struct State {
        float unit;
    };
    template <int kWm, int kNt>
    __device__ __forceinline__ State prepare(int, int, int) const { return {*unit}; }
    template <int kBm, int kBn, int kWavesM, int kWavesN, bool kAAlong, int kMt, int kNt>
    __device__ __forceinline__ void finish(f32x4 (&acc)[kMt][kNt], const State& s, int m0, int n0, TilePlace place, int wm, int wn,
                                           int lane, float2* part) const {
        constexpr int kWm = kBm / kWavesM, kWn = kBn / kWavesN;
        const float u = s.unit;
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            const int v = n0 + wn * kWn + j * 16 + (lane & 15);
            if (v >= vocab) continue;
#pragma unroll
            for (int i = 0; i < kMt; ++i) {
                const int d = m0 + wm * kWm + i * 16 + 4 * (lane >> 4);
                T* o = out + v * ld + d;
                T q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = from_f32<T>(acc[i][j][e] * u);
                if (vec && d + 4 <= dim) {
                    if constexpr (sizeof(T) == 4)
                        *reinterpret_cast<f32x4*>(o) = f32x4{q[0], q[1], q[2], q[3]};
                    else
                        *reinterpret_cast<uint2*>(o) = make_uint2(q[0] | static_cast<uint32_t>(q[1]) << 16,
                                                                  q[2] | static_cast<uint32_t>(q[3]) << 16);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (d + e < dim) o[e] = q[e];
                }
            }
        }
    }
};

// The parts of dhidden in order, rounded once; 0 for rows without a loss, also where weights
// that are no numbers met their zeros. A workgroup per 256 channels of a row.
template <typename T>
__global__ __launch_bounds__(256) void hidden_sum_kernel(const float* parts, int64_t ld, int64_t split, int splits, int dim,
                                                         const int32_t* targets, int vocab, const float* unit, T* out, int64_t out_ld) {
    const int d = blockIdx.x * 256 + threadIdx.x;
    if (d >= dim) return;
    const int64_t r = blockIdx.y;
    float s = 0.f;
    for (int i = 0; i < splits; ++i) s += parts[i * split + r * ld + d];
    const int t = targets[r];
    out[r * out_ld + d] = from_f32<T>(t >= 0 && t < vocab ? s * *unit : 0.f);
}

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
__global__ __launch_bounds__(256) void pack_kernel(const T* in, int64_t ld, unsigned rows, int dim, int kpad, T* out) {
    const int d = (blockIdx.x * blockDim.x + threadIdx.x) * 8;
    const int64_t r = blockIdx.y * blockDim.y + threadIdx.y;
    if (d >= kpad || r >= rows) return;
    pack_unit(in, ld, r, d, dim, kpad, out);
}

// The same of hidden states, zeros for rows without a loss. The last row of workgroups of
// a launch that gets `unit` finds the gradient's unit of all `all` rows meanwhile, which
// takes as long as a launch of its own.
template <typename T>
__global__ __launch_bounds__(256) void keep_kernel(const T* in, int64_t ld, unsigned rows, int dim, int kpad, T* out, const int32_t* targets,
                                                   int vocab, const float* grad, int all, float* unit) {
    if (unit && blockIdx.y == gridDim.y - 1) {
        if (blockIdx.x == 0) grad_unit<256>(grad, targets, all, vocab, unit, threadIdx.y * blockDim.x + threadIdx.x);
        return;
    }
    const int d = (blockIdx.x * blockDim.x + threadIdx.x) * 8;
    const int64_t r = blockIdx.y * blockDim.y + threadIdx.y;
    if (d >= kpad || r >= rows) return;
    const int t = targets[r];
    pack_unit(in, ld, r, d, t >= 0 && t < vocab ? dim : 0, kpad, out);
}

__global__ __launch_bounds__(256) void fill_zero_kernel(uint16_t* p, int64_t ld, int dim) {
    const int d = blockIdx.x * 256 + threadIdx.x;
    if (d < dim) p[blockIdx.y * ld + d] = 0;
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

template <typename T>
struct Call {
    const ge_loss_args& x;
    const LossPlan& plan;
    const Buffers& b;
    hipStream_t st;
    static constexpr bool kFast = sizeof(T) == 2;

    Operand operand(const T* p, int64_t ld, int64_t rows, bool packed, void* to) const {
        if (!packed) return Operand{p, ld, (rows - 1) * ld + x.dim};
        T* const out = static_cast<T*>(to);
        const int kpad = static_cast<int>(plan.kpad);
        for_units(rows, plan.kpad, [&](int64_t r, unsigned n, dim3 grid, dim3 block) {
            pack_kernel<T><<<grid, block, 0, st>>>(p + r * ld, ld, n, x.dim, kpad, out + r * plan.kpad);
        });
        return Operand{to, plan.kpad, rows * plan.kpad};
    }
    int64_t hidden_ld() const { return x.rows > 1 ? x.hidden_stride : x.dim; }
    Operand hidden() const { return operand(static_cast<const T*>(x.hidden), hidden_ld(), x.rows, plan.pack_h, b.hpack); }
    // Rows without a loss read as zeros, for the weights' gradient: it multiplies them by
    // zeros, and padding that is no number would be NaN in it all the same. The copy
    // takes 22 us for 4,096 rows of 2,816 channels, of 14.3 ms.
    Operand kept_hidden(float* unit) const {
        const T* const p = static_cast<const T*>(x.hidden);
        T* const out = reinterpret_cast<T*>(b.hpack);
        const int64_t ld = hidden_ld();
        for_units(x.rows, plan.kpad, [&](int64_t r, unsigned n, dim3 grid, dim3 block) {
            if (r == 0) ++grid.y;
            keep_kernel<T><<<grid, block, 0, st>>>(p + r * ld, ld, n, x.dim, static_cast<int>(plan.kpad), out + r * plan.kpad, x.targets + r,
                                                   x.vocab, x.grad, x.rows, r == 0 ? unit : nullptr);
        });
        return Operand{b.hpack, plan.kpad, x.rows * plan.kpad};
    }
    // Rows v0 .. v0 + n of the weights.
    Operand weights(int v0, int n) const {
        const int64_t ld = x.vocab > 1 ? x.weight_stride : x.dim;
        return operand(static_cast<const T*>(x.weight) + v0 * ld, ld, n, plan.pack_w, b.wpack);
    }
    Softcap softcap() const {
        if (!(x.softcap > 0.f)) return Softcap{0.f, 0.f, 0.f};
        // Finite for subnormal caps too: a logit of 0 times infinity would be NaN.
        constexpr float kMost = std::numeric_limits<float>::max();
        return Softcap{x.softcap, std::min(1.0f / x.softcap, kMost), std::min(2.0f * kLog2e / x.softcap, kMost)};
    }
    template <int kBm, int kBn, int kWm, int kWn, bool kA, bool kB, typename Epi>
    void run(const Operand& a, const Operand& bb, int64_t k, int m, int n, int splits, int group, const Epi& e) const {
        constexpr int kStep = sizeof(T) == 4 ? kStepK32 : kStepK;
        GemmArgs g{};
        g.a = a;
        g.b = bb;
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
    template <typename Epi>
    void logits(const Operand& w, const Operand& h, int n, const Epi& e) const {
        // A packed row's padding is zeros on both sides; a direct row ends at dim.
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
        } else if (plan.tile_n == kSmallTileN) {
            run<kSmallTileM, kSmallTileN, 4, 1, true, true>(w, h, k, n, x.rows, 1, 4, e);
        } else if (plan.tile_n == 128) {
            run<256, 128, 2, 2, true, true>(w, h, k, n, x.rows, 1, 6, e);
        } else {
            run<256, 256, 2, 2, true, true>(w, h, k, n, x.rows, 1, 6, e);
        }
    }
    void forward() const {
        const Operand h = hidden();
        const int tiles = (x.vocab + plan.tile_m - 1) / plan.tile_m;
        for (int v0 = 0; v0 < x.vocab; v0 += plan.pack_piece) {
            const int n = std::min(plan.pack_piece, x.vocab - v0);
            StatsEpi<kFast> e{softcap(), n, v0, x.rows, x.targets, b.row, reinterpret_cast<float2*>(b.stats), tiles, v0 / plan.tile_m};
            logits(weights(v0, n), h, n, e);
        }
        join_kernel<<<x.rows, 256, 0, st>>>(reinterpret_cast<const float2*>(b.stats), tiles, tiles, x.vocab, x.targets, b.row, x.loss, x.lse);
    }
    void backward() const {
        T* dw = static_cast<T*>(x.dweight);
        T* dh = static_cast<T*>(x.dhidden);
        const int64_t dw_ld = x.vocab > 1 ? x.dweight_stride : x.dim, dh_ld = x.rows > 1 ? x.dhidden_stride : x.dim;
        float* unit = b.row;
        const Operand h = dw ? kept_hidden(unit) : hidden();
        if (!dw) grad_unit_kernel<<<1, 1024, 0, st>>>(x.grad, x.targets, x.rows, x.vocab, unit);
        const int64_t ld = plan.dz_ld;
        constexpr int kTile = sizeof(T) == 4 ? 128 : 256;
        const int64_t hld = (x.dim + 3) / 4 * 4;
        const int64_t split = x.rows * hld;
        int splits = plan.splits;
        for (int v0 = 0; v0 < x.vocab; v0 += plan.piece) {
            const int n = std::min(plan.piece, x.vocab - v0);
            const Operand w = weights(v0, n);
            GradEpi<T> e{softcap(), v0, x.rows, x.vocab, n, x.targets, x.lse, x.grad, unit, reinterpret_cast<T*>(b.dlogits), ld};
            logits(w, h, n, e);
            // Rows past the batch read as zeros: they are no rows of the hidden states either.
            const Operand dz{b.dlogits, ld, x.rows * ld};
            if (dh) {
                HiddenEpi he{b.dhidden, hld, split, x.dim, x.rows, v0 > 0};
                if (sizeof(T) == 2 && x.rows <= 128)
                    run<kTile, 128, 2, 2, false, true>(w, dz, n, x.dim, x.rows, splits, 6, he);
                else
                    run<kTile, kTile, 2, 2, false, true>(w, dz, n, x.dim, x.rows, splits, 6, he);
            }
            if (dw) {
                WeightEpi<T> we{dw + v0 * dw_ld, dw_ld, x.dim, n, false, unit};
                we.vec = aligned_to(we.out, 4 * sizeof(T)) && (x.vocab <= 1 || dw_ld % 4 == 0);
                run<kTile, kTile, 2, 2, false, false>(h, dz, x.rows, x.dim, n, 1, 4, we);
            }
        }
        if (dh) {
            for_rows(x.rows, [&](int64_t r, unsigned n) {
                hidden_sum_kernel<T><<<dim3((x.dim + 255) / 256, n), 256, 0, st>>>(
                    b.dhidden + r * hld, hld, split, splits, x.dim, x.targets + r, x.vocab, unit, dh + r * dh_ld, dh_ld);
            });
        }
    }
};

}  // namespace

hipError_t launch_loss(const ge_loss_args& x, int dtype, const LossPlan& plan, const Buffers& b, hipStream_t st) {
    if (x.rows == 0) return hipSuccess;
    if (dtype == GE_DTYPE_F32)
        Call<float>{x, plan, b, st}.forward();
    else
        Call<uint16_t>{x, plan, b, st}.forward();
    return hipGetLastError();
}

hipError_t launch_loss_backward(const ge_loss_args& x, int dtype, const LossPlan& plan, const Buffers& b, hipStream_t st) {
    if (x.rows == 0) {  // no rows: the weights' gradient is zero
        if (x.dweight) {
            const int64_t ld = (x.vocab > 1 ? x.dweight_stride : x.dim) * elem_size(dtype) / 2;
            const int dim = x.dim * elem_size(dtype) / 2;
            for_rows(x.vocab, [&](int64_t r, unsigned n) {
                fill_zero_kernel<<<dim3((dim + 255) / 256, n), 256, 0, st>>>(static_cast<uint16_t*>(x.dweight) + r * ld, ld, dim);
            });
        }
        return hipGetLastError();
    }
    if (dtype == GE_DTYPE_F32)
        Call<float>{x, plan, b, st}.backward();
    else
        Call<uint16_t>{x, plan, b, st}.backward();
    return hipGetLastError();
}

}  // namespace head
}  // namespace ge

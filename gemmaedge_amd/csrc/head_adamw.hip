// One AdamW step over a list of tensors (include/gemmaedge_head.h): one launch,
// a workgroup per chunk of 4,096 elements, found through the table that the
// caller keeps on the device. Every element is read and written once, in pieces
// of up to 16 bytes a lane at any address (tensors need no alignment beyond
// their elements'), and a lane's loads are all issued before its first sum.
//
// Bound by memory, at 5.2 to 5.5 TB/s: 56 million elements in bf16 with float32
// masters and states in 297 us, 738 million in bf16 with 8-bit states in 1.42 ms
// (2.13 ms with loads converted where they are issued: each branch on a type
// then waits for its own).
#include <hip/hip_runtime.h>

#include "head_internal.h"

namespace ge {
namespace head {
namespace {

// What a step needs of its parameters, in the precision it is applied in.
struct AdamCoeff {
    float beta1, rest1, beta2, rest2, eps, decay, size, root, grad_scale;
    uint32_t seed_mul, step_mul;
    // The hardware's square root takes a subnormal v for 0. That stays below half an ulp
    // of sqrt(v) root + eps where eps is at least 2^24 times the root of 2^-126.
    __host__ __device__ bool fast() const { return eps >= root * 0x1p-39f; }
};

__host__ __device__ inline double power(double b, uint32_t n) {
    double r = 1.0;
    for (; n; n >>= 1, b *= b)
        if (n & 1) r *= b;
    return r;
}

__host__ __device__ inline AdamCoeff coefficients(const ge_adamw_params& p) {
    AdamCoeff c;
    c.beta1 = static_cast<float>(p.beta1);
    c.rest1 = static_cast<float>(1.0 - p.beta1);
    c.beta2 = static_cast<float>(p.beta2);
    c.rest2 = static_cast<float>(1.0 - p.beta2);
    c.eps = static_cast<float>(p.eps);
    c.decay = static_cast<float>(1.0 - p.lr * p.weight_decay);
    c.size = static_cast<float>(p.lr / (1.0 - power(p.beta1, p.step)));
    c.root = static_cast<float>(1.0 / sqrt(1.0 - power(p.beta2, p.step)));
    c.grad_scale = static_cast<float>(p.grad_scale);
    c.seed_mul = p.seed * 0x9E3779B9u;
    c.step_mul = p.step * 0x9E3779B9u;
    return c;
}

// A 32-bit hash: two rounds of xor-shift and a product with an odd constant
// (the fractions of the square roots of 3 and 2, times 2^32).
__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0xBB67AE85u;
    x = (x ^ (x >> 15)) * 0x6A09E667u;
    return x ^ (x >> 16);
}

// m and v of one element after the step.
__device__ __forceinline__ void moments(const AdamCoeff& c, float grad, float& m, float& v) {
    const float g = grad * c.grad_scale;
    m = m * c.beta1 + g * c.rest1;
    v = v * c.beta2 + g * g * c.rest2;
}
// The parameter after the step. kFast: the hardware's square root and reciprocal,
// 1 ulp each, instead of correctly rounded ones: some 20 instructions an element
// fewer, which is what 8-bit states are bound by; 32-bit states wait for memory.
template <bool kFast>
__device__ __forceinline__ float updated(const AdamCoeff& c, float m, float v, float p) {
    if (kFast) {
        const float d = __builtin_amdgcn_sqrtf(v) * c.root + c.eps;
        return p * c.decay - m * __builtin_amdgcn_rcpf(d) * c.size;
    }
    return p * c.decay - m / (sqrtf(v) * c.root + c.eps) * c.size;
}

// A tensor's elements: its address comes out of the table, so that it lies in
// global memory has to be said. kN neighbours at any address.
template <typename T>
using Global = __attribute__((address_space(1))) T*;
template <typename T, int kN>
using Some = T __attribute__((ext_vector_type(kN), aligned(sizeof(T))));

// `count` (at most kN) elements from element i on, zeros behind them; kFull: all kN are there.
template <bool kFull, int kN, typename T>
__device__ __forceinline__ void load_some(const void* base, int64_t i, int count, T (&x)[kN]) {
    const Global<const T> p = (Global<const T>)base + i;
    if (kFull || count >= kN) {
        const Some<T, kN> q = *(Global<const Some<T, kN>>)p;
#pragma unroll
        for (int j = 0; j < kN; ++j) x[j] = q[j];
    } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) x[j] = j < count ? p[j] : T(0);
    }
}
template <bool kFull, int kN, typename T>
__device__ __forceinline__ void store_some(void* base, int64_t i, int count, const T (&x)[kN]) {
    const Global<T> p = (Global<T>)base + i;
    if (kFull || count >= kN) {
        Some<T, kN> q;
#pragma unroll
        for (int j = 0; j < kN; ++j) q[j] = x[j];
        *(Global<Some<T, kN>>)p = q;
    } else {
#pragma unroll
        for (int j = 0; j < kN; ++j)
            if (j < count) p[j] = x[j];
    }
}
// The parameter, rounded to its type, and its master where there is one.
template <bool kFull, int kN>
__device__ __forceinline__ void store_param(const ge_adamw_tensor& t, int64_t i, int count, const float (&x)[kN]) {
    if (t.master) store_some<kFull>(t.master, i, count, x);
    if (t.param_dtype == GE_DTYPE_F32) {
        store_some<kFull>(t.param, i, count, x);
    } else {
        uint16_t h[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) h[j] = to_bf16(x[j]);
        store_some<kFull>(t.param, i, count, h);
    }
}

// 8-bit codes without sign. kMan mantissa bits, exponent bias kBias; normal
// codes from 2^(1 - kBias); `bits`: 16 random bits.
template <int kMan, int kBias, bool kUp>
__device__ __forceinline__ uint32_t encode(float y, uint32_t bits) {
    constexpr int kDrop = 23 - kMan;
    const float low = __builtin_bit_cast(float, static_cast<uint32_t>(127 + 1 - kBias) << 23);
    const bool up = kUp ? y > 0.f : static_cast<float>(bits) * (low / 65536.0f) < y;
    const uint32_t r = ((__builtin_bit_cast(uint32_t, y) + (bits << (kDrop - 16))) >> kDrop) - (static_cast<uint32_t>(127 - kBias) << kMan);
    return y < low ? (up ? 1u << kMan : 0u) : r;
}

// Largest value of 32 neighbouring lanes, in each of them.
__device__ __forceinline__ uint32_t half_wave_max(uint32_t v) {
    auto with = [&](int w) { v = v > static_cast<uint32_t>(w) ? v : static_cast<uint32_t>(w); };
    with(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xf, 0xf, true));   // lane ^ 1
    with(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xf, 0xf, true));   // lane ^ 2
    with(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xf, 0xf, true));  // mirrored in 8
    with(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xf, 0xf, true));  // mirrored in 16
    with(__shfl_xor(static_cast<int>(v), 16));
    return v;
}

// A block's scale and the factor that brings its values into the code's range.
// `big` by its bits: NaN and infinity are above every finite value.
__device__ __forceinline__ void block_scale(uint32_t big_bits, float top, float& scale, float& inv) {
    const float big = __builtin_bit_cast(float, big_bits);
    const bool dead = big < 0x1p-100f;
    const bool bad = big_bits >= 0x7f800000u;
    scale = dead ? 0.f : big * (1.0f / top);
    inv = dead ? 0.f : (1.0f / big) * top;
    if (bad) scale = __builtin_bit_cast(float, 0x7fc00000u);
}

// A chunk's elements. kFull: the tensor does not end in it; P and G: types of the
// value to update (the master's or the parameter's) and of the gradient. These
// are constants because a conversion inside a branch would wait for its load
// there, one tensor after another.
struct Chunk {
    const ge_adamw_tensor& t;
    int64_t first_block;  // of the tensor, in the whole list
    int32_t chunk;
};

// States of 32 bits: 4 elements a lane, 4 blocks a wave.
template <bool kFull, typename P, typename G>
__device__ __forceinline__ void step32(const AdamCoeff& c, const Chunk& ch) {
    const ge_adamw_tensor& t = ch.t;
    constexpr int kN = 4, kBlocks = kAdamBlocks / 4;
    const int64_t e0 = static_cast<int64_t>(ch.chunk) * kAdamChunk + threadIdx.x * kN;
    P p[kBlocks][kN];
    G g[kBlocks][kN];
    float m[kBlocks][kN], v[kBlocks][kN];
    int count[kBlocks];
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
        const int64_t i = e0 + u * 256 * kN;
        count[u] = t.n - i >= kN ? kN : t.n > i ? static_cast<int>(t.n - i) : 0;
        load_some<kFull>(t.master ? t.master : t.param, i, count[u], p[u]);
        load_some<kFull>(t.grad, i, count[u], g[u]);
        load_some<kFull>(t.m, i, count[u], m[u]);
        load_some<kFull>(t.v, i, count[u], v[u]);
    }
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
        const int64_t i = e0 + u * 256 * kN;
        float q[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            moments(c, to_f32(g[u][j]), m[u][j], v[u][j]);
            q[j] = updated<false>(c, m[u][j], v[u][j], to_f32(p[u][j]));
        }
        store_param<kFull>(t, i, count[u], q);
        store_some<kFull>(t.m, i, count[u], m[u]);
        store_some<kFull>(t.v, i, count[u], v[u]);
    }
}

// States of 8 bits: 8 elements a lane, a block on each half of a wave.
template <bool kFull, typename P, typename G>
__device__ __forceinline__ void step8(const AdamCoeff& c, const Chunk& ch) {
    const ge_adamw_tensor& t = ch.t;
    constexpr int kN = 8, kPasses = kAdamChunk / (256 * kN);
    const int place = (threadIdx.x & 31) * kN;  // of the lane's first element in its block
    P p[kPasses][kN];
    G g[kPasses][kN];
    float ms[kPasses], vs[kPasses];
    uint8_t qm[kPasses][kN], qv[kPasses][kN];
    int count[kPasses];
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const int64_t block = static_cast<int64_t>(ch.chunk) * kAdamBlocks + u * 8 + (threadIdx.x >> 5);
        const int64_t i = block * GE_ADAMW_BLOCK + place;
        count[u] = t.n - i >= kN ? kN : t.n > i ? static_cast<int>(t.n - i) : 0;
        load_some<kFull>(t.master ? t.master : t.param, i, count[u], p[u]);
        load_some<kFull>(t.grad, i, count[u], g[u]);
        load_some<kFull>(t.m, i, count[u], qm[u]);
        load_some<kFull>(t.v, i, count[u], qv[u]);
        const bool live = kFull || block * GE_ADAMW_BLOCK < t.n;
        ms[u] = live ? ((Global<const float>)t.m_scale)[block] : 0.f;
        vs[u] = live ? ((Global<const float>)t.v_scale)[block] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const int64_t block = static_cast<int64_t>(ch.chunk) * kAdamBlocks + u * 8 + (threadIdx.x >> 5);
        const int64_t i = block * GE_ADAMW_BLOCK + place;
        float m[kN], v[kN], q[kN];
        uint32_t mbig = 0, vbig = 0;
#pragma unroll
        for (int j = 0; j < kN; j += 4) {
            uint32_t wm, wv;
            __builtin_memcpy(&wm, qm[u] + j, 4);
            __builtin_memcpy(&wv, qv[u] + j, 4);
            const auto a0 = __builtin_amdgcn_cvt_pk_f32_fp8(wm, false), a1 = __builtin_amdgcn_cvt_pk_f32_fp8(wm, true);
            const auto b0 = __builtin_amdgcn_cvt_pk_f32_bf8(wv, false), b1 = __builtin_amdgcn_cvt_pk_f32_bf8(wv, true);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int e = j + k;
                m[e] = (k < 2 ? a0[k & 1] : a1[k & 1]) * ms[u];
                v[e] = (k < 2 ? b0[k & 1] : b1[k & 1]) * vs[u];
                moments(c, to_f32(g[u][e]), m[e], v[e]);
                // Elements behind the tensor's end are zeros and no largest value.
                mbig = max(mbig, __builtin_bit_cast(uint32_t, m[e]) & 0x7fffffffu);
                vbig = max(vbig, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
            }
        }
        if (c.fast()) {
#pragma unroll
            for (int e = 0; e < kN; ++e) q[e] = updated<true>(c, m[e], v[e], to_f32(p[u][e]));
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) q[e] = updated<false>(c, m[e], v[e], to_f32(p[u][e]));
        }
        store_param<kFull>(t, i, count[u], q);
        mbig = half_wave_max(mbig);
        vbig = half_wave_max(vbig);
        float mscale, minv, vscale, vinv;
        block_scale(mbig, 448.f, mscale, minv);
        block_scale(vbig, 57344.f, vscale, vinv);
        const uint32_t key = mix(mix(static_cast<uint32_t>(ch.first_block + block) + c.seed_mul) + c.step_mul) +
                             static_cast<uint32_t>(place) * 0x9E3779B9u;
        uint32_t cm[kN], cv[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const uint32_t bits = mix(key + static_cast<uint32_t>(j) * 0x9E3779B9u);
            cm[j] = encode<3, 7, false>(fminf(fabsf(m[j]) * minv, 448.f), bits & 0xffffu);
            cv[j] = encode<2, 15, true>(fminf(v[j] * vinv, 57344.f), bits >> 16);
        }
        if (mbig >= 0x7f800000u || vbig >= 0x7f800000u) {  // ones under a scale of NaN
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                if (mbig >= 0x7f800000u) cm[j] = 0x38u;
                if (vbig >= 0x7f800000u) cv[j] = 0x3cu;
            }
        }
        uint8_t om[kN], ov[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            om[j] = static_cast<uint8_t>(cm[j] | (m[j] < 0.f ? 0x80u : 0u));
            ov[j] = static_cast<uint8_t>(cv[j]);
        }
        store_some<kFull>(t.m, i, count[u], om);
        store_some<kFull>(t.v, i, count[u], ov);
        if (place == 0 && count[u] > 0) {
            ((Global<float>)t.m_scale)[block] = mscale;
            ((Global<float>)t.v_scale)[block] = vscale;
        }
    }
}

template <bool k8, bool kFull, typename P, typename G>
__device__ __forceinline__ void step_chunk(const AdamCoeff& c, const Chunk& ch) {
    if constexpr (k8)
        step8<kFull, P, G>(c, ch);
    else
        step32<kFull, P, G>(c, ch);
}

template <bool k8>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamTensor* tensors, const AdamChunk* chunks, AdamCoeff hc,
                                                    const ge_adamw_params* dp) {
    const AdamCoeff c = dp ? coefficients(*dp) : hc;
    const AdamChunk at = chunks[blockIdx.x];
    const AdamTensor& a = tensors[at.tensor];
    const ge_adamw_tensor t = a.t;
    const Chunk ch{t, a.first_block, at.chunk};
    const bool pf = t.master || t.param_dtype == GE_DTYPE_F32, gf = t.grad_dtype == GE_DTYPE_F32;
    if (t.n - static_cast<int64_t>(at.chunk) * kAdamChunk >= kAdamChunk) {
        if (pf && gf)
            step_chunk<k8, true, float, float>(c, ch);
        else if (pf)
            step_chunk<k8, true, float, uint16_t>(c, ch);
        else if (gf)
            step_chunk<k8, true, uint16_t, float>(c, ch);
        else
            step_chunk<k8, true, uint16_t, uint16_t>(c, ch);
    } else {
        if (pf && gf)
            step_chunk<k8, false, float, float>(c, ch);
        else if (pf)
            step_chunk<k8, false, float, uint16_t>(c, ch);
        else if (gf)
            step_chunk<k8, false, uint16_t, float>(c, ch);
        else
            step_chunk<k8, false, uint16_t, uint16_t>(c, ch);
    }
}

}  // namespace

hipError_t launch_adamw(const ge_adamw_args& x, int64_t chunks, hipStream_t st) {
    if (chunks == 0) return hipSuccess;
    const AdamTensor* t = static_cast<const AdamTensor*>(x.table);
    const AdamChunk* c = reinterpret_cast<const AdamChunk*>(t + x.count);
    const AdamCoeff coeff = x.device_params ? AdamCoeff{} : coefficients(x.params);
    auto* kernel = x.state_bits == 8 ? adamw_kernel<true> : adamw_kernel<false>;
    kernel<<<static_cast<unsigned>(chunks), 256, 0, st>>>(t, c, coeff, x.device_params);
    return hipGetLastError();
}

}  // namespace head
}  // namespace ge

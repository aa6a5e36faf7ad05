// One AdamW step over a list of tensors (include/gemmaedge_head.h): one launch,
// a workgroup per chunk of 4,096 elements, found through the table that the
// caller keeps on the device. Every element is read and written once.
//
// 8-bit states: a wave holds one block of 256 elements, 4 a lane, so the
// block's largest value is a reduction over the wave.
#include <hip/hip_runtime.h>

#include "head_internal.h"

namespace ge {
namespace head {
namespace {

// What a step needs of its parameters, in the precision it is applied in.
struct AdamCoeff {
    float beta1, rest1, beta2, rest2, eps, decay, size, root, grad_scale;
    uint32_t seed_mul, step_mul;
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

// m, v and p of one element after the step.
__device__ __forceinline__ void update(const AdamCoeff& c, float grad, float& m, float& v, float& p) {
    const float g = grad * c.grad_scale;
    m = m * c.beta1 + g * c.rest1;
    v = v * c.beta2 + g * g * c.rest2;
    p = p * c.decay - m / (sqrtf(v) * c.root + c.eps) * c.size;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
    return dtype == GE_DTYPE_F32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int dtype, float x) {
    if (dtype == GE_DTYPE_F32)
        static_cast<float*>(p)[i] = x;
    else
        static_cast<uint16_t*>(p)[i] = to_bf16(x);
}

// 8-bit codes without sign. kMan mantissa bits, exponent bias kBias; normal
// codes from 2^(1 - kBias); `bits`: 16 random bits.
template <int kMan, int kBias, bool kUp>
__device__ __forceinline__ uint32_t encode(float y, uint32_t bits) {
    constexpr int kDrop = 23 - kMan;
    const float low = __builtin_bit_cast(float, static_cast<uint32_t>(127 + 1 - kBias) << 23);
    if (y < low) {
        const bool up = kUp ? y > 0.f : static_cast<float>(bits) * (low / 65536.0f) < y;
        return up ? 1u << kMan : 0u;
    }
    const uint32_t r = (__builtin_bit_cast(uint32_t, y) + (bits << (kDrop - 16))) >> kDrop;
    return r - (static_cast<uint32_t>(127 - kBias) << kMan);
}
template <int kMan, int kBias>
__device__ __forceinline__ float decode(uint32_t code) {
    // Subnormal codes are whole numbers of 2^(1 - kBias - kMan).
    const uint32_t q = code & 0x7f;
    if (q < (1u << kMan))
        return static_cast<float>(q) * __builtin_bit_cast(float, static_cast<uint32_t>(127 + 1 - kBias - kMan) << 23);
    return __builtin_bit_cast(float, (q + (static_cast<uint32_t>(127 - kBias) << kMan)) << (23 - kMan));
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t w = static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o));
        v = v > w ? v : w;
    }
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

template <bool k8>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamTensor* tensors, const AdamChunk* chunks, ge_adamw_params hp,
                                                    const ge_adamw_params* dp) {
    const AdamCoeff c = coefficients(dp ? *dp : hp);
    const AdamChunk ch = chunks[blockIdx.x];
    const AdamTensor& at = tensors[ch.tensor];
    const ge_adamw_tensor t = at.t;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = wave; b < kAdamBlocks; b += 4) {
        const int64_t block = static_cast<int64_t>(ch.chunk) * kAdamBlocks + b;
        const int64_t e0 = block * GE_ADAMW_BLOCK;
        if (e0 >= t.n) return;
        float m[4], v[4];
        const float ms = k8 ? t.m_scale[block] : 1.f, vs = k8 ? t.v_scale[block] : 1.f;
        uint32_t mbig = 0, vbig = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = e0 + lane * 4 + j;
            m[j] = v[j] = 0.f;
            if (i >= t.n) continue;
            if (k8) {
                const uint32_t q = static_cast<const uint8_t*>(t.m)[i];
                const float a = decode<3, 7>(q) * ms;
                m[j] = q & 0x80 ? -a : a;
                v[j] = decode<2, 15>(static_cast<const uint8_t*>(t.v)[i]) * vs;
            } else {
                m[j] = static_cast<const float*>(t.m)[i];
                v[j] = static_cast<const float*>(t.v)[i];
            }
            float p = t.master ? t.master[i] : load_any(t.param, i, t.param_dtype);
            update(c, load_any(t.grad, i, t.grad_dtype), m[j], v[j], p);
            if (t.master) t.master[i] = p;
            store_any(t.param, i, t.param_dtype, p);
            if (!k8) {
                static_cast<float*>(t.m)[i] = m[j];
                static_cast<float*>(t.v)[i] = v[j];
            }
            mbig = max(mbig, __builtin_bit_cast(uint32_t, m[j]) & 0x7fffffffu);
            vbig = max(vbig, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
        }
        if (!k8) continue;
        mbig = wave_max(mbig);
        vbig = wave_max(vbig);
        float mscale, minv, vscale, vinv;
        block_scale(mbig, 448.f, mscale, minv);
        block_scale(vbig, 57344.f, vscale, vinv);
        const uint32_t key = mix(mix(static_cast<uint32_t>(at.first_block + block) + c.seed_mul) + c.step_mul);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = e0 + lane * 4 + j;
            if (i >= t.n) continue;
            const uint32_t bits = mix(key + static_cast<uint32_t>(lane * 4 + j) * 0x9E3779B9u);
            uint32_t qm = mbig >= 0x7f800000u ? 0x38u : encode<3, 7, false>(fminf(fabsf(m[j]) * minv, 448.f), bits & 0xffffu);
            if (m[j] < 0.f) qm |= 0x80u;
            const uint32_t qv = vbig >= 0x7f800000u ? 0x3cu : encode<2, 15, true>(fminf(v[j] * vinv, 57344.f), bits >> 16);
            static_cast<uint8_t*>(t.m)[i] = static_cast<uint8_t>(qm);
            static_cast<uint8_t*>(t.v)[i] = static_cast<uint8_t>(qv);
        }
        if (lane == 0) {
            t.m_scale[block] = mscale;
            t.v_scale[block] = vscale;
        }
    }
}

}  // namespace

hipError_t launch_adamw(const ge_adamw_args& x, int64_t chunks, hipStream_t st) {
    if (chunks == 0) return hipSuccess;
    const AdamTensor* t = static_cast<const AdamTensor*>(x.table);
    const AdamChunk* c = reinterpret_cast<const AdamChunk*>(t + x.count);
    if (x.state_bits == 8)
        adamw_kernel<true><<<static_cast<unsigned>(chunks), 256, 0, st>>>(t, c, x.params, x.device_params);
    else
        adamw_kernel<false><<<static_cast<unsigned>(chunks), 256, 0, st>>>(t, c, x.params, x.device_params);
    return hipGetLastError();
}

}  // namespace head
}  // namespace ge

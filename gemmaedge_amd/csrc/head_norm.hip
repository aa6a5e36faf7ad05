// The norm over a row's channels and its gradients (include/gemmaedge_head.h).
//
// Forward: a workgroup per row; sum, then the sum of squared differences from
// the mean (two passes: one pass of sum and sum of squares loses the variance
// of channels whose offset is large against their spread).
//
// Backward: dx needs two sums over the row, of a = dy w and of a xhat. The
// weights' gradients are sums over the rows of one column each; row groups sum
// their rows, and a second launch adds the groups in one fixed order, so the
// result does not depend on the order in which workgroups run.
#include <hip/hip_runtime.h>

#include "head_internal.h"

namespace ge {
namespace head {
namespace {

constexpr int kNormThreads = 256;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// Sum over the workgroup, the same value in every thread. `red` holds kNormThreads / 64 floats.
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kNormThreads / 64; ++i) s += red[i];
    return s;
}

template <typename T, typename W>
__global__ __launch_bounds__(kNormThreads) void norm_kernel(ge_norm_args x) {
    __shared__ float red[kNormThreads / 64];
    const int64_t r = blockIdx.x;
    const T* in = static_cast<const T*>(x.x) + r * x.x_stride;
    T* out = static_cast<T*>(x.y) + r * x.y_stride;
    const W* w = static_cast<const W*>(x.weight);
    const W* b = static_cast<const W*>(x.bias);
    const float inv = 1.0f / static_cast<float>(x.dim);
    float mean = 0.f;
    if (x.center) {
        float s = 0.f;
        for (int i = threadIdx.x; i < x.dim; i += kNormThreads) s += to_f32(in[i]);
        mean = block_sum(s, red) * inv;
    }
    float q = 0.f;
    for (int i = threadIdx.x; i < x.dim; i += kNormThreads) {
        const float d = to_f32(in[i]) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(block_sum(q, red) * inv + x.eps);
    for (int i = threadIdx.x; i < x.dim; i += kNormThreads) {
        const float h = (to_f32(in[i]) - mean) * rstd;
        out[i] = from_f32<T>(fmaf(h, to_f32(w[i]), b ? to_f32(b[i]) : 0.f));
    }
    if (threadIdx.x == 0) {
        x.rstd[r] = rstd;
        if (x.mean) x.mean[r] = mean;
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(kNormThreads) void norm_dx_kernel(ge_norm_args x) {
    __shared__ float red[kNormThreads / 64];
    const int64_t r = blockIdx.x;
    const T* in = static_cast<const T*>(x.x) + r * x.x_stride;
    const T* dy = static_cast<const T*>(x.dy) + r * x.dy_stride;
    T* dx = static_cast<T*>(x.dx) + r * x.dx_stride;
    const W* w = static_cast<const W*>(x.weight);
    const float inv = 1.0f / static_cast<float>(x.dim);
    const float mean = x.center ? x.mean[r] : 0.f, rstd = x.rstd[r];
    float sa = 0.f, sx = 0.f;
    for (int i = threadIdx.x; i < x.dim; i += kNormThreads) {
        const float a = to_f32(dy[i]) * to_f32(w[i]);
        sa += a;
        sx = fmaf(a, (to_f32(in[i]) - mean) * rstd, sx);
    }
    sx = block_sum(sx, red) * inv;
    sa = x.center ? block_sum(sa, red) * inv : 0.f;
    for (int i = threadIdx.x; i < x.dim; i += kNormThreads) {
        const float a = to_f32(dy[i]) * to_f32(w[i]);
        const float h = (to_f32(in[i]) - mean) * rstd;
        dx[i] = from_f32<T>(rstd * (a - sa - h * sx));
    }
}

// Rows part, part + parts, ... summed for each column of a workgroup's 256.
template <typename T>
__global__ __launch_bounds__(kNormThreads) void norm_dw_kernel(ge_norm_args x, float* parts) {
    const int c = blockIdx.x * kNormThreads + threadIdx.x;
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

template <typename W>
__global__ __launch_bounds__(kNormThreads) void norm_dw_sum_kernel(ge_norm_args x, const float* parts, int n) {
    const int c = blockIdx.x * kNormThreads + threadIdx.x;
    if (c >= x.dim) return;
    float sw = 0.f, sb = 0.f;
    for (int i = 0; i < n; ++i) {
        const float* p = parts + static_cast<int64_t>(i) * 2 * x.dim;
        sw += p[c];
        sb += p[x.dim + c];
    }
    if (x.dweight) static_cast<W*>(x.dweight)[c] = from_f32<W>(sw);
    if (x.dbias) static_cast<W*>(x.dbias)[c] = from_f32<W>(sb);
}

}  // namespace

template <typename T, typename W>
static void norm_forward(const ge_norm_args& x, hipStream_t st) {
    norm_kernel<T, W><<<x.rows, kNormThreads, 0, st>>>(x);
}

hipError_t launch_norm(const ge_norm_args& x, int dtype, hipStream_t st) {
    if (x.rows == 0) return hipSuccess;
    const bool xf = dtype == GE_DTYPE_F32, wf = x.weight_dtype == GE_DTYPE_F32;
    if (xf && wf) norm_forward<float, float>(x, st);
    if (xf && !wf) norm_forward<float, uint16_t>(x, st);
    if (!xf && wf) norm_forward<uint16_t, float>(x, st);
    if (!xf && !wf) norm_forward<uint16_t, uint16_t>(x, st);
    return hipGetLastError();
}

template <typename T, typename W>
static void norm_backward(const ge_norm_args& x, const Buffers& b, hipStream_t st) {
    if (x.dweight || x.dbias) {  // before dx, which may be written over dy
        const int cols = (x.dim + kNormThreads - 1) / kNormThreads;
        const int parts = x.rows < kNormParts ? x.rows : kNormParts;
        if (parts > 0) norm_dw_kernel<T><<<dim3(cols, parts), kNormThreads, 0, st>>>(x, b.norm);
        norm_dw_sum_kernel<W><<<cols, kNormThreads, 0, st>>>(x, b.norm, parts);
    }
    if (x.dx && x.rows > 0) norm_dx_kernel<T, W><<<x.rows, kNormThreads, 0, st>>>(x);
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

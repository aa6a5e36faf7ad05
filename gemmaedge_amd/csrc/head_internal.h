// Launches of the head's kernels (include/gemmaedge_head.h); arguments are
// checked by head_validate.h before they get here.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "head_validate.h"

namespace ge {

// Sets the calling thread's last message and returns `code`.
int report(int code, const char* msg);

namespace head {

// Device memory of a handle.
struct Buffers {
    float* stats;
    float* row;
    uint16_t* hpack;
    uint16_t* wpack;
    uint16_t* dlogits;
    float* dhidden;
    float* norm;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return __builtin_bit_cast(float, static_cast<uint32_t>(x) << 16); }
// bf16 to the nearest, ties to even; NaN stays NaN.
__device__ __forceinline__ uint16_t to_bf16(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
}
// Two of them, the first in the low half.
__device__ __forceinline__ uint32_t to_bf16(float x, float y) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
}
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ uint16_t from_f32<uint16_t>(float x) { return to_bf16(x); }

hipError_t launch_norm(const ge_norm_args& x, int dtype, hipStream_t st);
hipError_t launch_norm_backward(const ge_norm_args& x, int dtype, const Buffers& b, hipStream_t st);
hipError_t launch_loss(const ge_loss_args& x, int dtype, const LossPlan& plan, const Buffers& b, hipStream_t st);
hipError_t launch_loss_backward(const ge_loss_args& x, int dtype, const LossPlan& plan, const Buffers& b, hipStream_t st);

// The optimiser's table: `count` tensors, then one entry per chunk of elements.
constexpr int kAdamBlocks = 16;                              // blocks of GE_ADAMW_BLOCK in a chunk
constexpr int kAdamChunk = kAdamBlocks * GE_ADAMW_BLOCK;     // elements of a workgroup
struct AdamTensor {
    ge_adamw_tensor t;
    int64_t first_block;  // number of the tensor's first block in the whole list
};
struct AdamChunk {
    int32_t tensor;
    int32_t chunk;
};
hipError_t launch_adamw(const ge_adamw_args& x, int64_t chunks, hipStream_t st);

}  // namespace head
}  // namespace ge

// nt_layer_common.cuh -- element types and activations of the texel-layer operators (group
// normalisation, 4-bit microscaled matrices).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "nt_capi.h"

namespace nt {

void count_launch();
int sm_count();
cudaError_t set_smem_limit(const void *kernel, size_t bytes);
nt_status set_error(nt_status st, const char *fmt, ...);

#define NT_LAYER_REQUIRE(cond, ...)                                         \
    do {                                                                    \
        if (!(cond)) return nt::set_error(NT_ERR_INVALID_ARG, __VA_ARGS__); \
    } while (0)

inline bool is_aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// Bytes of a layer dtype, 0 for any other.
inline int layer_dtype_size(int32_t dt)
{
    return dt == NT_DTYPE_F32 ? 4 : (dt == NT_DTYPE_F16 || dt == NT_DTYPE_BF16) ? 2 : 0;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 1 / (1 + exp(-z)); exp(-z) = inf gives 0.
__device__ __forceinline__ float sigmoid_f32(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

// A NaN stays a NaN under every activation.
__device__ __forceinline__ float activate(float z, int act)
{
    switch (act) {
    case NT_ACT_RELU: return z < 0.f ? 0.f : z;
    case NT_ACT_SILU: return z * sigmoid_f32(z);
    case NT_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    default: return z;
    }
}

// d activation / dz
__device__ __forceinline__ float activation_slope(float z, int act)
{
    switch (act) {
    case NT_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case NT_ACT_SILU: {
        const float s = sigmoid_f32(z);
        return s * (1.f + z * (1.f - s));
    }
    case NT_ACT_GELU:
        return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * __expf(-0.5f * z * z);
    default: return 1.f;
    }
}

}  // namespace nt

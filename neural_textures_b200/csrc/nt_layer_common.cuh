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

// Launch order.  These kernels are launched so that the next one of them in a stream may be set up while
// this one runs: `after_previous` is where a kernel waits for everything queued before it, and nothing global is
// read or written before that point.
__device__ __forceinline__ void after_previous()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <class... P, class... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, unsigned cluster, const A &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) count_launch();
    return e;
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

// Two 16-bit values and their fp32 pair.
template <class T>
struct Pair;
template <>
struct Pair<__half> { using type = __half2; };
template <>
struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
__device__ __forceinline__ float2 pair_f32(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 pair_f32(__nv_bfloat162 v) { return __bfloat1622float2(v); }
template <class T>
__device__ __forceinline__ typename Pair<T>::type f32_pair(float2 v);
template <>
__device__ __forceinline__ __half2 f32_pair<__half>(float2 v) { return __float22half2_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat162 f32_pair<__nv_bfloat16>(float2 v) { return __float22bfloat162_rn(v); }

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

// 1 / a of both lanes with one reciprocal: 1 / (a.x a.y), times the other lane.  The special-function unit
// is the narrowest one that an activation uses.  |a| stays within 2^+-63.
__device__ __forceinline__ float2 rcp2(float2 a)
{
    const float r = rcp(a.x * a.y);
    return make_float2(a.y * r, a.x * r);
}

// 1 / (1 + exp(-z)) as e / (1 + e), e = exp(z): silu multiplies it by z, however far below 0, where e keeps its digits and
// ends at 0.  Above 43 it is 1, where e is held.
__device__ __forceinline__ float2 sigmoid2(float2 z)
{
    const float2 t = __fmul2_rn(make_float2(fminf(z.x, 43.f), fminf(z.y, 43.f)), f2(1.44269504f));
    const float2 e = make_float2(ex2(t.x), ex2(t.y));
    return __fmul2_rn(e, rcp2(__fadd2_rn(e, f2(1.f))));
}

// The normal distribution's integral Phi(z), and exp(-z^2 / 2).  With x = |z| / sqrt 2, t = 1 / (1 + p x):
// erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2) within 1.5e-7 (Abramowitz and Stegun, 7.1.26).
__device__ __forceinline__ float2 normal_cdf2(float2 z, float2 &bell)
{
    const float2 x = make_float2(fminf(fabsf(z.x), 64.f), fminf(fabsf(z.y), 64.f));
    const float2 t = rcp2(__ffma2_rn(x, f2(0.3275911f * 0.70710678f), f2(1.f)));
    const float2 q = __fmul2_rn(__fmul2_rn(x, x), f2(-0.5f * 1.44269504f));
    bell = make_float2(ex2(q.x), ex2(q.y));
    float2 s = __ffma2_rn(t, f2(0.5f * 1.061405429f), f2(0.5f * -1.453152027f));
    s = __ffma2_rn(s, t, f2(0.5f * 1.421413741f));
    s = __ffma2_rn(s, t, f2(0.5f * -0.284496736f));
    s = __ffma2_rn(s, t, f2(0.5f * 0.254829592f));
    const float2 tail = __fmul2_rn(__fmul2_rn(s, t), bell);  // Phi(-|z|)
    return make_float2(z.x < 0.f ? tail.x : 1.f - tail.x, z.y < 0.f ? tail.y : 1.f - tail.y);
}

// A NaN stays a NaN under every activation.
template <int ACT>
__device__ __forceinline__ float2 activate2(float2 z)
{
    if (ACT == NT_ACT_RELU) return make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y);
    if (ACT == NT_ACT_SILU) return __fmul2_rn(z, sigmoid2(z));
    if (ACT == NT_ACT_GELU) {
        float2 bell;
        return __fmul2_rn(z, normal_cdf2(z, bell));
    }
    return z;
}

__device__ __forceinline__ float2 activate2(float2 z, int act)
{
    switch (act) {
    case NT_ACT_RELU: return activate2<NT_ACT_RELU>(z);
    case NT_ACT_SILU: return activate2<NT_ACT_SILU>(z);
    case NT_ACT_GELU: return activate2<NT_ACT_GELU>(z);
    default: return z;
    }
}

__device__ __forceinline__ float activate1(float z, int act) { return activate2(make_float2(z, 0.f), act).x; }

// e d activation / dz
template <int ACT>
__device__ __forceinline__ float2 times_slope2(float2 e, float2 z)
{
    if (ACT == NT_ACT_RELU) return make_float2(z.x > 0.f ? e.x : e.x * 0.f, z.y > 0.f ? e.y : e.y * 0.f);
    if (ACT == NT_ACT_SILU) {  // s (1 + z (1 - s)) = s + y (1 - s), y = z s
        const float2 s = sigmoid2(z);
        return __fmul2_rn(e, __ffma2_rn(__fmul2_rn(z, s), __ffma2_rn(s, f2(-1.f), f2(1.f)), s));
    }
    if (ACT == NT_ACT_GELU) {
        float2 bell;
        const float2 cdf = normal_cdf2(z, bell);
        return __fmul2_rn(e, __ffma2_rn(__fmul2_rn(z, f2(0.39894228f)), bell, cdf));
    }
    return e;
}

}  // namespace nt

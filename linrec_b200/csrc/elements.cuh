// Element helpers of the channels-last operators: the logistic function, and loads and stores of a lane's
// two adjacent channels in any storage type.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace linrec {

// ---- logistic function ---------------------------------------------------------------------------------
// 1/d for d in [1, 2]: the hardware approximation and one Newton step.
__device__ __forceinline__ float newton_rcp(float d)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return fmaf(r, fmaf(-d, r, 1.0f), r);
}
__device__ __forceinline__ float approx_sqrt(float v)
{
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// s(v) and s(-v), both to full relative accuracy.
__device__ __forceinline__ void logistic_pair(float v, float& p, float& n)
{
    const float e = expf(-fabsf(v));
    const float r = newton_rcp(1.0f + e), s = e * r;
    p = v >= 0.0f ? r : s;
    n = v >= 0.0f ? s : r;
}
__device__ __forceinline__ float logistic(float v)
{
    float p, n;
    logistic_pair(v, p, n);
    return p;
}
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))); }

// ---- loads and stores of a lane's two channels ----------------------------------------------------------
template <typename ST>
__device__ __forceinline__ float to_f32(ST v)
{
    return (float)v;
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v)
{
    return __half2float(v);
}
template <typename ST>
__device__ __forceinline__ ST from_f32(float v)
{
    return (ST)v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v)
{
    return __float2half_rn(v);
}

template <typename ST>
__device__ __forceinline__ void load_two(const void* base, long long offset, int have, float* v)
{
    const ST* q = static_cast<const ST*>(base) + offset;
    v[0] = have > 0 ? to_f32<ST>(q[0]) : 0.0f;
    v[1] = have > 1 ? to_f32<ST>(q[1]) : 0.0f;
}
template <typename ST>
__device__ __forceinline__ void store_two(void* base, long long offset, int have, const float* v)
{
    ST* q = static_cast<ST*>(base) + offset;
    if (have > 0) q[0] = from_f32<ST>(v[0]);
    if (have > 1) q[1] = from_f32<ST>(v[1]);
}

}  // namespace linrec

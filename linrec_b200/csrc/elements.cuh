// Element helpers of the channels-last operators: the logistic function, and loads and stores of a lane's
// two adjacent channels in any storage type.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace linrec {

// ---- logistic function ---------------------------------------------------------------------------------
__device__ __forceinline__ float approx_rcp(float d)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}
__device__ __forceinline__ float approx_sqrt(float v)
{
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// exp(v) as a power of two.  The product v log2(e) is rounded, so the relative error is (4 + 1.3 |v|) 2^-24:
// far below half a step of a 16-bit result, not good enough for 32-bit storage.
__device__ __forceinline__ float fast_exp(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.44269504f));
    return r;
}
template <bool FAST>
__device__ __forceinline__ float exp_of(float v)
{
    return FAST ? fast_exp(v) : expf(v);
}
// s(v) and s(-v) to full relative accuracy: the smaller one as a quotient, the larger as its distance from one
// (a value next to one is then off by half its last place, whatever the reciprocal's error is).
template <bool FAST>
__device__ __forceinline__ void logistic_pair(float v, float& p, float& n)
{
    const float e = exp_of<FAST>(-fabsf(v)), d = 1.0f + e;
    float r = approx_rcp(d);
    if (!FAST) r = fmaf(r, fmaf(-d, r, 1.0f), r);
    const float s = e * r, l = 1.0f - s;
    p = v >= 0.0f ? l : s;
    n = v >= 0.0f ? s : l;
}
// s(v) alone; a value next to one may be off by two of its last places.
template <bool FAST>
__device__ __forceinline__ float logistic(float v)
{
    if (FAST) return approx_rcp(1.0f + fast_exp(-v));
    float p, n;
    logistic_pair<false>(v, p, n);
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

// ---- two channels at a time ---------------------------------------------------------------------------------
// Pairs of floats in one 64-bit register pair: sm_100 multiplies and adds both with one instruction, which is
// what operators with 16-bit operands need (they are bound by instruction issue before they are by memory).
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi)
{
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ F2 f2(float both) { return f2(both, both); }
__device__ __forceinline__ float2 f2_get(F2 a)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c)
{
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b)
{
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b)
{
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ float approx_exp2(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// logistic() and logistic_pair() of both channels.
template <bool FAST>
__device__ __forceinline__ F2 logistic2(F2 v)
{
    if (FAST) {
        const float2 t = f2_get(f2_mul(v, f2(-1.44269504f)));
        const float2 d = f2_get(f2_add(f2(approx_exp2(t.x), approx_exp2(t.y)), f2(1.0f)));
        return f2(approx_rcp(d.x), approx_rcp(d.y));
    }
    const float2 w = f2_get(v);
    return f2(logistic<false>(w.x), logistic<false>(w.y));
}
template <bool FAST>
__device__ __forceinline__ void logistic_pair2(F2 v, F2& p, F2& n)
{
    const float2 w = f2_get(v);
    if (FAST) {
        const F2 e = f2(fast_exp(-fabsf(w.x)), fast_exp(-fabsf(w.y)));
        const float2 d = f2_get(f2_add(e, f2(1.0f)));
        const F2 s2 = f2_mul(e, f2(approx_rcp(d.x), approx_rcp(d.y)));
        const float2 s = f2_get(s2), l = f2_get(f2_fma(s2, f2(-1.0f), f2(1.0f)));
        p = f2(w.x >= 0.0f ? l.x : s.x, w.y >= 0.0f ? l.y : s.y);
        n = f2(w.x >= 0.0f ? s.x : l.x, w.y >= 0.0f ? s.y : l.y);
    } else {
        float p0, n0, p1, n1;
        logistic_pair<false>(w.x, p0, n0);
        logistic_pair<false>(w.y, p1, n1);
        p = f2(p0, p1);
        n = f2(n0, n1);
    }
}

// s(v) and s(-v) = e^-v s(v) of both channels, for operands that are tested for NaN elsewhere (the bound on the
// exponent, which keeps 0 * inf out, lets NaN through as a number).
template <bool FAST>
__device__ __forceinline__ void logistic_both2(F2 v, F2& p, F2& n)
{
    if (FAST) {
        const float2 t = f2_get(f2_mul(v, f2(-1.44269504f)));
        const F2 e = f2(approx_exp2(fminf(t.x, 126.0f)), approx_exp2(fminf(t.y, 126.0f)));
        const float2 d = f2_get(f2_add(e, f2(1.0f)));
        p = f2(approx_rcp(d.x), approx_rcp(d.y));
        n = f2_mul(e, p);
    } else {
        logistic_pair2<false>(v, p, n);
    }
}
__device__ __forceinline__ float approx_rsqrt(float v)
{
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Two adjacent channels as one word of shared or global memory.
template <typename ST>
struct Two;
template <>
struct Two<float> {
    using Word = float2;
    __device__ static __forceinline__ void unpack(Word w, float* v) { v[0] = w.x, v[1] = w.y; }
    __device__ static __forceinline__ Word pack(const float* v) { return make_float2(v[0], v[1]); }
    __device__ static __forceinline__ F2 get(Word w) { return f2(w.x, w.y); }
    __device__ static __forceinline__ Word put(F2 v) { return f2_get(v); }
};
template <>
struct Two<__nv_bfloat16> {
    using Word = uint32_t;
    __device__ static __forceinline__ void unpack(Word w, float* v)
    {
        v[0] = __uint_as_float(w << 16);
        v[1] = __uint_as_float(w & 0xffff0000u);
    }
    __device__ static __forceinline__ Word pack(const float* v)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ static __forceinline__ F2 get(Word w)
    {
        float v[2];
        unpack(w, v);
        return f2(v[0], v[1]);
    }
    __device__ static __forceinline__ Word put(F2 v)
    {
        const float2 f = f2_get(v);
        const float w[2] = {f.x, f.y};
        return pack(w);
    }
};
template <>
struct Two<__half> {
    using Word = uint32_t;
    __device__ static __forceinline__ void unpack(Word w, float* v)
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        v[0] = f.x, v[1] = f.y;
    }
    __device__ static __forceinline__ Word pack(const float* v)
    {
        const __half2 h = __floats2half2_rn(v[0], v[1]);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ static __forceinline__ F2 get(Word w)
    {
        float v[2];
        unpack(w, v);
        return f2(v[0], v[1]);
    }
    __device__ static __forceinline__ Word put(F2 v)
    {
        const float2 f = f2_get(v);
        const float w[2] = {f.x, f.y};
        return pack(w);
    }
};
// `pair`: the two channels exist and lie at an address a whole word can be written to.
template <typename ST>
__device__ __forceinline__ void store_two(void* base, long long offset, int have, const float* v, bool pair)
{
    if (pair) *reinterpret_cast<typename Two<ST>::Word*>(static_cast<ST*>(base) + offset) = Two<ST>::pack(v);
    else store_two<ST>(base, offset, have, v);
}
template <typename ST>
__device__ __forceinline__ void store_two(void* base, long long offset, int have, F2 v, bool pair)
{
    const float2 f = f2_get(v);
    const float w[2] = {f.x, f.y};
    store_two<ST>(base, offset, have, w, pair);
}
__device__ __forceinline__ F2 load_state(const float* base, long long offset, int have)
{
    float v[2];
    load_two<float>(base, offset, have, v);
    return f2(v[0], v[1]);
}

}  // namespace linrec

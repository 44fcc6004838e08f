// Group norm of channels-last tensors with an activation, or with an activated gate, and its backward pass.
//
// x is (samples, positions, channels); a group is the channels [g c, (g+1) c) of all positions of a sample.
//   xhat = (x - mean) * inv,   z = xhat * w + b,   y = act(z)   or, with a gate,   y = z * act(gate)
// Backward, with dz the gradient that reaches z and k = dz w:
//   dx = inv (k - mean(k) - xhat mean(k xhat)),   dgate = dy z act'(gate),   dw = sum dz xhat,   db = sum dz
#pragma once
#include "elements.cuh"
#include "ptx.cuh"

namespace linrec {

constexpr int kActNone = 0, kActSilu = 1, kActSigmoid = 2;

struct NormParams {
    const void *x, *gate, *dy;
    long long sx, sg, sdy;        // elements between rows (a row = one position of one sample)
    const float *w, *b;           // [C] or null (ones, zeros)
    float eps;
    int act;
    long long n, L;               // samples, positions
    int C, G, c;                  // channels, groups, channels per group
    float2* stats;                // [n][G] (mean, inv): written forward, read backward
    void *y, *dx, *dgate;         // rows at stride C
    float2* part;                 // backward: [parts][C] sums of (dz xhat, dz)
    int parts;
    float *dw, *db;
};

// act(v) and its derivative.
template <bool FAST>
__device__ __forceinline__ void activate(int act, float v, float& value, float& slope)
{
    if (act == kActNone) {
        value = v;
        slope = 1.0f;
        return;
    }
    float p, n;
    logistic_pair<FAST>(v, p, n);
    if (act == kActSilu) {
        value = v * p;
        slope = p * fmaf(v, n, 1.0f);
    } else {
        value = p;
        slope = p * n;
    }
}

__device__ __forceinline__ float block_sum(float v, float* shared)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) v += shared[i];
    return v;
}

// One CTA per (sample, group).
template <typename ST>
__global__ void __launch_bounds__(256) norm_fwd_kernel(const NormParams p)
{
    __shared__ float shared[8];
    ptx::grid_dependency_wait();
    const long long unit = blockIdx.x;
    const long long n = unit / p.G;
    const int g = (int)(unit - n * p.G);
    const long long count = p.L * p.c, row0 = n * p.L;
    const ST* x = static_cast<const ST*>(p.x);
    const ST* gate = static_cast<const ST*>(p.gate);
    auto at = [&](long long i, long long& row, int& ch) {
        const long long l = i / p.c;
        row = row0 + l;
        ch = g * p.c + (int)(i - l * p.c);
    };
    long long row;
    int ch;
    float s = 0.0f;
    for (long long i = threadIdx.x; i < count; i += blockDim.x) {
        at(i, row, ch);
        s += to_f32<ST>(x[row * p.sx + ch]);
    }
    const float mean = block_sum(s, shared) / (float)count;
    s = 0.0f;
    for (long long i = threadIdx.x; i < count; i += blockDim.x) {
        at(i, row, ch);
        const float d = to_f32<ST>(x[row * p.sx + ch]) - mean;
        s = fmaf(d, d, s);
    }
    const float inv = 1.0f / sqrtf(block_sum(s, shared) / (float)count + p.eps);
    if (threadIdx.x == 0 && p.stats) p.stats[unit] = make_float2(mean, inv);
    for (long long i = threadIdx.x; i < count; i += blockDim.x) {
        at(i, row, ch);
        const float z = fmaf((to_f32<ST>(x[row * p.sx + ch]) - mean) * inv, p.w ? p.w[ch] : 1.0f, p.b ? p.b[ch] : 0.0f);
        float v, slope;
        activate<sizeof(ST) == 2>(p.act, gate ? to_f32<ST>(gate[row * p.sg + ch]) : z, v, slope);
        static_cast<ST*>(p.y)[row * p.C + ch] = from_f32<ST>(gate ? z * v : v);
    }
}

// What reaches one element: xhat, the gradient dz of z, and the gate's gradient.
template <typename ST>
__device__ __forceinline__ void norm_element(const NormParams& p, float2 st, long long row, int ch, float& xhat, float& dz, float& dgate)
{
    xhat = (to_f32<ST>(static_cast<const ST*>(p.x)[row * p.sx + ch]) - st.x) * st.y;
    const float z = fmaf(xhat, p.w ? p.w[ch] : 1.0f, p.b ? p.b[ch] : 0.0f);
    const float dy = to_f32<ST>(static_cast<const ST*>(p.dy)[row * p.sdy + ch]);
    float v, slope;
    if (p.gate) {
        activate<sizeof(ST) == 2>(p.act, to_f32<ST>(static_cast<const ST*>(p.gate)[row * p.sg + ch]), v, slope);
        dz = dy * v;
        dgate = dy * z * slope;
    } else {
        activate<sizeof(ST) == 2>(p.act, z, v, slope);
        dz = dy * slope;
        dgate = 0.0f;
    }
}

template <typename ST>
__global__ void __launch_bounds__(256) norm_bwd_kernel(const NormParams p)
{
    __shared__ float shared[8];
    ptx::grid_dependency_wait();
    const long long unit = blockIdx.x;
    const long long n = unit / p.G;
    const int g = (int)(unit - n * p.G);
    const long long count = p.L * p.c, row0 = n * p.L;
    const float2 st = p.stats[unit];
    float s1 = 0.0f, s2 = 0.0f, xhat, dz, dgate;
    for (long long i = threadIdx.x; i < count; i += blockDim.x) {
        const long long row = row0 + i / p.c;
        const int ch = g * p.c + (int)(i % p.c);
        norm_element<ST>(p, st, row, ch, xhat, dz, dgate);
        const float k = dz * (p.w ? p.w[ch] : 1.0f);
        s1 += k;
        s2 = fmaf(k, xhat, s2);
    }
    const float m1 = block_sum(s1, shared) / (float)count, m2 = block_sum(s2, shared) / (float)count;
    for (long long i = threadIdx.x; i < count; i += blockDim.x) {
        const long long row = row0 + i / p.c;
        const int ch = g * p.c + (int)(i % p.c);
        norm_element<ST>(p, st, row, ch, xhat, dz, dgate);
        const float k = dz * (p.w ? p.w[ch] : 1.0f);
        static_cast<ST*>(p.dx)[row * p.C + ch] = from_f32<ST>(st.y * (k - m1 - xhat * m2));
        if (p.gate) static_cast<ST*>(p.dgate)[row * p.C + ch] = from_f32<ST>(dgate);
    }
}

// Sums over a slice of the rows for every channel.
template <typename ST>
__global__ void __launch_bounds__(128) norm_param_kernel(const NormParams p)
{
    ptx::grid_dependency_wait();
    const int ch = (int)blockIdx.x * 128 + (int)threadIdx.x;
    if (ch >= p.C) return;
    float2 s = make_float2(0.0f, 0.0f);
    for (long long row = blockIdx.y; row < p.n * p.L; row += gridDim.y) {
        float xhat, dz, dgate;
        norm_element<ST>(p, p.stats[row / p.L * p.G + ch / p.c], row, ch, xhat, dz, dgate);
        s.x = fmaf(dz, xhat, s.x);
        s.y += dz;
    }
    p.part[(long long)blockIdx.y * p.C + ch] = s;
}

// Sums of all parts in a fixed order: 32 channels per CTA, eight warps along the parts.
static __global__ void __launch_bounds__(256) norm_param_sum_kernel(const float2* part, int parts, int C, float* dw, float* db)
{
    __shared__ double2 sums[8][32];
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, ch = (int)blockIdx.x * 32 + lane;
    ptx::grid_dependency_wait();
    double2 s = make_double2(0.0, 0.0);
    if (ch < C)
        for (int i = warp; i < parts; i += 8) {
            const float2 v = part[(long long)i * C + ch];
            s.x += v.x;
            s.y += v.y;
        }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && ch < C) {
        for (int i = 1; i < 8; ++i) {
            s.x += sums[i][lane].x;
            s.y += sums[i][lane].y;
        }
        if (dw) dw[ch] = (float)s.x;
        if (db) db[ch] = (float)s.y;
    }
}

}  // namespace linrec

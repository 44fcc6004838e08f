// Group norm of channels-last tensors with an activation, or with an activated gate, and its backward pass.
//
// x is (samples, positions, channels); a group is the channels [g c, (g+1) c) of all positions of a sample.
//   xhat = (x - mean) * inv,   z = xhat * w + b,   y = act(z)   or, with a gate,   y = z * act(gate)
// Backward, with dz the gradient that reaches z and k = dz w:
//   dx = inv (k - mean(k) - xhat mean(k xhat)),   dgate = dy z act'(gate),   dw = sum dz xhat,   db = sum dz
//
// Two ways, both bound by memory:
//   rows     one position per sample (what follows a recurrence) and groups of up to 1024 channels.  A group
//            stays in the registers of the 1 to 32 lanes that hold it, the sums are shuffles; everything is
//            read once and written once.  A thread keeps its channels from row to row, so that weights are
//            loaded once and the parameters' gradients are summed in registers.
//   planes   anything else.  A CTA takes a slice of a sample's positions and a block of its groups; one kernel
//            leaves a partial result per slice and group, the second combines a sample's partials at its
//            start and applies them.  What the second reads again comes from L2 where a sample fits there.
// Variances are never differences of large sums: rows take two passes over registers, planes sum squares about
// an element of the thread's own and combine (mean, squares about the mean, count) triples.  All sums have a
// fixed order.
#pragma once
#include "elements.cuh"
#include "ptx.cuh"

namespace linrec {

constexpr int kActNone = 0, kActSilu = 1, kActSigmoid = 2;
constexpr int kNormThreads = 256;

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
    float2* part;                 // backward: [parts][C] sums of (dz xhat, dz), or null: not wanted
    // rows
    int lanes;                    // lanes per group, a power of two
    int gb, rp;                   // groups per CTA, rows it works on at a time
    // planes
    int cpb, sub;                 // channels per CTA; CTAs that a group is spread over (1: a CTA holds whole groups)
    int slices, xblocks;          // slices of a sample's positions; CTAs across the channels
    float4* gpart;                // [n][slices * sub][G]: (mean, squares, count) forward, (sum k, sum k xhat) backward
};

// V elements of one row as floats; `VEC`: the address is on a 16-byte boundary and all V exist.
template <typename ST, int V>
__device__ __forceinline__ void norm_load(const void* base, long long offset, float* v)
{
    const ST* q = static_cast<const ST*>(base) + offset;
    if constexpr (V == 8 && sizeof(ST) == 2) {
        const uint4 w = *reinterpret_cast<const uint4*>(q);
        Two<ST>::unpack(w.x, v), Two<ST>::unpack(w.y, v + 2), Two<ST>::unpack(w.z, v + 4), Two<ST>::unpack(w.w, v + 6);
    } else if constexpr (V == 8) {
        const float4 a = *reinterpret_cast<const float4*>(q), b = *reinterpret_cast<const float4*>(q + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        v[0] = to_f32<ST>(*q);
    }
}
template <typename ST, int V>
__device__ __forceinline__ void norm_store(void* base, long long offset, const float* v)
{
    ST* q = static_cast<ST*>(base) + offset;
    if constexpr (V == 8 && sizeof(ST) == 2) {
        *reinterpret_cast<uint4*>(q) = make_uint4(Two<ST>::pack(v), Two<ST>::pack(v + 2), Two<ST>::pack(v + 4), Two<ST>::pack(v + 6));
    } else if constexpr (V == 8) {
        reinterpret_cast<float4*>(q)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(q)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *q = from_f32<ST>(v[0]);
    }
}
template <int V>
__device__ __forceinline__ void norm_param(const float* p, int ch, float missing, float* v)
{
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = p ? __ldg(p + ch + e) : missing;
}

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
template <bool FAST>
__device__ __forceinline__ float activated(int act, float v)
{
    if (act == kActNone) return v;
    const float p = logistic<FAST>(v);
    // (minus infinity times a logistic value of zero is taken as it is: NaN, as in v * s(v))
    return act == kActSilu ? v * p : p;
}

// One element forward.
template <bool FAST, bool GATE>
__device__ __forceinline__ float norm_value(int act, float x, float gate, float mean, float inv, float w, float b)
{
    const float z = fmaf((x - mean) * inv, w, b);
    return GATE ? z * activated<FAST>(act, gate) : activated<FAST>(act, z);
}
// One element backward: xhat, the gradient dz of z, and the gate's gradient.
template <bool FAST, bool GATE>
__device__ __forceinline__ void norm_gradient(int act, float x, float gate, float dy, float2 st, float w, float b, float& xhat, float& dz,
                                              float& dgate)
{
    xhat = (x - st.x) * st.y;
    const float z = fmaf(xhat, w, b);
    float v, slope;
    activate<FAST>(act, GATE ? gate : z, v, slope);
    dz = dy * (GATE ? v : slope);
    dgate = GATE ? dy * z * slope : 0.0f;
}

// ---- rows -----------------------------------------------------------------------------------------------
__device__ __forceinline__ float lanes_sum(float v, int lanes)
{
    for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Thread -> (row within the CTA's set, group, first of its V-element pieces); pieces are `lanes` apart.
struct NormSlot {
    int r, g, lane;
    bool active;
};
__device__ __forceinline__ NormSlot norm_slot(const NormParams& p)
{
    NormSlot s;
    const int slot = (int)threadIdx.x / p.lanes;
    s.lane = (int)threadIdx.x - slot * p.lanes;
    s.r = slot / p.gb;
    s.g = (int)blockIdx.x * p.gb + slot - s.r * p.gb;
    s.active = s.r < p.rp && s.g < p.G;
    return s;
}

// NV pieces of V elements per lane.  The next row's operands are requested before this row is worked on.
template <typename ST, int V, int NV, bool GATE>
__global__ void __launch_bounds__(kNormThreads) norm_rows_fwd_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    const NormSlot s = norm_slot(p);
    ptx::grid_dependency_wait();
    bool have[NV];
    int ch[NV];
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = (i * p.lanes + s.lane) * V;
        have[i] = s.active && e < p.c;
        ch[i] = s.g * p.c + e;
        if (have[i]) {
            norm_param<V>(p.w, ch[i], 1.0f, w[i]);
            norm_param<V>(p.b, ch[i], 0.0f, b[i]);
        }
    }
    const long long step = (long long)gridDim.y * p.rp;
    long long n = (long long)blockIdx.y * p.rp + s.r;
    const float count = 1.0f / (float)p.c;
    float x[NV][V], gt[NV][V];
    auto fetch = [&](long long row, float (&to)[NV][V], float (&tg)[NV][V]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = have[i] && row < p.n;
#pragma unroll
            for (int e = 0; e < V; ++e) to[i][e] = tg[i][e] = 0.0f;
            if (in) norm_load<ST, V>(p.x, row * p.sx + ch[i], to[i]);
            if (GATE && in) norm_load<ST, V>(p.gate, row * p.sg + ch[i], tg[i]);
        }
    };
    fetch(n, x, gt);
    // (all threads of a CTA take the same number of turns: the shuffles need whole warps)
    for (long long base = (long long)blockIdx.y * p.rp; base < p.n; base += step, n += step) {
        float nx[NV][V], ng[NV][V];
        fetch(n + step, nx, ng);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) sum += x[i][e];
        const float mean = lanes_sum(sum, p.lanes) * count;
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (have[i])
#pragma unroll
                for (int e = 0; e < V; ++e) sq = fmaf(x[i][e] - mean, x[i][e] - mean, sq);
        const float inv = 1.0f / sqrtf(fmaf(lanes_sum(sq, p.lanes), count, p.eps));
        if (n < p.n) {
            if (p.stats && s.lane == 0 && s.active) p.stats[n * p.G + s.g] = make_float2(mean, inv);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (have[i]) {
                    float y[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) y[e] = norm_value<kFast, GATE>(p.act, x[i][e], gt[i][e], mean, inv, w[i][e], b[i][e]);
                    norm_store<ST, V>(p.y, n * p.C + ch[i], y);
                }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) x[i][e] = nx[i][e], gt[i][e] = ng[i][e];
    }
}

template <typename ST, int V, int NV, bool GATE>
__global__ void __launch_bounds__(kNormThreads) norm_rows_bwd_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    extern __shared__ __align__(16) float2 norm_sums[];      // [gb * c][rp] sums of (dz xhat, dz), if rp > 1
    const NormSlot s = norm_slot(p);
    ptx::grid_dependency_wait();
    bool have[NV];
    int ch[NV];
    float w[NV][V], b[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e0 = (i * p.lanes + s.lane) * V;
        have[i] = s.active && e0 < p.c;
        ch[i] = s.g * p.c + e0;
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = b[i][e] = dw[i][e] = db[i][e] = 0.0f;
        if (have[i]) {
            norm_param<V>(p.w, ch[i], 1.0f, w[i]);
            norm_param<V>(p.b, ch[i], 0.0f, b[i]);
        }
    }
    const long long step = (long long)gridDim.y * p.rp;
    const float count = 1.0f / (float)p.c;
    long long n = (long long)blockIdx.y * p.rp + s.r;
    for (long long base = (long long)blockIdx.y * p.rp; base < p.n; base += step, n += step) {
        const bool row = n < p.n;
        const float2 st = row && s.active ? p.stats[n * p.G + s.g] : make_float2(0.0f, 0.0f);
        float xhat[NV][V], k[NV][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < V; ++e) xhat[i][e] = k[i][e] = 0.0f;
            if (have[i] && row) {
                float x[V], gt[V], dy[V], dg[V];
                norm_load<ST, V>(p.x, n * p.sx + ch[i], x);
                norm_load<ST, V>(p.dy, n * p.sdy + ch[i], dy);
                if (GATE) norm_load<ST, V>(p.gate, n * p.sg + ch[i], gt);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float dz;
                    norm_gradient<kFast, GATE>(p.act, x[e], GATE ? gt[e] : 0.0f, dy[e], st, w[i][e], b[i][e], xhat[i][e], dz, dg[e]);
                    dw[i][e] = fmaf(dz, xhat[i][e], dw[i][e]);
                    db[i][e] += dz;
                    k[i][e] = dz * w[i][e];
                    s1 += k[i][e];
                    s2 = fmaf(k[i][e], xhat[i][e], s2);
                }
                if (GATE) norm_store<ST, V>(p.dgate, n * p.C + ch[i], dg);
            }
        }
        const float m1 = lanes_sum(s1, p.lanes) * count, m2 = lanes_sum(s2, p.lanes) * count;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (have[i] && row) {
                float dx[V];
#pragma unroll
                for (int e = 0; e < V; ++e) dx[e] = st.y * (k[i][e] - m1 - xhat[i][e] * m2);
                norm_store<ST, V>(p.dx, n * p.C + ch[i], dx);
            }
    }
    if (!p.part) return;
    float2* out = p.part + (long long)blockIdx.y * p.C;
    if (p.rp == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (have[i])
#pragma unroll
                for (int e = 0; e < V; ++e) out[ch[i] + e] = make_float2(dw[i][e], db[i][e]);
        return;
    }
    const int c0 = (int)blockIdx.x * p.gb * p.c, nch = min(p.gb * p.c, p.C - c0);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (have[i])
#pragma unroll
            for (int e = 0; e < V; ++e) norm_sums[s.r * nch + ch[i] + e - c0] = make_float2(dw[i][e], db[i][e]);
    __syncthreads();
    for (int i = (int)threadIdx.x; i < nch; i += kNormThreads) {
        float2 v = norm_sums[i];
        for (int r = 1; r < p.rp; ++r) {
            const float2 u = norm_sums[r * nch + i];
            v.x += u.x;
            v.y += u.y;
        }
        out[c0 + i] = v;
    }
}

// ---- planes -----------------------------------------------------------------------------------------------
// What a CTA covers: channels [c0, c0 + nch) and positions [l0, l1) of one sample.  A thread owns V channels
// (V divides a group's width) and every Y-th position.
struct NormBlock {
    long long n, l0, l1;
    int c0, nch, g0, groups, slot;      // slot: where its partial results go
    int X, Y, tx, ty;
    bool active;
};
template <int V>
__device__ __forceinline__ NormBlock norm_block(const NormParams& p, long long item, int xblock)
{
    NormBlock k;
    const long long per = (p.L + p.slices - 1) / p.slices;
    k.n = item / p.slices;
    const int slice = (int)(item - k.n * p.slices);
    k.l0 = per * slice;
    k.l1 = min(p.L, k.l0 + per);
    if (p.sub == 1) {
        const int gb = p.cpb / p.c;
        k.g0 = xblock * gb;
        k.groups = min(gb, p.G - k.g0);
        k.c0 = k.g0 * p.c;
        k.nch = k.groups * p.c;
        k.slot = slice;
    } else {
        k.g0 = xblock / p.sub;
        const int part = xblock - k.g0 * p.sub;
        k.groups = 1;
        k.c0 = k.g0 * p.c + part * p.cpb;
        k.nch = min(p.cpb, p.c - part * p.cpb);
        k.slot = slice * p.sub + part;
    }
    k.X = k.nch / V;
    k.Y = kNormThreads / k.X;
    k.ty = (int)threadIdx.x / k.X;
    k.tx = (int)threadIdx.x - k.ty * k.X;
    k.active = k.ty < k.Y;
    return k;
}

// (mean, squares about it, count) of two disjoint sets together.
__device__ __forceinline__ float4 norm_merge(float4 a, float4 b)
{
    if (b.z == 0.0f) return a;
    if (a.z == 0.0f) return b;
    const float n = a.z + b.z, d = b.x - a.x, f = b.z / n;
    return make_float4(fmaf(d, f, a.x), a.y + fmaf(d * d, a.z * f, b.y), n, 0.0f);
}
__device__ __forceinline__ float4 norm_add(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, 0.0f, 0.0f); }
__device__ __forceinline__ float4 shfl_down4(float4 v, int o)
{
    return make_float4(__shfl_down_sync(0xffffffffu, v.x, o), __shfl_down_sync(0xffffffffu, v.y, o), __shfl_down_sync(0xffffffffu, v.z, o), 0.0f);
}

// Combines the threads' triples group by group (a warp per group) and leaves them in the partials.
template <int V, typename Merge>
__device__ __forceinline__ void norm_leave(const NormParams& p, const NormBlock& k, float4 mine, float4* shared, Merge merge)
{
    if (k.active) shared[threadIdx.x] = mine;
    __syncthreads();
    const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
    const int width = k.X / k.groups;      // threads of one position in one group
    for (int g = warp; g < k.groups; g += kNormThreads / 32) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i = lane; i < width * k.Y; i += 32) v = merge(v, shared[(i / width) * k.X + g * width + i % width]);
#pragma unroll
        for (int o = 16; o; o >>= 1) v = merge(v, shfl_down4(v, o));
        if (lane == 0) p.gpart[(k.n * p.slices * p.sub + k.slot) * p.G + k.g0 + g] = v;
    }
}
// The combination of all of a sample's partials, for the groups of this CTA, as (x, y) pairs in shared memory.
template <typename Merge, typename Finish>
__device__ __forceinline__ void norm_collect(const NormParams& p, const NormBlock& k, float2* result, Merge merge, Finish finish)
{
    const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31, slots = p.slices * p.sub;
    for (int g = warp; g < k.groups; g += kNormThreads / 32) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i = lane; i < slots; i += 32) v = merge(v, p.gpart[(k.n * slots + i) * p.G + k.g0 + g]);
#pragma unroll
        for (int o = 16; o; o >>= 1) v = merge(v, shfl_down4(v, o));
        if (lane == 0) {
            result[g] = finish(v);
            if (p.stats && k.slot == 0 && p.y) p.stats[k.n * p.G + k.g0 + g] = result[g];
        }
    }
    __syncthreads();
}

template <typename ST, int V>
__global__ void __launch_bounds__(kNormThreads) norm_planes_stats_kernel(const NormParams p)
{
    __shared__ float4 shared[kNormThreads];
    const NormBlock k = norm_block<V>(p, blockIdx.x / (unsigned)p.xblocks, (int)blockIdx.x % p.xblocks);
    ptx::grid_dependency_wait();
    const int ch = k.c0 + k.tx * V;
    float4 mine = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (k.active && k.l0 + k.ty < k.l1) {
        const long long row0 = k.n * p.L;
        float v[V], about = 0.0f, s = 0.0f, q = 0.0f;
        long long l = k.l0 + k.ty;
        norm_load<ST, V>(p.x, (row0 + l) * p.sx + ch, v);
        about = v[0];
        float count = 0.0f;
#pragma unroll 4
        for (; l < k.l1; l += k.Y) {
            norm_load<ST, V>(p.x, (row0 + l) * p.sx + ch, v);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = v[e] - about;
                s += d;
                q = fmaf(d, d, q);
            }
            count += (float)V;
        }
        mine = make_float4(about + s / count, fmaxf(fmaf(-s / count, s, q), 0.0f), count, 0.0f);
        if (!(q == q)) mine.y = q;      // (fmaxf drops NaN)
    }
    norm_leave<V>(p, k, mine, shared, norm_merge);
}

template <typename ST, int V, bool GATE>
__global__ void __launch_bounds__(kNormThreads) norm_planes_apply_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    __shared__ float2 st[kNormThreads * V];
    const NormBlock k = norm_block<V>(p, blockIdx.x / (unsigned)p.xblocks, (int)blockIdx.x % p.xblocks);
    ptx::grid_dependency_wait();
    norm_collect(p, k, st, norm_merge, [&](float4 v) { return make_float2(v.x, 1.0f / sqrtf(v.y / v.z + p.eps)); });
    if (!k.active) return;
    const int ch = k.c0 + k.tx * V;
    const float2 mine = st[k.groups > 1 ? k.tx * V / p.c : 0];
    float w[V], b[V];
    norm_param<V>(p.w, ch, 1.0f, w);
    norm_param<V>(p.b, ch, 0.0f, b);
    const long long row0 = k.n * p.L;
#pragma unroll 2
    for (long long l = k.l0 + k.ty; l < k.l1; l += k.Y) {
        float x[V], gt[V], y[V];
        norm_load<ST, V>(p.x, (row0 + l) * p.sx + ch, x);
        if (GATE) norm_load<ST, V>(p.gate, (row0 + l) * p.sg + ch, gt);
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = norm_value<kFast, GATE>(p.act, x[e], GATE ? gt[e] : 0.0f, mine.x, mine.y, w[e], b[e]);
        norm_store<ST, V>(p.y, (row0 + l) * p.C + ch, y);
    }
}

// Sums of k and k xhat per slice and group, and of (dz xhat, dz) per slice and channel.
template <typename ST, int V, bool GATE>
__global__ void __launch_bounds__(kNormThreads) norm_planes_sums_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    __shared__ float4 shared[kNormThreads];
    __shared__ float2 chan[kNormThreads * V];
    const int xblock = (int)blockIdx.x % p.xblocks;
    const long long items = p.n * p.slices, turns = gridDim.x / (unsigned)p.xblocks;
    NormBlock k = norm_block<V>(p, blockIdx.x / (unsigned)p.xblocks, xblock);
    ptx::grid_dependency_wait();
    const int ch = k.c0 + k.tx * V;
    float dw[V], db[V], w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.0f;
    if (k.active) {
        norm_param<V>(p.w, ch, 1.0f, w);
        norm_param<V>(p.b, ch, 0.0f, b);
    }
    // a CTA takes several samples where there are many: their channel sums share one part
    for (long long item = blockIdx.x / (unsigned)p.xblocks; item < items; item += turns) {
        k = norm_block<V>(p, item, xblock);
        float s1 = 0.0f, s2 = 0.0f;
        if (k.active) {
            const float2 st = p.stats[k.n * p.G + ch / p.c];
            const long long row0 = k.n * p.L;
#pragma unroll 2
            for (long long l = k.l0 + k.ty; l < k.l1; l += k.Y) {
                float x[V], gt[V], dy[V];
                norm_load<ST, V>(p.x, (row0 + l) * p.sx + ch, x);
                norm_load<ST, V>(p.dy, (row0 + l) * p.sdy + ch, dy);
                if (GATE) norm_load<ST, V>(p.gate, (row0 + l) * p.sg + ch, gt);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float xhat, dz, dg;
                    norm_gradient<kFast, GATE>(p.act, x[e], GATE ? gt[e] : 0.0f, dy[e], st, w[e], b[e], xhat, dz, dg);
                    const float t = dz * w[e];
                    s1 += t;
                    s2 = fmaf(t, xhat, s2);
                    dw[e] = fmaf(dz, xhat, dw[e]);
                    db[e] += dz;
                }
            }
        }
        norm_leave<V>(p, k, make_float4(s1, s2, 0.0f, 0.0f), shared, norm_add);
        __syncthreads();
    }
    if (k.active)
#pragma unroll
        for (int e = 0; e < V; ++e) chan[threadIdx.x * V + e] = make_float2(dw[e], db[e]);
    __syncthreads();
    if (!p.part) return;
    for (int i = (int)threadIdx.x; i < k.nch; i += kNormThreads) {
        float2 v = chan[i];
        for (int y = 1; y < k.Y; ++y) {
            const float2 u = chan[y * k.nch + i];
            v.x += u.x;
            v.y += u.y;
        }
        p.part[(long long)(blockIdx.x / (unsigned)p.xblocks) * p.C + k.c0 + i] = v;
    }
}

template <typename ST, int V, bool GATE>
__global__ void __launch_bounds__(kNormThreads) norm_planes_dx_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    __shared__ float2 means[kNormThreads * V];
    const NormBlock k = norm_block<V>(p, blockIdx.x / (unsigned)p.xblocks, (int)blockIdx.x % p.xblocks);
    ptx::grid_dependency_wait();
    const float count = 1.0f / ((float)p.L * (float)p.c);
    norm_collect(p, k, means, norm_add, [&](float4 v) { return make_float2(v.x * count, v.y * count); });
    if (!k.active) return;
    const int ch = k.c0 + k.tx * V;
    const float2 m = means[k.groups > 1 ? k.tx * V / p.c : 0];
    float w[V], b[V];
    norm_param<V>(p.w, ch, 1.0f, w);
    norm_param<V>(p.b, ch, 0.0f, b);
    const float2 st = p.stats[k.n * p.G + ch / p.c];
    const long long row0 = k.n * p.L;
#pragma unroll 2
    for (long long l = k.l0 + k.ty; l < k.l1; l += k.Y) {
        float x[V], gt[V], dy[V], dx[V], dg[V];
        norm_load<ST, V>(p.x, (row0 + l) * p.sx + ch, x);
        norm_load<ST, V>(p.dy, (row0 + l) * p.sdy + ch, dy);
        if (GATE) norm_load<ST, V>(p.gate, (row0 + l) * p.sg + ch, gt);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float xhat, dz;
            norm_gradient<kFast, GATE>(p.act, x[e], GATE ? gt[e] : 0.0f, dy[e], st, w[e], b[e], xhat, dz, dg[e]);
            dx[e] = st.y * (dz * w[e] - m.x - xhat * m.y);
        }
        norm_store<ST, V>(p.dx, (row0 + l) * p.C + ch, dx);
        if (GATE) norm_store<ST, V>(p.dgate, (row0 + l) * p.C + ch, dg);
    }
}

// Sums of all parts in a fixed order: 32 channels per CTA, 32 warps along the parts.
static __global__ void __launch_bounds__(1024) norm_param_sum_kernel(const float2* part, int parts, int C, float* dw, float* db)
{
    __shared__ float2 sums[32][33];
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, ch = (int)blockIdx.x * 32 + lane;
    ptx::grid_dependency_wait();
    float2 s = make_float2(0.0f, 0.0f);
    if (ch < C)
#pragma unroll 4
        for (int i = warp; i < parts; i += 32) {
            const float2 v = part[(long long)i * C + ch];
            s.x += v.x;
            s.y += v.y;
        }
    sums[warp][lane] = s;
    __syncthreads();
    s = sums[lane][warp];
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s.x += __shfl_down_sync(0xffffffffu, s.x, o);
        s.y += __shfl_down_sync(0xffffffffu, s.y, o);
    }
    const int out = (int)blockIdx.x * 32 + warp;
    if (lane == 0 && out < C) {
        if (dw) dw[out] = s.x;
        if (db) db[out] = s.y;
    }
}

}  // namespace linrec

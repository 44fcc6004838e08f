// Group norm of channels-last tensors with an activation, or with an activated gate, and its backward pass.
//
// x is (samples, positions, channels); a group is the channels [g c, (g+1) c) of all positions of a sample.
//   xhat = (x - mean) * inv,   z = xhat * w + b,   y = act(z)   or, with a gate,   y = z * act(gate)
// Backward, with dz the gradient that reaches z and k = dz w:
//   dx = inv (k - mean(k) - xhat mean(k xhat)),   dgate = dy z act'(gate),   dw = sum dz xhat,   db = sum dz
//
// Two ways:
//   rows     one position per sample (what follows a recurrence) and groups of up to 1024 channels.  A group
//            stays in the registers of the 1 to 32 lanes that hold it, the sums are shuffles; everything is
//            read once and written once.  A thread keeps its channels from row to row, so that weights are
//            loaded once and the parameters' gradients are summed in registers.
//   planes   anything else.  A CTA takes a slice of a sample's positions and a block of its groups; one kernel
//            leaves a partial result per slice and group, the second combines a sample's partials at its
//            start and applies them.  What the second reads again comes from L2 where a sample fits there.
// Variances are never differences of large sums: rows take two passes over registers, planes sum squares about
// an element of the thread's own, or its mean where that element is an outlier, and combine (mean, squares about
// the mean, count) triples.  All sums have a fixed order.
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
    long long per;                // positions in a slice
    float4* gpart;                // [n][slices * sub][G]: (mean, squares, count) forward, (sum k, sum k xhat) backward
};

// Operands are loaded as read-only data: a kernel's loads may then be issued ahead of its stores.
template <typename ST>
__device__ __forceinline__ float load_one(const void* base, long long offset)
{
    return to_f32<ST>(__ldg(static_cast<const ST*>(base) + offset));
}
// Eight adjacent elements on a 16-byte boundary: as loaded, and as pairs of floats.
template <typename ST>
struct Eight {
    uint4 w[sizeof(ST) / 2];
    __device__ __forceinline__ void load(const void* base, long long offset)
    {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const ST*>(base) + offset);
        w[0] = __ldg(q);
        if constexpr (sizeof(ST) == 4) w[1] = __ldg(q + 1);
    }
    __device__ __forceinline__ void clear()
    {
        w[0] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (sizeof(ST) == 4) w[1] = w[0];
    }
    __device__ __forceinline__ void get(F2 (&v)[4]) const
    {
        if constexpr (sizeof(ST) == 4) {
            v[0] = f2(__uint_as_float(w[0].x), __uint_as_float(w[0].y)), v[1] = f2(__uint_as_float(w[0].z), __uint_as_float(w[0].w));
            v[2] = f2(__uint_as_float(w[1].x), __uint_as_float(w[1].y)), v[3] = f2(__uint_as_float(w[1].z), __uint_as_float(w[1].w));
        } else {
            v[0] = Two<ST>::get(w[0].x), v[1] = Two<ST>::get(w[0].y), v[2] = Two<ST>::get(w[0].z), v[3] = Two<ST>::get(w[0].w);
        }
    }
};
template <typename ST>
__device__ __forceinline__ void store_eight(void* base, long long offset, const F2 (&v)[4])
{
    uint4* q = reinterpret_cast<uint4*>(static_cast<ST*>(base) + offset);
    if constexpr (sizeof(ST) == 4) {
        const float2 a = f2_get(v[0]), b = f2_get(v[1]), c = f2_get(v[2]), d = f2_get(v[3]);
        q[0] = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
        q[1] = make_uint4(__float_as_uint(c.x), __float_as_uint(c.y), __float_as_uint(d.x), __float_as_uint(d.y));
    } else {
        q[0] = make_uint4(Two<ST>::put(v[0]), Two<ST>::put(v[1]), Two<ST>::put(v[2]), Two<ST>::put(v[3]));
    }
}
__device__ __forceinline__ void param_eight(const float* p, int ch, float missing, F2 (&v)[4])
{
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
        const float4 q = p ? __ldg(reinterpret_cast<const float4*>(p + ch + 2 * e)) : make_float4(missing, missing, missing, missing);
        v[e] = f2(q.x, q.y);
        v[e + 1] = f2(q.z, q.w);
    }
}
__device__ __forceinline__ float f2_sum(F2 a)
{
    const float2 v = f2_get(a);
    return v.x + v.y;
}

// act(v), and act(v) with its derivative, of two elements.
template <bool FAST, int ACT>
__device__ __forceinline__ F2 activated2(F2 v)
{
    if (ACT == kActNone) return v;
    const F2 p = logistic2<FAST>(v);
    return ACT == kActSilu ? f2_mul(v, p) : p;
}
template <bool FAST, int ACT>
__device__ __forceinline__ void activate2(F2 v, F2& value, F2& slope)
{
    if (ACT == kActNone) {
        value = v;
        slope = f2(1.0f);
        return;
    }
    if (ACT == kActSilu) {
        // p (1 + v s(-v)); s(-v) as 1 - p: where that loses its bits it is next to nothing beside 1/v
        const F2 p = logistic2<FAST>(v), n = f2_fma(p, f2(-1.0f), f2(1.0f));
        value = f2_mul(v, p);
        slope = f2_fma(value, n, p);
    } else {
        F2 n;
        logistic_pair2<FAST>(v, value, n);
        slope = f2_mul(value, n);
    }
}

// One element forward and backward (rows that are off 16-byte boundaries).
template <bool FAST, bool GATE, int ACT>
__device__ __forceinline__ float norm_value(float x, float gate, float mean, float inv, float w, float b)
{
    const float z = fmaf((x - mean) * inv, w, b);
    const float a = f2_get(activated2<FAST, ACT>(f2(GATE ? gate : z))).x;
    return GATE ? z * a : a;
}
template <bool FAST, bool GATE, int ACT>
__device__ __forceinline__ void norm_gradient(float x, float gate, float dy, float2 st, float w, float b, float& xhat, float& dz, float& dgate)
{
    xhat = (x - st.x) * st.y;
    const float z = fmaf(xhat, w, b);
    F2 v2, s2;
    activate2<FAST, ACT>(f2(GATE ? gate : z), v2, s2);
    const float v = f2_get(v2).x, slope = f2_get(s2).x;
    dz = dy * (GATE ? v : slope);
    dgate = GATE ? dy * z * slope : 0.0f;
}
// Eight elements backward: xhat and the gradient dz of z, and the gate's gradient.
template <bool FAST, bool GATE, int ACT>
__device__ __forceinline__ void norm_gradient8(const F2 (&x)[4], const F2 (&gate)[4], const F2 (&dy)[4], float2 st, const F2 (&w)[4],
                                               const F2 (&b)[4], F2 (&xhat)[4], F2 (&dz)[4], F2 (&dgate)[4])
{
    const F2 inv = f2(st.y), off = f2(-st.x);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        xhat[e] = f2_mul(f2_add(x[e], off), inv);
        const F2 z = f2_fma(xhat[e], w[e], b[e]);
        F2 v, slope;
        activate2<FAST, ACT>(GATE ? gate[e] : z, v, slope);
        dz[e] = f2_mul(dy[e], GATE ? v : slope);
        if (GATE) dgate[e] = f2_mul(f2_mul(dy[e], z), slope);
    }
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

// NV pieces of eight elements per lane.  The next row's operands are in flight while a row is worked on, as they come
// (four registers for eight elements).  Bytes in flight bound both passes: forward four CTAs per SM with one row
// ahead (three with two: 80 us instead of 79 at (16384, 4096) bf16 with gate, fp32 86 instead of 70), backward two CTAs
// with two rows ahead (three with one: 160 us instead of 128).  So measured: 79 us (5.1 TB/s), issue slots 72 %, DRAM 54 % busy.
template <typename ST, int NV, bool GATE, int ACT>
__global__ void __launch_bounds__(kNormThreads, NV == 1 ? 4 : 2) norm_rows_fwd_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    const NormSlot s = norm_slot(p);
    ptx::grid_dependency_wait();
    bool have[NV];
    int ch[NV];
    F2 w[NV][4], b[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = (i * p.lanes + s.lane) * 8;
        have[i] = s.active && e < p.c;
        ch[i] = s.g * p.c + e;
        if (have[i]) {
            param_eight(p.w, ch[i], 1.0f, w[i]);
            param_eight(p.b, ch[i], 0.0f, b[i]);
        }
    }
    const long long step = (long long)gridDim.y * p.rp;
    long long n = (long long)blockIdx.y * p.rp + s.r;
    const float count = 1.0f / (float)p.c;
    constexpr int kAhead = 1;
    Eight<ST> rx[kAhead][NV], rg[kAhead][NV];
    auto fetch = [&](int set, long long row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            rx[set][i].clear();
            if (have[i] && row < p.n) {
                rx[set][i].load(p.x, row * p.sx + ch[i]);
                if (GATE) rg[set][i].load(p.gate, row * p.sg + ch[i]);
            }
        }
    };
    auto turn = [&](int set) {
        F2 x[NV][4];
        Eight<ST> gate[NV];
        F2 sum = f2(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            rx[set][i].get(x[i]);
            if (GATE) gate[i] = rg[set][i];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = f2_add(sum, x[i][e]);
        }
        fetch(set, n + kAhead * step);
        const float mean = lanes_sum(f2_sum(sum), p.lanes) * count;
        F2 sq = f2(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (have[i])
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[i][e] = f2_add(x[i][e], f2(-mean));
                    sq = f2_fma(x[i][e], x[i][e], sq);
                }
        const float inv = 1.0f / sqrtf(fmaf(lanes_sum(f2_sum(sq), p.lanes), count, p.eps));
        if (n < p.n) {
            if (p.stats && s.lane == 0 && s.active) p.stats[n * p.G + s.g] = make_float2(mean, inv);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (have[i]) {
                    F2 gt[4], y[4];
                    if (GATE) gate[i].get(gt);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const F2 z = f2_fma(f2_mul(x[i][e], f2(inv)), w[i][e], b[i][e]);
                        y[e] = GATE ? f2_mul(z, activated2<kFast, ACT>(gt[e])) : activated2<kFast, ACT>(z);
                    }
                    store_eight<ST>(p.y, n * p.C + ch[i], y);
                }
        }
        n += step;
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(k, n + k * step);
    // (all threads of a CTA take the same number of turns: the shuffles need whole warps)
    for (long long base = (long long)blockIdx.y * p.rp; base < p.n; base += kAhead * step)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) turn(k);
}

// One element per access, NV per lane (rows off 16-byte boundaries, or groups that are not whole sixteens of bytes).
// With many pieces per lane the operands of eight are loaded before any is worked on: behind the stores and branches of
// the piece before them they wait for memory one by one.  (16384, 4098) with gate, 6 groups, without and with:
// forward bf16 439 and 326 us, fp32 499 and 446; backward fp32 835 and 491, but bf16 447 and 472, and with few pieces
// ((16384, 4004), 91 groups, bf16) 265 / 365 and 282 / 478, which therefore load piece by piece.
template <typename ST, int NV, bool GATE, int ACT>
__global__ void __launch_bounds__(kNormThreads, NV > 8 ? 3 : 4) norm_rows1_fwd_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    const int lanes = NV > 8 ? 32 : p.lanes;      // (many pieces: a whole warp, and constant distances)
    const NormSlot s = norm_slot(p);
    ptx::grid_dependency_wait();
    const int ch0 = s.g * p.c, mine = s.active ? (p.c - s.lane + lanes - 1) / lanes : 0;      // elements of this lane
    const float *w = p.w + ch0 + s.lane, *b = p.b + ch0 + s.lane;
    const long long step = (long long)gridDim.y * p.rp;
    long long n = (long long)blockIdx.y * p.rp + s.r;
    const float count = 1.0f / (float)p.c;
    for (long long base = (long long)blockIdx.y * p.rp; base < p.n; base += step, n += step) {
        const bool row = n < p.n;
        const ST* x = static_cast<const ST*>(p.x) + n * p.sx + ch0 + s.lane;
        const ST* gate = static_cast<const ST*>(p.gate) + n * p.sg + ch0 + s.lane;
        ST* y = static_cast<ST*>(p.y) + n * p.C + ch0 + s.lane;
        float v[NV], sum = 0.0f, sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = row && i < mine ? load_one<ST>(x, i * lanes) : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) sum += v[i];
        const float mean = lanes_sum(sum, lanes) * count;
#pragma unroll
        for (int i = 0; i < NV; ++i) sq = i < mine ? fmaf(v[i] - mean, v[i] - mean, sq) : sq;
        const float inv = 1.0f / sqrtf(fmaf(lanes_sum(sq, lanes), count, p.eps));
        if (!row) continue;
        if (p.stats && s.lane == 0 && s.active) p.stats[n * p.G + s.g] = make_float2(mean, inv);
        if constexpr (NV > 8) {
#pragma unroll
            for (int i0 = 0; i0 < NV; i0 += 8) {
                float g[8], wi[8], bi[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = i0 + j;
                    g[j] = GATE && i < mine ? load_one<ST>(gate, i * lanes) : 0.0f;
                    wi[j] = p.w && i < mine ? __ldg(w + i * lanes) : 1.0f;
                    bi[j] = p.b && i < mine ? __ldg(b + i * lanes) : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const ST r = from_f32<ST>(norm_value<kFast, GATE, ACT>(v[i0 + j], g[j], mean, inv, wi[j], bi[j]));
                    if (i0 + j < mine) y[(i0 + j) * lanes] = r;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i < mine)
                    y[i * lanes] = from_f32<ST>(norm_value<kFast, GATE, ACT>(v[i], GATE ? load_one<ST>(gate, i * lanes) : 0.0f, mean, inv,
                                                                             p.w ? __ldg(w + i * lanes) : 1.0f, p.b ? __ldg(b + i * lanes) : 0.0f));
        }
    }
}

// The sums of (dz xhat, dz) of a CTA's rows, which lie as [rp][channels of the CTA] in shared memory, to the parts.
__device__ __forceinline__ void norm_rows_leave(const NormParams& p, const float2* sums)
{
    __syncthreads();
    const int c0 = (int)blockIdx.x * p.gb * p.c, nch = min(p.gb * p.c, p.C - c0);
    for (int i = (int)threadIdx.x; i < nch; i += kNormThreads) {
        float2 v = sums[i];
        for (int r = 1; r < p.rp; ++r) {
            const float2 u = sums[r * nch + i];
            v.x += u.x;
            v.y += u.y;
        }
        p.part[(long long)blockIdx.y * p.C + c0 + i] = v;
    }
}

template <typename ST, int NV, bool GATE, int ACT>
__global__ void __launch_bounds__(kNormThreads, NV == 1 ? 2 : 1) norm_rows_bwd_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    extern __shared__ __align__(16) float2 norm_sums[];
    const NormSlot s = norm_slot(p);
    ptx::grid_dependency_wait();
    bool have[NV];
    int ch[NV];
    F2 w[NV][4], b[NV][4], dw[NV][4], db[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e0 = (i * p.lanes + s.lane) * 8;
        have[i] = s.active && e0 < p.c;
        ch[i] = s.g * p.c + e0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[i][e] = b[i][e] = dw[i][e] = db[i][e] = f2(0.0f);
        if (have[i]) {
            param_eight(p.w, ch[i], 1.0f, w[i]);
            param_eight(p.b, ch[i], 0.0f, b[i]);
        }
    }
    const long long step = (long long)gridDim.y * p.rp;
    const float count = 1.0f / (float)p.c;
    long long n = (long long)blockIdx.y * p.rp + s.r;
    constexpr int kAhead = NV == 1 ? 2 : 1;
    Eight<ST> rx[kAhead][NV], rg[kAhead][NV], rd[kAhead][NV];
    float2 rst[kAhead];
    auto fetch = [&](int set, long long row) {
        rst[set] = row < p.n && s.active ? __ldg(p.stats + row * p.G + s.g) : make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (have[i] && row < p.n) {
                rx[set][i].load(p.x, row * p.sx + ch[i]);
                rd[set][i].load(p.dy, row * p.sdy + ch[i]);
                if (GATE) rg[set][i].load(p.gate, row * p.sg + ch[i]);
            } else {
                rx[set][i].clear(), rd[set][i].clear(), rg[set][i].clear();
            }
        }
    };
    auto turn = [&](int set) {
        const bool row = n < p.n;
        const float2 st = rst[set];
        F2 xhat[NV][4], k[NV][4], s1 = f2(0.0f), s2 = f2(0.0f);
        Eight<ST> cx[NV], cg[NV], cd[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) cx[i] = rx[set][i], cg[i] = rg[set][i], cd[i] = rd[set][i];
        fetch(set, n + kAhead * step);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            F2 x[4], gt[4], dy[4], dg[4];
            cx[i].get(x);
            cd[i].get(dy);
            if (GATE) cg[i].get(gt);
            norm_gradient8<kFast, GATE, ACT>(x, gt, dy, st, w[i], b[i], xhat[i], k[i], dg);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (rows and pieces that do not exist have dy = 0 and therefore add nothing)
                dw[i][e] = f2_fma(k[i][e], xhat[i][e], dw[i][e]);
                db[i][e] = f2_add(db[i][e], k[i][e]);
                k[i][e] = f2_mul(k[i][e], w[i][e]);
                s1 = f2_add(s1, k[i][e]);
                s2 = f2_fma(k[i][e], xhat[i][e], s2);
            }
            if (GATE && have[i] && row) store_eight<ST>(p.dgate, n * p.C + ch[i], dg);
        }
        const float m1 = lanes_sum(f2_sum(s1), p.lanes) * count, m2 = lanes_sum(f2_sum(s2), p.lanes) * count;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (have[i] && row) {
                F2 dx[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) dx[e] = f2_mul(f2_fma(xhat[i][e], f2(-m2), f2_add(k[i][e], f2(-m1))), f2(st.y));
                store_eight<ST>(p.dx, n * p.C + ch[i], dx);
            }
        n += step;
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(k, n + k * step);
    for (long long base = (long long)blockIdx.y * p.rp; base < p.n; base += kAhead * step)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) turn(k);
    if (!p.part) return;
    const int c0 = (int)blockIdx.x * p.gb * p.c, nch = min(p.gb * p.c, p.C - c0);
    float2* out = p.rp == 1 ? p.part + (long long)blockIdx.y * p.C : norm_sums + s.r * nch - c0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (have[i])
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 a = f2_get(dw[i][e]), c = f2_get(db[i][e]);
                out[ch[i] + 2 * e] = make_float2(a.x, c.x);
                out[ch[i] + 2 * e + 1] = make_float2(a.y, c.y);
            }
    if (p.rp > 1) norm_rows_leave(p, norm_sums);
}

// One element per access; the sums of (dz xhat, dz) live in shared memory, every thread at its own places.
template <typename ST, int NV, bool GATE, int ACT>
__global__ void __launch_bounds__(kNormThreads, NV > 8 ? 3 : 4) norm_rows1_bwd_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    const int lanes = NV > 8 ? 32 : p.lanes;      // (many pieces: a whole warp, and constant distances)
    extern __shared__ __align__(16) float2 norm_sums[];
    const NormSlot s = norm_slot(p);
    ptx::grid_dependency_wait();
    const int c0 = (int)blockIdx.x * p.gb * p.c, nch = min(p.gb * p.c, p.C - c0);
    const int ch0 = s.g * p.c, mine = s.active ? (p.c - s.lane + lanes - 1) / lanes : 0;
    float2* sums = norm_sums + s.r * nch + ch0 - c0 + s.lane;
    if (p.part)
        for (int i = 0; i < mine; ++i) sums[i * lanes] = make_float2(0.0f, 0.0f);
    const float *w = p.w + ch0 + s.lane, *b = p.b + ch0 + s.lane;
    const long long step = (long long)gridDim.y * p.rp;
    const float count = 1.0f / (float)p.c;
    long long n = (long long)blockIdx.y * p.rp + s.r;
    for (long long base = (long long)blockIdx.y * p.rp; base < p.n; base += step, n += step) {
        const bool row = n < p.n;
        const float2 st = row && s.active ? p.stats[n * p.G + s.g] : make_float2(0.0f, 0.0f);
        const ST* x = static_cast<const ST*>(p.x) + n * p.sx + ch0 + s.lane;
        const ST* dy = static_cast<const ST*>(p.dy) + n * p.sdy + ch0 + s.lane;
        const ST* gate = static_cast<const ST*>(p.gate) + n * p.sg + ch0 + s.lane;
        ST* dx = static_cast<ST*>(p.dx) + n * p.C + ch0 + s.lane;
        ST* dgate = static_cast<ST*>(p.dgate) + n * p.C + ch0 + s.lane;
        float xhat[NV], k[NV], s1 = 0.0f, s2 = 0.0f;
        auto take = [&](int i, float xv, float g, float d, float wi, float bi) {
            float dz, dg;
            norm_gradient<kFast, GATE, ACT>(xv, g, d, st, wi, bi, xhat[i], dz, dg);
            if (p.part) {
                float2 v = sums[i * lanes];
                v.x = fmaf(dz, xhat[i], v.x);
                v.y += dz;
                sums[i * lanes] = v;
            }
            k[i] = dz * wi;
            s1 += k[i];
            s2 = fmaf(k[i], xhat[i], s2);
            if (GATE) dgate[i * lanes] = from_f32<ST>(dg);
        };
        if constexpr (NV > 8 && sizeof(ST) == 4) {
#pragma unroll
            for (int i0 = 0; i0 < NV; i0 += 8) {
                float xv[8], g[8], d[8], wi[8], bi[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = i0 + j;
                    const bool have = row && i < mine;
                    xv[j] = have ? load_one<ST>(x, i * lanes) : 0.0f;
                    g[j] = GATE && have ? load_one<ST>(gate, i * lanes) : 0.0f;
                    d[j] = have ? load_one<ST>(dy, i * lanes) : 0.0f;
                    wi[j] = p.w && have ? __ldg(w + i * lanes) : 1.0f;
                    bi[j] = p.b && have ? __ldg(b + i * lanes) : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    xhat[i0 + j] = k[i0 + j] = 0.0f;
                    if (row && i0 + j < mine) take(i0 + j, xv[j], g[j], d[j], wi[j], bi[j]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                xhat[i] = k[i] = 0.0f;
                if (row && i < mine) {
                    const float wi = p.w ? __ldg(w + i * lanes) : 1.0f;
                    take(i, load_one<ST>(x, i * lanes), GATE ? load_one<ST>(gate, i * lanes) : 0.0f, load_one<ST>(dy, i * lanes), wi,
                         p.b ? __ldg(b + i * lanes) : 0.0f);
                }
            }
        }
        const float m1 = lanes_sum(s1, lanes) * count, m2 = lanes_sum(s2, lanes) * count;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (row && i < mine) dx[i * lanes] = from_f32<ST>(st.y * (k[i] - m1 - xhat[i] * m2));
    }
    if (p.part) norm_rows_leave(p, norm_sums);
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
    k.n = (unsigned)item / (unsigned)p.slices;
    const int slice = (int)((unsigned)item - (unsigned)k.n * (unsigned)p.slices);
    k.l0 = p.per * slice;
    k.l1 = min(p.L, k.l0 + p.per);
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
    const float n = a.z + b.z, d = b.x - a.x, f = __fdividef(b.z, n);
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
    __shared__ float4 some[kNormThreads / 32][32];
    const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31, slots = p.slices * p.sub;
    // neighbouring lanes take neighbouring groups, the warps share the slices
    for (int g0 = 0; g0 < k.groups; g0 += 32) {
        const int g = g0 + lane;
        const bool in = g < k.groups;
        const float4* from = p.gpart + k.n * slots * p.G + k.g0 + g;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (in)
#pragma unroll 4
            for (int i = warp; i < slots; i += kNormThreads / 32) v = merge(v, from[(long long)i * p.G]);
        some[warp][lane] = v;
        __syncthreads();
        if (warp == 0 && in) {
            for (int i = 1; i < kNormThreads / 32; ++i) v = merge(v, some[i][lane]);
            result[g] = finish(v);
            if (p.stats && k.slot == 0 && p.y) p.stats[k.n * p.G + k.g0 + g] = result[g];
        }
        __syncthreads();
    }
}

template <typename ST, int V>
__global__ void __launch_bounds__(kNormThreads, 3) norm_planes_stats_kernel(const NormParams p)
{
    __shared__ float4 shared[kNormThreads];
    const NormBlock k = norm_block<V>(p, blockIdx.x / (unsigned)p.xblocks, (int)blockIdx.x % p.xblocks);
    ptx::grid_dependency_wait();
    const int ch = k.c0 + k.tx * V;
    float4 mine = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const long long first = k.l0 + k.ty;
    if (k.active && first < k.l1) {
        const long long row0 = k.n * p.L;
        const float count = (float)V * (float)((k.l1 - first + k.Y - 1) / k.Y);
        float about = load_one<ST>(p.x, (row0 + first) * p.sx + ch), m, squares;
        // A second time, about the thread's mean, where the first element lies so far from the others that the squares are
        // less than a 32nd of the sum they are a difference of (within five standard deviations they are more).  (223, 600, 2048) fp32, 32 groups, every sample's first position at 1000: results were off by 1.1 %, now by
        // 2e-6; no time where it does not occur ((8, 8192, 2048) bf16 177 us with and without).
        for (bool again = false;; again = true) {
            float s, q;
            if constexpr (V == 8) {
                const F2 off = f2(-about);
                F2 s2 = f2(0.0f), q2 = f2(0.0f);
#pragma unroll 4
                for (long long l = first; l < k.l1; l += k.Y) {
                    Eight<ST> r;
                    F2 v[4];
                    r.load(p.x, (row0 + l) * p.sx + ch);
                    r.get(v);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const F2 d = f2_add(v[e], off);
                        s2 = f2_add(s2, d);
                        q2 = f2_fma(d, d, q2);
                    }
                }
                s = f2_sum(s2), q = f2_sum(q2);
            } else {
                s = q = 0.0f;
#pragma unroll 4
                for (long long l = first; l < k.l1; l += k.Y) {
                    const float d = load_one<ST>(p.x, (row0 + l) * p.sx + ch) - about;
                    s += d;
                    q = fmaf(d, d, q);
                }
            }
            m = s / count, squares = fmaf(-m, s, q);
            if (again || !(q > 32.0f * squares)) break;
            about += m;
        }
        mine = make_float4(about + m, squares < 0.0f ? 0.0f : squares, count, 0.0f);
    }
    norm_leave<V>(p, k, mine, shared, [](float4 a, float4 b) { return norm_merge(a, b); });
}

template <typename ST, int V, bool GATE, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3) norm_planes_apply_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    __shared__ float2 st[kNormThreads * V];
    const NormBlock k = norm_block<V>(p, blockIdx.x / (unsigned)p.xblocks, (int)blockIdx.x % p.xblocks);
    ptx::grid_dependency_wait();
    norm_collect(p, k, st, [](float4 a, float4 b) { return norm_merge(a, b); },
                 [&](float4 v) { return make_float2(v.x, 1.0f / sqrtf(v.y / v.z + p.eps)); });
    if (!k.active) return;
    const int ch = k.c0 + k.tx * V;
    const float2 mine = st[k.groups > 1 ? k.tx * V / p.c : 0];
    const long long row0 = k.n * p.L;
    if constexpr (V == 8) {
        F2 w[4], b[4];
        param_eight(p.w, ch, 1.0f, w);
        param_eight(p.b, ch, 0.0f, b);
#pragma unroll 2
        for (long long l = k.l0 + k.ty; l < k.l1; l += k.Y) {
            Eight<ST> rx, rg;
            F2 x[4], gt[4], y[4];
            rx.load(p.x, (row0 + l) * p.sx + ch);
            if (GATE) rg.load(p.gate, (row0 + l) * p.sg + ch);
            rx.get(x);
            if (GATE) rg.get(gt);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const F2 z = f2_fma(f2_mul(f2_add(x[e], f2(-mine.x)), f2(mine.y)), w[e], b[e]);
                y[e] = GATE ? f2_mul(z, activated2<kFast, ACT>(gt[e])) : activated2<kFast, ACT>(z);
            }
            store_eight<ST>(p.y, (row0 + l) * p.C + ch, y);
        }
    } else {
        const float w = p.w ? p.w[ch] : 1.0f, b = p.b ? p.b[ch] : 0.0f;
#pragma unroll 4
        for (long long l = k.l0 + k.ty; l < k.l1; l += k.Y)
            static_cast<ST*>(p.y)[(row0 + l) * p.C + ch] = from_f32<ST>(norm_value<kFast, GATE, ACT>(
                load_one<ST>(p.x, (row0 + l) * p.sx + ch),
                GATE ? load_one<ST>(p.gate, (row0 + l) * p.sg + ch) : 0.0f, mine.x, mine.y, w, b));
    }
}

// Sums of k and k xhat per slice and group, and of (dz xhat, dz) per slice and channel.
template <typename ST, int V, bool GATE, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3) norm_planes_sums_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    constexpr int H = V == 8 ? 4 : 1;
    __shared__ float4 shared[kNormThreads];
    __shared__ float2 chan[kNormThreads * V];
    const int xblock = (int)blockIdx.x % p.xblocks;
    const long long items = p.n * p.slices, turns = gridDim.x / (unsigned)p.xblocks;
    NormBlock k = norm_block<V>(p, blockIdx.x / (unsigned)p.xblocks, xblock);
    ptx::grid_dependency_wait();
    const int ch = k.c0 + k.tx * V;
    F2 dw[H], db[H], w[4], b[4];
#pragma unroll
    for (int e = 0; e < H; ++e) dw[e] = db[e] = f2(0.0f);
    if (k.active) {
        if constexpr (V == 8) {
            param_eight(p.w, ch, 1.0f, w);
            param_eight(p.b, ch, 0.0f, b);
        } else {
            w[0] = f2(p.w ? p.w[ch] : 1.0f);
            b[0] = f2(p.b ? p.b[ch] : 0.0f);
        }
    }
    // a CTA takes several samples where there are many: their channel sums share one part
    for (long long item = blockIdx.x / (unsigned)p.xblocks; item < items; item += turns) {
        k = norm_block<V>(p, item, xblock);
        F2 s1 = f2(0.0f), s2 = f2(0.0f);
        if (k.active) {
            const float2 st = p.stats[k.n * p.G + ch / p.c];
            const long long row0 = k.n * p.L;
#pragma unroll 2
            for (long long l = k.l0 + k.ty; l < k.l1; l += k.Y) {
                if constexpr (V == 8) {
                    Eight<ST> rx, rg, rd;
                    F2 x[4], gt[4], dy[4], xhat[4], dz[4], dg[4];
                    rx.load(p.x, (row0 + l) * p.sx + ch);
                    rd.load(p.dy, (row0 + l) * p.sdy + ch);
                    if (GATE) rg.load(p.gate, (row0 + l) * p.sg + ch);
                    rx.get(x);
                    rd.get(dy);
                    if (GATE) rg.get(gt);
                    norm_gradient8<kFast, GATE, ACT>(x, gt, dy, st, w, b, xhat, dz, dg);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const F2 t = f2_mul(dz[e], w[e]);
                        s1 = f2_add(s1, t);
                        s2 = f2_fma(t, xhat[e], s2);
                        dw[e] = f2_fma(dz[e], xhat[e], dw[e]);
                        db[e] = f2_add(db[e], dz[e]);
                    }
                } else {
                    float xhat, dz, dg;
                    norm_gradient<kFast, GATE, ACT>(load_one<ST>(p.x, (row0 + l) * p.sx + ch),
                                                    GATE ? load_one<ST>(p.gate, (row0 + l) * p.sg + ch) : 0.0f,
                                                    load_one<ST>(p.dy, (row0 + l) * p.sdy + ch), st, f2_get(w[0]).x,
                                                    f2_get(b[0]).x, xhat, dz, dg);
                    // both sums of the channel in one pair, (dz xhat, dz)
                    dw[0] = f2_fma(f2(dz), f2(xhat, 1.0f), dw[0]);
                    s1 = f2_fma(f2(dz * f2_get(w[0]).x), f2(1.0f, xhat), s1);
                }
            }
        }
        const float2 a = f2_get(s1);
        norm_leave<V>(p, k, V == 8 ? make_float4(a.x + a.y, f2_sum(s2), 0.0f, 0.0f) : make_float4(a.x, a.y, 0.0f, 0.0f), shared,
                      [](float4 a, float4 b) { return norm_add(a, b); });
        __syncthreads();
    }
    if (!p.part) return;
    if (k.active) {
        if constexpr (V == 8) {
#pragma unroll
            for (int e = 0; e < H; ++e) {
                const float2 a = f2_get(dw[e]), c = f2_get(db[e]);
                chan[threadIdx.x * 8 + 2 * e] = make_float2(a.x, c.x);
                chan[threadIdx.x * 8 + 2 * e + 1] = make_float2(a.y, c.y);
            }
        } else {
            chan[threadIdx.x] = f2_get(dw[0]);
        }
    }
    __syncthreads();
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

template <typename ST, int V, bool GATE, int ACT>
__global__ void __launch_bounds__(kNormThreads, 3) norm_planes_dx_kernel(const NormParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    __shared__ float2 means[kNormThreads * V];
    const NormBlock k = norm_block<V>(p, blockIdx.x / (unsigned)p.xblocks, (int)blockIdx.x % p.xblocks);
    ptx::grid_dependency_wait();
    const float count = 1.0f / ((float)p.L * (float)p.c);
    norm_collect(p, k, means, [](float4 a, float4 b) { return norm_add(a, b); }, [&](float4 v) { return make_float2(v.x * count, v.y * count); });
    if (!k.active) return;
    const int ch = k.c0 + k.tx * V;
    const float2 m = means[k.groups > 1 ? k.tx * V / p.c : 0];
    const float2 st = p.stats[k.n * p.G + ch / p.c];
    const long long row0 = k.n * p.L;
    if constexpr (V == 8) {
        F2 w[4], b[4];
        param_eight(p.w, ch, 1.0f, w);
        param_eight(p.b, ch, 0.0f, b);
#pragma unroll 2
        for (long long l = k.l0 + k.ty; l < k.l1; l += k.Y) {
            Eight<ST> rx, rg, rd;
            F2 x[4], gt[4], dy[4], xhat[4], dz[4], dg[4];
            rx.load(p.x, (row0 + l) * p.sx + ch);
            rd.load(p.dy, (row0 + l) * p.sdy + ch);
            if (GATE) rg.load(p.gate, (row0 + l) * p.sg + ch);
            rx.get(x);
            rd.get(dy);
            if (GATE) rg.get(gt);
            norm_gradient8<kFast, GATE, ACT>(x, gt, dy, st, w, b, xhat, dz, dg);
#pragma unroll
            for (int e = 0; e < 4; ++e) dz[e] = f2_mul(f2_fma(xhat[e], f2(-m.y), f2_fma(dz[e], w[e], f2(-m.x))), f2(st.y));
            store_eight<ST>(p.dx, (row0 + l) * p.C + ch, dz);
            if (GATE) store_eight<ST>(p.dgate, (row0 + l) * p.C + ch, dg);
        }
    } else {
        const float w = p.w ? p.w[ch] : 1.0f, b = p.b ? p.b[ch] : 0.0f;
#pragma unroll 4
        for (long long l = k.l0 + k.ty; l < k.l1; l += k.Y) {
            float xhat, dz, dg;
            norm_gradient<kFast, GATE, ACT>(load_one<ST>(p.x, (row0 + l) * p.sx + ch),
                                            GATE ? load_one<ST>(p.gate, (row0 + l) * p.sg + ch) : 0.0f,
                                            load_one<ST>(p.dy, (row0 + l) * p.sdy + ch), st, w, b, xhat, dz, dg);
            static_cast<ST*>(p.dx)[(row0 + l) * p.C + ch] = from_f32<ST>(st.y * (dz * w - m.x - xhat * m.y));
            if (GATE) static_cast<ST*>(p.dgate)[(row0 + l) * p.C + ch] = from_f32<ST>(dg);
        }
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

// Gated linear recurrence on channels-last tensors, with its backward pass and its one-token step.
//
//     h[t] = a[t] * h[t-1] + b[t] * u[t],     y[t] = h[t] rounded once,     state in fp32
//   forget form   a = s(f),   b = s(-f),                                  u = x
//   decay form    log a = -k softplus(L) s(f),   b = sqrt(1 - a^2),       u = s(i) x       (L per channel)
// with s the logistic function and f, i logits.  The multiplier is formed in fp32 and never stored:
// rounded to 16 bits a multiplier next to one would be off by more than its distance from one.
//
// Layout of the work.  All sequences lie along ONE scan axis of rows (a packed buffer as it is, a batch
// of equal lengths either as one axis per batch entry or, for short sequences, packed as well).  A row
// where a sequence starts has its multiplier taken out of the chain (the initial state enters through
// the added term instead), a row that belongs to no sequence is an element (0, 0): nothing but these two
// rules tells ragged from dense, so the tiles are the same size whatever the lengths are.  Positions are
// counted in scan order; a reversed scan only changes the memory row a position stands for.
//
// A tile is 64 channels x R positions for one CTA of eight warps: a lane owns two adjacent channels, a
// warp K consecutive positions, kept in registers as (a, b u) pairs, so that the gates are evaluated
// once.  Each thread folds its run into a (P, Y) pair, the eight runs meet in shared memory, and 64
// threads link the tile to its predecessor along the axis by decoupled look-back (one 16-byte descriptor
// per channel and tile; tickets are handed out position-major, so the predecessor is `units` tickets
// older and a wait is only ever for a ticket that a running CTA holds).  The runs are then walked again
// from the true state.  Reads and writes every element once.
//
// The cut is carried as a multiplier of minus zero, which products of multipliers (all >= 0) keep, and it
// selects rather than multiplies: 0 * NaN would let one sequence's infinities into its neighbour.
//
// The backward pass recomputes h from fp32 checkpoints that the forward pass leaves every 64 positions
// (never from the rounded outputs) and scans the adjoint against the direction of the forward pass:
//   w[t] = dy[t] + q[t+1],   q[t] = a[t] w[t]      (q enters the state gradient where a sequence starts)
// whose multiplier is the element's own, so one product P serves both directions.
#pragma once
#include "column_kernels.cuh"
#include "elements.cuh"

namespace linrec {

constexpr int kGatedWarps = 8;
constexpr int kGatedChannels = 64;      // channels per tile: 32 lanes x 2
constexpr int kGatedCheckpoint = 64;    // positions between two checkpoints
constexpr int kGatedThreads = kGatedWarps * 32;

struct GatedParams {
    const void *x, *f, *ig, *dy;        // (rows, D) with the row strides below; ig: decay form only; dy: backward only
    long long sx, sf, si, sdy;          // elements between rows
    void *y, *dx, *df, *di;             // results, rows at stride D
    const float* decay;                 // [D], decay form
    float scale;
    const float* h0;                    // [nseq][D] or null
    float* hT;                          // [nseq][D] or null (forward)
    const float* dhT;                   // [nseq][D] or null (backward)
    float* dh0;                         // [nseq][D] or null (backward)
    float* ckpt;                        // [nb * nck][D]: state that enters positions 0, 64, 128, ...; null: not wanted
    float* dlam;                        // [nb * nk][D]: sums of d(log a) log a over a tile (backward, decay form)
    const void* cu;                     // nseq + 1 offsets, or null: sequences of `seqlen` rows
    int cu64;
    int nseq;
    long long seqlen;
    long long nrows;                    // rows per axis
    int nb;                             // axes (batch entries scanned side by side)
    int D, dtiles, units;               // units = nb * dtiles
    int nk, nck;                        // tiles, checkpoints per axis
    long long ntickets;                 // nk * units
    int reverse;
    uint32_t* header;
    TileDesc* desc;                     // [nk][units][64]
    long long wait_budget;
};

// ---- gates ------------------------------------------------------------------------------------------
// sqrt(1 - exp(2 la)) for la <= 0: the Taylor series of 1 - exp(-z) where the difference would cancel.
__device__ __forceinline__ float decay_input_factor(float la, float a)
{
    const float z = -2.0f * la;
    float s = fmaf(z, -1.0f / 7.0f, 1.0f);
    s = fmaf(z * s, -1.0f / 6.0f, 1.0f);
    s = fmaf(z * s, -1.0f / 5.0f, 1.0f);
    s = fmaf(z * s, -1.0f / 4.0f, 1.0f);
    s = fmaf(z * s, -1.0f / 3.0f, 1.0f);
    s = fmaf(z * s, -1.0f / 2.0f, 1.0f);
    return approx_sqrt(z < 0.25f ? z * s : fmaf(-a, a, 1.0f));
}

// ---- the pair operator with cuts ------------------------------------------------------------------------
constexpr float kCut = -0.0f;
__device__ __forceinline__ bool is_cut(float p) { return __float_as_uint(p) == 0x80000000u; }
__device__ __forceinline__ float enter(float in, Pair s) { return is_cut(s.p) ? s.y : fmaf(in, s.p, s.y); }
__device__ __forceinline__ Pair join(Pair far, Pair near)
{
    return Pair{enter(far.y, near), is_cut(near.p) ? near.p : far.p * near.p};
}

// ---- where sequences start and end --------------------------------------------------------------------
// Positions [s0, s0 + K) of one warp's run: bit j of `start` / `end` / `valid` describes position s0 + j
// (`cut`: nothing enters it from the position before); lane j keeps the index of the sequence that
// position belongs to.
struct GatedRun {
    uint32_t start, end, valid, cut;
    int seq;
};

__device__ __forceinline__ long long gated_offset(const GatedParams& p, int i)
{
    return p.cu64 ? __ldg(static_cast<const long long*>(p.cu) + i) : (long long)__ldg(static_cast<const int*>(p.cu) + i);
}

template <int K>
__device__ __forceinline__ GatedRun gated_run(const GatedParams& p, int b, long long s0, int lane)
{
    GatedRun r;
    bool st = false, en = false, ok = false;
    int q = 0;
    const long long s = s0 + lane;
    if (lane < K && s < p.nrows) {
        if (p.cu) {
            // the last sequence whose offset is not behind the row (bounded whatever the offsets hold)
            const long long row = p.reverse ? p.nrows - 1 - s : s;
            int lo = 0, hi = p.nseq + 1;          // first index with offset > row lies in [lo, hi]
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (gated_offset(p, mid) <= row) lo = mid + 1;
                else hi = mid;
            }
            q = lo - 1;
            if (q >= 0 && q < p.nseq) {
                ok = true;
                const long long first = gated_offset(p, q), last = gated_offset(p, q + 1) - 1;
                st = row == (p.reverse ? last : first);
                en = row == (p.reverse ? first : last);
            }
        } else {
            ok = true;
            if (p.nb > 1 || p.seqlen == p.nrows) {   // one sequence per axis
                q = b;
                st = s == 0;
                en = s == p.nrows - 1;
            } else {
                const long long i = s / p.seqlen, o = s - i * p.seqlen;
                q = (int)(p.reverse ? p.nseq - 1 - i : i);
                st = o == 0;
                en = o == p.seqlen - 1;
            }
        }
    }
    r.start = __ballot_sync(0xffffffffu, st);
    r.end = __ballot_sync(0xffffffffu, en);
    r.valid = __ballot_sync(0xffffffffu, ok);
    r.cut = r.start | ~r.valid;
    r.seq = q;
    return r;
}

// ---- linking a tile to its predecessor -----------------------------------------------------------------
// Waits (bounded) until descriptor `d` of tile `n` holds something; false when the budget ran out.
__device__ __forceinline__ bool gated_await(const TileDesc* d, int n, uint4& w, uint32_t epoch, long long budget, uint32_t* status)
{
    if (w.z != 0u && w.w == (uint32_t)n) return true;
    const long long t0 = clock64();
    while (true) {
        w = desc_load(d, epoch);
        if (w.z != 0u && w.w == (uint32_t)n) return true;
        if (clock64() - t0 > budget) {
            atomicOr(status, kStatusLookbackTimeout);
            return false;
        }
        __nanosleep(20);
    }
}

// What enters tile `k` of one channel.  Walks back to the nearest predecessor that holds an inclusive value,
// then folds FORWARD from there, one tile after the other: the value is the one that the predecessors'
// own chain of inclusive values gives, bit for bit, whichever of them were finished when it was read, so
// results do not depend on timing.  `d` is the descriptor of tile k - 1; tile 0 is always inclusive.
// Descriptors are requested a window at a time (independent loads, one round trip).
__device__ __forceinline__ float gated_lookback(const TileDesc* d, long long stride, int k, uint32_t epoch, long long budget, uint32_t* status)
{
    constexpr int W = 8;
    uint4 w[W];
    int dist = 0;          // tiles k - 1, ..., k - dist hold aggregates
    bool found = false;
    while (!found) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = dist + i < k ? desc_load(d - (long long)(dist + i) * stride, epoch) : make_uint4(0u, 0u, 2u, 0u);
        int here = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if (found || dist + i >= k) continue;
            if (!gated_await(d - (long long)(dist + i) * stride, k - 1 - dist - i, w[i], epoch, budget, status)) return 0.0f;
            if (w[i].z == 2u) found = true;
            else ++here;
        }
        dist += here;
        if (found && here == dist) {   // all of the walk is in this window
            float v = 0.0f;
#pragma unroll
            for (int i = W - 1; i >= 0; --i) {
                if (i == here) v = __uint_as_float(w[i].x);
                else if (i < here) v = enter(v, desc_pair(w[i]));
            }
            return v;
        }
        if (dist >= k) return 0.0f;    // not reached: tile 0 is inclusive
    }
    float v = __uint_as_float(desc_load(d - (long long)dist * stride, epoch).x);
    for (int far = dist - 1; far >= 0; far -= W) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (far - i >= 0) w[i] = desc_load(d - (long long)(far - i) * stride, epoch);
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (far - i >= 0) v = w[i].z == 2u ? __uint_as_float(w[i].x) : enter(v, desc_pair(w[i]));
    }
    return v;
}

// Run by 64 threads, one channel each: returns the value that enters the tile and publishes the one that
// leaves it.  `k` counts tiles along the axis in the direction of the scan; `d` is this tile's descriptor.
__device__ __forceinline__ float gated_link(const GatedParams& p, TileDesc* d, uint4 seen, int k, Pair total, uint32_t epoch)
{
    const long long stride = (long long)p.units * kGatedChannels;
    const bool more = k + 1 < p.nk;
    float in = 0.0f;
    bool done = false;
    if (k > 0) {
        if (seen.z == 2u && seen.w == (uint32_t)(k - 1)) {
            in = __uint_as_float(seen.x);
        } else {
            // a total that forgets what enters (a sequence starts in the tile) is final already
            if (more) {
                done = is_cut(total.p);
                col_publish(d, total.y, total.p, done ? 2u : 1u, epoch, (uint32_t)k);
            }
            in = gated_lookback(d - stride, stride, k, epoch, p.wait_budget, p.header + 1);
        }
    }
    if (more && !done) col_publish(d, enter(in, total), 0.0f, 2u, epoch, (uint32_t)k);
    return in;
}

// ---- forward ------------------------------------------------------------------------------------------
template <typename ST>
struct GatedTile {
    static constexpr int kRunFwd = sizeof(ST) == 4 ? 8 : 16;      // positions per thread
    static constexpr int kRunBwd = 8;
    static constexpr int kRowsFwd = kRunFwd * kGatedWarps;
    static constexpr int kRowsBwd = kRunBwd * kGatedWarps;
};

template <typename ST, bool DECAY>
__global__ void __launch_bounds__(kGatedThreads) gated_fwd_kernel(const GatedParams p)
{
    constexpr int K = GatedTile<ST>::kRunFwd, R = GatedTile<ST>::kRowsFwd;
    __shared__ float4 runs[2][kGatedWarps][32];      // (Y, P) of both channels of every thread
    __shared__ float entering[kGatedChannels];
    __shared__ uint32_t next_ticket;

    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    ptx::grid_dependency_wait();
    const uint32_t epoch = read_epoch(p.header);

    for (int it = 0;; ++it) {
        if (tid == 0) next_ticket = atomicAdd(p.header, 1u);
        __syncthreads();
        const uint32_t ticket = next_ticket;
        if ((long long)ticket >= p.ntickets) break;
        const int k = (int)(ticket / (uint32_t)p.units);
        const int unit = (int)(ticket - (uint32_t)k * (uint32_t)p.units);
        const int b = unit / p.dtiles, dt = unit - b * p.dtiles;
        const int ch = dt * kGatedChannels + 2 * lane;
        const int have = p.D - ch;
        const long long s0 = (long long)k * R + warp * K;
        const GatedRun run = gated_run<K>(p, b, s0, lane);
        TileDesc* desc = p.desc + ((long long)ticket * kGatedChannels + tid);
        uint4 seen = make_uint4(0u, 0u, 0u, 0u);
        if (tid < kGatedChannels && k > 0) seen = desc_load(desc - (long long)p.units * kGatedChannels, epoch);
        const long long row0 = (long long)b * p.nrows + (p.reverse ? p.nrows - 1 - s0 : s0);
        const int step = p.reverse ? -1 : 1;

        float nsp[2] = {0.0f, 0.0f};
        if (DECAY) {
#pragma unroll
            for (int v = 0; v < 2; ++v)
                if (v < have) nsp[v] = -p.scale * softplus(p.decay[ch + v]);
        }
        float a[K][2], u[K][2];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            float xv[2] = {0.0f, 0.0f}, fv[2] = {0.0f, 0.0f}, iv[2] = {0.0f, 0.0f};
            if (run.valid >> j & 1u) {
                const long long row = row0 + (long long)j * step;
                load_two<ST>(p.x, row * p.sx + ch, have, xv);
                load_two<ST>(p.f, row * p.sf + ch, have, fv);
                if (DECAY) load_two<ST>(p.ig, row * p.si + ch, have, iv);
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                float g, n;
                logistic_pair(fv[v], g, n);
                if (DECAY) {
                    const float la = nsp[v] * g;
                    a[j][v] = expf(la);
                    u[j][v] = decay_input_factor(la, a[j][v]) * (logistic(iv[v]) * xv[v]);
                } else {
                    a[j][v] = g;
                    u[j][v] = n * xv[v];
                }
            }
            if (!(run.valid >> j & 1u)) u[j][0] = u[j][1] = 0.0f;
            if (run.start >> j & 1u) {
                const int q = __shfl_sync(0xffffffffu, run.seq, j);
                float hv[2] = {0.0f, 0.0f};
                if (p.h0) load_two<float>(p.h0, (long long)q * p.D + ch, have, hv);
#pragma unroll
                for (int v = 0; v < 2; ++v) u[j][v] = fmaf(a[j][v], hv[v], u[j][v]);
            }
        }
        Pair agg[2] = {pair_identity(), pair_identity()};
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const bool cut = run.cut >> j & 1u;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                agg[v].y = cut ? u[j][v] : fmaf(a[j][v], agg[v].y, u[j][v]);
                agg[v].p = cut ? kCut : agg[v].p * a[j][v];
            }
        }
        float4(*set)[32] = runs[it & 1];
        set[warp][lane] = make_float4(agg[0].y, agg[0].p, agg[1].y, agg[1].p);
        __syncthreads();

        if (tid < kGatedChannels) {
            Pair total = pair_identity();
#pragma unroll
            for (int i = 0; i < kGatedWarps; ++i) {
                const float2 w = reinterpret_cast<const float2*>(&set[i][tid >> 1])[tid & 1];
                total = join(total, Pair{w.x, w.y});
            }
            entering[tid] = gated_link(p, desc, seen, k, total, epoch);
        }
        Pair before[2] = {pair_identity(), pair_identity()};
        for (int i = 0; i < warp; ++i) {
            const float4 w = set[i][lane];
            before[0] = join(before[0], Pair{w.x, w.y});
            before[1] = join(before[1], Pair{w.z, w.w});
        }
        __syncthreads();
        float h[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) h[v] = enter(entering[2 * lane + v], before[v]);
        if (p.ckpt && s0 % kGatedCheckpoint == 0 && s0 < p.nrows)
            store_two<float>(p.ckpt, ((long long)b * p.nck + s0 / kGatedCheckpoint) * p.D + ch, have, h);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (s0 + j >= p.nrows) break;
#pragma unroll
            for (int v = 0; v < 2; ++v) h[v] = (run.cut >> j & 1u) ? u[j][v] : fmaf(a[j][v], h[v], u[j][v]);
            store_two<ST>(p.y, (row0 + (long long)j * step) * p.D + ch, have, h);
            if (p.hT && (run.end >> j & 1u)) {
                const int q = __shfl_sync(0xffffffffu, run.seq, j);
                store_two<float>(p.hT, (long long)q * p.D + ch, have, h);
            }
        }
    }
    if (tid == 0) finish_launch(p.header, epoch);
}

// ---- backward -----------------------------------------------------------------------------------------
template <typename ST, bool DECAY>
__global__ void __launch_bounds__(kGatedThreads) gated_bwd_kernel(const GatedParams p)
{
    constexpr int K = GatedTile<ST>::kRunBwd, R = GatedTile<ST>::kRowsBwd;
    static_assert(R == kGatedCheckpoint, "one checkpoint per tile");
    __shared__ float4 runs[2][kGatedWarps][32];      // (Y, P) of both channels, forward direction
    __shared__ float2 back[2][kGatedWarps][32];      // Y of both channels, adjoint direction (same P)
    __shared__ float entering[kGatedChannels];
    __shared__ float2 dsum[kGatedWarps][32];
    __shared__ uint32_t next_ticket;

    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    ptx::grid_dependency_wait();
    const uint32_t epoch = read_epoch(p.header);

    for (int it = 0;; ++it) {
        if (tid == 0) next_ticket = atomicAdd(p.header, 1u);
        __syncthreads();
        const uint32_t ticket = next_ticket;
        if ((long long)ticket >= p.ntickets) break;
        const int g = (int)(ticket / (uint32_t)p.units);      // tiles in adjoint order
        const int unit = (int)(ticket - (uint32_t)g * (uint32_t)p.units);
        const int k = p.nk - 1 - g;
        const int b = unit / p.dtiles, dt = unit - b * p.dtiles;
        const int ch = dt * kGatedChannels + 2 * lane;
        const int have = p.D - ch;
        const long long s0 = (long long)k * R + warp * K;
        const GatedRun run = gated_run<K>(p, b, s0, lane);
        TileDesc* desc = p.desc + ((long long)ticket * kGatedChannels + tid);
        uint4 seen = make_uint4(0u, 0u, 0u, 0u);
        if (tid < kGatedChannels && g > 0) seen = desc_load(desc - (long long)p.units * kGatedChannels, epoch);
        const long long row0 = (long long)b * p.nrows + (p.reverse ? p.nrows - 1 - s0 : s0);
        const int step = p.reverse ? -1 : 1;

        float nsp[2] = {0.0f, 0.0f};
        float h[2];
        load_two<float>(p.ckpt, ((long long)b * p.nck + k) * p.D + ch, have, h);
        if (DECAY) {
#pragma unroll
            for (int v = 0; v < 2; ++v)
                if (v < have) nsp[v] = -p.scale * softplus(p.decay[ch + v]);
        }
        float a[K][2], bb[K][2], x[K][2], dyv[K][2], sn[K][2], gi[K][2], la[K][2], hs[K][2];
        Pair agg[2] = {pair_identity(), pair_identity()};
#pragma unroll
        for (int j = 0; j < K; ++j) {
            float fv[2] = {0.0f, 0.0f}, iv[2] = {0.0f, 0.0f};
            x[j][0] = x[j][1] = dyv[j][0] = dyv[j][1] = hs[j][0] = hs[j][1] = 0.0f;
            const bool ok = run.valid >> j & 1u;
            if (ok) {
                const long long row = row0 + (long long)j * step;
                load_two<ST>(p.x, row * p.sx + ch, have, x[j]);
                load_two<ST>(p.f, row * p.sf + ch, have, fv);
                if (DECAY) load_two<ST>(p.ig, row * p.si + ch, have, iv);
                load_two<ST>(p.dy, row * p.sdy + ch, have, dyv[j]);
                if (p.dhT && (run.end >> j & 1u)) {
                    const int q = __shfl_sync(0xffffffffu, run.seq, j);
                    float e[2] = {0.0f, 0.0f};
                    load_two<float>(p.dhT, (long long)q * p.D + ch, have, e);
                    dyv[j][0] += e[0];
                    dyv[j][1] += e[1];
                }
                if (p.h0 && (run.start >> j & 1u)) {
                    const int q = __shfl_sync(0xffffffffu, run.seq, j);
                    load_two<float>(p.h0, (long long)q * p.D + ch, have, hs[j]);
                }
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                float s;
                logistic_pair(fv[v], s, sn[j][v]);
                float uv = x[j][v];
                if (DECAY) {
                    la[j][v] = nsp[v] * s;
                    a[j][v] = expf(la[j][v]);
                    bb[j][v] = decay_input_factor(la[j][v], a[j][v]);
                    gi[j][v] = logistic(iv[v]);
                    uv *= gi[j][v];
                } else {
                    a[j][v] = s;
                    bb[j][v] = sn[j][v];
                }
                if (!ok) a[j][v] = bb[j][v] = 0.0f;
                const bool cut = run.cut >> j & 1u;
                agg[v].y = fmaf(a[j][v], cut ? hs[j][v] : agg[v].y, bb[j][v] * uv);
                agg[v].p = cut ? kCut : agg[v].p * a[j][v];
            }
        }
        float qv[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = K - 1; j >= 0; --j)
#pragma unroll
            for (int v = 0; v < 2; ++v) qv[v] = (run.cut >> j & 1u) ? 0.0f : a[j][v] * (dyv[j][v] + qv[v]);
        float4(*set)[32] = runs[it & 1];
        float2(*bset)[32] = back[it & 1];
        set[warp][lane] = make_float4(agg[0].y, agg[0].p, agg[1].y, agg[1].p);
        bset[warp][lane] = make_float2(qv[0], qv[1]);
        __syncthreads();

        if (tid < kGatedChannels) {
            Pair total = pair_identity();
#pragma unroll
            for (int i = kGatedWarps - 1; i >= 0; --i) {
                const float P = reinterpret_cast<const float2*>(&set[i][tid >> 1])[tid & 1].y;
                const float Y = reinterpret_cast<const float*>(&bset[i][tid >> 1])[tid & 1];
                total = join(total, Pair{Y, P});
            }
            entering[tid] = gated_link(p, desc, seen, g, total, epoch);
        }
        // the state that enters this run, from the checkpoint
        for (int i = 0; i < warp; ++i) {
            const float4 w = set[i][lane];
            h[0] = enter(h[0], Pair{w.x, w.y});
            h[1] = enter(h[1], Pair{w.z, w.w});
        }
        Pair after[2] = {pair_identity(), pair_identity()};
        for (int i = kGatedWarps - 1; i > warp; --i) {
            const float4 w = set[i][lane];
            const float2 y = bset[i][lane];
            after[0] = join(after[0], Pair{y.x, w.y});
            after[1] = join(after[1], Pair{y.y, w.w});
        }
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float before = (run.cut >> j & 1u) ? hs[j][v] : h[v];
                hs[j][v] = before;
                float uv = x[j][v];
                if (DECAY) uv *= gi[j][v];
                h[v] = fmaf(a[j][v], before, bb[j][v] * uv);
            }
        __syncthreads();
        float q[2], dl[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < 2; ++v) q[v] = enter(entering[2 * lane + v], after[v]);
#pragma unroll
        for (int j = K - 1; j >= 0; --j) {
            const bool cut = run.cut >> j & 1u, ok = run.valid >> j & 1u;
            float odx[2], odf[2], odi[2], oq[2];
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float w = dyv[j][v] + q[v];
                oq[v] = a[j][v] * w;
                q[v] = cut ? 0.0f : oq[v];
                if (DECAY) {
                    const float u = gi[j][v] * x[j][v];
                    const float aa = a[j][v], slope = bb[j][v] > 0.0f ? __fdividef(aa * aa, bb[j][v]) : 0.0f;
                    const float dla = w * fmaf(aa, hs[j][v], -u * slope);
                    const float t = dla * la[j][v];
                    dl[v] += ok ? t : 0.0f;
                    odx[v] = w * bb[j][v] * gi[j][v];
                    odi[v] = w * bb[j][v] * (u * (1.0f - gi[j][v]));
                    odf[v] = t * sn[j][v];
                } else {
                    odx[v] = w * bb[j][v];
                    odf[v] = oq[v] * bb[j][v] * (hs[j][v] - x[j][v]);
                }
            }
            if (s0 + j < p.nrows) {
                const long long at = (row0 + (long long)j * step) * p.D + ch;
                if (!ok) odx[0] = odx[1] = odf[0] = odf[1] = odi[0] = odi[1] = 0.0f;
                store_two<ST>(p.dx, at, have, odx);
                store_two<ST>(p.df, at, have, odf);
                if (DECAY) store_two<ST>(p.di, at, have, odi);
                if (p.dh0 && (run.start >> j & 1u)) {
                    const int n = __shfl_sync(0xffffffffu, run.seq, j);
                    store_two<float>(p.dh0, (long long)n * p.D + ch, have, oq);
                }
            }
        }
        if (DECAY) {
            dsum[warp][lane] = make_float2(dl[0], dl[1]);
            __syncthreads();
            if (tid < kGatedChannels && dt * kGatedChannels + tid < p.D) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < kGatedWarps; ++i) s += reinterpret_cast<const float*>(&dsum[i][tid >> 1])[tid & 1];
                p.dlam[((long long)b * p.nk + k) * p.D + dt * kGatedChannels + tid] = s;
            }
        }
    }
    if (tid == 0) finish_launch(p.header, epoch);
}

// Gradient of the decay parameter from the tiles' sums, in a fixed order: d L = s(L)/softplus(L) * sum.
// One warp-wide column of 32 channels per CTA, eight warps along the tiles.
static __global__ void __launch_bounds__(256) gated_decay_grad_kernel(const float* part, long long tiles, int D, const float* decay, float* out)
{
    __shared__ double sums[8][32];
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
    const int ch = (int)blockIdx.x * 32 + lane;
    ptx::grid_dependency_wait();
    double s = 0.0;
    if (ch < D)
        for (long long t = warp; t < tiles; t += 8) s += (double)part[t * D + ch];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && ch < D) {
        for (int i = 1; i < 8; ++i) s += sums[i][lane];
        const float L = decay[ch], sp = softplus(L);
        out[ch] = (float)s * (sp > 0.0f ? logistic(L) / sp : 1.0f);
    }
}

// ---- one token ------------------------------------------------------------------------------------------
struct GatedStepParams {
    const void *x, *f, *ig;
    long long sx, sf, si;
    void* y;                      // rows at stride D
    const float* decay;
    float scale;
    float* state;                 // [nslots] rows at stride `sstate`
    long long sstate;
    const void* slots;            // [rows] or null: row r owns state row r
    int slots64;
    int rows, nslots, D;
};

__device__ __forceinline__ long long step_slot(const GatedStepParams& p, int r)
{
    if (!p.slots) return r;
    const long long s = p.slots64 ? __ldg(static_cast<const long long*>(p.slots) + r) : (long long)__ldg(static_cast<const int*>(p.slots) + r);
    return s >= 0 && s < p.nslots ? s : -1;
}

// One row per block row; a thread owns V channels.  A slot that several rows name holds ONE sequence whose
// tokens are the rows in order: the first of them walks through all, the others leave.
template <typename ST, bool DECAY>
__global__ void __launch_bounds__(128) gated_step_kernel(const GatedStepParams p)
{
    __shared__ int nearest;
    const int tid = (int)threadIdx.x;
    const int ch = ((int)blockIdx.y * 128 + tid) * 2;
    const int have = p.D - ch;
    int row = (int)blockIdx.x;
    ptx::grid_dependency_wait();
    const long long slot = step_slot(p, row);
    if (slot < 0) {
        const float zero[2] = {0.0f, 0.0f};
        store_two<ST>(p.y, (long long)row * p.D + ch, have, zero);
        return;
    }
    bool earlier = false, later = false;
    if (p.slots)
        for (int r = tid; r < p.rows; r += 128)
            if (r != row && step_slot(p, r) == slot) (r < row ? earlier : later) = true;
    if (__syncthreads_or(earlier)) return;
    const bool chain = __syncthreads_or(later);

    float h[2] = {0.0f, 0.0f}, nsp[2] = {0.0f, 0.0f};
    load_two<float>(p.state, slot * p.sstate + ch, have, h);
    if (DECAY) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
            if (v < have) nsp[v] = -p.scale * softplus(p.decay[ch + v]);
    }
    while (true) {
        float xv[2], fv[2], iv[2];
        load_two<ST>(p.x, (long long)row * p.sx + ch, have, xv);
        load_two<ST>(p.f, (long long)row * p.sf + ch, have, fv);
        if (DECAY) load_two<ST>(p.ig, (long long)row * p.si + ch, have, iv);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            float s, n;
            logistic_pair(fv[v], s, n);
            if (DECAY) {
                const float la = nsp[v] * s, a = expf(la);
                h[v] = fmaf(a, h[v], decay_input_factor(la, a) * (logistic(iv[v]) * xv[v]));
            } else {
                h[v] = fmaf(s, h[v], n * xv[v]);
            }
        }
        store_two<ST>(p.y, (long long)row * p.D + ch, have, h);
        if (!chain) break;
        __syncthreads();
        if (tid == 0) nearest = 0x7fffffff;
        __syncthreads();
        for (int r = row + 1 + tid; r < p.rows; r += 128)
            if (step_slot(p, r) == slot) {
                atomicMin(&nearest, r);
                break;
            }
        __syncthreads();
        if (nearest == 0x7fffffff) break;
        row = nearest;
    }
    store_two<float>(p.state, slot * p.sstate + ch, have, h);
}

}  // namespace linrec

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

#include <type_traits>

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
    int pair;                           // results may be written two channels at a time
};

// ---- gates ------------------------------------------------------------------------------------------
// a = exp(-y) and b^2 = 1 - a^2 = (1 - a)(1 + a) from y = -log a >= 0.  Below 1/4 the distance 1 - a comes from
// its Taylor series (truncated at y^6/7! = 5e-8 relative) and a from it: an error of the multiplier is
// kept for 1/(1 - a) positions, so next to one it has to be right to half its last place.  SMALL: y is known to be below 1/4.
template <bool FAST, bool SMALL>
__device__ __forceinline__ void decay_factors(float y, float& a, float& b2)
{
    float s = fmaf(y, -1.0f / 720.0f, 1.0f / 120.0f);
    s = fmaf(y, s, -1.0f / 24.0f);
    s = fmaf(y, s, 1.0f / 6.0f);
    s = fmaf(y, s, -0.5f);
    float d = y * fmaf(y, s, 1.0f);
    a = 1.0f - d;
    if (!SMALL && !(y < 0.25f)) {
        a = exp_of<FAST>(-y);
        d = 1.0f - a;
    }
    b2 = d * (1.0f + a);
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

// ---- the tile ---------------------------------------------------------------------------------------------
// How operands reach shared memory, where every thread finds the words of its own two channels and K
// positions:
//   kLoadTma    one bulk-tensor copy per operand through a ring of stages, issued by the last warp as soon as a
//               barrier of the tile shows a stage free (rows on 16-byte boundaries); a ninth warp for the
//               copies would cost every thread a quarter of its registers
//   kLoadWord   4-byte asynchronous copies, every thread its own words, one tile ahead (4-byte boundaries)
//   kLoadAny    plain loads by the thread, stored to the same place (any alignment)
constexpr int kLoadTma = 0, kLoadWord = 1, kLoadAny = 2;

template <typename ST, bool DECAY, bool BWD>
struct GatedTile {
    static constexpr bool kFast = sizeof(ST) == 2;                     // 16-bit results: fast exponentials will do
    static constexpr int K = BWD || sizeof(ST) == 4 ? 8 : 16;          // positions per thread
    static constexpr int R = K * kGatedWarps;                          // positions per tile
    static constexpr int kArrays = (DECAY ? 3 : 2) + (BWD ? 1 : 0);    // x, f(, i)(, dy)
    static constexpr int kArrayBytes = R * kGatedChannels * (int)sizeof(ST);
    static constexpr int kStageBytes = kArrays * kArrayBytes;
    // forward: a stage is free once the gates are in registers; backward: only when the next tile has begun
    static constexpr int kStages = BWD && sizeof(ST) == 2 ? 3 : 2;
    static constexpr int kDynSmem = kStages * kStageBytes + 128;
    using Word = typename Two<ST>::Word;
};

struct GatedMaps {
    CUtensorMap x, f, i, dy;
};

struct GatedWhere {
    int k;            // tile along the axis, in forward scan order
    int g;            // the same in the order of this pass
    int b, dt;        // axis, channel block
};
template <bool BWD>
__device__ __forceinline__ GatedWhere gated_where(const GatedParams& p, uint32_t ticket)
{
    GatedWhere w;
    w.g = (int)(ticket / (uint32_t)p.units);
    const int unit = (int)(ticket - (uint32_t)w.g * (uint32_t)p.units);
    w.b = unit / p.dtiles;
    w.dt = unit - w.b * p.dtiles;
    w.k = BWD ? p.nk - 1 - w.g : w.g;
    return w;
}

// A thread's own words of one tile, by asynchronous 4-byte copies or plain loads.
template <typename ST, bool DECAY, bool BWD, int LOAD>
__device__ __forceinline__ void gated_fetch(const GatedParams& p, const GatedWhere& w, typename Two<ST>::Word* stage, int warp, int lane)
{
    using T = GatedTile<ST, DECAY, BWD>;
    const void* src[4] = {p.x, p.f, DECAY ? p.ig : p.dy, p.dy};
    const long long stride[4] = {p.sx, p.sf, DECAY ? p.si : p.sdy, p.sdy};
    const int ch = w.dt * kGatedChannels + 2 * lane, have = p.D - ch;
    const long long s0 = (long long)w.k * T::R + warp * T::K;
    const long long row0 = (long long)w.b * p.nrows + (p.reverse ? p.nrows - 1 - s0 : s0);
    const int step = p.reverse ? -1 : 1;
#pragma unroll
    for (int a = 0; a < T::kArrays; ++a) {
        const ST* from = static_cast<const ST*>(src[a]) + ch;
#pragma unroll
        for (int j = 0; j < T::K; ++j) {
            const int sl = warp * T::K + j, r = p.reverse ? T::R - 1 - sl : sl;
            typename Two<ST>::Word* to = stage + (a * T::R + r) * 32 + lane;
            const ST* at = from + (row0 + (long long)j * step) * stride[a];
            const bool in = s0 + j < p.nrows;
            if (LOAD == kLoadWord) {
                if (sizeof(ST) == 4) {
                    if (in && have > 0) ptx::cp_async_4(to, at);
                    if (in && have > 1) ptx::cp_async_4(reinterpret_cast<char*>(to) + 4, at + 1);
                } else if (in && have > 1) {
                    ptx::cp_async_4(to, at);
                } else if (in && have > 0) {   // the last channel of an odd number
                    float v[2];
                    load_two<ST>(at, 0, have, v);
                    *to = Two<ST>::pack(v);
                }
            } else {
                float v[2] = {0.0f, 0.0f};
                if (in) load_two<ST>(at, 0, have, v);
                *to = Two<ST>::pack(v);
            }
        }
    }
}

// The last warp's side of the ring: tickets (drawn one ahead, so that the counter's latency is hidden), copies,
// and the block's decay parameters, which the other warps find beside the operands.
template <typename ST, bool DECAY, bool BWD>
struct GatedRing {
    using T = GatedTile<ST, DECAY, BWD>;
    const GatedParams& p;
    const GatedMaps& maps;
    char* stages;
    uint64_t* full;
    uint32_t* tickets;
    float (*rates)[kGatedChannels];
    int lane;
    uint32_t ahead, issued;
    bool drained;

    __device__ __forceinline__ void draw()
    {
        if (lane == 0) ahead = atomicAdd(p.header, 1u);
    }
    __device__ __forceinline__ void refill()
    {
        if (drained) return;
        const int s = (int)(issued % T::kStages);
        const uint32_t ticket = __shfl_sync(0xffffffffu, ahead, 0);
        if ((long long)ticket >= p.ntickets) {
            drained = true;
            if (lane == 0) {
                tickets[s] = 0xffffffffu;
                ptx::mbar_arrive(&full[s]);
            }
            return;
        }
        ++issued;
        const GatedWhere w = gated_where<BWD>(p, ticket);
        if (lane == 0) {
            // (operands first: the barrier completes when the arrival below has come as well)
            tickets[s] = ticket;
            const int row = p.reverse ? (int)(p.nrows - (long long)(w.k + 1) * T::R) : w.k * T::R;
            char* to = stages + s * T::kStageBytes;
            if (DECAY) ptx::mbar_expect_tx(&full[s], (uint32_t)T::kStageBytes);
            else ptx::mbar_arrive_expect_tx(&full[s], (uint32_t)T::kStageBytes);
            ptx::tma_load_3d(to, &maps.x, &full[s], w.dt * kGatedChannels, row, w.b);
            ptx::tma_load_3d(to + T::kArrayBytes, &maps.f, &full[s], w.dt * kGatedChannels, row, w.b);
            if (DECAY) ptx::tma_load_3d(to + 2 * T::kArrayBytes, &maps.i, &full[s], w.dt * kGatedChannels, row, w.b);
            if (BWD) ptx::tma_load_3d(to + (T::kArrays - 1) * T::kArrayBytes, &maps.dy, &full[s], w.dt * kGatedChannels, row, w.b);
        }
        draw();
        if (DECAY) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int ch = w.dt * kGatedChannels + v * 32 + lane;
                rates[s][v * 32 + lane] = ch < p.D ? p.scale * softplus(p.decay[ch]) : 0.0f;
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&full[s]);
        }
    }
};

// What both passes have in common: the pipeline of tiles around `body`, which calls `refill` behind its first
// barrier and returns false to stop (all threads alike).
template <typename ST, bool DECAY, bool BWD, int LOAD, typename Body>
__device__ __forceinline__ void gated_tiles(const GatedParams& p, const GatedMaps& maps, Body body)
{
    using T = GatedTile<ST, DECAY, BWD>;
    using Word = typename T::Word;
    extern __shared__ char gated_smem[];
    char* stages = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(gated_smem) + 127) & ~(uintptr_t)127);
    __shared__ __align__(8) uint64_t full[T::kStages];
    __shared__ uint32_t tickets[T::kStages];
    __shared__ float rates[T::kStages][kGatedChannels];
    __shared__ int abort_flag;
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (LOAD == kLoadTma) {
        if (tid == 0) {
#pragma unroll
            for (int s = 0; s < T::kStages; ++s) {
                ptx::mbar_init(&full[s], 1u);
                tickets[s] = 0u;
            }
            abort_flag = 0;
            ptx::fence_mbar_init();
        }
        __syncthreads();
        ptx::grid_dependency_wait();
        const uint32_t epoch = read_epoch(p.header);
        GatedRing<ST, DECAY, BWD> ring{p, maps, stages, full, tickets, rates, lane, 0u, 0u, false};
        const bool issuer = warp == kGatedWarps - 1;
        if (issuer) {
            ring.draw();
            for (int s = 0; s < T::kStages - (BWD ? 1 : 0); ++s) ring.refill();
        }
        uint32_t it = 0;
        bool gave_up = false;
        for (;; ++it) {
            const int s = (int)(it % T::kStages);
            if (!ptx::mbar_wait_bounded(&full[s], (it / T::kStages) & 1u, p.wait_budget)) {
                // keeps step with the other warps up to the next barrier, where all of them see the flag
                *(volatile int*)&abort_flag = 1;
                atomicOr(p.header + 1, kStatusCopyTimeout);
            }
            const uint32_t ticket = *(volatile uint32_t*)&tickets[s];
            if (ticket == 0xffffffffu) break;
            if (!body(gated_where<BWD>(p, ticket), ticket, it, epoch, reinterpret_cast<const Word*>(stages + s * T::kStageBytes), rates[s],
                      [&] { if (issuer) ring.refill(); }, (volatile int*)&abort_flag)) {
                gave_up = true;
                break;
            }
        }
        if (issuer) {
            // no copy may land in this CTA's shared memory after it has left
            if (gave_up)
                for (uint32_t i = it; i < ring.issued; ++i) (void)ptx::mbar_wait_bounded(&full[i % T::kStages], (i / T::kStages) & 1u, p.wait_budget);
            if (lane == 0) finish_launch(p.header, epoch);
        }
        return;
    }
    ptx::grid_dependency_wait();
    const uint32_t epoch = read_epoch(p.header);
    if (tid == 0) {
        tickets[0] = atomicAdd(p.header, 1u);
        abort_flag = 0;
    }
    __syncthreads();
    uint32_t ticket = tickets[0];
    if ((long long)ticket < p.ntickets) gated_fetch<ST, DECAY, BWD, LOAD>(p, gated_where<BWD>(p, ticket), reinterpret_cast<Word*>(stages), warp, lane);
    ptx::cp_async_commit();
    for (uint32_t it = 0; (long long)ticket < p.ntickets; ++it) {
        if (tid == 0) tickets[(it + 1) & 1] = atomicAdd(p.header, 1u);
        const GatedWhere w = gated_where<BWD>(p, ticket);
        if (DECAY && tid < kGatedChannels) {
            const int ch = w.dt * kGatedChannels + tid;
            rates[it & 1][tid] = ch < p.D ? p.scale * softplus(p.decay[ch]) : 0.0f;
        }
        __syncthreads();
        const uint32_t next = tickets[(it + 1) & 1];
        if ((long long)next < p.ntickets)
            gated_fetch<ST, DECAY, BWD, LOAD>(p, gated_where<BWD>(p, next), reinterpret_cast<Word*>(stages + ((it + 1) & 1) * T::kStageBytes), warp, lane);
        ptx::cp_async_commit();
        ptx::cp_async_wait_group<1>();
        body(w, ticket, it, epoch, reinterpret_cast<const Word*>(stages + (it & 1) * T::kStageBytes), rates[it & 1], [] {}, (volatile int*)&abort_flag);
        ticket = next;
    }
    if (tid == 0) finish_launch(p.header, epoch);
}

// ---- forward ------------------------------------------------------------------------------------------
template <typename ST, bool DECAY, int LOAD>
__global__ void __launch_bounds__(kGatedThreads, 2)
    gated_fwd_kernel(const GatedParams p, const __grid_constant__ GatedMaps maps)
{
    using T = GatedTile<ST, DECAY, false>;
    constexpr int K = T::K, R = T::R;
    __shared__ float4 runs[2][kGatedWarps][32];      // (Y, P) of both channels of every thread
    __shared__ float entering[kGatedChannels];
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;

    gated_tiles<ST, DECAY, false, LOAD>(p, maps, [&](const GatedWhere& w, uint32_t ticket, uint32_t it, uint32_t epoch,
                                                     const typename T::Word* stage, const float* rates, auto refill, volatile int* abort_flag) {
        const int ch = w.dt * kGatedChannels + 2 * lane;
        const int have = p.D - ch;
        const long long s0 = (long long)w.k * R + warp * K;
        TileDesc* desc = p.desc + ((long long)ticket * kGatedChannels + tid);
        uint4 seen = make_uint4(0u, 0u, 0u, 0u);
        if (tid < kGatedChannels && w.g > 0) seen = desc_load(desc - (long long)p.units * kGatedChannels, epoch);
        const GatedRun run = gated_run<K>(p, w.b, s0, lane);
        const typename T::Word* words = stage + (p.reverse ? R - 1 - warp * K : warp * K) * 32 + lane;
        const int wstep = p.reverse ? -32 : 32;

        float a[K][2], u[K][2];
        auto gates = [&](auto small) {
            float rate[2] = {0.0f, 0.0f};
            if (DECAY) rate[0] = rates[2 * lane], rate[1] = rates[2 * lane + 1];
#pragma unroll
            for (int j = 0; j < K; ++j) {
                float xv[2], fv[2], iv[2];
                Two<ST>::unpack(words[j * wstep], xv);
                Two<ST>::unpack(words[j * wstep + R * 32], fv);
                if (DECAY) Two<ST>::unpack(words[j * wstep + 2 * R * 32], iv);
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    if (DECAY) {
                        float b2;
                        decay_factors<T::kFast, decltype(small)::value>(rate[v] * logistic<T::kFast>(fv[v]), a[j][v], b2);
                        u[j][v] = approx_sqrt(b2) * (logistic<T::kFast>(iv[v]) * xv[v]);
                    } else {
                        float n;
                        logistic_pair<T::kFast>(fv[v], a[j][v], n);
                        u[j][v] = n * xv[v];
                    }
                }
            }
        };
        // a slow decay (rate below 1/4 in all of the warp's channels) never needs the exponential
        if (DECAY && !__all_sync(0xffffffffu, rates[2 * lane] < 0.25f && rates[2 * lane + 1] < 0.25f)) gates(std::false_type{});
        else gates(std::true_type{});
        if (run.cut) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if (!(run.valid >> j & 1u)) u[j][0] = u[j][1] = 0.0f;
                if (p.h0 && (run.start >> j & 1u)) {
                    const int q = __shfl_sync(0xffffffffu, run.seq, j);
                    float hv[2];
                    load_two<float>(p.h0, (long long)q * p.D + ch, have, hv);
#pragma unroll
                    for (int v = 0; v < 2; ++v) u[j][v] = fmaf(a[j][v], hv[v], u[j][v]);
                }
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
        if (LOAD == kLoadTma && *abort_flag) return false;
        refill();

        if (tid < kGatedChannels) {
            Pair total = pair_identity();
#pragma unroll
            for (int i = 0; i < kGatedWarps; ++i) {
                const float2 r = reinterpret_cast<const float2*>(&set[i][tid >> 1])[tid & 1];
                total = join(total, Pair{r.x, r.y});
            }
            entering[tid] = gated_link(p, desc, seen, w.g, total, epoch);
        }
        Pair before[2] = {pair_identity(), pair_identity()};
        for (int i = 0; i < warp; ++i) {
            const float4 r = set[i][lane];
            before[0] = join(before[0], Pair{r.x, r.y});
            before[1] = join(before[1], Pair{r.z, r.w});
        }
        __syncthreads();
        float h[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) h[v] = enter(entering[2 * lane + v], before[v]);
        if (p.ckpt && s0 % kGatedCheckpoint == 0 && s0 < p.nrows)
            store_two<float>(p.ckpt, ((long long)w.b * p.nck + s0 / kGatedCheckpoint) * p.D + ch, have, h);
        const bool pair = (LOAD == kLoadTma || p.pair) && have > 1;
        const long long row0 = (long long)w.b * p.nrows + (p.reverse ? p.nrows - 1 - s0 : s0);
        ST* y = static_cast<ST*>(p.y) + row0 * p.D + ch;
        const long long ystep = p.reverse ? -(long long)p.D : p.D;
        const int rows = (int)min((long long)K, p.nrows - s0);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (j >= rows) break;
#pragma unroll
            for (int v = 0; v < 2; ++v) h[v] = (run.cut >> j & 1u) ? u[j][v] : fmaf(a[j][v], h[v], u[j][v]);
            store_two<ST>(y, j * ystep, have, h, pair);
            if (p.hT && (run.end >> j & 1u)) {
                const int q = __shfl_sync(0xffffffffu, run.seq, j);
                store_two<float>(p.hT, (long long)q * p.D + ch, have, h);
            }
        }
        return true;
    });
}

// ---- backward -----------------------------------------------------------------------------------------
// Between the two halves of a tile a thread keeps a, b, s(i) and the state in front of each of its elements;
// x, dy and the logits stay in shared memory and what else is needed is evaluated again from them (two
// exponentials cheaper than the registers: keeping everything leaves one CTA per SM).
template <typename ST, bool DECAY, int LOAD>
__global__ void __launch_bounds__(kGatedThreads, 2)
    gated_bwd_kernel(const GatedParams p, const __grid_constant__ GatedMaps maps)
{
    using T = GatedTile<ST, DECAY, true>;
    constexpr int K = T::K, R = T::R;
    static_assert(R == kGatedCheckpoint, "one checkpoint per tile");
    constexpr int kDy = (T::kArrays - 1) * R * 32;
    __shared__ float4 runs[2][kGatedWarps][32];      // (Y, P) of both channels, forward direction
    __shared__ float2 back[2][kGatedWarps][32];      // Y of both channels, adjoint direction (same P)
    __shared__ float entering[kGatedChannels];
    __shared__ float2 dsum[kGatedWarps][32];
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;

    gated_tiles<ST, DECAY, true, LOAD>(p, maps, [&](const GatedWhere& w, uint32_t ticket, uint32_t it, uint32_t epoch,
                                                    const typename T::Word* stage, const float* rates, auto refill, volatile int* abort_flag) {
        const int ch = w.dt * kGatedChannels + 2 * lane;
        const int have = p.D - ch;
        const long long s0 = (long long)w.k * R + warp * K;
        TileDesc* desc = p.desc + ((long long)ticket * kGatedChannels + tid);
        uint4 seen = make_uint4(0u, 0u, 0u, 0u);
        if (tid < kGatedChannels && w.g > 0) seen = desc_load(desc - (long long)p.units * kGatedChannels, epoch);
        float h[2];
        load_two<float>(p.ckpt, ((long long)w.b * p.nck + w.k) * p.D + ch, have, h);
        const GatedRun run = gated_run<K>(p, w.b, s0, lane);
        const typename T::Word* words = stage + (p.reverse ? R - 1 - warp * K : warp * K) * 32 + lane;
        const int wstep = p.reverse ? -32 : 32;
        float rate[2] = {0.0f, 0.0f};
        if (DECAY) rate[0] = rates[2 * lane], rate[1] = rates[2 * lane + 1];

        // add: b u, later the state in front of the element
        float a[K][2], bb[K][2], gi[K][2], add[K][2];
        auto gates = [&](auto small) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                float xv[2], fv[2], iv[2];
                Two<ST>::unpack(words[j * wstep], xv);
                Two<ST>::unpack(words[j * wstep + R * 32], fv);
                if (DECAY) Two<ST>::unpack(words[j * wstep + 2 * R * 32], iv);
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    if (DECAY) {
                        float b2;
                        decay_factors<T::kFast, decltype(small)::value>(rate[v] * logistic<T::kFast>(fv[v]), a[j][v], b2);
                        bb[j][v] = approx_sqrt(b2);
                        gi[j][v] = logistic<T::kFast>(iv[v]);
                        add[j][v] = bb[j][v] * (gi[j][v] * xv[v]);
                    } else {
                        logistic_pair<T::kFast>(fv[v], a[j][v], bb[j][v]);
                        add[j][v] = bb[j][v] * xv[v];
                    }
                }
            }
        };
        if (DECAY && !__all_sync(0xffffffffu, rate[0] < 0.25f && rate[1] < 0.25f)) gates(std::false_type{});
        else gates(std::true_type{});
        // initial states and final gradients of sequences that start or end in this run
        auto state_of = [&](const float* states, uint32_t mask, int j, float* v) {
            v[0] = v[1] = 0.0f;
            if (states && (mask >> j & 1u)) {
                const int q = __shfl_sync(0xffffffffu, run.seq, j);
                load_two<float>(states, (long long)q * p.D + ch, have, v);
            }
        };
        auto gradient = [&](int j, float* v) {
            Two<ST>::unpack(words[j * wstep + kDy], v);
            if (p.dhT && (run.end >> j & 1u)) {
                float e[2];
                state_of(p.dhT, run.end, j, e);
                v[0] += e[0];
                v[1] += e[1];
            }
        };
        if (~run.valid & ((1u << K) - 1u)) {
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (!(run.valid >> j & 1u)) {
                    a[j][0] = a[j][1] = bb[j][0] = bb[j][1] = add[j][0] = add[j][1] = 0.0f;
                    if (DECAY) gi[j][0] = gi[j][1] = 0.0f;
                }
        }
        Pair agg[2] = {pair_identity(), pair_identity()};
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const bool cut = run.cut >> j & 1u;
            float start[2] = {0.0f, 0.0f};
            if (cut) state_of(p.h0, run.start, j, start);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                agg[v].y = fmaf(a[j][v], cut ? start[v] : agg[v].y, add[j][v]);
                agg[v].p = cut ? kCut : agg[v].p * a[j][v];
            }
        }
        float q[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = K - 1; j >= 0; --j) {
            float dy[2];
            gradient(j, dy);
#pragma unroll
            for (int v = 0; v < 2; ++v) q[v] = (run.cut >> j & 1u) ? 0.0f : a[j][v] * (dy[v] + q[v]);
        }
        float4(*set)[32] = runs[it & 1];
        float2(*bset)[32] = back[it & 1];
        set[warp][lane] = make_float4(agg[0].y, agg[0].p, agg[1].y, agg[1].p);
        bset[warp][lane] = make_float2(q[0], q[1]);
        __syncthreads();
        if (LOAD == kLoadTma && *abort_flag) return false;
        refill();

        if (tid < kGatedChannels) {
            Pair total = pair_identity();
#pragma unroll
            for (int i = kGatedWarps - 1; i >= 0; --i) {
                const float P = reinterpret_cast<const float2*>(&set[i][tid >> 1])[tid & 1].y;
                const float Y = reinterpret_cast<const float*>(&bset[i][tid >> 1])[tid & 1];
                total = join(total, Pair{Y, P});
            }
            entering[tid] = gated_link(p, desc, seen, w.g, total, epoch);
        }
        // the state that enters this run, from the checkpoint
        for (int i = 0; i < warp; ++i) {
            const float4 r = set[i][lane];
            h[0] = enter(h[0], Pair{r.x, r.y});
            h[1] = enter(h[1], Pair{r.z, r.w});
        }
        Pair after[2] = {pair_identity(), pair_identity()};
        for (int i = kGatedWarps - 1; i > warp; --i) {
            const float4 r = set[i][lane];
            const float2 y = bset[i][lane];
            after[0] = join(after[0], Pair{y.x, r.y});
            after[1] = join(after[1], Pair{y.y, r.w});
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (run.cut >> j & 1u) state_of(p.h0, run.start, j, h);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float before = h[v];
                h[v] = fmaf(a[j][v], before, add[j][v]);
                add[j][v] = before;
            }
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < 2; ++v) q[v] = enter(entering[2 * lane + v], after[v]);
        float dl[2] = {0.0f, 0.0f};
        const bool pair = (LOAD == kLoadTma || p.pair) && have > 1;
        const long long row0 = (long long)w.b * p.nrows + (p.reverse ? p.nrows - 1 - s0 : s0);
        const long long at0 = row0 * p.D + ch, astep = p.reverse ? -(long long)p.D : p.D;
#pragma unroll
        for (int j = K - 1; j >= 0; --j) {
            const bool cut = run.cut >> j & 1u, ok = run.valid >> j & 1u;
            float xv[2], fv[2], dy[2], odx[2], odf[2], odi[2], oq[2];
            Two<ST>::unpack(words[j * wstep], xv);
            gradient(j, dy);
            if (DECAY) Two<ST>::unpack(words[j * wstep + R * 32], fv);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float grad = dy[v] + q[v], b = bb[j][v], hp = add[j][v];
                oq[v] = a[j][v] * grad;
                q[v] = cut ? 0.0f : oq[v];
                const float wb = grad * b;
                if (DECAY) {
                    float s, n;
                    logistic_pair<T::kFast>(fv[v], s, n);
                    const float u = gi[j][v] * xv[v];
                    const float slope = b > 0.0f ? a[j][v] * approx_rcp(b) : 0.0f;
                    // d(log a) * log a, with log a = -rate s
                    const float t = oq[v] * fmaf(-u, slope, hp) * (-rate[v] * s);
                    if (ok) dl[v] += t;
                    odx[v] = wb * gi[j][v];
                    odi[v] = wb * (u * (1.0f - gi[j][v]));
                    odf[v] = t * n;
                } else {
                    odx[v] = wb;
                    odf[v] = oq[v] * b * (hp - xv[v]);
                }
            }
            if (s0 + j < p.nrows) {
                if (!ok) odx[0] = odx[1] = odf[0] = odf[1] = odi[0] = odi[1] = 0.0f;
                store_two<ST>(p.dx, at0 + j * astep, have, odx, pair);
                store_two<ST>(p.df, at0 + j * astep, have, odf, pair);
                if (DECAY) store_two<ST>(p.di, at0 + j * astep, have, odi, pair);
                if (p.dh0 && (run.start >> j & 1u)) {
                    const int n = __shfl_sync(0xffffffffu, run.seq, j);
                    store_two<float>(p.dh0, (long long)n * p.D + ch, have, oq);
                }
            }
        }
        if (DECAY) {
            dsum[warp][lane] = make_float2(dl[0], dl[1]);
            __syncthreads();
            if (tid < kGatedChannels && w.dt * kGatedChannels + tid < p.D) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < kGatedWarps; ++i) s += reinterpret_cast<const float*>(&dsum[i][tid >> 1])[tid & 1];
                p.dlam[((long long)w.b * p.nk + w.k) * p.D + w.dt * kGatedChannels + tid] = s;
            }
        }
        return true;
    });
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
        out[ch] = (float)s * (sp > 0.0f ? logistic<false>(L) / sp : 1.0f);
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
    constexpr bool kFast = sizeof(ST) == 2;
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

    float h[2] = {0.0f, 0.0f}, rate[2] = {0.0f, 0.0f};
    load_two<float>(p.state, slot * p.sstate + ch, have, h);
    if (DECAY) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
            if (v < have) rate[v] = p.scale * softplus(p.decay[ch + v]);
    }
    while (true) {
        float xv[2], fv[2], iv[2];
        load_two<ST>(p.x, (long long)row * p.sx + ch, have, xv);
        load_two<ST>(p.f, (long long)row * p.sf + ch, have, fv);
        if (DECAY) load_two<ST>(p.ig, (long long)row * p.si + ch, have, iv);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            if (DECAY) {
                float a, b2;
                decay_factors<kFast, false>(rate[v] * logistic<kFast>(fv[v]), a, b2);
                h[v] = fmaf(a, h[v], approx_sqrt(b2) * (logistic<kFast>(iv[v]) * xv[v]));
            } else {
                float s, n;
                logistic_pair<kFast>(fv[v], s, n);
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

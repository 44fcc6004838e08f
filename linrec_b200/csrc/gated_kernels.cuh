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
// A tile is 64 channels x R positions for one CTA of four or eight warps: a lane owns two adjacent channels, a
// warp K consecutive positions, kept in registers as (a, b u) pairs.  Each thread folds its run into a (P, Y)
// pair, the warps' runs meet in shared memory, and the tile is linked to its predecessor along the axis: by the CTA
// itself within a job of tiles, by the cluster's shared memory, or by decoupled look-back (one 16-byte
// descriptor per channel and job; tickets are handed out position-major, so the predecessor is `units`
// tickets older and a wait is only ever for a ticket that a running CTA holds).  The runs are then walked
// again from the true state.  Reads and writes every element once.
//
// The cut is carried as a multiplier of minus zero, and it selects rather than multiplies: 0 * NaN would let one
// sequence's infinities into its neighbour.  Within a run it is set from the positions of the cuts; from run to run
// products of multipliers (all >= 0) keep it, but for NaN ones: the run they are in has a NaN sum beside them, so that
// they reach no more than their own sequence.
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

constexpr int kGatedChannels = 64;      // channels per tile: 32 lanes x 2
constexpr int kGatedCheckpoint = 64;    // positions between two checkpoints

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
    float* dlam;                        // [nb * jobs][D]: sums of d(log a) log a over a job (backward, decay form)
    const void* cu;                     // nseq + 1 offsets, or null: sequences of `seqlen` rows
    int cu64;
    int nseq;
    long long seqlen;
    long long nrows;                    // rows per axis
    int nb;                             // axes (batch entries scanned side by side)
    int D, dtiles, units;               // units = nb * dtiles
    int nk, nck;                        // tiles, checkpoints per axis
    int cluster;                        // kLoadCluster: CTAs that share a column
    int tiles_per_job, jobs;            // a ticket is a job: consecutive tiles of one column; jobs per column
    long long ntickets;                 // jobs * units
    int reverse;
    uint32_t* header;
    TileDesc* desc;                     // [jobs][units][64]
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

// The same for two channels: a and b^2.
template <bool FAST, bool SMALL>
__device__ __forceinline__ void decay_factors2(F2 y, F2& a, F2& b2)
{
    if (SMALL) {
        F2 s = f2_fma(y, f2(-1.0f / 720.0f), f2(1.0f / 120.0f));
        s = f2_fma(y, s, f2(-1.0f / 24.0f));
        s = f2_fma(y, s, f2(1.0f / 6.0f));
        s = f2_fma(y, s, f2(-0.5f));
        const F2 d = f2_mul(y, f2_fma(y, s, f2(1.0f)));
        a = f2_fma(d, f2(-1.0f), f2(1.0f));
        b2 = f2_fma(d, a, d);
    } else {
        const float2 w = f2_get(y);
        float a0, a1, b0, b1;
        decay_factors<FAST, false>(w.x, a0, b0);
        decay_factors<FAST, false>(w.y, a1, b1);
        a = f2(a0, a1);
        b2 = f2(b0, b1);
    }
}
constexpr float kSmallestNormal = 1.17549435e-38f;
__device__ __forceinline__ F2 root2(F2 v)
{
    const float2 w = f2_get(v);
    return f2(approx_sqrt(w.x), approx_sqrt(w.y));
}
// b s(i).  Fast: with d = 1 + e^-i it is b^2 / sqrt(b^2 d^2), one special function for a root and a reciprocal
// (they bound the forward pass).  A gate that is shut gives exactly nothing: so does a b^2 below the smallest normal
// number, which the root would take for zero (its reciprocal is infinite there, and d >= 1 keeps all larger ones out of
// that range), as the root of the other passes does.  A NaN is neither and goes through.  An input gate below e^-44 counts
// as shut as well: b^2 d^2 overflows.
template <bool FAST>
__device__ __forceinline__ F2 gated_factor2(F2 b2, F2 i)
{
    if (FAST) {
        const float2 t = f2_get(f2_mul(i, f2(-1.44269504f)));
        const F2 d = f2_add(f2(approx_exp2(t.x), approx_exp2(t.y)), f2(1.0f));
        const float2 q = f2_get(b2), r = f2_get(f2_mul(f2_mul(b2, d), d));
        const float2 g = f2_get(f2_mul(b2, f2(approx_rsqrt(r.x), approx_rsqrt(r.y))));
        return f2(q.x < kSmallestNormal ? 0.0f : g.x, q.y < kSmallestNormal ? 0.0f : g.y);
    }
    return f2_mul(root2(b2), logistic2<false>(i));
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

// Is there a cut among a run's first j + 1 positions?  Their product is the cut then, whatever multipliers follow it: minus
// zero times NaN would be NaN, and would let the multipliers of a sequence into the adjoint of the one before it.
__device__ __forceinline__ bool gated_is_cut(const GatedRun& r, int j) { return r.cut & ((2u << j) - 1u); }

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
    r.cut = (r.start | ~r.valid) & ((1u << K) - 1u);
    r.seq = q;
    return r;
}

// ---- tiles and jobs ------------------------------------------------------------------------------------
// One tile: `k` along the axis in forward scan order (< 0: no more tiles), its job in the order of this pass,
// axis, channel block; `first` and `last` of its job.
struct GatedWhere {
    int k, job, b, dt;
    static constexpr int kFirst = 1 << 30, kLast = 1 << 29;
    __device__ __forceinline__ int block() const { return dt & (kLast - 1); }
    __device__ __forceinline__ bool first() const { return dt & kFirst; }
    __device__ __forceinline__ bool last() const { return dt & kLast; }
};
template <bool BWD>
__device__ __forceinline__ GatedWhere gated_where(const GatedParams& p, uint32_t ticket, int t)
{
    GatedWhere w;
    w.job = (int)(ticket / (uint32_t)p.units);
    const int unit = (int)(ticket - (uint32_t)w.job * (uint32_t)p.units);
    const int g = w.job * p.tiles_per_job + t;
    w.b = unit / p.dtiles;
    w.dt = unit - w.b * p.dtiles;
    if (t == 0) w.dt |= GatedWhere::kFirst;
    if (t + 1 == p.tiles_per_job || g + 1 == p.nk) w.dt |= GatedWhere::kLast;
    w.k = BWD ? p.nk - 1 - g : g;
    return w;
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
// Descriptors are requested a window at a time, and a window with holes again as a whole: waiting for one
// descriptor after the other costs a round trip for each.  The wait is bounded; on expiry the status word is flagged and nothing enters.
__device__ __forceinline__ float gated_lookback(const TileDesc* d, long long stride, int k, uint32_t epoch, long long budget, uint32_t* status)
{
    constexpr int W = 8;
    uint4 w[W];
    int dist = 0;          // tiles k - 1, ..., k - dist are known to hold aggregates
    const long long t0 = clock64();
    while (true) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if (dist + i >= k) w[i] = make_uint4(0u, 0u, 2u, 0u);
            else w[i] = desc_load(d - (long long)(dist + i) * stride, epoch);
        }
        int here = 0;              // aggregates in front of the first inclusive value or hole
        bool found = false, hole = false;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            // (a descriptor of this epoch that another job of the launch wrote cannot be: each has its own place)
            if (found || hole) continue;
            if (w[i].z == 0u) hole = true;
            else if (w[i].z == 2u) found = true;
            else ++here;
        }
        if (found && dist == 0) {
            float v = 0.0f;
#pragma unroll
            for (int i = W - 1; i >= 0; --i) {
                if (i == here) v = __uint_as_float(w[i].x);
                else if (i < here) v = enter(v, desc_pair(w[i]));
            }
            return v;
        }
        if (found) {
            dist += here;
            break;
        }
        if (!hole) {
            dist += W;
        } else if (clock64() - t0 > budget) {
            atomicOr(status, kStatusLookbackTimeout);
            return 0.0f;
        } else {
            __nanosleep(100);
        }
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

// Run by 64 threads, one channel each, in the first tile of a job: returns the value that enters it.  `d` is
// the job's descriptor, `seen` what its predecessor's held a while ago.  Jobs of one tile publish their total
// before they look back (decoupled look-back); a longer job, of which the first tile says nothing about the
// whole, waits for its predecessor, which was handed out `units` tickets earlier.
__device__ __forceinline__ float gated_link(const GatedParams& p, TileDesc* d, uint4 seen, int job, Pair total, uint32_t epoch, bool& published)
{
    published = false;
    if (job == 0) return 0.0f;
    if (seen.z == 2u && seen.w == (uint32_t)(job - 1)) return __uint_as_float(seen.x);
    const long long stride = (long long)p.units * kGatedChannels;
    if (p.tiles_per_job > 1) {
        seen.z = 0u;
        return gated_await(d - stride, job - 1, seen, epoch, p.wait_budget, p.header + 1) ? __uint_as_float(seen.x) : 0.0f;
    }
    if (job + 1 < p.jobs) {
        // a total that forgets what enters (a sequence starts in the tile) is final already
        published = is_cut(total.p);
        col_publish(d, total.y, total.p, published ? 2u : 1u, epoch, (uint32_t)job);
    }
    return gated_lookback(d - stride, stride, job, epoch, p.wait_budget, p.header + 1);
}

// The 64 threads' part of every tile: what enters it (beside `now`, where the first tile of a job finds it only
// behind the next barrier) and what leaves it, for the next tile and the next job.
__device__ __forceinline__ void gated_carry(const GatedParams& p, const GatedWhere& w, TileDesc* d, uint4 seen, Pair total, uint32_t epoch,
                                            float* now, float* then)
{
    float in;
    bool published = false;
    if (w.first()) *now = in = gated_link(p, d, seen, w.job, total, epoch, published);
    else in = *now;
    const float out = enter(in, total);
    *then = out;
    if (w.last() && !published && w.job + 1 < p.jobs) col_publish(d, out, 0.0f, 2u, epoch, (uint32_t)w.job);
}

// ---- the tile ---------------------------------------------------------------------------------------------
// How operands reach shared memory, where every thread finds the words of its own two channels and K
// positions:
//   kLoadTma    one bulk-tensor copy per operand through a ring of stages, issued by a warp of its own (rows on
//               16-byte boundaries)
//   kLoadWord   32-bit elements: 4-byte asynchronous copies, every thread its own words, one tile ahead
//   kLoadAny    16-bit elements: plain loads by the thread, stored to the same place
//   kLoadCluster  as kLoadTma, for fewer columns than SMs: the CTAs of a cluster take consecutive tiles of ONE column
//               and tell one another their totals through shared memory, so that a column's carry never
//               leaves its cluster and nobody looks back through global memory
constexpr int kLoadTma = 0, kLoadWord = 1, kLoadAny = 2, kLoadCluster = 3;
__host__ __device__ constexpr bool gated_bulk(int load) { return load == kLoadTma || load == kLoadCluster; }
constexpr int kGatedClusterMost = 8;

// Two shapes of a CTA.  SHAPE 0: four warps, several CTAs per SM, whose phases (gates, which the special
// function unit bounds, and the exchange between warps, which latency bounds) overlap each other's.  SHAPE 1:
// eight warps and longer tiles, one CTA per SM: half as many tiles wait for one another along a column, which
// counts when there are few columns, and it is the shape that fits 32-bit operands.
// Measured when both linked tiles by look-back and jobs alone, forward / backward us, 16-bit decay form:
// (8, 4096, 4096), 512 columns: 247 / 614 and 292 / 689; (1, 32768, 2048), 32 columns: 269 / 735 and 240 / 598.
// The sides that are taken now measure 228 / 559 and, in clusters, 170 / 427.
template <typename ST, bool DECAY, bool BWD, int SHAPE>
struct GatedTile {
    static constexpr bool kFast = sizeof(ST) == 2;                     // 16-bit results: fast exponentials will do
    static constexpr int W = SHAPE ? 8 : 4;                            // warps
    static constexpr int K = SHAPE && BWD ? 8 : 16;                    // positions per thread
    static constexpr int R = K * W;                                    // positions per tile
    static constexpr int kCtas = SHAPE ? 1 : BWD ? 2 : 3;              // per SM, for the register budget
    static_assert(R % kGatedCheckpoint == 0, "workspaces hold descriptors for tiles of that many positions, the shortest");
    static constexpr int kArrays = (DECAY ? 3 : 2) + (BWD ? 1 : 0);    // x, f(, i)(, dy)
    static constexpr int kArrayBytes = R * kGatedChannels * (int)sizeof(ST);
    static constexpr int kStageBytes = kArrays * kArrayBytes;
    // forward: a stage is free once the gates are in registers; backward: only when the next tile has begun
    static constexpr int kStages = SHAPE && BWD ? 3 : 2;
    static constexpr int kDynSmem = kStages * kStageBytes;
    using Word = typename Two<ST>::Word;
    static constexpr int threads(int load) { return (W + (gated_bulk(load) ? 1 : 0)) * 32; }
};

// A barrier of the warps that own positions.
template <int W>
__device__ __forceinline__ void gated_sync()
{
    asm volatile("bar.sync 1, %0;" ::"n"(W * 32) : "memory");
}

// The totals of a cluster's turn: every CTA sends its 64 channels' (Y, P) to all of the cluster, each transfer
// counted on the receiver's barrier.  Two sets take turns: a CTA sends its next but one total only after it
// has received this CTA's next one, which is sent after this one's set has been read.
struct GatedNoExchange {
    __device__ __forceinline__ void open() {}
};
struct GatedExchange {
    float2 totals[2][kGatedClusterMost][kGatedChannels];
    uint64_t arrived[2];
    int failed;      // a wait ran out: this launch's numbers are void, and it waits for nobody any more
    __device__ __forceinline__ void open()
    {
        failed = 0;
        ptx::mbar_init(&arrived[0], 1u);
        ptx::mbar_init(&arrived[1], 1u);
    }
    // Run by 64 threads, one channel each: returns what enters this CTA's tile, `carry` is what entered the turn and
    // becomes what enters the next.
    __device__ __forceinline__ float turn(const GatedParams& p, uint32_t n, int tid, Pair total, float& carry)
    {
        float in = carry;
        if (p.cluster == 1) {
            carry = enter(carry, total);
            return in;
        }
        const int set = (int)(n & 1u), rank = (int)(blockIdx.x % (unsigned)p.cluster);
        if (tid == 0) ptx::mbar_arrive_expect_tx(&arrived[set], (uint32_t)(p.cluster * kGatedChannels * sizeof(float2)));
        for (int c = 0; c < p.cluster; ++c) ptx::st_async_f32x2(&totals[set][rank][tid], &arrived[set], c, total.y, total.p);
        if (!*(volatile int*)&failed && !ptx::mbar_wait_bounded_cluster(&arrived[set], (n >> 1) & 1u, p.wait_budget)) {
            failed = 1;
            atomicOr(p.header + 1, kStatusLookbackTimeout);
        }
        for (int c = 0; c < p.cluster; ++c) {
            const float2 v = totals[set][c][tid];
            if (c == rank) in = carry;
            carry = enter(carry, Pair{v.x, v.y});
        }
        return in;
    }
};

template <int W>
__device__ __forceinline__ bool gated_any(const int* flags)
{
    int any = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) any |= flags[i];
    return any != 0;
}
__device__ __forceinline__ F2 gated_enter(float2 in, F2 Y, F2 P, bool cut)
{
    if (!cut) return f2_fma(f2(in.x, in.y), P, Y);
    const float2 y = f2_get(Y), p = f2_get(P);
    return f2(enter(in.x, Pair{y.x, p.x}), enter(in.y, Pair{y.y, p.y}));
}

struct GatedMaps {
    CUtensorMap x, f, i, dy;
};

// A cluster's turn t in a column: its CTA `rank` has tile t * cluster + rank (k = nk: none, the column is at its end).
template <bool BWD>
__device__ __forceinline__ GatedWhere gated_turn(const GatedParams& p, uint32_t column, int t, int rank)
{
    GatedWhere w;
    w.job = 0;
    w.b = (int)column / p.dtiles;
    w.dt = (int)column - w.b * p.dtiles;
    const int g = t * p.cluster + rank;
    w.k = g >= p.nk ? p.nk : BWD ? p.nk - 1 - g : g;
    if (t == 0) w.dt |= GatedWhere::kFirst;
    if ((t + 1) * p.cluster >= p.nk) w.dt |= GatedWhere::kLast;
    return w;
}

// A thread's own words of one tile, by asynchronous 4-byte copies or plain loads.
template <typename ST, bool DECAY, bool BWD, int SHAPE, int LOAD>
__device__ __forceinline__ void gated_fetch(const GatedParams& p, const GatedWhere& w, typename Two<ST>::Word* stage, int warp, int lane)
{
    using T = GatedTile<ST, DECAY, BWD, SHAPE>;
    const void* src[4] = {p.x, p.f, DECAY ? p.ig : p.dy, p.dy};
    const long long stride[4] = {p.sx, p.sf, DECAY ? p.si : p.sdy, p.sdy};
    const int ch = w.block() * kGatedChannels + 2 * lane, have = p.D - ch;
    const long long s0 = (long long)w.k * T::R + warp * T::K;
    const long long row0 = (long long)w.b * p.nrows + (p.reverse ? p.nrows - 1 - s0 : s0);
    const int step = p.reverse ? -1 : 1;
#pragma unroll
    for (int a = 0; a < T::kArrays; ++a) {
        const ST* from = static_cast<const ST*>(src[a]) + ch;
        auto place = [&](int j) {
            const int sl = warp * T::K + j, r = p.reverse ? T::R - 1 - sl : sl;
            return stage + (a * T::R + r) * 32 + lane;
        };
        auto at = [&](int j) { return from + (row0 + (long long)j * step) * stride[a]; };
        if (LOAD == kLoadWord) {
#pragma unroll
            for (int j = 0; j < T::K; ++j) {
                const bool in = s0 + j < p.nrows;
                typename Two<ST>::Word* to = place(j);
                if (in && have > 0) ptx::cp_async_4(to, at(j));
                if (in && have > 1) ptx::cp_async_4(reinterpret_cast<char*>(to) + 4, at(j) + 1);
            }
        } else {
            // eight rows at a time: all of their loads, then all of their stores
#pragma unroll
            for (int j0 = 0; j0 < T::K; j0 += 8) {
                ST v[8][2];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool in = s0 + j0 + j < p.nrows;
                    v[j][0] = v[j][1] = from_f32<ST>(0.0f);
                    if (in && have > 0) v[j][0] = __ldg(at(j0 + j));
                    if (in && have > 1) v[j][1] = __ldg(at(j0 + j) + 1);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float f[2] = {to_f32<ST>(v[j][0]), to_f32<ST>(v[j][1])};
                    *place(j0 + j) = Two<ST>::pack(f);
                }
            }
        }
    }
}

// What GatedRun says, for all positions of a tile, found by the warp that issues the copies (a search through the
// offsets is 1600 cycles of round trips, which the other warps would all stand still for) and left beside them.
// Used in clusters, where a column's tiles follow one another (packed (16384, 4096): forward 286 us without,
// 256 with); where tickets are drawn the launch gets slower by it ((4, 4096, 4096) fp32: 128 / 240 us without).
template <int R>
struct GatedMarks {
    uint32_t start[R / 32], end[R / 32], valid[R / 32];
    int seq[R];
    // Run by a warp: lane l has positions l, 32 + l, ...; their searches go step by step together.
    __device__ __forceinline__ void find(const GatedParams& p, int b, long long s0, int lane)
    {
        constexpr int N = R / 32;
        int q[N];
        bool ok[N], st[N], en[N];
        if (p.cu) {
            int lo[N], hi[N];
#pragma unroll
            for (int i = 0; i < N; ++i) lo[i] = 0, hi[i] = p.nseq + 1;
            for (int step = 32 - __clz(p.nseq + 1); step > 0; --step)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const long long s = s0 + 32 * i + lane, row = p.reverse ? p.nrows - 1 - s : s;
                    const int mid = (lo[i] + hi[i]) >> 1;
                    if (lo[i] < hi[i]) {
                        if (gated_offset(p, mid) <= row) lo[i] = mid + 1;
                        else hi[i] = mid;
                    }
                }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const long long s = s0 + 32 * i + lane, row = p.reverse ? p.nrows - 1 - s : s;
                q[i] = lo[i] - 1;
                ok[i] = s < p.nrows && q[i] >= 0 && q[i] < p.nseq;
                const long long first = ok[i] ? gated_offset(p, q[i]) : 0, last = ok[i] ? gated_offset(p, q[i] + 1) - 1 : 0;
                st[i] = ok[i] && row == (p.reverse ? last : first);
                en[i] = ok[i] && row == (p.reverse ? first : last);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const long long s = s0 + 32 * i + lane;
                ok[i] = s < p.nrows;
                long long n = b, o = s;
                if (p.nb == 1 && p.seqlen < p.nrows) {
                    n = s / p.seqlen;
                    o = s - n * p.seqlen;
                    if (p.reverse) n = p.nseq - 1 - n;
                }
                q[i] = (int)n;
                st[i] = ok[i] && o == 0;
                en[i] = ok[i] && o == p.seqlen - 1;
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t a = __ballot_sync(0xffffffffu, st[i]), c = __ballot_sync(0xffffffffu, en[i]), v = __ballot_sync(0xffffffffu, ok[i]);
            if (lane == 0) start[i] = a, end[i] = c, valid[i] = v;
            seq[32 * i + lane] = q[i];
        }
    }
    template <int K>
    __device__ __forceinline__ GatedRun run(int warp, int lane) const
    {
        constexpr uint32_t kMask = (1u << K) - 1u;
        const int word = warp * K >> 5, shift = warp * K & 31;
        GatedRun r;
        r.start = start[word] >> shift & kMask;
        r.end = end[word] >> shift & kMask;
        r.valid = valid[word] >> shift & kMask;
        r.cut = (r.start | ~r.valid) & kMask;
        r.seq = (r.start | r.end) ? seq[warp * K + (lane & (K - 1))] : 0;
        return r;
    }
};

// The warp behind the others: draws tickets (one ahead, so that the counter's latency is hidden), issues the
// copies, and evaluates the block's decay parameters, which the other warps find beside the operands.
template <typename ST, bool DECAY, bool BWD, int SHAPE, int LOAD>
__device__ __forceinline__ void gated_produce(const GatedParams& p, const GatedMaps& maps, char* stages, uint64_t* full, uint64_t* empty,
                                              GatedWhere* items, GatedMarks<GatedTile<ST, DECAY, BWD, SHAPE>::R>* marks,
                                              float (*rates)[kGatedChannels], volatile int* abort_flag, uint32_t epoch)
{
    using T = GatedTile<ST, DECAY, BWD, SHAPE>;
    const int lane = (int)threadIdx.x & 31;
    uint32_t ahead = 0, j = 0, ticket = 0;
    if (LOAD != kLoadCluster && lane == 0) ahead = atomicAdd(p.header, 1u);
    bool gave_up = false, more = true;
    const int rank = LOAD == kLoadCluster ? (int)(blockIdx.x % (unsigned)p.cluster) : 0;
    const uint32_t clusters = LOAD == kLoadCluster ? gridDim.x / (unsigned)p.cluster : 1u;
    uint32_t column = LOAD == kLoadCluster ? blockIdx.x / (unsigned)p.cluster : 0u;      // this cluster's columns: every `clusters`-th
    float rate[2] = {0.0f, 0.0f};
    GatedWhere w;
    w.dt = GatedWhere::kLast;
    for (int t = 0;; ++j, ++t) {
        const int s = (int)(j % T::kStages);
        if (LOAD == kLoadCluster) {
            // (a job is the whole column, its tiles are dealt out to the cluster's CTAs in turn)
            if (j > 0 && w.last()) {
                t = 0;
                column += clusters;
            }
            more = column < (uint32_t)p.units;
            w = gated_turn<BWD>(p, column, t, rank);
        } else {
            if (w.last()) {
                t = 0;
                ticket = __shfl_sync(0xffffffffu, ahead, 0);
                more = (long long)ticket < p.ntickets;
                if (more && lane == 0) ahead = atomicAdd(p.header, 1u);
            }
            w = gated_where<BWD>(p, ticket, t);
        }
        const int block = w.block() * kGatedChannels;
        if (DECAY && more && w.first()) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int ch = block + v * 32 + lane;
                rate[v] = ch < p.D ? p.scale * softplus(__ldg(p.decay + ch)) : 0.0f;
            }
        }
        if (j >= (uint32_t)T::kStages && !ptx::mbar_wait_bounded(&empty[s], ((j / T::kStages) - 1u) & 1u, p.wait_budget)) gave_up = true;
        gave_up = __any_sync(0xffffffffu, gave_up || *abort_flag);
        if (gave_up) break;
        if (DECAY) {
            rates[s][lane] = rate[0];
            rates[s][32 + lane] = rate[1];
            __syncwarp();
        }
        if (lane == 0) {
            items[s] = more ? w : GatedWhere{-1, 0, 0, 0};
            if (more && w.k < p.nk) {
                const int row = p.reverse ? (int)(p.nrows - (long long)(w.k + 1) * T::R) : w.k * T::R;
                char* to = stages + s * T::kStageBytes;
                if (LOAD == kLoadCluster) ptx::mbar_expect_tx(&full[s], (uint32_t)T::kStageBytes);
                else ptx::mbar_arrive_expect_tx(&full[s], (uint32_t)T::kStageBytes);
                ptx::tma_load_3d(to, &maps.x, &full[s], block, row, w.b);
                ptx::tma_load_3d(to + T::kArrayBytes, &maps.f, &full[s], block, row, w.b);
                if (DECAY) ptx::tma_load_3d(to + 2 * T::kArrayBytes, &maps.i, &full[s], block, row, w.b);
                if (BWD) ptx::tma_load_3d(to + (T::kArrays - 1) * T::kArrayBytes, &maps.dy, &full[s], block, row, w.b);
            } else if (LOAD != kLoadCluster) {
                ptx::mbar_arrive(&full[s]);
            }
        }
        if (LOAD == kLoadCluster) {
            if (more) marks[s].find(p, w.b, (long long)w.k * T::R, lane);
            // the arrival that lets the stage be used once the copies have landed as well
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&full[s]);
        }
        if (!more) break;
    }
    if (gave_up) {
        *abort_flag = 1;
        if (lane == 0) atomicOr(p.header + 1, kStatusCopyTimeout);
        // no copy may land in this CTA's shared memory after it has left
        for (uint32_t i = j > (uint32_t)T::kStages ? j - T::kStages : 0u; i < j; ++i)
            (void)ptx::mbar_wait_bounded(&full[i % T::kStages], (i / T::kStages) & 1u, p.wait_budget);
    }
    if (LOAD != kLoadCluster && lane == 0) finish_launch(p.header, epoch);
}

// What both passes have in common: the pipeline of tiles around `body`, which calls `next` behind its first
// barrier (where a stage is free: forward its own, backward the one of the tile before) and returns false to
// stop (all threads alike).
template <typename ST, bool DECAY, bool BWD, int SHAPE, int LOAD, typename Exchange, typename Body>
__device__ __forceinline__ void gated_tiles(const GatedParams& p, const GatedMaps& maps, Exchange& exchange, Body body)
{
    using T = GatedTile<ST, DECAY, BWD, SHAPE>;
    using Word = typename T::Word;
    // (used as it is: rounding the address up would hide from the compiler that it is shared memory)
    extern __shared__ __align__(128) char gated_smem[];
    char* const stages = gated_smem;
    __shared__ __align__(8) uint64_t full[T::kStages], empty[T::kStages];
    __shared__ uint32_t tickets[2];
    __shared__ __align__(16) GatedWhere items[T::kStages];
    __shared__ __align__(8) float rates[T::kStages][kGatedChannels];
    __shared__ GatedMarks<T::R> marks[LOAD == kLoadCluster ? T::kStages : 1];
    __shared__ int abort_flag;
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (gated_bulk(LOAD)) {
        if (tid == 0) {
#pragma unroll
            for (int s = 0; s < T::kStages; ++s) {
                ptx::mbar_init(&full[s], 1u);
                ptx::mbar_init(&empty[s], 1u);
                items[s] = GatedWhere{0, 0, 0, 0};
            }
            abort_flag = 0;
            exchange.open();
            ptx::fence_mbar_init();
        }
        __syncthreads();
        if (LOAD == kLoadCluster && p.cluster > 1) ptx::cluster_sync();      // the others' barriers exist
        ptx::grid_dependency_wait();
        const uint32_t epoch = LOAD == kLoadCluster ? 0u : read_epoch(p.header);
        if (warp == T::W) {
            gated_produce<ST, DECAY, BWD, SHAPE, LOAD>(p, maps, stages, full, empty, items, marks, rates, &abort_flag, epoch);
            if (LOAD == kLoadCluster && p.cluster > 1) {
                __syncwarp();
                ptx::cluster_sync();      // nobody sends here any more
            }
            return;
        }
        for (uint32_t it = 0;; ++it) {
            const int s = (int)(it % T::kStages);
            if (!ptx::mbar_wait_bounded(&full[s], (it / T::kStages) & 1u, p.wait_budget)) {
                // keeps step with the other warps up to the next barrier, where all of them see the flag
                *(volatile int*)&abort_flag = 1;
                atomicOr(p.header + 1, kStatusCopyTimeout);
            }
            const int4 item = *reinterpret_cast<const int4*>(&items[s]);
            if (item.x < 0) break;
            const bool on = body(GatedWhere{item.x, item.y, item.z, item.w}, it, epoch, reinterpret_cast<const Word*>(stages + s * T::kStageBytes), rates[s],
                                 [&] {
                                     if constexpr (LOAD == kLoadCluster) return marks[s].template run<T::K>(warp, lane);
                                     else return gated_run<T::K>(p, item.z, (long long)item.x * T::R + warp * T::K, lane);
                                 },
                                 [&] {
                                     const uint32_t done = BWD ? it - 1u : it;
                                     if (tid == 0 && (!BWD || it > 0)) ptx::mbar_arrive(&empty[done % T::kStages]);
                                 },
                                 (volatile int*)&abort_flag);
            if (!on) break;
        }
        if (LOAD == kLoadCluster && p.cluster > 1) {
            __syncwarp();
            ptx::cluster_sync();
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
    int t = 0;
    GatedWhere w = gated_where<BWD>(p, ticket, 0);
    bool more = (long long)ticket < p.ntickets;
    if (more) gated_fetch<ST, DECAY, BWD, SHAPE, LOAD>(p, w, reinterpret_cast<Word*>(stages), warp, lane);
    ptx::cp_async_commit();
    for (uint32_t it = 0; more; ++it) {
        if (tid == 0 && w.last()) tickets[(it + 1) & 1] = atomicAdd(p.header, 1u);
        if (DECAY && tid < kGatedChannels) {
            const int ch = w.block() * kGatedChannels + tid;
            rates[it & 1][tid] = ch < p.D ? p.scale * softplus(p.decay[ch]) : 0.0f;
        }
        __syncthreads();
        ++t;
        if (w.last()) {
            t = 0;
            ticket = tickets[(it + 1) & 1];
            more = (long long)ticket < p.ntickets;
        }
        const GatedWhere next = gated_where<BWD>(p, ticket, t);
        if (more) gated_fetch<ST, DECAY, BWD, SHAPE, LOAD>(p, next, reinterpret_cast<Word*>(stages + ((it + 1) & 1) * T::kStageBytes), warp, lane);
        ptx::cp_async_commit();
        ptx::cp_async_wait_group<1>();
        body(w, it, epoch, reinterpret_cast<const Word*>(stages + (it & 1) * T::kStageBytes), rates[it & 1],
             [&] { return gated_run<T::K>(p, w.b, (long long)w.k * T::R + warp * T::K, lane); }, [] {}, (volatile int*)&abort_flag);
        w = next;
    }
    if (tid == 0) finish_launch(p.header, epoch);
}

// ---- forward ------------------------------------------------------------------------------------------
// 6 (forget) or 8 (decay) bytes per element in 16 bits.  (8, 4096, 4096) bf16: 168 us (4.8 TB/s) and 228 us (4.7 TB/s).
// Decay form there: issue 61 %, special functions 53 %, DRAM 55 % busy, 37 instructions per element; in the other shape
// ((4, 4096, 4096)) 46, 44 and 44 %.  Latency between them bounds it, no unit alone.
template <typename ST, bool DECAY, int SHAPE, int LOAD>
__global__ void __launch_bounds__(GatedTile<ST, DECAY, false, SHAPE>::threads(LOAD), GatedTile<ST, DECAY, false, SHAPE>::kCtas)
    gated_fwd_kernel(const GatedParams p, const __grid_constant__ GatedMaps maps)
{
    using T = GatedTile<ST, DECAY, false, SHAPE>;
    constexpr int K = T::K, R = T::R;
    __shared__ float4 runs[2][T::W][32];      // every thread's Y of both channels, then P
    __shared__ int cuts[2][T::W];             // does a sequence start in a warp's run?
    __shared__ __align__(8) float entering[2][kGatedChannels];      // tiles take turns
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;

    __shared__ __align__(16) std::conditional_t<LOAD == kLoadCluster, GatedExchange, GatedNoExchange> exchange;
    float carry = 0.0f;      // of a cluster's column, in the 64 threads that link
    gated_tiles<ST, DECAY, false, SHAPE, LOAD>(p, maps, exchange, [&](const GatedWhere& w, uint32_t it, uint32_t epoch,
                                                     const typename T::Word* stage, const float* rates, auto marked, auto next, volatile int* abort_flag) {
        const int ch = w.block() * kGatedChannels + 2 * lane;
        const int have = p.D - ch;
        const long long s0 = (long long)w.k * R + warp * K;
        TileDesc* desc = p.desc + (((long long)w.job * p.units + w.b * p.dtiles + w.block()) * kGatedChannels + tid);
        uint4 seen = make_uint4(0u, 0u, 0u, 0u);
        if (LOAD != kLoadCluster && tid < kGatedChannels && w.job > 0 && w.first()) seen = desc_load(desc - (long long)p.units * kGatedChannels, epoch);
        const GatedRun run = marked();
        const typename T::Word* words = stage + (p.reverse ? R - 1 - warp * K : warp * K) * 32 + lane;
        const int wstep = p.reverse ? -32 : 32;

        F2 a[K], u[K];
        auto gates = [&](auto small) {
            F2 rate = f2(0.0f);
            if (DECAY) rate = f2(rates[2 * lane], rates[2 * lane + 1]);
            const typename T::Word* at = words;
#pragma unroll
            for (int j = 0; j < K; ++j, at += wstep) {
                const F2 xv = Two<ST>::get(at[0]), fv = Two<ST>::get(at[R * 32]);
                if (DECAY) {
                    F2 b2;
                    decay_factors2<T::kFast, decltype(small)::value>(f2_mul(rate, logistic2<T::kFast>(fv)), a[j], b2);
                    u[j] = f2_mul(gated_factor2<T::kFast>(b2, Two<ST>::get(at[2 * R * 32])), xv);
                } else {
                    F2 n;
                    logistic_pair2<T::kFast>(fv, a[j], n);
                    u[j] = f2_mul(n, xv);
                }
            }
        };
        // a slow decay (rate below 1/4 in all of the warp's channels) never needs the exponential
        if (DECAY && !__all_sync(0xffffffffu, rates[2 * lane] < 0.25f && rates[2 * lane + 1] < 0.25f)) gates(std::false_type{});
        else gates(std::true_type{});
        // a run in which sequences start, or rows belong to none, takes a path of its own: it selects where
        // the common one multiplies
        F2 Y = f2(0.0f), P = f2(1.0f);
        if (run.cut) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if (!(run.valid >> j & 1u)) u[j] = f2(0.0f);
                if (p.h0 && (run.start >> j & 1u)) u[j] = f2_fma(a[j], load_state(p.h0, (long long)__shfl_sync(0xffffffffu, run.seq, j) * p.D + ch, have), u[j]);
                const bool cut = run.cut >> j & 1u;
                Y = cut ? u[j] : f2_fma(a[j], Y, u[j]);
                P = gated_is_cut(run, j) ? f2(kCut) : f2_mul(P, a[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                Y = f2_fma(a[j], Y, u[j]);
                P = f2_mul(P, a[j]);
            }
        }
        float4(*set)[32] = runs[it & 1];
        const float2 y2 = f2_get(Y), p2 = f2_get(P);
        set[warp][lane] = make_float4(y2.x, y2.y, p2.x, p2.y);
        if (lane == 0) cuts[it & 1][warp] = run.cut != 0u;
        gated_sync<T::W>();
        if (gated_bulk(LOAD) && *abort_flag) return false;
        next();

        if (tid < kGatedChannels) {
            Pair total = pair_identity();
#pragma unroll
            for (int i = 0; i < T::W; ++i) {
                const float* r = reinterpret_cast<const float*>(&set[i][tid >> 1]) + (tid & 1);
                total = join(total, Pair{r[0], r[2]});
            }
            if constexpr (LOAD == kLoadCluster) {
                if (w.first()) carry = 0.0f;
                entering[it & 1][tid] = exchange.turn(p, it, tid, total, carry);
            } else {
                gated_carry(p, w, desc, seen, total, epoch, &entering[it & 1][tid], &entering[(it + 1) & 1][tid]);
            }
        }
        // the warps in front of this one, joined; without a cut in the tile no selection is needed
        F2 bY = f2(0.0f), bP = f2(1.0f);
        const bool any_cut = gated_any<T::W>(cuts[it & 1]);
        if (any_cut) {
            Pair before[2] = {pair_identity(), pair_identity()};
            for (int i = 0; i < warp; ++i) {
                const float4 r = set[i][lane];
                before[0] = join(before[0], Pair{r.x, r.z});
                before[1] = join(before[1], Pair{r.y, r.w});
            }
            bY = f2(before[0].y, before[1].y);
            bP = f2(before[0].p, before[1].p);
        } else {
#pragma unroll
            for (int i = 0; i < T::W - 1; ++i) {
                const float4 r = set[i][lane];
                if (i < warp) {
                    bY = f2_fma(bY, f2(r.z, r.w), f2(r.x, r.y));
                    bP = f2_mul(bP, f2(r.z, r.w));
                }
            }
        }
        if (LOAD == kLoadCluster || w.first()) gated_sync<T::W>();
        const float* in = entering[it & 1];
        F2 h = gated_enter(*reinterpret_cast<const float2*>(in + 2 * lane), bY, bP, any_cut);
        if (p.ckpt && s0 % kGatedCheckpoint == 0 && s0 < p.nrows)
            store_two<float>(p.ckpt, ((long long)w.b * p.nck + s0 / kGatedCheckpoint) * p.D + ch, have, h, false);
        const bool pair = (gated_bulk(LOAD) || p.pair) && have > 1;
        const long long row0 = (long long)w.b * p.nrows + (p.reverse ? p.nrows - 1 - s0 : s0);
        ST* y = static_cast<ST*>(p.y) + row0 * p.D + ch;
        const long long ystep = p.reverse ? -(long long)p.D : p.D;
        if (run.cut | run.end) {
            const int rows = (int)min((long long)K, p.nrows - s0);
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if (j >= rows) break;
                h = (run.cut >> j & 1u) ? u[j] : f2_fma(a[j], h, u[j]);
                store_two<ST>(y + j * ystep, 0, have, h, pair);
                if (p.hT && (run.end >> j & 1u)) store_two<float>(p.hT, (long long)__shfl_sync(0xffffffffu, run.seq, j) * p.D + ch, have, h, false);
            }
        } else if (pair) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                h = f2_fma(a[j], h, u[j]);
                *reinterpret_cast<typename T::Word*>(y) = Two<ST>::put(h);
                y += ystep;
            }
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                h = f2_fma(a[j], h, u[j]);
                store_two<ST>(y, 0, have, h, false);
                y += ystep;
            }
        }
        return true;
    });
}

// ---- backward -----------------------------------------------------------------------------------------
// Between the two halves of a tile a thread keeps a, b and the state in front of each of its elements; x, dy
// and the logits stay in shared memory and what else is needed is evaluated again from them.
// 10 or 14 bytes per element in 16 bits.  (8, 4096, 4096) bf16: forget 347 us (3.9 TB/s), decay 559 us (3.4 TB/s).
// Decay form there: issue 47 %, special functions 54 %, DRAM 40 % busy, 71 instructions per element; in the other shape
// ((4, 4096, 4096)) 44, 43 and 31 %, 82 instructions.
template <typename ST, bool DECAY, int SHAPE, int LOAD>
__global__ void __launch_bounds__(GatedTile<ST, DECAY, true, SHAPE>::threads(LOAD), GatedTile<ST, DECAY, true, SHAPE>::kCtas)
    gated_bwd_kernel(const GatedParams p, const __grid_constant__ GatedMaps maps)
{
    using T = GatedTile<ST, DECAY, true, SHAPE>;
    constexpr int K = T::K, R = T::R;
    static_assert(R % kGatedCheckpoint == 0, "a checkpoint where a tile starts");
    constexpr int kDy = (T::kArrays - 1) * R * 32;
    __shared__ float4 runs[2][T::W][32];      // every thread's Y of both channels, forward direction, then P
    __shared__ int cuts[2][T::W];             // does a sequence start in a warp's run?
    __shared__ float2 back[2][T::W][32];      // Y of both channels, adjoint direction (same P)
    __shared__ __align__(8) float entering[2][kGatedChannels];      // tiles take turns
    __shared__ float2 dsum[T::W][32];
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;

    F2 dl = f2(0.0f);      // this thread's share of the decay gradient, over a job

    __shared__ __align__(16) std::conditional_t<LOAD == kLoadCluster, GatedExchange, GatedNoExchange> exchange;
    float carry = 0.0f;      // of a cluster's column, in the 64 threads that link
    gated_tiles<ST, DECAY, true, SHAPE, LOAD>(p, maps, exchange, [&](const GatedWhere& w, uint32_t it, uint32_t epoch,
                                                    const typename T::Word* stage, const float* rates, auto marked, auto next, volatile int* abort_flag) {
        const int ch = w.block() * kGatedChannels + 2 * lane;
        const int have = p.D - ch;
        const long long s0 = (long long)w.k * R + warp * K;
        TileDesc* desc = p.desc + (((long long)w.job * p.units + w.b * p.dtiles + w.block()) * kGatedChannels + tid);
        uint4 seen = make_uint4(0u, 0u, 0u, 0u);
        if (LOAD != kLoadCluster && tid < kGatedChannels && w.job > 0 && w.first()) seen = desc_load(desc - (long long)p.units * kGatedChannels, epoch);
        const float2 h0 = f2_get(load_state(p.ckpt, ((long long)w.b * p.nck + (long long)w.k * (R / kGatedCheckpoint)) * p.D + ch, w.k < p.nk ? have : 0));
        const GatedRun run = marked();
        const typename T::Word* words = stage + (p.reverse ? R - 1 - warp * K : warp * K) * 32 + lane;
        const int wstep = p.reverse ? -32 : 32;
        F2 rate = f2(0.0f);
        if (DECAY) rate = f2(rates[2 * lane], rates[2 * lane + 1]);

        // add: b u, later the state in front of the element
        F2 a[K], bb[K], add[K];
        auto gates = [&](auto small) {
            const typename T::Word* at = words;
#pragma unroll
            for (int j = 0; j < K; ++j, at += wstep) {
                const F2 xv = Two<ST>::get(at[0]), fv = Two<ST>::get(at[R * 32]);
                if (DECAY) {
                    F2 b2;
                    decay_factors2<T::kFast, decltype(small)::value>(f2_mul(rate, logistic2<T::kFast>(fv)), a[j], b2);
                    bb[j] = root2(b2);
                    add[j] = f2_mul(bb[j], f2_mul(logistic2<T::kFast>(Two<ST>::get(at[2 * R * 32])), xv));
                } else {
                    logistic_pair2<T::kFast>(fv, a[j], bb[j]);
                    add[j] = f2_mul(bb[j], xv);
                }
            }
        };
        if (DECAY && !__all_sync(0xffffffffu, rates[2 * lane] < 0.25f && rates[2 * lane + 1] < 0.25f)) gates(std::false_type{});
        else gates(std::true_type{});
        // `edge`: sequences start or end in this run, or rows belong to none
        const bool edge = run.cut || run.end;
        auto of_sequence = [&](const float* states, int j) {
            return load_state(states, (long long)__shfl_sync(0xffffffffu, run.seq, j) * p.D + ch, have);
        };
        const typename T::Word* const words_end = words + (K - 1) * wstep;
        auto gradient = [&](const typename T::Word* at, int j, bool edge) {
            F2 dy = Two<ST>::get(at[kDy]);
            if (edge && p.dhT && (run.end >> j & 1u)) dy = f2_add(dy, of_sequence(p.dhT, j));
            return dy;
        };
        F2 Y = f2(0.0f), P = f2(1.0f), q = f2(0.0f);
        const typename T::Word* at = words_end;
        if (edge) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const bool cut = run.cut >> j & 1u;
                if (!(run.valid >> j & 1u)) a[j] = bb[j] = add[j] = f2(0.0f);
                if (cut) Y = p.h0 && (run.start >> j & 1u) ? of_sequence(p.h0, j) : f2(0.0f);
                Y = f2_fma(a[j], Y, add[j]);
                P = gated_is_cut(run, j) ? f2(kCut) : f2_mul(P, a[j]);
            }
#pragma unroll
            for (int j = K - 1; j >= 0; --j, at -= wstep) q = (run.cut >> j & 1u) ? f2(0.0f) : f2_mul(a[j], f2_add(gradient(at, j, true), q));
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                Y = f2_fma(a[j], Y, add[j]);
                P = f2_mul(P, a[j]);
            }
#pragma unroll
            for (int j = K - 1; j >= 0; --j, at -= wstep) q = f2_mul(a[j], f2_add(gradient(at, j, false), q));
        }
        float4(*set)[32] = runs[it & 1];
        float2(*bset)[32] = back[it & 1];
        const float2 y2 = f2_get(Y), p2 = f2_get(P);
        set[warp][lane] = make_float4(y2.x, y2.y, p2.x, p2.y);
        if (lane == 0) cuts[it & 1][warp] = run.cut != 0u;
        bset[warp][lane] = f2_get(q);
        gated_sync<T::W>();
        if (gated_bulk(LOAD) && *abort_flag) return false;
        next();

        if (tid < kGatedChannels) {
            Pair total = pair_identity();
#pragma unroll
            for (int i = T::W - 1; i >= 0; --i) {
                const float P = reinterpret_cast<const float*>(&set[i][tid >> 1])[2 + (tid & 1)];
                const float Y = reinterpret_cast<const float*>(&bset[i][tid >> 1])[tid & 1];
                total = join(total, Pair{Y, P});
            }
            if constexpr (LOAD == kLoadCluster) {
                if (w.first()) carry = 0.0f;
                entering[it & 1][tid] = exchange.turn(p, it, tid, total, carry);
            } else {
                gated_carry(p, w, desc, seen, total, epoch, &entering[it & 1][tid], &entering[(it + 1) & 1][tid]);
            }
        }
        // the state that enters this run, from the checkpoint
        F2 h = f2(h0.x, h0.y), aY = f2(0.0f), aP = f2(1.0f);
        const bool any_cut = gated_any<T::W>(cuts[it & 1]);
        if (any_cut) {
            float hx = h0.x, hy = h0.y;
            for (int i = 0; i < warp; ++i) {
                const float4 r = set[i][lane];
                hx = enter(hx, Pair{r.x, r.z});
                hy = enter(hy, Pair{r.y, r.w});
            }
            h = f2(hx, hy);
            Pair after[2] = {pair_identity(), pair_identity()};
            for (int i = T::W - 1; i > warp; --i) {
                const float4 r = set[i][lane];
                const float2 y = bset[i][lane];
                after[0] = join(after[0], Pair{y.x, r.z});
                after[1] = join(after[1], Pair{y.y, r.w});
            }
            aY = f2(after[0].y, after[1].y);
            aP = f2(after[0].p, after[1].p);
        } else {
#pragma unroll
            for (int i = 0; i < T::W - 1; ++i) {
                const float4 r = set[i][lane];
                if (i < warp) h = f2_fma(h, f2(r.z, r.w), f2(r.x, r.y));
            }
#pragma unroll
            for (int i = T::W - 1; i > 0; --i) {
                const float4 r = set[i][lane];
                const float2 y = bset[i][lane];
                if (i > warp) {
                    aY = f2_fma(aY, f2(r.z, r.w), f2(y.x, y.y));
                    aP = f2_mul(aP, f2(r.z, r.w));
                }
            }
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (edge && (run.cut >> j & 1u)) h = p.h0 && (run.start >> j & 1u) ? of_sequence(p.h0, j) : f2(0.0f);
            const F2 before = h;
            h = f2_fma(a[j], before, add[j]);
            add[j] = before;
        }
        if (LOAD == kLoadCluster || w.first()) gated_sync<T::W>();
        const float* in = entering[it & 1];
        q = gated_enter(*reinterpret_cast<const float2*>(in + 2 * lane), aY, aP, any_cut);
        if (w.first()) dl = f2(0.0f);
        const bool pair = (gated_bulk(LOAD) || p.pair) && have > 1;
        const long long row0 = (long long)w.b * p.nrows + (p.reverse ? p.nrows - 1 - s0 : s0);
        const long long at0 = row0 * p.D + ch, astep = p.reverse ? -(long long)p.D : p.D;
        // gradients of element j; q becomes what flows on to the element before it
        at = words_end;
        auto element = [&](int j, bool edge, F2& odx, F2& odf, F2& odi) {
            const F2 xv = Two<ST>::get(at[0]);
            const F2 grad = f2_add(gradient(at, j, edge), q), hp = add[j];
            q = f2_mul(a[j], grad);
            const F2 wb = f2_mul(grad, bb[j]);
            if (DECAY) {
                F2 s, n;
                logistic_both2<T::kFast>(Two<ST>::get(at[R * 32]), s, n);
                const float2 b = f2_get(bb[j]);
                // -a/b, left out where the factor b has vanished (its share is the root of a log a below 1e-38)
                const F2 minus_slope = f2_mul(a[j], f2(b.x > 0.0f ? -approx_rcp(b.x) : 0.0f, b.y > 0.0f ? -approx_rcp(b.y) : 0.0f));
                const F2 gi = logistic2<T::kFast>(Two<ST>::get(at[2 * R * 32])), u = f2_mul(gi, xv);
                // d(log a) * log a, with log a = -rate s
                const F2 t = f2_mul(f2_mul(q, f2_fma(u, minus_slope, hp)), f2_mul(f2_mul(rate, f2(-1.0f)), s));
                odx = f2_mul(wb, gi);
                odi = f2_mul(wb, f2_mul(u, f2_fma(gi, f2(-1.0f), f2(1.0f))));
                odf = f2_mul(t, n);
                if (!edge || (run.valid >> j & 1u)) dl = f2_add(dl, t);
            } else {
                odx = wb;
                odf = f2_mul(f2_mul(q, bb[j]), f2_fma(xv, f2(-1.0f), hp));
                odi = odx;
            }
        };
        if (edge || !pair) {
#pragma unroll
            for (int j = K - 1; j >= 0; --j, at -= wstep) {
                F2 odx, odf, odi;
                element(j, true, odx, odf, odi);
                if (p.dh0 && (run.start >> j & 1u)) store_two<float>(p.dh0, (long long)__shfl_sync(0xffffffffu, run.seq, j) * p.D + ch, have, q, false);
                if (run.cut >> j & 1u) q = f2(0.0f);
                if (s0 + j < p.nrows) {
                    if (!(run.valid >> j & 1u)) odx = odf = odi = f2(0.0f);
                    store_two<ST>(p.dx, at0 + j * astep, have, odx, pair);
                    store_two<ST>(p.df, at0 + j * astep, have, odf, pair);
                    if (DECAY) store_two<ST>(p.di, at0 + j * astep, have, odi, pair);
                }
            }
        } else {
            long long to = at0 + (K - 1) * astep;
#pragma unroll
            for (int j = K - 1; j >= 0; --j, at -= wstep) {
                F2 odx, odf, odi;
                element(j, false, odx, odf, odi);
                *reinterpret_cast<typename T::Word*>(static_cast<ST*>(p.dx) + to) = Two<ST>::put(odx);
                *reinterpret_cast<typename T::Word*>(static_cast<ST*>(p.df) + to) = Two<ST>::put(odf);
                if (DECAY) *reinterpret_cast<typename T::Word*>(static_cast<ST*>(p.di) + to) = Two<ST>::put(odi);
                to -= astep;
            }
        }
        if (DECAY && w.last()) {
            dsum[warp][lane] = f2_get(dl);
            gated_sync<T::W>();
            if (tid < kGatedChannels && w.block() * kGatedChannels + tid < p.D) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < T::W; ++i) s += reinterpret_cast<const float*>(&dsum[i][tid >> 1])[tid & 1];
                p.dlam[((long long)w.b * p.jobs + (LOAD == kLoadCluster ? (int)(blockIdx.x % (unsigned)p.cluster) : w.job)) * p.D + w.block() * kGatedChannels + tid] = s;
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

// V adjacent channels of a row (V = 4: one access, on a boundary of four elements).
template <typename ST, int V>
__device__ __forceinline__ void step_load(const void* base, long long offset, float* v)
{
    const ST* q = static_cast<const ST*>(base) + offset;
    if constexpr (V == 4 && sizeof(ST) == 4) {
        const float4 w = *reinterpret_cast<const float4*>(q);
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else if constexpr (V == 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(q);
        Two<ST>::unpack(w.x, v), Two<ST>::unpack(w.y, v + 2);
    } else {
        v[0] = to_f32<ST>(*q);
    }
}
template <typename ST, int V>
__device__ __forceinline__ void step_store(void* base, long long offset, const float* v)
{
    ST* q = static_cast<ST*>(base) + offset;
    if constexpr (V == 4 && sizeof(ST) == 4) *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(q) = make_uint2(Two<ST>::pack(v), Two<ST>::pack(v + 2));
    else *q = from_f32<ST>(v[0]);
}

constexpr int kStepThreads = 128;

// ROWS rows and 128 V channels per CTA.  Bound by memory: an element moves 6 or 8 bytes of operands and results
// in 16 bits and 8 of state; several rows per CTA keep that much more in flight and share the decay parameters and
// the search below.
// A slot that several rows name holds ONE sequence whose tokens are the rows in order: the first of them walks
// through all, the others leave them to it.  Every CTA compares its rows' slots with all rows'.
// (512, 8192) bf16 replayed in a graph: decay form with slots 17.5 us (31.8 before rows shared a CTA),
// forget form without 8.1 us (7.2 TB/s, above the copy bandwidth: part of it comes from L2).
template <typename ST, bool DECAY, int V, int ROWS>
__global__ void __launch_bounds__(kStepThreads) gated_step_kernel(const GatedStepParams p)
{
    constexpr bool kFast = sizeof(ST) == 2;
    __shared__ unsigned shared_flags;      // bit r: an earlier row has row r's slot; bit 16 + r: a later one
    __shared__ int nearest;
    const int tid = (int)threadIdx.x;
    const int ch = ((int)blockIdx.y * kStepThreads + tid) * V;
    const bool have = ch < p.D;
    const int row0 = (int)blockIdx.x * ROWS;
    if (tid == 0) shared_flags = 0u;
    ptx::grid_dependency_wait();
    long long slot[ROWS];
    float x[ROWS][V], f[ROWS][V], g[ROWS][V], h[ROWS][V], rate[V];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        slot[r] = row0 + r < p.rows ? step_slot(p, row0 + r) : -1;
        if (slot[r] >= 0 && have) {
            step_load<float, V>(p.state, slot[r] * p.sstate + ch, h[r]);
            step_load<ST, V>(p.x, (long long)(row0 + r) * p.sx + ch, x[r]);
            step_load<ST, V>(p.f, (long long)(row0 + r) * p.sf + ch, f[r]);
            if (DECAY) step_load<ST, V>(p.ig, (long long)(row0 + r) * p.si + ch, g[r]);
        }
    }
    if (DECAY && have)
#pragma unroll
        for (int v = 0; v < V; ++v) rate[v] = p.scale * softplus(__ldg(p.decay + ch + v));
    unsigned flags = 0u;
    if (p.slots) {
        for (int n = tid; n < p.rows; n += kStepThreads) {
            const long long other = step_slot(p, n);
            if (other < 0) continue;
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (other == slot[r] && n != row0 + r) flags |= n < row0 + r ? 1u << r : 65536u << r;
        }
        flags = __reduce_or_sync(0xffffffffu, flags);
        __syncthreads();
        if ((tid & 31) == 0 && flags) atomicOr(&shared_flags, flags);
        __syncthreads();
        flags = shared_flags;
    }
    auto advance = [&](const float* xv, const float* fv, const float* gv, float* hv) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (DECAY) {
                float a, b2;
                decay_factors<kFast, false>(rate[v] * logistic<kFast>(fv[v]), a, b2);
                hv[v] = fmaf(a, hv[v], approx_sqrt(b2) * (logistic<kFast>(gv[v]) * xv[v]));
            } else {
                float s, n;
                logistic_pair<kFast>(fv[v], s, n);
                hv[v] = fmaf(s, hv[v], n * xv[v]);
            }
        }
    };
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        int row = row0 + r;
        if (row >= p.rows || (flags >> r & 1u)) continue;
        if (slot[r] < 0) {
            const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (have) step_store<ST, V>(p.y, (long long)row * p.D + ch, zero);
            continue;
        }
        if (have) {
            advance(x[r], f[r], g[r], h[r]);
            step_store<ST, V>(p.y, (long long)row * p.D + ch, h[r]);
        }
        while (flags >> (16 + r) & 1u) {      // the sequence's next token, if there is one
            __syncthreads();
            if (tid == 0) nearest = 0x7fffffff;
            __syncthreads();
            for (int n = row + 1 + tid; n < p.rows; n += kStepThreads)
                if (step_slot(p, n) == slot[r]) {
                    atomicMin(&nearest, n);
                    break;
                }
            __syncthreads();
            row = nearest;
            if (row == 0x7fffffff) break;
            if (have) {
                float xn[V], fn[V], gn[V];
                step_load<ST, V>(p.x, (long long)row * p.sx + ch, xn);
                step_load<ST, V>(p.f, (long long)row * p.sf + ch, fn);
                if (DECAY) step_load<ST, V>(p.ig, (long long)row * p.si + ch, gn);
                advance(xn, fn, gn, h[r]);
                step_store<ST, V>(p.y, (long long)row * p.D + ch, h[r]);
            }
        }
        if (have) step_store<float, V>(p.state, slot[r] * p.sstate + ch, h[r]);
    }
}

}  // namespace linrec

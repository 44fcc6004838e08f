// Host side of the gated recurrence (include/linrec_b200.h): argument checks, how the sequences are laid
// on scan axes, launches.
#include "gated_variants.h"
#include "host.h"

#include <cstdio>
#include <cstring>

namespace {

using linrec::GatedParams;
using linrec::GatedStepParams;
using linrec::kGatedChannels;
using linrec::kGatedCheckpoint;
using linrec_host::DeviceInfo;

bool known_dtype(int dtype)
{
    return dtype == LINREC_DTYPE_F32 || dtype == LINREC_DTYPE_BF16 || dtype == LINREC_DTYPE_F16;
}

struct Axes {
    int nb;            // scan axes side by side
    int64_t nrows;     // rows per axis
};

// A batch of equal lengths gets one axis per entry, whose tiles depend on nothing but their own sequence,
// unless the entries are so short that the last tile of each would be mostly empty; those, and packed
// sequences, share one axis.  128 positions: the longest tile of any type, so that the choice (which the
// checkpoints depend on) is the same in both passes.
Axes axes_of(const linrec_gated_args& a)
{
    if (!a.cu_seqlens && a.nseq > 1 && (a.seqlen >= 512 || a.seqlen % 128 == 0)) return Axes{(int)a.nseq, a.seqlen};
    return Axes{1, a.nrows};
}

int check(const linrec_gated_args* a)
{
    if (!a || a->nseq < 0 || a->nrows < 0 || a->nchan < 0 || (!a->cu_seqlens && a->seqlen < 0)) return LINREC_ERR_INVALID_ARG;
    if (!known_dtype(a->dtype)) return LINREC_ERR_NOT_IMPLEMENTED;
    if (!a->decay != !a->input_gate) return LINREC_ERR_INVALID_ARG;
    if (a->nseq >= 0x7fffffffLL || a->nrows >= 0x40000000LL || a->nchan >= 0x40000000LL) return LINREC_ERR_INVALID_ARG;
    if (!a->cu_seqlens && (a->seqlen > a->nrows || a->nseq * a->seqlen != a->nrows)) return LINREC_ERR_INVALID_ARG;
    const int64_t rows = a->nrows / kGatedCheckpoint + 1, chans = (a->nchan + 63) / 64;
    if ((rows + a->nseq) * chans >= 0x7f000000LL) return LINREC_ERR_INVALID_ARG;   // tickets are 32-bit
    return LINREC_OK;
}

int parse(const linrec_opts* o, int& wait_ms)
{
    wait_ms = 2000;
    if (!o || o->n_opts == 0) return LINREC_OK;
    if (o->n_opts < 0 || !o->names || !o->values) return LINREC_ERR_INVALID_ARG;
    for (int i = 0; i < o->n_opts; ++i) {
        if (!o->names[i]) return LINREC_ERR_INVALID_ARG;
        if (strcmp(o->names[i], "waitBudgetMs")) return LINREC_ERR_NOT_IMPLEMENTED;
        wait_ms = o->values[i];
    }
    return LINREC_OK;
}

// Rows of `width` bytes, `step` apart.  Do two sets share memory, or does one lie among the other's rows in any other way than
// in columns of its own?
struct Rows {
    const void* p;
    int64_t n, step, width;
};
bool rows_meet(const Rows& a, const Rows& b)
{
    if (!a.p || !b.p || a.n == 0 || b.n == 0) return false;
    const intptr_t a0 = reinterpret_cast<intptr_t>(a.p), b0 = reinterpret_cast<intptr_t>(b.p);
    if (a0 + (a.n - 1) * a.step + a.width <= b0 || b0 + (b.n - 1) * b.step + b.width <= a0) return false;
    if (a.step != b.step) return true;
    const int64_t at = ((a0 - b0) % b.step + b.step) % b.step;      // of a's columns, from b's on
    return at < b.width || at + a.width > b.step;
}

bool on_boundary(const void* p, int64_t stride, int size, int bytes)
{
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * size % bytes == 0;
}

// Rank-3 view (channels, positions, axes) of rows at `stride`, no swizzle; box = one tile.  Positions outside
// an axis and channels outside the rows read as zero.
int make_map(CUtensorMap* map, const void* ptr, int64_t stride, const GatedParams& p, int rows, int dtype)
{
    linrec_host::EncodeTiledFn enc = linrec_host::encode_tiled_fn();
    if (!enc) {
        linrec_host::note_cuda_error("cudaGetDriverEntryPoint", "cuTensorMapEncodeTiled not found");
        return LINREC_ERR_CUDA;
    }
    const int size = dtype == LINREC_DTYPE_F32 ? 4 : 2;
    const cuuint64_t dims[3] = {(cuuint64_t)p.D, (cuuint64_t)p.nrows, (cuuint64_t)p.nb};
    const cuuint64_t strides[2] = {(cuuint64_t)(stride * size), (cuuint64_t)(stride * size * p.nrows)};
    const cuuint32_t box[3] = {(cuuint32_t)kGatedChannels, (cuuint32_t)rows, 1u};
    const cuuint32_t ones[3] = {1, 1, 1};
    const CUresult r = enc(map, dtype == LINREC_DTYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                           : dtype == LINREC_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           3, const_cast<void*>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return LINREC_OK;
    char msg[64];
    snprintf(msg, sizeof(msg), "driver error %d", (int)r);
    linrec_host::note_cuda_error("cuTensorMapEncodeTiled", msg);
    return LINREC_ERR_CUDA;
}

// How many consecutive tiles of a column one CTA takes.  Jobs of four tiles where there are about as many
// columns as CTAs at least (a job waits for its predecessor, handed out `units` jobs earlier); when it was chosen (8, 4096, 4096)
// forward, 512 columns on 444 CTAs, took 306 us as single tiles, 247 in fours, 259 in eights (now 228 in fours).
// Fewer columns are single tiles linked by decoupled look-back ((1, 32768, 2048), 32 columns, then: 240 us, 530 in fours).
int tiles_per_job(long long units, int nk, long long slots)
{
    const int want = 7 * units >= 6 * slots ? 4 : 1;
    return want < nk ? want : nk;
}

// How many CTAs of a cluster share each column (0: not this way): as many as keep all columns running at a
// time, if that fills a good part of the device.
int cluster_size(const linrec_variants::GatedKernel& k, long long units, int nk, int sms, int& size)
{
    size = 0;
    long long want = sms / units;
    if (want > linrec::kGatedClusterMost) want = linrec::kGatedClusterMost;
    if (want > nk) want = nk;
    for (; want > 0; --want) {
        int active = sms;      // of single CTAs, one per SM
        const int rc = want == 1 ? LINREC_OK : linrec_host::active_clusters(reinterpret_cast<const void*>(k.fn), k.threads, (size_t)k.smem, (int)want, active);
        if (rc != LINREC_OK) return rc;
        if (active >= units) break;
    }
    // (16384, 512) bf16 decay form: 8 columns in clusters of 8 take 47 / 115 us, linked by look-back 41 / 102;
    // (16384, 1280), 20 columns in clusters of 7: 49 / 97 and 74 / 133
    if (2 * want * units >= sms) size = (int)want;
    return LINREC_OK;
}

int launch_gated(bool bwd, const linrec_gated_args* args, const linrec_opts* opts, void* workspace, size_t workspace_bytes, void* stream_)
{
    int rc = check(args);
    if (rc != LINREC_OK) return rc;
    const linrec_gated_args& a = *args;
    const bool decay = a.decay != nullptr;
    int wait_ms;
    rc = parse(opts, wait_ms);
    if (rc != LINREC_OK) return rc;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (a.nchan == 0) return LINREC_OK;
    if (a.nrows == 0) {
        if (bwd && decay && a.ddecay && cudaMemsetAsync(a.ddecay, 0, (size_t)a.nchan * 4, stream) != cudaSuccess) {
            linrec_host::note_cuda_error("cudaMemsetAsync", cudaGetErrorString(cudaGetLastError()));
            return LINREC_ERR_CUDA;
        }
        return LINREC_OK;
    }
    if (!a.x || !a.forget || a.x_stride < a.nchan || a.forget_stride < a.nchan) return LINREC_ERR_INVALID_ARG;
    if (decay && a.input_gate_stride < a.nchan) return LINREC_ERR_INVALID_ARG;
    if (!bwd && !a.y) return LINREC_ERR_INVALID_ARG;
    if (bwd && (!a.dy || a.dy_stride < a.nchan || !a.dx || !a.dforget || !a.checkpoints)) return LINREC_ERR_INVALID_ARG;
    if (bwd && decay && (!a.dinput_gate || !a.ddecay || !a.scratch || a.scratch_bytes < linrec_b200_gated_scratch_size(args)))
        return LINREC_ERR_INVALID_ARG;
    if (!linrec_host::on_elements({a.x, a.forget, a.input_gate, a.y, a.dy, a.dx, a.dforget, a.dinput_gate}, a.dtype == LINREC_DTYPE_F32 ? 4 : 2) ||
        !linrec_host::on_elements({a.decay, a.initial_state, a.checkpoints, a.final_state, a.d_final_state, a.ddecay, a.d_initial_state, a.scratch}, 4) ||
        !linrec_host::on_elements({a.cu_seqlens}, a.cu_is_64 ? 8 : 4))
        return LINREC_ERR_INVALID_ARG;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < linrec_b200_gated_workspace_size(args))
        return LINREC_ERR_WORKSPACE;
    DeviceInfo dev;
    rc = linrec_host::device_facts(dev);
    if (rc != LINREC_OK) return rc;

    const Axes ax = axes_of(a);
    GatedParams p{};
    p.x = a.x; p.f = a.forget; p.ig = a.input_gate; p.dy = a.dy;
    p.sx = a.x_stride; p.sf = a.forget_stride; p.si = a.input_gate_stride; p.sdy = a.dy_stride;
    p.y = a.y; p.dx = a.dx; p.df = a.dforget; p.di = a.dinput_gate;
    p.decay = a.decay; p.scale = a.decay_scale;
    p.h0 = a.initial_state; p.hT = a.final_state; p.dhT = a.d_final_state; p.dh0 = a.d_initial_state;
    p.ckpt = a.checkpoints;
    p.dlam = static_cast<float*>(a.scratch);
    p.cu = a.cu_seqlens; p.cu64 = a.cu_is_64; p.nseq = (int)a.nseq; p.seqlen = a.seqlen;
    p.nrows = ax.nrows; p.nb = ax.nb;
    p.D = (int)a.nchan; p.dtiles = linrec_host::ceil_div_i(a.nchan, kGatedChannels); p.units = p.dtiles * p.nb;
    p.nck = linrec_host::ceil_div_i(ax.nrows, kGatedCheckpoint);
    p.reverse = a.reverse != 0;
    p.header = static_cast<uint32_t*>(workspace);
    p.desc = reinterpret_cast<linrec::TileDesc*>(static_cast<char*>(workspace) + linrec::kHeaderBytes);
    p.wait_budget = (long long)wait_ms * (long long)dev.clock_khz;

    const int size = a.dtype == LINREC_DTYPE_F32 ? 4 : 2;
    const void* in[4] = {a.x, a.forget, decay ? a.input_gate : a.x, bwd ? a.dy : a.x};
    const int64_t stride[4] = {a.x_stride, a.forget_stride, decay ? a.input_gate_stride : a.x_stride, bwd ? a.dy_stride : a.x_stride};
    const void* out[4] = {bwd ? a.dx : a.y, bwd ? a.dforget : a.y, bwd && decay ? a.dinput_gate : a.y, a.y};
    p.pair = 1;
    for (int i = 0; i < (bwd ? (decay ? 3 : 2) : 1); ++i) p.pair &= on_boundary(out[i], a.nchan, size, 2 * size);
    int load = linrec::kLoadTma;
    for (int i = 0; i < 4; ++i) {
        if (!on_boundary(in[i], stride[i], size, 4)) load = linrec::kLoadAny;
        else if (load == linrec::kLoadTma &&
                 (!on_boundary(in[i], stride[i], size, 16) || !p.pair || (double)stride[i] * size * (double)ax.nrows >= 1e12))
            load = linrec::kLoadWord;
    }
    // (4-byte copies of 16-bit rows, two bytes to a channel, are slower than plain loads, eight rows of them at a time:
    // (4, 4096, 4002) bf16 forget form 197 / 559 us and 173 / 347)
    if (load == linrec::kLoadWord && size == 2) load = linrec::kLoadAny;
    // as many columns as the small CTAs of an SM-filling grid, or fewer, larger ones
    const int shape = p.units < (bwd ? 2 : 3) * dev.sm_count;
    auto pick = [&](int how) {
        return a.dtype == LINREC_DTYPE_F32 ? linrec_variants::gated_kernel_f32(bwd, decay, how, shape)
             : a.dtype == LINREC_DTYPE_BF16 ? linrec_variants::gated_kernel_bf16(bwd, decay, how, shape)
                                            : linrec_variants::gated_kernel_f16(bwd, decay, how, shape);
    };
    linrec_variants::GatedKernel kernel = pick(load);
    if (load == linrec::kLoadTma && p.units <= dev.sm_count) {
        const linrec_variants::GatedKernel of_cluster = pick(linrec::kLoadCluster);
        rc = cluster_size(of_cluster, p.units, linrec_host::ceil_div_i(ax.nrows, of_cluster.rows), dev.sm_count, p.cluster);
        if (rc != LINREC_OK) return rc;
        if (p.cluster > 0) {
            load = linrec::kLoadCluster;
            kernel = of_cluster;
        }
    }
    p.nk = linrec_host::ceil_div_i(ax.nrows, kernel.rows);
    int occ = 0;
    rc = linrec_host::occupancy(reinterpret_cast<const void*>(kernel.fn), kernel.threads, (size_t)kernel.smem, occ);
    if (rc != LINREC_OK) return rc;
    const long long slots = (long long)dev.sm_count * occ;
    p.tiles_per_job = tiles_per_job(p.units, p.nk, slots);
    p.jobs = p.cluster > 0 ? p.cluster : linrec_host::ceil_div_i(p.nk, p.tiles_per_job);
    p.ntickets = (long long)p.jobs * p.units;
    linrec::GatedMaps maps{};
    if (linrec::gated_bulk(load)) {
        CUtensorMap* to[4] = {&maps.x, &maps.f, &maps.i, &maps.dy};
        for (int i = 0; i < 4; ++i) {
            if ((i == 2 && !decay) || (i == 3 && !bwd)) continue;
            rc = make_map(to[i], in[i], stride[i], p, kernel.rows, a.dtype);
            if (rc != LINREC_OK) return rc;
        }
    }
    long long grid = slots;
    if (grid > p.ntickets) grid = p.ntickets;
    if (p.cluster > 0) grid = (long long)p.units * p.cluster;
    // (a cluster of one is a plain CTA: it exchanges nothing)
    rc = linrec_host::launch_clusters("gated recurrence", p.cluster > 1 ? p.cluster : 0, kernel.fn, dim3((unsigned)grid), (unsigned)kernel.threads,
                                      (size_t)kernel.smem, stream, p, maps);
    if (rc != LINREC_OK || !bwd || !decay) return rc;
    return linrec_host::launch("decay gradient", linrec::gated_decay_grad_kernel, dim3((unsigned)linrec_host::ceil_div_i(a.nchan, 32)), 256, 0,
                               stream, (const float*)p.dlam, (long long)p.jobs * p.nb, p.D, p.decay, a.ddecay);
}

template <typename ST, int V, int ROWS>
int launch_step(const GatedStepParams& p, cudaStream_t stream)
{
    const dim3 grid((unsigned)linrec_host::ceil_div_i(p.rows, ROWS), (unsigned)linrec_host::ceil_div_i(p.D, linrec::kStepThreads * V));
    return linrec_host::launch("gated step", p.decay ? linrec::gated_step_kernel<ST, true, V, ROWS> : linrec::gated_step_kernel<ST, false, V, ROWS>,
                               grid, linrec::kStepThreads, 0, stream, p);
}
// Four channels per access where every row allows it; four rows per CTA once that still leaves 8 CTAs per SM
// ((512, 8192) bf16 decay form over a padded cache: 31.8 us with one row and single elements, 17.5 with these).
template <typename ST>
int launch_step(const GatedStepParams& p, bool four, int sms, cudaStream_t stream)
{
    const long long ctas = (long long)linrec_host::ceil_div_i(p.rows, 4) * linrec_host::ceil_div_i(p.D, linrec::kStepThreads * (four ? 4 : 1));
    const bool rows4 = ctas >= 8LL * sms;
    if (four) return rows4 ? launch_step<ST, 4, 4>(p, stream) : launch_step<ST, 4, 1>(p, stream);
    return rows4 ? launch_step<ST, 1, 4>(p, stream) : launch_step<ST, 1, 1>(p, stream);
}

}  // namespace

extern "C" {

size_t linrec_b200_gated_workspace_size(const linrec_gated_args* args)
{
    size_t n = linrec::kHeaderBytes;
    if (check(args) == LINREC_OK) {
        const Axes ax = axes_of(*args);
        const size_t tiles = (size_t)((ax.nrows + kGatedCheckpoint - 1) / kGatedCheckpoint) * ax.nb * (size_t)((args->nchan + kGatedChannels - 1) / kGatedChannels);
        n += tiles * kGatedChannels * sizeof(linrec::TileDesc);
    }
    return n;
}

size_t linrec_b200_gated_scratch_size(const linrec_gated_args* args)
{
    if (check(args) != LINREC_OK || !args->decay) return 0;
    return (size_t)linrec_b200_gated_checkpoint_rows(args) * (size_t)args->nchan * sizeof(float);
}

int64_t linrec_b200_gated_checkpoint_rows(const linrec_gated_args* args)
{
    if (check(args) != LINREC_OK) return 0;
    const Axes ax = axes_of(*args);
    return (ax.nrows + kGatedCheckpoint - 1) / kGatedCheckpoint * ax.nb;
}

int linrec_b200_gated_fwd(const linrec_gated_args* args, const linrec_opts* opts, void* workspace, size_t workspace_bytes, void* stream)
{
    return linrec_host::guarded([&] { return launch_gated(false, args, opts, workspace, workspace_bytes, stream); });
}

int linrec_b200_gated_bwd(const linrec_gated_args* args, const linrec_opts* opts, void* workspace, size_t workspace_bytes, void* stream)
{
    return linrec_host::guarded([&] { return launch_gated(true, args, opts, workspace, workspace_bytes, stream); });
}

int linrec_b200_gated_step(const void* x, const void* forget, const void* input_gate, int64_t x_stride, int64_t forget_stride,
                           int64_t input_gate_stride, const float* decay, float decay_scale, void* y, float* state,
                           int64_t state_stride, int64_t nslots, const void* slots, int slots_are_64, int64_t nrows, int64_t nchan,
                           int dtype, void* stream)
{
    return linrec_host::guarded([&]() -> int {
        if (!known_dtype(dtype)) return LINREC_ERR_NOT_IMPLEMENTED;
        if (nrows < 0 || nchan < 0 || nslots < 0 || nrows >= 0x7fffffffLL || nslots >= 0x7fffffffLL || nchan > 128LL * 65535)
            return LINREC_ERR_INVALID_ARG;
        if (!decay != !input_gate) return LINREC_ERR_INVALID_ARG;
        if (nrows == 0 || nchan == 0) return LINREC_OK;
        if (!x || !forget || !y || (!state && nslots > 0) || x_stride < nchan || forget_stride < nchan || state_stride < nchan ||
            (decay && input_gate_stride < nchan) || (!slots && nrows > nslots))
            return LINREC_ERR_INVALID_ARG;
        // blocks would read what others have already advanced
        const int size = dtype == LINREC_DTYPE_F32 ? 4 : 2;
        const Rows of_state{state, nslots, state_stride * 4, nchan * 4};
        for (const Rows& r : {Rows{x, nrows, x_stride * size, nchan * size}, Rows{forget, nrows, forget_stride * size, nchan * size},
                              Rows{input_gate, nrows, input_gate_stride * size, nchan * size}, Rows{y, nrows, nchan * size, nchan * size},
                              Rows{decay, 1, nchan * 4, nchan * 4}, Rows{slots, 1, nrows * (slots_are_64 ? 8 : 4), nrows * (slots_are_64 ? 8 : 4)}})
            if (rows_meet(r, of_state)) return LINREC_ERR_OVERLAP;
        if (!linrec_host::on_elements({x, forget, input_gate, y}, dtype == LINREC_DTYPE_F32 ? 4 : 2) || !linrec_host::on_elements({decay, state}, 4) ||
            !linrec_host::on_elements({slots}, slots_are_64 ? 8 : 4))
            return LINREC_ERR_INVALID_ARG;
        DeviceInfo dev;
        const int rc = linrec_host::device_facts(dev);
        if (rc != LINREC_OK) return rc;
        GatedStepParams p{};
        p.x = x; p.f = forget; p.ig = input_gate; p.sx = x_stride; p.sf = forget_stride; p.si = input_gate_stride;
        p.y = y; p.decay = decay; p.scale = decay_scale; p.state = state; p.sstate = state_stride;
        p.slots = slots; p.slots64 = slots_are_64; p.rows = (int)nrows; p.nslots = (int)nslots; p.D = (int)nchan;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool four = nchan % 4 == 0 && on_boundary(x, x_stride, size, 4 * size) && on_boundary(forget, forget_stride, size, 4 * size) &&
                          (!decay || on_boundary(input_gate, input_gate_stride, size, 4 * size)) && on_boundary(y, nchan, size, 4 * size) &&
                          on_boundary(state, state_stride, 4, 16);
        return dtype == LINREC_DTYPE_F32 ? launch_step<float>(p, four, dev.sm_count, s)
             : dtype == LINREC_DTYPE_BF16 ? launch_step<__nv_bfloat16>(p, four, dev.sm_count, s) : launch_step<__half>(p, four, dev.sm_count, s);
    });
}

}  // extern "C"

// Host side of the group norm (include/linrec_b200.h): argument checks and launches.
#include "norm_variants.h"
#include "host.h"

namespace {

using linrec::NormParams;

int check(const linrec_group_norm_args* a)
{
    if (!a || a->nsamples < 0 || a->positions < 0 || a->nchan < 0 || a->groups <= 0) return LINREC_ERR_INVALID_ARG;
    if (a->dtype != LINREC_DTYPE_F32 && a->dtype != LINREC_DTYPE_BF16 && a->dtype != LINREC_DTYPE_F16) return LINREC_ERR_NOT_IMPLEMENTED;
    if (a->activation < 0 || a->activation > 2) return LINREC_ERR_NOT_IMPLEMENTED;
    if (a->nchan % a->groups || a->nchan >= 0x40000000LL || !(a->eps > 0.0f)) return LINREC_ERR_INVALID_ARG;
    if (a->nsamples > 0 && a->positions > 0x3fffffffffffLL / a->nsamples) return LINREC_ERR_INVALID_ARG;
    if (a->nsamples > 0 && a->groups > 0x7fffffffLL / a->nsamples) return LINREC_ERR_INVALID_ARG;
    return LINREC_OK;
}

// How a problem is laid out; the scratch sizes follow from it, so it depends on sizes and alignment alone (the
// grid is sized for 148 SMs whatever the device).
constexpr long long kCtas = 148 * 3;

struct Plan {
    bool rows;
    int V;               // elements per thread and access: 8 on 16-byte boundaries, else 1
    int many;            // rows: 0 few, 1 many pieces per lane
    int lanes, gb, rp;   // rows
    int cpb, sub, slices, xblocks;
    long long yblocks;   // rows: CTAs along the rows; planes: slices of all samples
    long long parts;     // partial sums of the parameters' gradients
};

bool on_16(const void* p, int64_t stride, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0; }

Plan plan_of(const linrec_group_norm_args& a, bool aligned, bool bwd)
{
    Plan p{};
    const int c = (int)(a.nchan / a.groups);
    const int size = a.dtype == LINREC_DTYPE_F32 ? 4 : 2;
    p.V = aligned && c % 8 == 0 && a.nchan * size % 16 == 0 ? 8 : 1;
    const int pieces = (c + p.V - 1) / p.V;
    if (a.positions == 1 && pieces <= (p.V == 8 ? 128 : 1024)) {
        p.rows = true;
        const int* nv = linrec_variants::kNormPieces[p.V == 8];
        p.many = pieces > 32 * nv[0];
        // (with many single elements per lane the kernels take a group to be a whole warp)
        p.lanes = p.many && p.V == 1 ? 32 : 1;
        while (p.lanes < 32 && p.lanes * nv[p.many] < pieces) p.lanes *= 2;
        const int slots = linrec::kNormThreads / p.lanes;
        p.gb = (int)(a.groups < slots ? a.groups : slots);
        p.rp = slots / p.gb;
        p.xblocks = linrec_host::ceil_div_i(a.groups, p.gb);
        // as many CTAs as are resident at a time, so that all of them take the same number of rows
        const long long ctas = 148 * (p.V == 1 ? (p.many ? 3 : 4) : p.many ? (bwd ? 1 : 2) : bwd ? 2 : 4);
        const long long want = ctas / p.xblocks > 0 ? ctas / p.xblocks : 1, most = (a.nsamples + p.rp - 1) / p.rp;
        p.yblocks = p.parts = most < want ? most : want;
        return p;
    }
    const int wide = linrec::kNormThreads * p.V;
    if (c <= wide) {
        p.cpb = (int)(a.groups < wide / c ? a.groups : wide / c) * c;
        p.sub = 1;
        p.xblocks = linrec_host::ceil_div_i(a.nchan, p.cpb);
    } else {
        p.cpb = wide;
        p.sub = (c + wide - 1) / wide;
        p.xblocks = (int)a.groups * p.sub;
    }
    // slices of at least four rounds of a CTA's threads, and no more CTAs than fill the device once
    const int threads_per_row = p.cpb / p.V, Y = linrec::kNormThreads / threads_per_row > 0 ? linrec::kNormThreads / threads_per_row : 1;
    long long want = kCtas / ((long long)p.xblocks * a.nsamples), most = a.positions / (4 * Y);
    if (want > most) want = most;
    p.slices = (int)(want < 1 ? 1 : want);
    p.yblocks = a.nsamples * p.slices;
    const long long full = kCtas / p.xblocks > 0 ? kCtas / p.xblocks : 1;
    p.parts = p.yblocks < full ? p.yblocks : full;
    return p;
}

// Room for either alignment: a caller asks for the size before the kernels see the pointers.
size_t part_bytes(const linrec_group_norm_args& a, const Plan& p) { return (size_t)p.parts * (size_t)a.nchan * sizeof(float2); }
size_t group_bytes(const linrec_group_norm_args& a, const Plan& p)
{
    return p.rows ? 0 : (size_t)p.yblocks * p.sub * (size_t)a.groups * sizeof(float4);
}

int run(bool bwd, const NormParams& p, const Plan& pl, const linrec_variants::NormKernels& k, cudaStream_t stream)
{
    if (pl.rows) {
        const dim3 grid((unsigned)pl.xblocks, (unsigned)pl.yblocks);
        if (!bwd) return linrec_host::launch("group norm", k.rows_fwd[pl.many], grid, linrec::kNormThreads, 0, stream, p);
        const linrec_variants::NormFn fn = k.rows_bwd[pl.many];
        const size_t sums = (size_t)p.rp * p.gb * p.c * sizeof(float2), smem = p.part && (p.rp > 1 || pl.V == 1) ? sums : 0;
        int occ = 0;      // raises the limit of shared memory to the most the kernel can be asked for
        const int most = linrec::kNormThreads * pl.V * linrec_variants::kNormPieces[pl.V == 8][pl.many] * (int)sizeof(float2);
        const int rc = linrec_host::occupancy(reinterpret_cast<const void*>(fn), linrec::kNormThreads, (size_t)most, occ);
        if (rc != LINREC_OK) return rc;
        return linrec_host::launch("group norm backward", fn, grid, linrec::kNormThreads, smem, stream, p);
    }
    const dim3 grid((unsigned)(pl.xblocks * pl.yblocks));
    int rc;
    if (!bwd) {
        rc = linrec_host::launch("group norm statistics", k.stats, grid, linrec::kNormThreads, 0, stream, p);
        if (rc != LINREC_OK) return rc;
        return linrec_host::launch("group norm", k.apply, grid, linrec::kNormThreads, 0, stream, p);
    }
    rc = linrec_host::launch("group norm sums", k.sums, dim3((unsigned)(pl.xblocks * pl.parts)), linrec::kNormThreads, 0, stream, p);
    if (rc != LINREC_OK) return rc;
    return linrec_host::launch("group norm backward", k.dx, grid, linrec::kNormThreads, 0, stream, p);
}

int launch_norm(bool bwd, const linrec_group_norm_args* args, void* stream_)
{
    int rc = check(args);
    if (rc != LINREC_OK) return rc;
    const linrec_group_norm_args& a = *args;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (a.nchan == 0) return LINREC_OK;
    if (a.nsamples == 0 || a.positions == 0) {
        for (float* p : {a.dweight, a.dbias})
            if (bwd && p && cudaMemsetAsync(p, 0, (size_t)a.nchan * 4, stream) != cudaSuccess) {
                linrec_host::note_cuda_error("cudaMemsetAsync", cudaGetErrorString(cudaGetLastError()));
                return LINREC_ERR_CUDA;
            }
        return LINREC_OK;
    }
    if (!a.x || a.x_stride < a.nchan || (a.gate && a.gate_stride < a.nchan)) return LINREC_ERR_INVALID_ARG;
    if (!bwd && !a.y) return LINREC_ERR_INVALID_ARG;
    if (bwd && (!a.dy || a.dy_stride < a.nchan || !a.dx || !a.stats || (a.gate && !a.dgate))) return LINREC_ERR_INVALID_ARG;
    if (!linrec_host::on_elements({a.x, a.gate, a.y, a.dy, a.dx, a.dgate}, a.dtype == LINREC_DTYPE_F32 ? 4 : 2) ||
        !linrec_host::on_elements({a.weight, a.bias, a.dweight, a.dbias}, 4) || !linrec_host::on_elements({a.stats}, 8))
        return LINREC_ERR_INVALID_ARG;
    const size_t need = linrec_b200_group_norm_scratch_size(args, bwd);
    if (need && (!a.scratch || a.scratch_bytes < need || reinterpret_cast<uintptr_t>(a.scratch) % 16 != 0)) return LINREC_ERR_WORKSPACE;
    linrec_host::DeviceInfo dev;
    rc = linrec_host::device_facts(dev);
    if (rc != LINREC_OK) return rc;

    const int size = a.dtype == LINREC_DTYPE_F32 ? 4 : 2;
    bool aligned = on_16(a.x, a.x_stride, size) && (!a.gate || on_16(a.gate, a.gate_stride, size));
    if (!bwd) aligned = aligned && on_16(a.y, a.nchan, size);
    else aligned = aligned && on_16(a.dy, a.dy_stride, size) && on_16(a.dx, a.nchan, size) && (!a.gate || on_16(a.dgate, a.nchan, size));
    aligned = aligned && on_16(a.weight, 0, 1) && on_16(a.bias, 0, 1);
    const Plan pl = plan_of(a, aligned, bwd);
    if (!pl.rows && pl.yblocks > 0x7fffffffLL / pl.xblocks) return LINREC_ERR_INVALID_ARG;
    NormParams p{};
    p.x = a.x; p.gate = a.gate; p.dy = a.dy;
    p.sx = a.x_stride; p.sg = a.gate_stride; p.sdy = a.dy_stride;
    p.w = a.weight; p.b = a.bias; p.eps = a.eps; p.act = a.activation;
    p.n = a.nsamples; p.L = a.positions; p.C = (int)a.nchan; p.G = (int)a.groups; p.c = (int)(a.nchan / a.groups);
    p.stats = reinterpret_cast<float2*>(a.stats);
    p.y = bwd ? nullptr : a.y; p.dx = a.dx; p.dgate = a.dgate;
    p.lanes = pl.lanes; p.gb = pl.gb; p.rp = pl.rp; p.cpb = pl.cpb; p.sub = pl.sub; p.slices = pl.slices; p.xblocks = pl.xblocks; p.per = pl.slices > 0 ? (a.positions + pl.slices - 1) / pl.slices : 0;
    char* scratch = static_cast<char*>(a.scratch);
    p.gpart = reinterpret_cast<float4*>(scratch);
    const bool params = bwd && (a.dweight || a.dbias);
    p.part = params ? reinterpret_cast<float2*>(scratch + group_bytes(a, pl)) : nullptr;
    const bool gate = a.gate != nullptr;
    rc = run(bwd, p, pl, a.dtype == LINREC_DTYPE_F32 ? linrec_variants::norm_kernels_f32(pl.V, gate, a.activation)
                       : a.dtype == LINREC_DTYPE_BF16 ? linrec_variants::norm_kernels_bf16(pl.V, gate, a.activation)
                                                      : linrec_variants::norm_kernels_f16(pl.V, gate, a.activation), stream);
    if (rc != LINREC_OK || !params) return rc;
    return linrec_host::launch("group norm parameters", linrec::norm_param_sum_kernel, dim3((unsigned)linrec_host::ceil_div_i(p.C, 32)), 1024, 0,
                               stream, (const float2*)p.part, (int)pl.parts, p.C, a.dweight, a.dbias);
}

}  // namespace

extern "C" {

size_t linrec_b200_group_norm_scratch_size(const linrec_group_norm_args* args, int bwd)
{
    if (check(args) != LINREC_OK || args->nsamples == 0 || args->positions == 0 || args->nchan == 0) return 0;
    size_t most = 0;
    for (bool aligned : {false, true}) {
        const Plan p = plan_of(*args, aligned, bwd != 0);
        const size_t n = group_bytes(*args, p) + (bwd && (args->dweight || args->dbias) ? part_bytes(*args, p) : 0);
        most = n > most ? n : most;
    }
    return most;
}

int linrec_b200_group_norm_fwd(const linrec_group_norm_args* args, void* stream) { return linrec_host::guarded([&] { return launch_norm(false, args, stream); }); }
int linrec_b200_group_norm_bwd(const linrec_group_norm_args* args, void* stream) { return linrec_host::guarded([&] { return launch_norm(true, args, stream); }); }

}  // extern "C"

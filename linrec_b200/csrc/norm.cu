// Host side of the group norm (include/linrec_b200.h): argument checks and launches.
#include "norm_kernels.cuh"
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

int parts_of(const linrec_group_norm_args& a)
{
    const long long rows = a.nsamples * a.positions;
    return (int)(rows < 256 ? (rows > 0 ? rows : 1) : 256);
}

NormParams params_of(const linrec_group_norm_args& a)
{
    NormParams p{};
    p.x = a.x; p.gate = a.gate; p.dy = a.dy;
    p.sx = a.x_stride; p.sg = a.gate_stride; p.sdy = a.dy_stride;
    p.w = a.weight; p.b = a.bias; p.eps = a.eps; p.act = a.activation;
    p.n = a.nsamples; p.L = a.positions; p.C = (int)a.nchan; p.G = (int)a.groups; p.c = (int)(a.nchan / a.groups);
    p.stats = reinterpret_cast<float2*>(a.stats);
    p.y = a.y; p.dx = a.dx; p.dgate = a.dgate;
    p.part = static_cast<float2*>(a.scratch); p.parts = parts_of(a);
    p.dw = a.dweight; p.db = a.dbias;
    return p;
}

template <typename ST>
int run(bool bwd, const NormParams& p, cudaStream_t stream)
{
    const dim3 units((unsigned)(p.n * p.G));
    if (!bwd) return linrec_host::launch("group norm", linrec::norm_fwd_kernel<ST>, units, 256, 0, stream, p);
    int rc = linrec_host::launch("group norm backward", linrec::norm_bwd_kernel<ST>, units, 256, 0, stream, p);
    if (rc != LINREC_OK || (!p.dw && !p.db)) return rc;
    rc = linrec_host::launch("group norm parameters", linrec::norm_param_kernel<ST>,
                             dim3((unsigned)linrec_host::ceil_div_i(p.C, 128), (unsigned)p.parts), 128, 0, stream, p);
    if (rc != LINREC_OK) return rc;
    return linrec_host::launch("group norm parameters", linrec::norm_param_sum_kernel, dim3((unsigned)linrec_host::ceil_div_i(p.C, 32)), 256,
                               0, stream, (const float2*)p.part, p.parts, p.C, p.dw, p.db);
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
    if (bwd && (a.dweight || a.dbias) && (!a.scratch || a.scratch_bytes < linrec_b200_group_norm_scratch_size(args)))
        return LINREC_ERR_INVALID_ARG;
    linrec_host::DeviceInfo dev;
    rc = linrec_host::device_facts(dev);
    if (rc != LINREC_OK) return rc;
    const NormParams p = params_of(a);
    return a.dtype == LINREC_DTYPE_F32 ? run<float>(bwd, p, stream)
         : a.dtype == LINREC_DTYPE_BF16 ? run<__nv_bfloat16>(bwd, p, stream) : run<__half>(bwd, p, stream);
}

}  // namespace

extern "C" {

size_t linrec_b200_group_norm_scratch_size(const linrec_group_norm_args* args)
{
    if (check(args) != LINREC_OK) return 0;
    return (size_t)parts_of(*args) * (size_t)args->nchan * sizeof(float2);
}

int linrec_b200_group_norm_fwd(const linrec_group_norm_args* args, void* stream) { return launch_norm(false, args, stream); }
int linrec_b200_group_norm_bwd(const linrec_group_norm_args* args, void* stream) { return launch_norm(true, args, stream); }

}  // extern "C"

// What the host files of the library share: device facts, launch bookkeeping and error texts, defined in
// capi.cu (gated.cu and norm.cu hold the host side of the operators of those names).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

#include "../../include/linrec_b200.h"

namespace linrec_host {

struct DeviceInfo {
    int sm_count = 0;
    int clock_khz = 0;
    int max_smem_optin = 0;
};

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

int device_facts(DeviceInfo& out);
// Resident CTAs per SM; the first query for a kernel also raises its dynamic shared-memory limit.
int occupancy(const void* fn, int threads, size_t smem, int& out);
// Clusters of `size` CTAs that can be resident at a time.
int active_clusters(const void* fn, int threads, size_t smem, int size, int& out);
EncodeTiledFn encode_tiled_fn();
void note_cuda_error(const char* where, const char* what);
// Result of a kernel launch: reads (and clears) the runtime's last error.
int launch_result(const char* where);
void count_launch();

// Body of a C entry point: no C++ exception leaves it.
template <typename Body>
int guarded(Body body) noexcept
{
    try {
        return body();
    } catch (...) {
        note_cuda_error("host", "out of memory or another C++ exception");
        return LINREC_ERR_CUDA;
    }
}

// Do all of the pointers (null ones included) lie on boundaries of `size` bytes?  Kernels that meet another address fault.
inline bool on_elements(std::initializer_list<const void*> pointers, int size)
{
    for (const void* p : pointers)
        if (reinterpret_cast<uintptr_t>(p) % (unsigned)size != 0) return false;
    return true;
}

inline int ceil_div_i(long long a, long long b) { return (int)((a + b - 1) / b); }

// Launch with the programmatic-stream-serialization attribute: the kernels call griddepcontrol.wait before
// their first access to global memory (ptx.cuh).
template <typename... KArgs, typename... Args>
int launch_clusters(const char* where, int cluster, void (*fn)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t stream, Args&&... args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1u;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    (void)cudaLaunchKernelEx(&cfg, fn, static_cast<Args&&>(args)...);
    const int rc = launch_result(where);
    if (rc == LINREC_OK) count_launch();
    return rc;
}

template <typename... KArgs, typename... Args>
int launch(const char* where, void (*fn)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t stream, Args&&... args)
{
    return launch_clusters(where, 0, fn, grid, block, smem, stream, static_cast<Args&&>(args)...);
}

}  // namespace linrec_host

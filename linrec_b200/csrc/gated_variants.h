// The compiled kernels of the gated recurrence: one translation unit per storage type (variants_gated_*.cu).
#pragma once
#include "gated_kernels.cuh"

namespace linrec_variants {

using GatedFn = void (*)(const linrec::GatedParams, const linrec::GatedMaps);

struct GatedKernel {
    GatedFn fn;
    int smem;        // dynamic shared memory
    int rows;        // positions per tile
    int threads;
};

// shape: 0 or 1 (GatedTile); 32-bit operands and rows off 16-byte boundaries have one shape each.
GatedKernel gated_kernel_f32(bool bwd, bool decay, int load, int shape);
GatedKernel gated_kernel_bf16(bool bwd, bool decay, int load, int shape);
GatedKernel gated_kernel_f16(bool bwd, bool decay, int load, int shape);

template <typename ST, bool DECAY, int SHAPE, int LOAD>
GatedKernel gated_pick(bool bwd)
{
    using namespace linrec;
    using F = GatedTile<ST, DECAY, false, SHAPE>;
    using B = GatedTile<ST, DECAY, true, SHAPE>;
    if (bwd) return {gated_bwd_kernel<ST, DECAY, SHAPE, LOAD>, B::kDynSmem, B::R, B::threads(LOAD)};
    return {gated_fwd_kernel<ST, DECAY, SHAPE, LOAD>, F::kDynSmem, F::R, F::threads(LOAD)};
}

template <typename ST, bool DECAY>
GatedKernel gated_pick(bool bwd, int load, int shape)
{
    using namespace linrec;
    if constexpr (sizeof(ST) == 4) {
        // 32-bit elements always lie on 4-byte boundaries
        if (load == kLoadCluster) return gated_pick<ST, DECAY, 1, kLoadCluster>(bwd);
        if (load == kLoadTma) return gated_pick<ST, DECAY, 1, kLoadTma>(bwd);
        return gated_pick<ST, DECAY, 1, kLoadWord>(bwd);
    } else {
        if (load == kLoadCluster) return gated_pick<ST, DECAY, 1, kLoadCluster>(bwd);
        if (load == kLoadTma) return shape ? gated_pick<ST, DECAY, 1, kLoadTma>(bwd) : gated_pick<ST, DECAY, 0, kLoadTma>(bwd);
        return gated_pick<ST, DECAY, 0, kLoadAny>(bwd);
    }
}

template <typename ST>
GatedKernel gated_pick(bool bwd, bool decay, int load, int shape)
{
    return decay ? gated_pick<ST, true>(bwd, load, shape) : gated_pick<ST, false>(bwd, load, shape);
}

}  // namespace linrec_variants

// The compiled kernels of the gated recurrence: one translation unit per storage type (variants_gated_*.cu).
#pragma once
#include "gated_kernels.cuh"

namespace linrec_variants {

using GatedFn = void (*)(const linrec::GatedParams, const linrec::GatedMaps);

struct GatedKernel {
    GatedFn fn;
    int smem;        // dynamic shared memory
    int rows;        // positions per tile
};

GatedKernel gated_kernel_f32(bool bwd, bool decay, int load);
GatedKernel gated_kernel_bf16(bool bwd, bool decay, int load);
GatedKernel gated_kernel_f16(bool bwd, bool decay, int load);

template <typename ST, bool DECAY, int LOAD>
GatedKernel gated_pick(bool bwd)
{
    using namespace linrec;
    if (bwd) return {gated_bwd_kernel<ST, DECAY, LOAD>, GatedTile<ST, DECAY, true>::kDynSmem, GatedTile<ST, DECAY, true>::R};
    return {gated_fwd_kernel<ST, DECAY, LOAD>, GatedTile<ST, DECAY, false>::kDynSmem, GatedTile<ST, DECAY, false>::R};
}

template <typename ST>
GatedKernel gated_pick(bool bwd, bool decay, int load)
{
    using namespace linrec;
    if (load == kLoadTma) return decay ? gated_pick<ST, true, kLoadTma>(bwd) : gated_pick<ST, false, kLoadTma>(bwd);
    // 32-bit elements always lie on 4-byte boundaries
    if (sizeof(ST) == 4 || load == kLoadWord) return decay ? gated_pick<ST, true, kLoadWord>(bwd) : gated_pick<ST, false, kLoadWord>(bwd);
    if constexpr (sizeof(ST) == 2) return decay ? gated_pick<ST, true, kLoadAny>(bwd) : gated_pick<ST, false, kLoadAny>(bwd);
}

}  // namespace linrec_variants

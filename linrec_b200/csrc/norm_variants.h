// The compiled kernels of the group norm: one translation unit per storage type (variants_norm_*.cu).
#pragma once
#include "norm_kernels.cuh"

namespace linrec_variants {

using NormFn = void (*)(const linrec::NormParams);

// Entry points for one combination of access width, gate and activation.
struct NormKernels {
    NormFn rows_fwd[2], rows_bwd[2];      // few / many pieces per lane
    NormFn stats, apply, sums, dx;        // planes
};

NormKernels norm_kernels_f32(int V, bool gate, int act);
NormKernels norm_kernels_bf16(int V, bool gate, int act);
NormKernels norm_kernels_f16(int V, bool gate, int act);

constexpr int kNormPieces[2][2] = {{8, 32}, {1, 4}};      // [V == 8][few / many]

template <typename ST, int V, bool GATE, int ACT>
NormKernels norm_pick()
{
    using namespace linrec;
    NormKernels k;
    if constexpr (V == 8) {
        k.rows_fwd[0] = norm_rows_fwd_kernel<ST, 1, GATE, ACT>;
        k.rows_fwd[1] = norm_rows_fwd_kernel<ST, 4, GATE, ACT>;
        k.rows_bwd[0] = norm_rows_bwd_kernel<ST, 1, GATE, ACT>;
        k.rows_bwd[1] = norm_rows_bwd_kernel<ST, 4, GATE, ACT>;
    } else {
        k.rows_fwd[0] = norm_rows1_fwd_kernel<ST, 8, GATE, ACT>;
        k.rows_fwd[1] = norm_rows1_fwd_kernel<ST, 32, GATE, ACT>;
        k.rows_bwd[0] = norm_rows1_bwd_kernel<ST, 8, GATE, ACT>;
        k.rows_bwd[1] = norm_rows1_bwd_kernel<ST, 32, GATE, ACT>;
    }
    k.stats = norm_planes_stats_kernel<ST, V>;
    k.apply = norm_planes_apply_kernel<ST, V, GATE, ACT>;
    k.sums = norm_planes_sums_kernel<ST, V, GATE, ACT>;
    k.dx = norm_planes_dx_kernel<ST, V, GATE, ACT>;
    return k;
}

template <typename ST, int V, bool GATE>
NormKernels norm_pick(int act)
{
    using namespace linrec;
    return act == kActNone ? norm_pick<ST, V, GATE, kActNone>() : act == kActSilu ? norm_pick<ST, V, GATE, kActSilu>()
                                                                                  : norm_pick<ST, V, GATE, kActSigmoid>();
}

template <typename ST>
NormKernels norm_pick(int V, bool gate, int act)
{
    if (V == 8) return gate ? norm_pick<ST, 8, true>(act) : norm_pick<ST, 8, false>(act);
    return gate ? norm_pick<ST, 1, true>(act) : norm_pick<ST, 1, false>(act);
}

}  // namespace linrec_variants

#include "norm_variants.h"

namespace linrec_variants {
NormKernels norm_kernels_bf16(int V, bool gate, int act) { return norm_pick<__nv_bfloat16>(V, gate, act); }
}  // namespace linrec_variants

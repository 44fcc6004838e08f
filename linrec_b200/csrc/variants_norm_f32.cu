#include "norm_variants.h"

namespace linrec_variants {
NormKernels norm_kernels_f32(int V, bool gate, int act) { return norm_pick<float>(V, gate, act); }
}  // namespace linrec_variants

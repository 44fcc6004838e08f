#include "norm_variants.h"

namespace linrec_variants {
NormKernels norm_kernels_f16(int V, bool gate, int act) { return norm_pick<__half>(V, gate, act); }
}  // namespace linrec_variants

#include "gated_variants.h"

namespace linrec_variants {
GatedKernel gated_kernel_bf16(bool bwd, bool decay, int load, int shape) { return gated_pick<__nv_bfloat16>(bwd, decay, load, shape); }
}  // namespace linrec_variants

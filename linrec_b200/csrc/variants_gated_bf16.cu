#include "gated_variants.h"

namespace linrec_variants {
GatedKernel gated_kernel_bf16(bool bwd, bool decay, int load) { return gated_pick<__nv_bfloat16>(bwd, decay, load); }
}  // namespace linrec_variants

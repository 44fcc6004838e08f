#include "gated_variants.h"

namespace linrec_variants {
GatedKernel gated_kernel_f32(bool bwd, bool decay, int load) { return gated_pick<float>(bwd, decay, load); }
}  // namespace linrec_variants

#include "gated_variants.h"

namespace linrec_variants {
GatedKernel gated_kernel_f16(bool bwd, bool decay, int load, int shape) { return gated_pick<__half>(bwd, decay, load, shape); }
}  // namespace linrec_variants

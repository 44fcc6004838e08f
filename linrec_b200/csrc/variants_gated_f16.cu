#include "gated_variants.h"

namespace linrec_variants {
GatedKernel gated_kernel_f16(bool bwd, bool decay, int load) { return gated_pick<__half>(bwd, decay, load); }
}  // namespace linrec_variants

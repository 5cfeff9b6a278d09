// layer_norm_f16.hip -- the layer norm kernels for f16 rows.
#include "layer_norm_kernel.h"

namespace spc {
hipError_t ln_forward_f16(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_forward<SPC_F16>(s, p, blocks);
}
hipError_t ln_backward_f16(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_backward<SPC_F16>(s, p, blocks);
}
}  // namespace spc

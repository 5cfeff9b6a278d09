// layer_norm_bf16.hip -- the layer norm kernels for bf16 rows.
#include "layer_norm_kernel.h"

namespace spc {
hipError_t ln_forward_bf16(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_forward<SPC_BF16>(s, p, blocks);
}
hipError_t ln_backward_bf16(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_backward<SPC_BF16>(s, p, blocks);
}
}  // namespace spc

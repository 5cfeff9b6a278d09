// layer_norm_f32.hip -- the layer norm kernels for f32 rows.
#include "layer_norm_kernel.h"

namespace spc {
hipError_t ln_forward_f32(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_forward<SPC_F32>(s, p, blocks);
}
hipError_t ln_backward_f32(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_backward<SPC_F32>(s, p, blocks);
}
}  // namespace spc

// lora_f32.hip -- the adapters' kernels for f32 rows.
#include "lora_kernel.h"

namespace spc {
hipError_t lora_forward_f32(hipStream_t s, const LoraArgs& p, int mode, int mt, dim3 grid) {
    return lora_forward<SPC_F32>(s, p, mode, mt, grid);
}
hipError_t lora_back_out_f32(hipStream_t s, const LoraBackArgs& p, dim3 grid) {
    return lora_back_out<SPC_F32>(s, p, grid);
}
hipError_t lora_back_in_f32(hipStream_t s, const LoraBackArgs& p, dim3 grid) {
    return lora_back_in<SPC_F32>(s, p, grid);
}
}  // namespace spc

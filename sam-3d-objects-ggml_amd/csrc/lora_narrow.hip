// lora_narrow.hip -- rows of fewer than eight elements, narrower than the 16 bytes
// that lora_kernel.h's loads take of one, copied to rows of eight in the workspace
// (zeros behind the row's end add nothing to any sum), and results back.
#include <algorithm>

#include "lora_kernel.h"

namespace spc {

namespace {

// A thread an element of the copies; grid y: the arrays.
template <typename S>
__global__ __launch_bounds__(kLoraThreads) void lora_copy_kernel(LoraCopies q) {
    const LoraCopy p = q.job[blockIdx.y];
    const uint32_t all = (uint32_t)(p.rows * p.fill);
    for (uint32_t i = blockIdx.x * kLoraThreads + threadIdx.x; i < all; i += gridDim.x * kLoraThreads) {
        const uint32_t row = i / (uint32_t)p.fill, col = i - row * (uint32_t)p.fill;
        S v = 0;
        if ((int)col < p.width) v = static_cast<const S*>(p.src)[(int64_t)row * p.src_stride + col];
        static_cast<S*>(p.dst)[(int64_t)row * p.dst_stride + col] = v;
    }
}

}  // namespace

hipError_t lora_copy(hipStream_t s, int dt, const LoraCopies& q) {
    int64_t most = 0;
    for (int i = 0; i < q.jobs; ++i) most = std::max(most, q.job[i].rows * q.job[i].fill);
    if (!most) return hipSuccess;
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div(most, kLoraThreads), 1 << 14), (unsigned)q.jobs);
    if (dt == SPC_F32) lora_copy_kernel<uint32_t><<<grid, kLoraThreads, 0, s>>>(q);
    else lora_copy_kernel<uint16_t><<<grid, kLoraThreads, 0, s>>>(q);
    return hipGetLastError();
}

}  // namespace spc

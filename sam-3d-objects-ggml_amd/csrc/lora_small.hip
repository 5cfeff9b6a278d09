// lora_small.hip -- the adapters where the rows' or the outputs' width is below
// eight, narrower than the 16 bytes that lora_kernel.h's loads take of a row: plain
// sums, a block a row, a thread an element of the gradients (sums in 64 bits).
// Launches and the rows' latency bound them (1000 x 4 -> 4, rank 4).
#include <algorithm>

#include "lora_kernel.h"

namespace spc {

namespace {

template <int DT>
__device__ __forceinline__ float lora_get(const void* p, int64_t i) {
    if constexpr (DT == SPC_F32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == SPC_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}

template <int DT>
__device__ __forceinline__ void lora_put(void* p, int64_t i, float v) {
    if constexpr (DT == SPC_F32) static_cast<float*>(p)[i] = v;
    else if constexpr (DT == SPC_BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(v);
    else static_cast<uint16_t*>(p)[i] = f32_to_f16_bits(v);
}

struct LoraDrop {
    const int64_t* seed;
    uint32_t drop;
    float factor;

    __device__ float apply(float v, int64_t row, int64_t col, int64_t c) const {
        if (!drop) return v;
        const u32x4 ones = drop_ones(philox7(drop_key(seed), (uint64_t)(row * ((c + 7) / 8) + col / 8)), drop);
        return ones[col % 8 / 2] >> (16 * (col & 1)) & 1 ? v * factor : 0.0f;
    }
};

// out[row, j] = s sum over i of d(x)[row, i] w_a(i, j); one block a row.
template <int DT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraItems it, const void* x, int64_t stride,
                                                          int64_t c, const void* w, int64_t w_i, int64_t w_j,
                                                          int64_t r, const float* scale, LoraDrop d,
                                                          float* out) {
    for (int64_t row = blockIdx.x; row < it.n; row += gridDim.x) {
        const int64_t a = it.find<1>(row, 0).adapter;
        for (int64_t j = threadIdx.x / 64; j < r; j += 4) {
            float sum = 0.0f;
            if (a >= 0)
                for (int64_t i = threadIdx.x % 64; i < c; i += 64)
                    sum += d.apply(lora_get<DT>(x, row * stride + i), row, i, c) *
                           lora_get<DT>(w, a * c * r + i * w_i + j * w_j);
            for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
            if (a >= 0 && scale) sum *= scale[a];
            if (threadIdx.x % 64 == 0) out[row * r + j] = sum;
        }
    }
}

// y[row, i] = base[row, i] + d(s sum over j of h[row, j] w_a(i, j)).
template <int DT>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraItems it, const float* h, int64_t r,
                                                          const void* w, int64_t w_i, int64_t w_j,
                                                          const float* scale, LoraDrop d, const void* base,
                                                          int64_t base_stride, int64_t c, void* y) {
    for (int64_t row = blockIdx.x; row < it.n; row += gridDim.x) {
        const int64_t a = it.find<1>(row, 0).adapter;
        for (int64_t i = threadIdx.x; i < c; i += 256) {
            float sum = 0.0f;
            if (a >= 0) {
                for (int64_t j = 0; j < r; ++j) sum += h[row * r + j] * lora_get<DT>(w, a * c * r + i * w_i + j * w_j);
                if (scale) sum *= scale[a];
                sum = d.apply(sum, row, i, c);
            }
            if (base) {
                const float b = lora_get<DT>(base, row * base_stride + i);
                sum = a >= 0 ? sum + b : b;
            }
            lora_put<DT>(y, row * c + i, sum);
        }
    }
}

// dw_a(i, j) = s_a sum over a's rows of d(x)[row, i] g[row, j]; a thread an
// element.
template <int DT>
__global__ __launch_bounds__(256) void lora_weight_kernel(LoraItems it, const void* x, int64_t stride, int64_t c,
                                                          const float* g, int64_t r, const float* scale,
                                                          LoraDrop d, int64_t w_i, int64_t w_j, void* dw) {
    const int64_t a = blockIdx.y, t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= c * r) return;
    const int64_t i = t / r, j = t % r;
    double sum = 0.0;
    for (int64_t k = 0; k < it.items; ++k) {
        const int64_t v = it.off ? k + 1 : k;
        if (it.adapter(v) != a) continue;
        for (int64_t row = it.begin(v); row < it.end(v); ++row)
            sum += (double)d.apply(lora_get<DT>(x, row * stride + i), row, i, c) * g[row * r + j];
    }
    lora_put<DT>(dw, a * c * r + i * w_i + j * w_j, (float)(scale ? sum * scale[a] : sum));
}

template <int DT>
void small_forward(hipStream_t s, const LoraArgs& p) {
    const unsigned blocks = (unsigned)std::min<int64_t>(p.it.n, 1 << 16);
    const LoraDrop d = {p.seed, p.drop, p.factor};
    float* h = p.hidden ? p.hidden : p.part;
    lora_shrink_kernel<DT><<<blocks, 256, 0, s>>>(p.it, p.x, p.xs, p.c, p.down, 1, p.c, p.r, nullptr, d, h);
    lora_expand_kernel<DT><<<blocks, 256, 0, s>>>(p.it, h, p.r, p.up, p.r, 1, p.scale, LoraDrop{}, p.base, p.bs, p.o, p.y);
}

template <int DT>
void small_backward(hipStream_t s, const LoraBackArgs& p, void* ddown, void* dup) {
    const unsigned blocks = (unsigned)std::min<int64_t>(p.it.n, 1 << 16);
    const LoraDrop d = {p.seed, p.drop, p.factor};
    auto grid = [&](int64_t c) { return dim3((unsigned)ceil_div(c * p.r, 256), (unsigned)p.it.adapters); };
    if (blocks && p.u)
        lora_shrink_kernel<DT><<<blocks, 256, 0, s>>>(p.it, p.dy, p.dys, p.o, p.up, p.r, 1, p.r, p.scale, LoraDrop{}, p.u);
    if (blocks && p.dx)
        lora_expand_kernel<DT><<<blocks, 256, 0, s>>>(p.it, p.u, p.r, p.down, 1, p.c, nullptr, d, p.base, p.bs, p.c, p.dx);
    if (ddown) lora_weight_kernel<DT><<<grid(p.c), 256, 0, s>>>(p.it, p.x, p.xs, p.c, p.u, p.r, nullptr, d, 1, p.c, ddown);
    if (dup)
        lora_weight_kernel<DT><<<grid(p.o), 256, 0, s>>>(p.it, p.dy, p.dys, p.o, p.hidden, p.r, p.scale, LoraDrop{}, p.r, 1, dup);
}

}  // namespace

hipError_t lora_small_forward(hipStream_t s, int dt, const LoraArgs& p) {
    if (dt == SPC_BF16) small_forward<SPC_BF16>(s, p);
    else if (dt == SPC_F16) small_forward<SPC_F16>(s, p);
    else small_forward<SPC_F32>(s, p);
    return hipGetLastError();
}

hipError_t lora_small_backward(hipStream_t s, int dt, const LoraBackArgs& p, void* ddown, void* dup) {
    if (dt == SPC_BF16) small_backward<SPC_BF16>(s, p, ddown, dup);
    else if (dt == SPC_F16) small_backward<SPC_F16>(s, p, ddown, dup);
    else small_backward<SPC_F32>(s, p, ddown, dup);
    return hipGetLastError();
}

}  // namespace spc

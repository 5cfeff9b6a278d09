// lora.hip -- low-rank adapters of many batch items beside a shared projection
// (spc_lora) and their gradients (spc_lora_backward).  With a the adapter of a
// row's item, d = dropout (dropout.hip's mask; 1 without),
//
//   h = d(x) down_a^T,  y = base + s_a h up_a^T
//   u = s_a dy up_a,    dx = dx_base + d(u down_a)
//   ddown_a = sum over a's rows of u^T d(x),  dup_a = s_a sum of dy^T h
#include <algorithm>

#include "rows8.h"

namespace spc {

namespace {

constexpr int64_t kLoraMaxRank = 128, kLoraMaxItems = 65535, kLoraMaxAdapters = 65535;
constexpr int64_t kLoraMaxWidth = 1 << 24;

// Where the items' rows and adapters are.
struct LoraItems {
    const int64_t* off;    // [items + 1] or null: one item of all rows
    const int32_t* which;  // [items] or null: adapter 0
    int64_t items, adapters, n;

    // The adapter of a row, -1 for none.
    __device__ int64_t of_row(int64_t row) const {
        int64_t i = 0;
        if (off) {
            int64_t lo = 0, hi = items + 1;  // the number of offsets that are at most `row`
            while (lo < hi) {
                const int64_t m = (lo + hi) / 2;
                if (off[m] <= row) lo = m + 1;
                else hi = m;
            }
            i = lo - 1;
            if (i < 0 || i >= items) return -1;
        }
        const int64_t a = which ? which[i] : 0;
        return a >= 0 && a < adapters ? a : -1;
    }
    __device__ int64_t begin(int64_t i) const { return off ? min(max(off[i], (int64_t)0), n) : 0; }
    __device__ int64_t end(int64_t i) const { return off ? min(max(off[i + 1], (int64_t)0), n) : n; }
};

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
        const u32x4 w = philox7(drop_key(seed), (uint64_t)(row * ((c + 7) / 8) + col / 8));
        return drop_keeps(w, (int)(col % 8), drop) ? v * factor : 0.0f;
    }
};

// out[row, j] = s sum over i of d(x)[row, i] w_a(i, j); one block a row.
template <int DT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraItems it, const void* x, int64_t stride,
                                                          int64_t c, const void* w, int64_t w_i, int64_t w_j,
                                                          int64_t r, const float* scale, LoraDrop d,
                                                          float* out) {
    for (int64_t row = blockIdx.x; row < it.n; row += gridDim.x) {
        const int64_t a = it.of_row(row);
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
        const int64_t a = it.of_row(row);
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
        if ((it.which ? it.which[k] : 0) != a) continue;
        for (int64_t row = it.begin(k); row < it.end(k); ++row)
            sum += (double)d.apply(lora_get<DT>(x, row * stride + i), row, i, c) * g[row * r + j];
    }
    lora_put<DT>(dw, a * c * r + i * w_i + j * w_j, (float)(scale ? sum * scale[a] : sum));
}

// Checks what both entry points share.
int lora_args(const char* fn, int dtype, const void* x, int64_t x_stride, int64_t n,
              const spc_lora_params* q, LoraItems* it, LoraDrop* d) {
    if (!q || n < 0 || n > INT32_MAX || x_stride < 0 || q->in_features < 1 || q->out_features < 1 ||
        q->in_features > kLoraMaxWidth || q->out_features > kLoraMaxWidth || q->rank < 1 ||
        q->rank > kLoraMaxRank || q->n_adapters < 1 || q->n_adapters > kLoraMaxAdapters || q->n_items < 1 ||
        q->n_items > kLoraMaxItems) {
        set_last_error("%s: unsupported shape (below 2^31 rows, widths 1 to 2^24, ranks 1 to 128, 1 to 65535 "
                       "adapters and items) or a negative stride", fn);
        return SPC_BAD_SHAPE;
    }
    if (!float_dtype(dtype)) {
        set_last_error("%s: unknown dtype %d", fn, dtype);
        return SPC_BAD_ARG;
    }
    if (!(q->p >= 0.0 && q->p <= 1.0)) {
        set_last_error("%s: p must lie in [0, 1]", fn);
        return SPC_BAD_ARG;
    }
    if ((!q->offsets && q->n_items != 1) || (!q->adapters && q->n_adapters != 1)) {
        set_last_error("%s: more than one item needs offsets, more than one adapter the items' adapters", fn);
        return SPC_BAD_ARG;
    }
    const int64_t e = float_size(dtype);
    auto off = [](const void* p, int64_t by) { return (uintptr_t)p % by != 0; };
    d->drop = drop_threshold(q->p);
    d->factor = drop_factor(d->drop);
    d->seed = q->seed;
    if (!q->down || !q->up || (d->drop && !q->seed) || (n > 0 && !x) || off(x, e) || off(q->down, e) ||
        off(q->up, e) || off(q->scale, 4) || off(q->offsets, 8) || off(q->adapters, 4) || off(q->seed, 8)) {
        set_last_error("%s: null or misaligned pointer", fn);
        return SPC_BAD_ARG;
    }
    *it = LoraItems{q->offsets, q->adapters, q->n_items, q->n_adapters, n};
    return SPC_OK;
}

template <int DT>
void lora_forward(hipStream_t s, const LoraItems& it, const LoraDrop& d, const void* x, int64_t x_stride,
                  const spc_lora_params& q, const void* base, int64_t base_stride, void* y, float* hidden) {
    const unsigned blocks = (unsigned)std::min<int64_t>(it.n, 1 << 16);
    const int64_t in = q.in_features, out = q.out_features, r = q.rank;
    lora_shrink_kernel<DT><<<blocks, 256, 0, s>>>(it, x, x_stride, in, q.down, 1, in, r, nullptr, d, hidden);
    lora_expand_kernel<DT><<<blocks, 256, 0, s>>>(it, hidden, r, q.up, r, 1, q.scale, LoraDrop{}, base,
                                                  base_stride, out, y);
}

template <int DT>
void lora_backward(hipStream_t s, const LoraItems& it, const LoraDrop& d, const void* dy, int64_t dy_stride,
                   const void* x, int64_t x_stride, const float* hidden, const spc_lora_params& q,
                   const void* base, int64_t base_stride, void* dx, void* ddown, void* dup, float* u) {
    const unsigned blocks = (unsigned)std::min<int64_t>(it.n, 1 << 16);
    const int64_t in = q.in_features, out = q.out_features, r = q.rank;
    if (blocks && (dx || ddown))
        lora_shrink_kernel<DT><<<blocks, 256, 0, s>>>(it, dy, dy_stride, out, q.up, r, 1, r, q.scale,
                                                      LoraDrop{}, u);
    if (blocks && dx)
        lora_expand_kernel<DT><<<blocks, 256, 0, s>>>(it, u, r, q.down, 1, in, nullptr, d, base, base_stride,
                                                      in, dx);
    if (ddown)
        lora_weight_kernel<DT><<<dim3((unsigned)ceil_div(in * r, 256), (unsigned)q.n_adapters), 256, 0, s>>>(
            it, x, x_stride, in, u, r, nullptr, d, 1, in, ddown);
    if (dup)
        lora_weight_kernel<DT><<<dim3((unsigned)ceil_div(out * r, 256), (unsigned)q.n_adapters), 256, 0, s>>>(
            it, dy, dy_stride, out, hidden, r, q.scale, LoraDrop{}, r, 1, dup);
}

}  // namespace

}  // namespace spc

using namespace spc;

extern "C" {

size_t spc_lora_workspace_bytes(int dtype, int64_t n, int64_t n_items, int64_t in_features,
                                int64_t out_features, int64_t rank, int backward) {
    (void)backward;
    if (!float_dtype(dtype) || n < 0 || n > INT32_MAX || rank < 1 || rank > kLoraMaxRank || n_items < 1 ||
        n_items > kLoraMaxItems || in_features < 1 || in_features > kLoraMaxWidth || out_features < 1 ||
        out_features > kLoraMaxWidth)
        return 0;
    return (size_t)std::max<int64_t>(n, 1) * rank * sizeof(float);
}

int spc_lora(spc_stream_t stream, int dtype, const void* x, int64_t x_stride, int64_t n,
             const spc_lora_params* params, const void* base, int64_t base_stride, void* y, float* hidden,
             void* workspace, size_t workspace_bytes) {
    const char* fn = "spc_lora";
    hipStream_t s = static_cast<hipStream_t>(stream);
    LoraItems it;
    LoraDrop d;
    const int st = lora_args(fn, dtype, x, x_stride, n, params, &it, &d);
    if (st != SPC_OK) return st;
    if (n == 0) return SPC_OK;
    const spc_lora_params& q = *params;
    const int64_t e = float_size(dtype);
    auto off = [](const void* p, int64_t by) { return (uintptr_t)p % by != 0; };
    if (!y || off(y, e) || off(base, e) || off(hidden, 4) || base_stride < 0) {
        set_last_error("%s: null or misaligned pointer, or a negative stride", fn);
        return SPC_BAD_ARG;
    }
    if (!workspace || off(workspace, 16) ||
        workspace_bytes < spc_lora_workspace_bytes(dtype, n, q.n_items, q.in_features, q.out_features, q.rank, 0)) {
        set_last_error("%s: workspace missing, misaligned or too small", fn);
        return SPC_BAD_ARG;
    }
    float* h = hidden ? hidden : static_cast<float*>(workspace);
    if (dtype == SPC_BF16) lora_forward<SPC_BF16>(s, it, d, x, x_stride, q, base, base_stride, y, h);
    else if (dtype == SPC_F16) lora_forward<SPC_F16>(s, it, d, x, x_stride, q, base, base_stride, y, h);
    else lora_forward<SPC_F32>(s, it, d, x, x_stride, q, base, base_stride, y, h);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? SPC_OK : hip_status(err, "spc_lora launch");
}

int spc_lora_backward(spc_stream_t stream, int dtype, const void* dy, int64_t dy_stride, const void* x,
                      int64_t x_stride, const float* hidden, int64_t n, const spc_lora_params* params,
                      const void* dx_base, int64_t dx_base_stride, void* dx, void* ddown, void* dup,
                      void* workspace, size_t workspace_bytes) {
    const char* fn = "spc_lora_backward";
    hipStream_t s = static_cast<hipStream_t>(stream);
    LoraItems it;
    LoraDrop d;
    const int st = lora_args(fn, dtype, x, x_stride, n, params, &it, &d);
    if (st != SPC_OK) return st;
    const spc_lora_params& q = *params;
    const int64_t e = float_size(dtype);
    auto off = [](const void* p, int64_t by) { return (uintptr_t)p % by != 0; };
    if ((n > 0 && (!dy || (dup && !hidden))) || off(dy, e) || off(hidden, 4) || off(dx_base, e) || off(dx, e) ||
        off(ddown, e) || off(dup, e) || dy_stride < 0 || dx_base_stride < 0) {
        set_last_error("%s: null or misaligned pointer, or a negative stride", fn);
        return SPC_BAD_ARG;
    }
    if (!dx && !ddown && !dup) return SPC_OK;
    if (!workspace || off(workspace, 16) ||
        workspace_bytes < spc_lora_workspace_bytes(dtype, n, q.n_items, q.in_features, q.out_features, q.rank, 1)) {
        set_last_error("%s: workspace missing, misaligned or too small", fn);
        return SPC_BAD_ARG;
    }
    float* u = static_cast<float*>(workspace);
    if (dtype == SPC_BF16)
        lora_backward<SPC_BF16>(s, it, d, dy, dy_stride, x, x_stride, hidden, q, dx_base, dx_base_stride, dx, ddown, dup, u);
    else if (dtype == SPC_F16)
        lora_backward<SPC_F16>(s, it, d, dy, dy_stride, x, x_stride, hidden, q, dx_base, dx_base_stride, dx, ddown, dup, u);
    else
        lora_backward<SPC_F32>(s, it, d, dy, dy_stride, x, x_stride, hidden, q, dx_base, dx_base_stride, dx, ddown, dup, u);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? SPC_OK : hip_status(err, "spc_lora_backward launch");
}

}  // extern "C"

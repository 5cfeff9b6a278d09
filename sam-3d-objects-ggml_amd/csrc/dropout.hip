// dropout.hip -- y = residual + dropout(x), the mask computed from (seed, row,
// column) and never stored (spc_dropout); its gradient is the same call on dy.
//
// Bound by the rows' bytes: 62,710 x 1024 BF16 onto a residual 68 us (385 MB, 5.7 TB/s;
// a large copy 5.15), without 40; 21,766 x 101 F32 6 us (17.6 MB, partly from the
// memory's cache).  A mask kept as bytes would be an eighth to a quarter more of them
// in each direction.  The seven rounds of a group of eight, some 14 products of
// 32 by 32 bits, hide behind the loads.
#include <algorithm>

#include "rows8.h"

namespace spc {

namespace {

constexpr int kDropThreads = 256;

struct DropArgs {
    const void* x;
    int64_t x_stride;
    const void* res;
    int64_t res_stride;
    void* y;
    int64_t n, c, groups;          // groups of eight columns a row
    int64_t step_rows, step_group; // the grid's threads as rows and groups
    const int64_t* seed;
    uint32_t drop;
    float factor;
};

// A thread takes groups of eight columns, the grid's threads apart.
template <int DT, bool RES>
__global__ __launch_bounds__(kDropThreads) void drop_kernel(DropArgs p) {
    using R = Row8<DT>;
    using S = typename R::S;
    // (2^28 threads at most, and as many groups a row: spc_dropout's largest width)
    const uint32_t first = blockIdx.x * kDropThreads + threadIdx.x, groups = (uint32_t)p.groups;
    const DropKey key = p.drop ? drop_key(p.seed) : DropKey{};
    int64_t row = first / groups, g = first % groups;
    while (row < p.n) {
        const int64_t left = p.c - 8 * g;
        R x, r;
        x.load(static_cast<const S*>(p.x) + row * p.x_stride + 8 * g, left);
        if (RES) r.load(static_cast<const S*>(p.res) + row * p.res_stride + 8 * g, left);
        // (a dropped value counts as zero even if it is not finite)
        if (p.drop) x.mask(drop_ones(philox7(key, (uint64_t)(row * p.groups + g)), p.drop));
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float k = x.get(e) * p.factor;
            v[e] = RES ? k + r.get(e) : k;
        }
        x.set(v);
        x.store(static_cast<S*>(p.y) + row * p.c + 8 * g, left);
        row += p.step_rows;
        g += p.step_group;
        if (g >= p.groups) {
            g -= p.groups;
            ++row;
        }
    }
}

template <int DT>
void drop_launch(hipStream_t s, const DropArgs& p, unsigned blocks) {
    if (p.res) drop_kernel<DT, true><<<blocks, kDropThreads, 0, s>>>(p);
    else drop_kernel<DT, false><<<blocks, kDropThreads, 0, s>>>(p);
}

}  // namespace

}  // namespace spc

using namespace spc;

extern "C" int spc_dropout(spc_stream_t stream, int dtype, const void* x, int64_t x_stride, int64_t n,
                           int64_t c, double p, const int64_t* seed, const void* residual,
                           int64_t residual_stride, void* y) {
    const char* fn = "spc_dropout";
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n < 0 || n > INT32_MAX || c <= 0 || c > INT32_MAX || x_stride < 0 || residual_stride < 0) {
        set_last_error("%s: unsupported shape n=%lld c=%lld (below 2^31 rows, 1 to 2^31 - 1 columns) or "
                       "a negative stride", fn, (long long)n, (long long)c);
        return SPC_BAD_SHAPE;
    }
    if (!float_dtype(dtype)) {
        set_last_error("%s: unknown dtype %d", fn, dtype);
        return SPC_BAD_ARG;
    }
    if (!(p >= 0.0 && p <= 1.0)) {
        set_last_error("%s: p must lie in [0, 1]", fn);
        return SPC_BAD_ARG;
    }
    if (n == 0) return SPC_OK;
    DropArgs a{};
    a.drop = drop_threshold(p);
    auto off = [](const void* q, int64_t by) { return (uintptr_t)q % by != 0; };
    const int64_t e = float_size(dtype);
    if (!x || !y || (a.drop && !seed) || off(x, e) || off(y, e) || off(residual, e) || off(seed, 8)) {
        set_last_error("%s: null or misaligned pointer", fn);
        return SPC_BAD_ARG;
    }
    a.x = x;
    a.x_stride = x_stride;
    a.res = residual;
    a.res_stride = residual_stride;
    a.y = y;
    a.n = n;
    a.c = c;
    a.groups = ceil_div(c, 8);
    a.seed = seed;
    a.factor = drop_factor(a.drop);
    // (a group a thread: 62,710 x 1024 onto a residual 67.7 us, by 16,384 blocks 69.8, 8192
    // 71.0, 4096 74.1; beyond 2^20 blocks in turn)
    const int64_t blocks = std::min<int64_t>(ceil_div(n * a.groups, kDropThreads), 1 << 20);
    a.step_rows = blocks * kDropThreads / a.groups;
    a.step_group = blocks * kDropThreads % a.groups;
    if (dtype == SPC_BF16) drop_launch<SPC_BF16>(s, a, (unsigned)blocks);
    else if (dtype == SPC_F16) drop_launch<SPC_F16>(s, a, (unsigned)blocks);
    else drop_launch<SPC_F32>(s, a, (unsigned)blocks);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? SPC_OK : hip_status(err, "spc_dropout launch");
}

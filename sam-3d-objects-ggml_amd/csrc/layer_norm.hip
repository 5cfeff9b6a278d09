// layer_norm.hip -- entry points of the general row layer norm and its
// gradient (kernels: layer_norm_kernel.h).
#include <algorithm>

#include "layer_norm_kernel.h"

namespace spc {

namespace {

// Rows a block takes, a number of rounds of its teams.  Forward: up to four, so
// that the coefficients' loads and the first rows' latency are shared, as long
// as three blocks to a CU are left (us with 1 / 2 / 4 / 8 rounds: 62,710 x 128
// bf16 9.5 / 7.6 / 7.2 / -, x 512 29 / - / 22.0 / 21.6, x 1024 53 / - / 46.3 / 50.2;
// 11,774 x 2048 modulated 26.0 / 20.4 / 18.5 (3) / -).
// A launch holds below 2^32 threads, so rows past 2^23 blocks take more rounds.
inline int64_t ln_forward_rows(int64_t n, int teams) {
    const int64_t rounds = std::min<int64_t>(4, std::max<int64_t>(1, ceil_div(n, teams) / 768));
    return std::max(rounds, ceil_div(n, (int64_t)teams << 23)) * teams;
}

// Backward: 512 blocks, since every block ends by writing its channels' two
// sums, which the second kernel reads again (62,710 x 512 bf16: 40.4 + 6.4 us
// with 1,024 blocks, 39.7 + 4.1).
constexpr int64_t kLnBackwardBlocks = 512;
inline int64_t ln_backward_rows(int64_t n, int teams) {
    return std::max<int64_t>(1, ceil_div(n, kLnBackwardBlocks * teams)) * teams;
}

// Sums the slots of each item's chunks (16 channels and all of an item's
// slots a block, in a fixed order; eight slots in flight a thread: the pass is
// the latency of its loads) and forms the parameters' gradients from
// A = sum dz h, B = sum dz:
//   modulated: dscale = gamma A + beta B, dshift = B, and for the weight and
//   bias (1 + scale) A, (1 + scale) B into `sums`, added over the items by
//   ln_sum_items_kernel;  affine alone: dgamma = A, dbeta = B.
constexpr int kLnFinalChannels = 16, kLnFinalThreads = 1024;

struct LnFinal {
    const float* part;
    const int64_t* off;
    int64_t n;
    int rows_per;
    int c;
    const void *gamma, *beta, *scale;
    int p_dtype, m_dtype;
    int64_t m_stride;
    void *dgamma, *dbeta, *dscale, *dshift;
    float* sums;  // [items][2][c] or null
};

__global__ __launch_bounds__(kLnFinalThreads) void ln_finalize_kernel(LnFinal p) {
    constexpr int C = kLnFinalChannels, L = kLnFinalThreads / C, W = kLnFinalThreads / 64, DEEP = 8;
    __shared__ float ls[2][W][C];
    const int64_t item = blockIdx.y;
    const int cl = threadIdx.x % C, l = threadIdx.x / C;
    const int ch = blockIdx.x * C + cl;
    const int64_t lo = p.off ? min(max(p.off[item], (int64_t)0), p.n) : 0;
    const int64_t hi = p.off ? min(max(p.off[item + 1], (int64_t)0), p.n) : p.n;
    float a = 0.0f, b = 0.0f;
    if (lo < hi && ch < p.c) {
        const int64_t j1 = (hi - 1) / p.rows_per;
        for (int64_t j = lo / p.rows_per + l; j <= j1; j += DEEP * L) {
            float u[DEEP], v[DEEP];
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                const int64_t jj = j + i * L;
                const float* s = p.part + (min(jj, j1) + item) * 2 * p.c + ch;
                u[i] = jj <= j1 ? s[0] : 0.0f;
                v[i] = jj <= j1 ? s[p.c] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                a += u[i];
                b += v[i];
            }
        }
    }
#pragma unroll
    for (int o = C; o < 64; o <<= 1) {
        a += __shfl_xor(a, o);
        b += __shfl_xor(b, o);
    }
    if ((threadIdx.x & 63) < C) {
        ls[0][threadIdx.x >> 6][cl] = a;
        ls[1][threadIdx.x >> 6][cl] = b;
    }
    __syncthreads();
    if (l != 0 || ch >= p.c) return;
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        a += ls[0][w][cl];
        b += ls[1][w][cl];
    }
    if (p.scale && lo >= hi) {  // no row met this item's coefficients, whatever they hold
        if (p.dscale) ln_put(p.dscale, p.m_dtype, item * p.c + ch, 0.0f);
        if (p.dshift) ln_put(p.dshift, p.m_dtype, item * p.c + ch, 0.0f);
        if (p.sums) p.sums[item * 2 * p.c + ch] = p.sums[(item * 2 + 1) * p.c + ch] = 0.0f;
    } else if (p.scale) {
        const float g = p.gamma ? ln_param(p.gamma, p.p_dtype, ch) : 1.0f;
        const float t = p.beta ? ln_param(p.beta, p.p_dtype, ch) : 0.0f;
        if (p.dscale) ln_put(p.dscale, p.m_dtype, item * p.c + ch, g * a + t * b);
        if (p.dshift) ln_put(p.dshift, p.m_dtype, item * p.c + ch, b);
        if (p.sums) {
            const float s = 1.0f + ln_param(p.scale, p.m_dtype, item * p.m_stride + ch);
            p.sums[item * 2 * p.c + ch] = s * a;
            p.sums[(item * 2 + 1) * p.c + ch] = s * b;
        }
    } else {
        if (p.dgamma) ln_put(p.dgamma, p.p_dtype, ch, a);
        if (p.dbeta) ln_put(p.dbeta, p.p_dtype, ch, b);
    }
}

__global__ __launch_bounds__(256) void ln_sum_items_kernel(const float* sums, int64_t items, int c,
                                                           int p_dtype, void* dgamma, void* dbeta) {
    const int ch = blockIdx.x * 256 + threadIdx.x;
    if (ch >= c) return;
    float a = 0.0f, b = 0.0f;
#pragma unroll 4
    for (int64_t i = 0; i < items; ++i) {
        a += sums[i * 2 * c + ch];
        b += sums[(i * 2 + 1) * c + ch];
    }
    if (dgamma) ln_put(dgamma, p_dtype, ch, a);
    if (dbeta) ln_put(dbeta, p_dtype, ch, b);
}

inline bool ln_float_dtype(int dt) { return dt == SPC_F32 || dt == SPC_F16 || dt == SPC_BF16; }
inline int64_t ln_size(int dt) { return dt == SPC_F32 ? 4 : 2; }

// Checks what both entry points share and fills the kernel's arguments.
int ln_args(const char* fn, int dtype, const void* x, int64_t x_stride, int64_t n, int64_t c,
            const spc_layer_norm_params* q, LnArgs* p) {
    if (n < 0 || n > INT32_MAX || c <= 0 || c > kLnMaxC || x_stride < 0) {
        set_last_error("%s: unsupported shape n=%lld c=%lld (below 2^31 rows, 1 to %d channels)", fn,
                       (long long)n, (long long)c, kLnMaxC);
        return SPC_BAD_SHAPE;
    }
    if (!ln_float_dtype(dtype)) {
        set_last_error("%s: unknown dtype %d", fn, dtype);
        return SPC_BAD_ARG;
    }
    if (!q || !(q->eps >= 0.0f)) {
        set_last_error("%s: needs parameters with eps >= 0", fn);
        return SPC_BAD_ARG;
    }
    const bool affine = q->gamma || q->beta, mod = q->scale || q->shift;
    auto known = [&](int dt) { return dt == SPC_F32 || dt == dtype; };
    if ((affine && !known(q->param_dtype)) || (mod && !known(q->mod_dtype))) {
        set_last_error("%s: parameters must be F32 or of the rows' dtype", fn);
        return SPC_BAD_ARG;
    }
    if (mod && (!q->scale || !q->shift || q->n_batch < 1 || q->n_batch > 65535 || q->mod_stride < 0 ||
                (!q->offsets && q->n_batch != 1))) {
        set_last_error("%s: a modulation needs scale and shift of 1 to 65535 items, and offsets for "
                       "more than one", fn);
        return SPC_BAD_ARG;
    }
    if (!mod && q->offsets) {
        set_last_error("%s: offsets without scale and shift", fn);
        return SPC_BAD_ARG;
    }
    const int64_t e = ln_size(dtype), pe = ln_size(q->param_dtype), me = ln_size(q->mod_dtype);
    auto off = [](const void* a, int64_t by) { return (uintptr_t)a % by != 0; };
    if (off(x, e) || (affine && (off(q->gamma, pe) || off(q->beta, pe))) ||
        (mod && (off(q->scale, me) || off(q->shift, me))) || off(q->offsets, 8)) {
        set_last_error("%s: misaligned pointer", fn);
        return SPC_BAD_ARG;
    }
    *p = LnArgs{};
    p->x = x;
    p->x_stride = x_stride;
    p->n = n;
    p->c = (int)c;
    p->gamma = q->gamma;
    p->beta = q->beta;
    p->p_dtype = q->param_dtype;
    p->scale = q->scale;
    p->shift = q->shift;
    p->m_stride = q->mod_stride;
    p->m_dtype = q->mod_dtype;
    p->off = q->offsets;
    p->nb = mod ? q->n_batch : 1;
    p->eps = q->eps;
    p->silu = q->silu;
    return SPC_OK;
}

// Whether one block takes all rows, its sums being the gradients: that saves the
// second kernel (3 us) and its launch (3 us of the host).  Up to four rounds of a
// block's teams, two where a row takes half a block or more (us alone / with the
// second kernel: 16 x 192 4.1 / 6.4, 16 x 1024 7.0 / 7.3, 8 x 2048 8.6 / 7.9).
inline bool ln_one_block(int64_t n, int teams) { return n > 0 && n <= (teams > 2 ? 4 : 2) * teams; }

// Chunks the backward's row pass makes of n rows.
inline int64_t ln_backward_chunks(int64_t n, int teams) {
    return ceil_div(n, ln_backward_rows(n, teams));
}

}  // namespace

}  // namespace spc

using namespace spc;

extern "C" {

int spc_layer_norm(spc_stream_t stream, int dtype, const void* x, int64_t x_stride, int64_t n,
                   int64_t c, const spc_layer_norm_params* params, void* y, float* stats) {
    const char* fn = "spc_layer_norm";
    hipStream_t s = static_cast<hipStream_t>(stream);
    LnArgs p;
    const int st = ln_args(fn, dtype, x, x_stride, n, c, params, &p);
    if (st != SPC_OK) return st;
    if (n == 0) return SPC_OK;
    if (!x || !y || (uintptr_t)y % ln_size(dtype) || (uintptr_t)stats % 4) {
        set_last_error("%s: null or misaligned pointer", fn);
        return SPC_BAD_ARG;
    }
    p.y = y;
    p.stats = stats;
    p.rows_per = (int)ln_forward_rows(n, ln_teams(dtype, p.c, false));
    const unsigned blocks = (unsigned)ceil_div(n, p.rows_per);
    const hipError_t e = dtype == SPC_BF16  ? ln_forward_bf16(s, p, blocks)
                         : dtype == SPC_F16 ? ln_forward_f16(s, p, blocks)
                                            : ln_forward_f32(s, p, blocks);
    return e == hipSuccess ? SPC_OK : hip_status(e, "spc_layer_norm launch");
}

size_t spc_layer_norm_backward_workspace_bytes(int dtype, int64_t n, int64_t c, int64_t n_batch) {
    if (!ln_float_dtype(dtype) || n < 0 || n > INT32_MAX || c <= 0 || c > kLnMaxC || n_batch < 1 ||
        n_batch > 65535)
        return 0;
    const int64_t slots = ln_backward_chunks(n, ln_teams(dtype, (int)c, true)) + n_batch;
    return (size_t)((slots + n_batch) * 2 * c * (int64_t)sizeof(float));
}

int spc_layer_norm_backward(spc_stream_t stream, int dtype, const void* dy, int64_t dy_stride,
                            const void* x, int64_t x_stride, const float* stats, int64_t n, int64_t c,
                            const spc_layer_norm_params* params, void* dx, void* dgamma, void* dbeta,
                            void* dscale, void* dshift, void* workspace, size_t workspace_bytes) {
    const char* fn = "spc_layer_norm_backward";
    hipStream_t s = static_cast<hipStream_t>(stream);
    LnArgs p;
    const int st = ln_args(fn, dtype, x, x_stride, n, c, params, &p);
    if (st != SPC_OK) return st;
    const bool affine = p.gamma || p.beta, mod = p.scale != nullptr;
    const bool sums = dgamma || dbeta || dscale || dshift;
    if (dy_stride < 0 || (!affine && (dgamma || dbeta)) || (!mod && (dscale || dshift))) {
        set_last_error("%s: gradients of parameters that were not given, or a negative stride", fn);
        return SPC_BAD_ARG;
    }
    const int64_t e = ln_size(dtype), pe = ln_size(p.p_dtype), me = ln_size(p.m_dtype);
    auto off = [](const void* a, int64_t by) { return (uintptr_t)a % by != 0; };
    if ((n > 0 && (!x || !dy || !stats)) || off(dy, e) || off(stats, 4) || off(dx, e) ||
        off(dgamma, pe) || off(dbeta, pe) || off(dscale, me) || off(dshift, me)) {
        set_last_error("%s: null or misaligned pointer", fn);
        return SPC_BAD_ARG;
    }
    if (!dx && !sums) return SPC_OK;
    const int teams = ln_teams(dtype, p.c, true);
    const int64_t chunks = ln_backward_chunks(n, teams);
    // (offsets: rows of no item, and an empty item's zeros, are the second kernel's)
    const bool alone = sums && ln_one_block(n, teams) && affine != mod && !p.off;
    if (sums && (!workspace || off(workspace, 4) ||
                 workspace_bytes < spc_layer_norm_backward_workspace_bytes(dtype, n, c, p.nb))) {
        set_last_error("%s: workspace missing, misaligned or too small", fn);
        return SPC_BAD_ARG;
    }
    if (alone) {
        p.grad_a = mod ? dscale : dgamma;
        p.grad_b = mod ? dshift : dbeta;
        p.grad_dtype = mod ? p.m_dtype : p.p_dtype;
    } else if (sums) {
        p.part = static_cast<float*>(workspace);
    }
    p.y = dx;
    p.dy = dy;
    p.dy_stride = dy_stride;
    p.stats = const_cast<float*>(stats);
    p.rows_per = (int)(alone ? n : ln_backward_rows(n, teams));
    if (n > 0) {
        const unsigned blocks = alone ? 1 : (unsigned)chunks;
        const hipError_t err = dtype == SPC_BF16  ? ln_backward_bf16(s, p, blocks)
                               : dtype == SPC_F16 ? ln_backward_f16(s, p, blocks)
                                                  : ln_backward_f32(s, p, blocks);
        if (err != hipSuccess) return hip_status(err, "spc_layer_norm_backward launch");
    }
    if (!sums || alone) return SPC_OK;
    LnFinal f{};
    f.part = p.part;
    f.off = p.off;
    f.n = n;
    f.rows_per = p.rows_per;
    f.c = p.c;
    f.gamma = p.gamma;
    f.beta = p.beta;
    f.scale = p.scale;
    f.p_dtype = p.p_dtype;
    f.m_dtype = p.m_dtype;
    f.m_stride = p.m_stride;
    f.dgamma = dgamma;
    f.dbeta = dbeta;
    f.dscale = dscale;
    f.dshift = dshift;
    f.sums = mod && (dgamma || dbeta) ? p.part + (chunks + p.nb) * 2 * p.c : nullptr;
    ln_finalize_kernel<<<dim3((unsigned)ceil_div(c, kLnFinalChannels), (unsigned)p.nb), kLnFinalThreads,
                         0, s>>>(f);
    if (f.sums)
        ln_sum_items_kernel<<<(unsigned)ceil_div(c, 256), 256, 0, s>>>(f.sums, p.nb, p.c, p.p_dtype,
                                                                       dgamma, dbeta);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? SPC_OK : hip_status(err, "spc_layer_norm_backward launch");
}

}  // extern "C"

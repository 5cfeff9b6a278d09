// lora_few.hip -- the adapters' gradients of few rows (a batch's modulation rows,
// requests of one row each): two launches and no partial sums, since a block can
// see all rows of its columns.  The first forms u, a block a row and share of the
// outputs; the second takes 64 columns and an adapter a block, holds the adapter's
// sums in registers and writes its gradients, and its rows' dx on the way.  Plain
// F32 arithmetic: for rows in the tens the adapters' bytes and the launches are
// what there is to wait for (7 rows of 1024 to 2048, rank 8 F16: 6 + 8 us, 13 in a
// graph).
#include <algorithm>

#include "lora_kernel.h"

namespace spc {

namespace {

constexpr int kFewRows = 32;   // rows at a time

// RJ values times f, `left` of which are the row's.
template <int DT, int RJ>
__device__ __forceinline__ void few_put_ranks(void* p, int64_t at, const float (&v)[RJ], float f, int left) {
    using S = typename LoraNum<DT>::S;
    constexpr int V = LoraNum<DT>::V;
    if constexpr (RJ >= V) {
#pragma unroll
        for (int i = 0; i < RJ; i += V) {
            float z[V];
#pragma unroll
            for (int e = 0; e < V; ++e) z[e] = f * v[i + e];
            if (i < left) lora_store(static_cast<S*>(p) + at + i, lora_round<DT>(z), left - i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < RJ; ++i)
            if (i < left) lora_put<DT>(p, at + i, f * v[i]);
    }
}

// Threads along the ranks (V each, to a power of two of them), the rest along the
// outputs.
template <int DT>
__host__ __device__ inline int few_chunks(int r) {
    int c = 1;
    while (c * LoraNum<DT>::V < r) c *= 2;
    return c;
}

// u[share][row] = s_a sum over the share's outputs of dy[row] up_a; of a row without an
// adapter dx, the base, a share of its columns.  (Left to few_columns_kernel, whose block of
// 64 columns would gather such rows 32 at a time, 512 of them were 169 us of 1024 columns.)
template <int DT>
__global__ __launch_bounds__(kLoraThreads) void few_u_kernel(LoraBackArgs p, int o_per) {
    using N = LoraNum<DT>;
    using S = typename N::S;
    constexpr int V = N::V, UN = 4;
    __shared__ float red[4][kLoraMaxRank];
    const LoraItems& it = p.it;
    const int64_t row = blockIdx.x, a = it.find(row, 1, 0).adapter;
    if (a < 0) {
        const int per = (p.c / 8 / (int)gridDim.y + 1) * 8, c0 = min((int)blockIdx.y * per, p.c);
        if (p.dx) lora_pass<DT>(p.dx, p.c, p.base, p.bs, row, 1, c0, min(c0 + per, p.c));
        return;
    }
    const int chunks = few_chunks<DT>(p.r), lines = kLoraThreads / chunks, t = threadIdx.x;
    const int j = t % chunks * V, o1 = min((int)(blockIdx.y + 1) * o_per, p.o);
    const S* up = static_cast<const S*>(p.up);
    const int64_t all = it.adapters * p.o * p.r;
    float s[V] = {};
    for (int o = blockIdx.y * o_per + t / chunks; o < o1; o += UN * lines) {
        u32x4 w[UN];
        float d[UN];
#pragma unroll
        for (int k = 0; k < UN; ++k) {
            const int q = min(o + k * lines, o1 - 1);
            w[k] = lora_fetch_short(up, (a * p.o + q) * p.r + j, all);
            d[k] = lora_get<DT>(p.dy, row * p.dys + q);
        }
#pragma unroll
        for (int k = 0; k < UN; ++k) {
            if (o + k * lines >= o1) continue;
            const u32x4 v = lora_edge_short<S>(w[k], (a * p.o + o + k * lines) * p.r + j, all, p.r - j);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += d[k] * lora_value<DT>(v, e);
        }
    }
    for (int k = 32; k >= chunks; k >>= 1)
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += __shfl_xor(s[e], k);
    if ((t & 63) < chunks)
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (j + e < p.r) red[t >> 6][j + e] = s[e];
    __syncthreads();
    if (t < p.r) {
        const float z = (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]);
        p.u[(blockIdx.y * it.n + row) * p.r + t] = p.scale ? p.scale[a] * z : z;
    }
}

// Blocks along x: 64 columns of x (dx, ddown), then of dy (dup); along y: adapters.
// The adapter's rows are gathered from
// the segments 32 at a time, so that one wait serves as many.  A wave loads eight
// of them and holds RJ ranks' sums over all.
template <int DT, int RJ, bool DROP>
__global__ __launch_bounds__(kLoraThreads) void few_columns_kernel(LoraBackArgs p, int in_blocks, void* ddown, void* dup) {
    __shared__ __attribute__((aligned(16))) float us[kFewRows][4 * RJ];
    __shared__ float xs[kFewRows][64], part[4][kFewRows][64];
    __shared__ int list[kFewRows];
    const LoraItems& it = p.it;
    const bool in = (int)blockIdx.x < in_blocks;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, j0 = w * RJ;
    const int width = in ? p.c : p.o, col = (in ? blockIdx.x : blockIdx.x - in_blocks) * 64 + lane;
    const bool on = col < width, dx = in && p.dx, drop = DROP && in;
    const int at = min(col, width - 1);
    const void* x = in ? p.x : p.dy;
    const int64_t stride = in ? p.xs : p.dys;
    void* grad = in ? ddown : dup;
    const DropKey key = DROP ? drop_key(p.seed) : DropKey{};
    for (int64_t a = blockIdx.y; a < it.adapters; a += gridDim.y) {
        float acc[RJ] = {}, wt[RJ] = {};
        if (dx)
#pragma unroll
            for (int i = 0; i < RJ; ++i)
                if (j0 + i < p.r) wt[i] = lora_get<DT>(p.down, (a * p.r + j0 + i) * p.c + at);
        int64_t v0 = -64;
        uint64_t m = 0;
        int b = 0, e = 0, row = 0, end = 0;
        for (;;) {
            int count = 0;
            while (count < kFewRows) {
                if (row < end) {
                    const int k = min(kFewRows - count, end - row);
                    if ((int)threadIdx.x < k) list[count + threadIdx.x] = row + threadIdx.x;
                    row += k;
                    count += k;
                } else if (m) {
                    const int k = __builtin_ctzll(m);
                    row = __shfl(b, k);
                    end = __shfl(e, k);
                    m &= m - 1;
                } else {
                    v0 += 64;
                    if (v0 >= it.segments()) break;
                    const int64_t v = v0 + lane;
                    b = e = 0;
                    if (v < it.segments() && it.adapter(v) == a) {
                        b = (int)it.begin(v);
                        e = (int)it.end(v);
                    }
                    m = __ballot(b < e);
                }
            }
            if (!count) break;
            __syncthreads();
            int64_t rows[8];
            float xv[8], bv[8];
            uint32_t kept = 0;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                rows[t] = list[min(8 * w + t, count - 1)];
                bv[t] = dx && p.base ? lora_get<DT>(p.base, rows[t] * p.bs + at) : 0.0f;
                xv[t] = grad ? lora_get<DT>(x, rows[t] * stride + at) : 0.0f;
            }
            for (int i = threadIdx.x; i < kFewRows * 4 * RJ; i += kLoraThreads) {
                const int t = i / (4 * RJ), j = i % (4 * RJ);
                float z = 0.0f;
                if (t < count && j < p.r) {
                    const int64_t f = (int64_t)list[t] * p.r + j;
                    if (in) for (int q = 0; q < p.u_parts; ++q) z += p.u[(int64_t)q * it.n * p.r + f];
                    else z = p.hidden[f];
                }
                us[t][j] = z;
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                if (8 * w + t >= count) continue;
                const bool k = !drop || lora_keeps(lora_ones(key, p.drop, rows[t], at, p.c), at);
                kept |= (uint32_t)k << t;
                xs[8 * w + t][lane] = k ? xv[t] : 0.0f;
            }
            __syncthreads();
            for (int t = 0; t < count; ++t) {
                const float xt = xs[t][lane];
                float d = 0.0f;
#pragma unroll
                for (int i = 0; i < RJ; ++i) {
                    const float u = us[t][j0 + i];
                    acc[i] += u * xt;
                    d += u * wt[i];
                }
                if (dx) part[w][t][lane] = d;
            }
            if (!dx) continue;
            __syncthreads();
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const int q = 8 * w + t;
                if (q >= count || !on) continue;
                float z = 0.0f;
                if (kept >> t & 1) {
                    z = (part[0][q][lane] + part[1][q][lane]) + (part[2][q][lane] + part[3][q][lane]);
                    if (drop) z *= p.factor;
                }
                lora_put<DT>(p.dx, rows[t] * p.c + col, z + bv[t]);
            }
        }
        __syncthreads();
        if (!grad || !on) continue;
        const float f = in ? (drop ? p.factor : 1.0f) : p.scale ? p.scale[a] : 1.0f;
        if (in) {
#pragma unroll
            for (int i = 0; i < RJ; ++i)
                if (j0 + i < p.r) lora_put<DT>(grad, (a * p.r + j0 + i) * p.c + col, f * acc[i]);
        } else {
            // (a column's ranks stand together: 16 bytes of them in a store, 34 one-row items of
            // 17 to 3712, rank 128 and 16 adapters 79 us one by one, so 46)
            few_put_ranks<DT, RJ>(grad, (a * p.o + col) * p.r + j0, acc, f, p.r - j0);
        }
    }
}

template <int DT, int RJ>
void few_columns(hipStream_t s, const LoraBackArgs& p, dim3 grid, int in_blocks, void* ddown, void* dup) {
    if (p.drop) few_columns_kernel<DT, RJ, true><<<grid, kLoraThreads, 0, s>>>(p, in_blocks, ddown, dup);
    else few_columns_kernel<DT, RJ, false><<<grid, kLoraThreads, 0, s>>>(p, in_blocks, ddown, dup);
}

template <int DT>
void few_backward(hipStream_t s, const LoraBackArgs& p, int o_per, void* ddown, void* dup) {
    if (p.it.n > 0 && p.u) few_u_kernel<DT><<<dim3((unsigned)p.it.n, (unsigned)p.u_parts), kLoraThreads, 0, s>>>(p, o_per);
    const int in_blocks = p.dx || ddown ? (int)ceil_div(p.c, 64) : 0, out_blocks = dup ? (int)ceil_div(p.o, 64) : 0;
    const int64_t x = in_blocks + out_blocks;
    // (at most 65,535 along y, as the adapters)
    const dim3 grid((unsigned)x, (unsigned)std::min<int64_t>(p.it.adapters, std::max<int64_t>(1, (1 << 18) / x)));
    const int rt = lora_rank_tiles(p.r);
    if (rt == 1) few_columns<DT, 4>(s, p, grid, in_blocks, ddown, dup);
    else if (rt == 2) few_columns<DT, 8>(s, p, grid, in_blocks, ddown, dup);
    else if (rt == 4) few_columns<DT, 16>(s, p, grid, in_blocks, ddown, dup);
    else few_columns<DT, 32>(s, p, grid, in_blocks, ddown, dup);
}

}  // namespace

hipError_t lora_few_backward(hipStream_t s, int dt, const LoraBackArgs& p, int o_per, void* ddown, void* dup) {
    if (dt == SPC_BF16) few_backward<SPC_BF16>(s, p, o_per, ddown, dup);
    else if (dt == SPC_F16) few_backward<SPC_F16>(s, p, o_per, ddown, dup);
    else few_backward<SPC_F32>(s, p, o_per, ddown, dup);
    return hipGetLastError();
}

}  // namespace spc

// lora.hip -- entry points of the low-rank adapters and their gradients
// (kernels: lora_kernel.h).
#include <algorithm>
#include <type_traits>

#include "lora_kernel.h"

namespace spc {

namespace {

// Gradients from the slots that the row passes left: adapter a's is the sum over
// its items and their chunks (lora_chunk_row), in a fixed order.  A block
// takes 1024 / G of a slot's floats, G slots at a time.  Where the slots hold a part of
// the chunks at a time (kLoraSlotBytes), sums are carried in F32 from part to part.
struct LoraSum {
    const float* part;
    void* dst;
    float* carry;  // like dst
    int64_t slot;  // floats
    int64_t first, chunks, all;  // chunks of this part, and of all
    int c;         // columns
    int along;     // dst [r][c], else [c][r]
    int rows_per;
};

template <int DT, int G>
__global__ __launch_bounds__(kLoraThreads) void lora_sum_kernel(LoraItems it, LoraSum first, LoraSum second, int r, int rt) {
    constexpr int V = LoraNum<DT>::V, T = kLoraThreads / G;
    __shared__ floatx4 ls[G][T];
    const LoraSum p = blockIdx.y ? second : first;
    if (!p.dst) return;
    const int tx = threadIdx.x % T, ty = threadIdx.x / T, lane = threadIdx.x & 63;
    const int64_t blocks = p.slot / (4 * T), last = p.first + p.chunks - 1;
    const bool begins = p.first == 0, ends = last >= p.all - 1;
    int64_t from = 0, to = it.items;  // items that may have chunks here
    if (!begins || !ends) {
        from = max(it.find(p.first, p.rows_per, 1).v - (it.off ? 1 : 0), (int64_t)0) & ~63;
        to = min(it.find(last, p.rows_per, 1).v + 1, it.items);
    }
    for (int64_t w = blockIdx.x; w < blocks * it.adapters; w += gridDim.x) {
        const int64_t a = w / blocks, e0 = w % blocks * (4 * T) + 4 * tx;
        floatx4 s = {0, 0, 0, 0};
        uint64_t any = 0;
        for (int64_t i0 = from; i0 < to; i0 += 64) {
            const int64_t i = i0 + lane, v = it.off ? i + 1 : i;
            int64_t b = 0, e = 0;
            if (i < it.items && it.adapter(v) == a) {
                b = it.begin(v);
                e = it.end(v);
            }
            const int mine0 = (int)b / p.rows_per, more = (int)(e - b - 1) / p.rows_per;
            uint64_t m = __ballot(b < e);
            for (any |= m; m; m &= m - 1) {
                const int k = __builtin_ctzll(m);
                const int64_t seg = i0 + k + (it.off ? 1 : 0);
                int64_t j0 = __shfl(mine0, k) + seg, j1 = min(j0 + __shfl(more, k), last) - p.first;
                j0 = max(j0 - p.first, (int64_t)0);
#pragma unroll 4
                for (int64_t j = j0 + ((ty - j0) & (G - 1)); j <= j1; j += G)
                    s += *reinterpret_cast<const floatx4*>(p.part + j * p.slot + e0);
            }
        }
        if (!any && !begins && !ends) continue;  // (what is carried stays as it is)
        ls[ty][tx] = s;
        __syncthreads();
        if (threadIdx.x < 4 * T) {
            const int64_t at = w % blocks * (4 * T) + threadIdx.x, tile = at >> 8;
            const int i = threadIdx.x & 3, n = (int)(at >> 2) & 63;
            const int64_t col = tile / (V * rt) * (16 * V) + V * (4 * (n >> 4) + i) + tile % V;
            const int rank = (int)(tile / V % rt) * 16 + (n & 15);
            float z = 0.0f;
#pragma unroll
            for (int q = 0; q < G; ++q) z += ls[q][threadIdx.x >> 2][i];
            if (col < p.c && rank < r) {
                const int64_t d = a * p.c * r + (p.along ? rank * (int64_t)p.c + col : col * r + rank);
                if (!begins) z += p.carry[d];
                if (ends) lora_put<DT>(p.dst, d, z);
                else p.carry[d] = z;
            }
        }
        __syncthreads();
    }
}

// The sum of u's shares in the first one's place.
__global__ __launch_bounds__(kLoraThreads) void lora_add_u_kernel(float* u, int64_t n, int parts) {
    for (int64_t i = (int64_t)blockIdx.x * kLoraThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kLoraThreads) {
        float s = u[i];
#pragma unroll 16
        for (int q = 1; q < parts; ++q) s += u[q * n + i];
        u[i] = s;
    }
}

inline size_t lora_round_up(size_t floats) { return (floats + 63) / 64 * 64; }

// How a call is split, from its sizes alone.
struct LoraPlan {
    int mt, mode;     // mode: kLoraFused, or kLoraShrink and kLoraExpand
    int64_t tiles;    // tile numbers of the grid
    int splits, k_per, col_per, col_blocks;
};

LoraPlan lora_plan(int dt, int64_t n, int64_t items, int64_t c, int64_t o, int64_t r) {
    LoraPlan q{};
    const int step = dt == SPC_F32 ? 16 : 32;
    // Tiles of 32 rows halve the adapters' traffic, tiles of 16 give twice the blocks
    // (us in a graph, 1024 -> 1024 rank 16 bf16, 32 / 16: 4096 rows 14.8 / 10.9, 16,384
    // 22.6 / 25.4; 30,000 rank 32 38.5 / 54.1).
    q.mt = n / items >= 32 && n >= 384 * 32 ? kLoraRowTiles : 1;
    // Ranks 33 to 64, whose adapters are most of a tile's traffic and whose sums still fit LDS
    // twice (us, tiles of 64 / 32: 1024 -> 1024 rank 64 bf16 20,000 rows 46 / 42, 30,000 48 / 55,
    // 50,000 97 / 90; 16,000 of 2048 -> 512 33 / 37, 25,000 51 / 63; f16 20,000 56 / 52, 30,000 60 / 62,
    // 50,000 106 / 105; f32 30,000 136 / 142).
    if (lora_rank_tiles(r) == 4 && n / items >= 64 && n >= 384 * 64) q.mt = 2 * kLoraRowTiles;
    const int64_t rows = 16 * q.mt, busy = std::max<int64_t>(1, std::max(ceil_div(n, rows), std::min(items, n)));
    q.tiles = n / rows + items + 3;
    // One kernel, each of whose column blocks forms the tile's hidden rows again, or two:
    // one where the tiles fill the device or are little work (us, one / two: 1024 x 1024 ->
    // 1024 rank 16 8.1 / 8.5, 4 items 1024 -> 4096 rank 64 9.0 / 9.1, 1024 x 4096 -> 1024
    // rank 32 27 / 14, 8 items 8192 -> 16,384 rank 64 f16 70 / 13.2).
    q.mode = q.mt > 1 || busy >= 256 || c * (16 + r) * float_size(dt) <= 200000 ? kLoraFused : kLoraShrink;
    auto share = [&](int64_t width, int64_t unit, int64_t want) {  // columns a block
        const int64_t blocks = std::min(std::max<int64_t>(want / busy, 1), ceil_div(width, unit));
        return ceil_div(ceil_div(width, blocks), unit) * unit;
    };
    // Blocks that share a tile, each of 8 steps of columns or more (us in a graph): by 128 /
    // 256 / 384 / 512 / 1024 of them 64 one-row requests 1024 -> 4096 rank 16 12.5 / 10.2 / 9.2
    // / 9.3 / 10.5; in two kernels, 256 / 512 / 1024, 8 of 8192 -> 16,384 rank 64 14.7 / 13.3 /
    // 13.2; one row of 1024 -> 2048, 8 steps / 16, 5.1 / 5.8.
    q.splits = 1;
    q.k_per = (int)c;
    if (q.mode == kLoraShrink) {
        q.k_per = (int)share(c, 8 * step, 512);
        q.splits = (int)ceil_div(c, q.k_per);
    }
    q.col_per = (int)share(o, 8 * step, q.mode == kLoraShrink ? 512 : 384);
    q.col_blocks = (int)ceil_div(o, q.col_per);
    return q;
}

// Of the slots of one weight's gradient; more chunks than they hold go in parts of 8192
// blocks and more.  (65,535 one-row items would fill 4 GB at 1024 columns, rank 16.)
constexpr int64_t kLoraSlotBytes = 1 << 29;

struct LoraBackPlan {
    bool few;                   // lora_few.hip, u in `shares` of o_per outputs
    int shares, o_per;
    int rows_o, rows_c;         // rows of a chunk
    int64_t chunks_o, chunks_c, blocks_o, blocks_c;
    int64_t slot_o, slot_c;     // floats
    int64_t held_o, held_c;     // chunks that the slots hold
    size_t u, pu, pd;           // floats, with what is carried from part to part
};

LoraBackPlan lora_back_plan(int dt, int64_t n, int64_t items, int64_t adapters, int64_t c, int64_t o, int64_t r) {
    LoraBackPlan q{};
    // Tiles of 32 rows of one item cost some 0.2 us an item, however short, and the sums
    // behind them; gathered, an adapter's rows wait one after the other, some 14 us for each
    // 32 of them.  How many those are is the device's to know, so that the rule stays where
    // rows spread evenly over the adapters gain and all rows of one adapter lose less than
    // twice (us, gathered / tiles, even; gathered / tiles, all of one; 1024 -> 1024 rank 16 bf16:
    // 64 one-row items of 4 adapters 22 / 31; 42 / 39. 256 of 8 30 / 83; 130 / 112. 256 items of 2
    // rows and 8 36 / 82; 178 / 113. 1024 of 2 and 64 79 / 198; 677 / 342. 4096 one-row items of 8
    // 296 / 906; 1946 / 1501, of 1024 1333 / 2306; 2043 / 2202, and of one adapter 1940 / 1380.
    // Left to tiles: 256 of 4 rows and 32 38 / 69; 279 / 105. 64 of 30 and 64 50 / 43; 401 / 49. 2048 of
    // 4 and 8 350 / 459; 2404 / 749. 1024 of 8 and 1024 666 / 667; 2152 / 613. 16 of 32 and 8 27 / 24).
    q.few = n <= std::min({32 * items, std::min(items, adapters) * (32 + items / 2), 180 + 2 * items});
    if (q.few) {
        int64_t chunks = 1;
        while (chunks * (dt == SPC_F32 ? 4 : 8) < r) chunks *= 2;
        const int64_t lines = kLoraThreads / chunks;
        // A row's u by one block is one wait after the other along the outputs (us of the call by
        // one block / 128 over the rows: 1 row 8192 -> 16,384 rank 64 109 / 28, 7 of 8192 -> 8192
        // 63 / 24, 16 of 4096 -> 4096 rank 16 18.6 / 14.8).
        q.shares = (int)std::min({(int64_t)8, ceil_div(o, lines * 8), std::max<int64_t>(1, 128 / std::max<int64_t>(n, 1))});
        q.o_per = (int)ceil_div(o, q.shares);
        q.u = (size_t)(q.shares * n * r);
        return q;
    }
    q.blocks_o = ceil_div(o, (int64_t)lora_col_waves(dt, r, o) * lora_wave_cols(dt));
    q.blocks_c = ceil_div(c, (int64_t)lora_col_waves(dt, r, c) * lora_wave_cols(dt));
    // Some two blocks a CU: the registers hold no more of them at once, and every further
    // chunk is a slot to write and add (us by 256 / 384 / 512 / 640 / 1024 blocks: 30,000 x 1024
    // rank 16 bf16 without dx_base 73 / 66 / 60 / 74 / 77, rank 64 170 / 142 / 120 / 138 / 138, 21,766 x
    // 768 rank 8 f32 71 / 73 / 65 / 65 / 73).
    // A block's chunk is of one item, whose last is shorter: some chunks fewer, so that those
    // do not make a second round.
    auto rows = [&](int64_t blocks, int64_t width) {
        const int64_t tile = kLoraRows * lora_row_waves(dt, r, width);
        const int64_t chunks = std::max<int64_t>(1, 512 / blocks), more = std::min(items, chunks / 2);
        const int64_t per = ceil_div(ceil_div(n, chunks - more), tile) * tile;
        return (int)per;
    };
    q.rows_o = rows(q.blocks_o, o);
    q.rows_c = rows(q.blocks_c, c);
    q.chunks_o = n / q.rows_o + items + 3;
    q.chunks_c = n / q.rows_c + items + 3;
    q.u = (size_t)(q.blocks_o * n * r);
    q.slot_o = lora_slot(o, lora_wave_cols(dt), lora_rank_tiles(r));
    q.slot_c = lora_slot(c, lora_wave_cols(dt), lora_rank_tiles(r));
    auto held = [&](int64_t chunks, int64_t slot) {
        return std::min(chunks, std::max<int64_t>(1, kLoraSlotBytes / (slot * (int64_t)sizeof(float))));
    };
    q.held_o = held(q.chunks_o, q.slot_o);
    q.held_c = held(q.chunks_c, q.slot_c);
    // (F32 gradients carry their own)
    auto floats = [&](int64_t held, int64_t chunks, int64_t slot, int64_t width) {
        return lora_round_up((size_t)(held * slot)) + (held < chunks && dt != SPC_F32 ? (size_t)(adapters * r * width) : 0);
    };
    q.pu = floats(q.held_o, q.chunks_o, q.slot_o, o);
    q.pd = floats(q.held_c, q.chunks_c, q.slot_c, c);
    return q;
}

// Widths below eight as the kernels take them: arrays of rows of eight behind the rest
// of the workspace (`at`; null: their bytes are counted only).  A launch before and one
// after, against plain sums over narrow rows (us of rank 8 bf16, so / plain: 21,766 x
// 1024 to 4 19 / 174 forward, 45 / 12,276 backward; 100,000 x 4 to 64 21 / 175, 41 /
// 56,246; 333 x 6 to 32 7.5 / 7.3, 23 / 131).
struct LoraNarrow {
    int dt;
    char* at;
    size_t bytes = 0;
    LoraCopies in{}, out{};

    LoraNarrow(int dt, void* at) : dt(dt), at(static_cast<char*>(at)) {}
    static int64_t width(int64_t c) { return std::max<int64_t>(c, 8); }

    void* take(int64_t elements) {
        void* p = at ? at + bytes : nullptr;
        bytes += lora_round_up((size_t)(elements * float_size(dt) + 3) / 4) * sizeof(float);
        return p;
    }
    // Rows of `width` as rows of `fill`, in `dst`; and results back.
    void* widen(void* dst, const void* src, int64_t rows, int64_t stride, int64_t width, int64_t fill) {
        if (src) in.job[in.jobs++] = {src, dst, rows, stride, fill, (int)width, (int)fill};
        return dst;
    }
    void narrow(void* dst, const void* src, int64_t rows, int64_t width, int64_t fill) {
        if (dst) out.job[out.jobs++] = {src, dst, rows, fill, width, (int)width, (int)width};
    }
    const void* rows(const void* src, int64_t rows, int64_t* stride, int64_t width) {
        const void* p = widen(take(rows * 8), src, rows, *stride, width, 8);
        *stride = 8;
        return p;
    }

    // The adapters, of c and o features.
    void adapters(const void** down, const void** up, int64_t k, int64_t r, int64_t c, int64_t o) {
        int64_t stride = c;
        if (c < 8) *down = rows(*down, k * r, &stride, c);
        if (o < 8) *up = widen(take(k * 8 * r), *up, k, o * r, o * r, 8 * r);
    }
    // y (dx), onto whose wide rows base is copied.
    void sum(void** y, const void** base, int64_t* stride, int64_t n, int64_t width) {
        void* wide = take(n * 8);
        if (*base) *base = widen(wide, *base, n, *stride, width, 8);
        *stride = 8;
        narrow(*y, wide, n, width, 8);
        if (*y) *y = wide;
    }
    void forward(LoraArgs* p, int64_t k, int64_t r, int64_t c, int64_t o) {
        adapters(&p->down, &p->up, k, r, c, o);
        if (c < 8) p->x = rows(p->x, p->it.n, &p->xs, c);
        if (o < 8) sum(&p->y, &p->base, &p->bs, p->it.n, o);
    }
    void backward(LoraBackArgs* p, void** ddown, void** dup, int64_t k, int64_t r, int64_t c, int64_t o) {
        adapters(&p->down, &p->up, k, r, c, o);
        if (c < 8) {
            p->x = rows(p->x, p->it.n, &p->xs, c);
            sum(&p->dx, &p->base, &p->bs, p->it.n, c);
            void* wide = take(k * r * 8);
            narrow(*ddown, wide, k * r, c, 8);
            if (*ddown) *ddown = wide;
        }
        if (o < 8) {
            p->dy = rows(p->dy, p->it.n, &p->dys, o);
            void* wide = take(k * 8 * r);
            narrow(*dup, wide, k, o * r, 8 * r);
            if (*dup) *dup = wide;
        }
    }
};

// Checks what both entry points share.
int lora_args(const char* fn, int dtype, const void* x, int64_t x_stride, int64_t n,
              const spc_lora_params* q, LoraItems* it, uint32_t* drop) {
    if (!q || n < 0 || n > kLoraMaxRows || x_stride < 0 || q->in_features < 1 || q->out_features < 1 ||
        q->in_features > kLoraMaxWidth || q->out_features > kLoraMaxWidth || q->rank < 1 ||
        q->rank > kLoraMaxRank || q->n_adapters < 1 || q->n_adapters > kLoraMaxAdapters || q->n_items < 1 ||
        q->n_items > kLoraMaxItems) {
        set_last_error("%s: unsupported shape (up to 2^27 rows, widths 1 to 2^24, ranks 1 to 128, 1 to 65535 "
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
    if ((!q->offsets && n % q->n_items) || (!q->adapters && q->n_adapters != 1)) {
        set_last_error("%s: items of unequal rows need offsets, more than one adapter the items' adapters", fn);
        return SPC_BAD_ARG;
    }
    const int64_t e = float_size(dtype);
    auto off = [](const void* p, int64_t by) { return (uintptr_t)p % by != 0; };
    *drop = drop_threshold(q->p);
    if (!q->down || !q->up || (*drop && !q->seed) || (n > 0 && !x) || off(x, e) || off(q->down, e) ||
        off(q->up, e) || off(q->scale, 4) || off(q->offsets, 8) || off(q->adapters, 4) || off(q->seed, 8)) {
        set_last_error("%s: null or misaligned pointer", fn);
        return SPC_BAD_ARG;
    }
    *it = LoraItems{q->offsets, q->adapters, q->n_items, q->n_adapters, n, n / q->n_items};
    return SPC_OK;
}

}  // namespace

}  // namespace spc

using namespace spc;

extern "C" {

size_t spc_lora_workspace_bytes(int dtype, int64_t n, int64_t n_items, int64_t n_adapters, int64_t in_features,
                                int64_t out_features, int64_t rank, int backward) {
    if (!float_dtype(dtype) || n < 0 || n > kLoraMaxRows || rank < 1 || rank > kLoraMaxRank || n_items < 1 ||
        n_items > kLoraMaxItems || n_adapters < 1 || n_adapters > kLoraMaxAdapters || in_features < 1 ||
        in_features > kLoraMaxWidth || out_features < 1 || out_features > kLoraMaxWidth)
        return 0;
    const int64_t c = LoraNarrow::width(in_features), o = LoraNarrow::width(out_features);
    LoraNarrow narrow(dtype, nullptr);
    size_t floats = 0;
    if (backward) {
        const LoraBackPlan b = lora_back_plan(dtype, n, n_items, n_adapters, c, o, rank);
        floats = lora_round_up(b.u) + lora_round_up(b.pu) + b.pd;
        LoraBackArgs p{};
        void *ddown = nullptr, *dup = nullptr;
        p.it.n = n;
        narrow.backward(&p, &ddown, &dup, n_adapters, rank, in_features, out_features);
    } else {
        const LoraPlan f = lora_plan(dtype, n, n_items, c, o, rank);
        if (f.mode == kLoraShrink) floats = (size_t)f.splits * n * rank;
        LoraArgs p{};
        p.it.n = n;
        narrow.forward(&p, n_adapters, rank, in_features, out_features);
    }
    return (narrow.bytes ? lora_round_up(floats) : floats) * sizeof(float) + narrow.bytes;
}

int spc_lora(spc_stream_t stream, int dtype, const void* x, int64_t x_stride, int64_t n,
             const spc_lora_params* params, const void* base, int64_t base_stride, void* y, float* hidden,
             void* workspace, size_t workspace_bytes) {
    const char* fn = "spc_lora";
    hipStream_t s = static_cast<hipStream_t>(stream);
    LoraArgs p{};
    const int st = lora_args(fn, dtype, x, x_stride, n, params, &p.it, &p.drop);
    if (st != SPC_OK) return st;
    if (n == 0) return SPC_OK;
    const spc_lora_params& q = *params;
    const int64_t e = float_size(dtype);
    auto off = [](const void* a, int64_t by) { return (uintptr_t)a % by != 0; };
    if (!y || off(y, e) || off(base, e) || off(hidden, 4) || base_stride < 0) {
        set_last_error("%s: null or misaligned pointer, or a negative stride", fn);
        return SPC_BAD_ARG;
    }
    const size_t need = spc_lora_workspace_bytes(dtype, n, q.n_items, q.n_adapters, q.in_features, q.out_features, q.rank, 0);
    if (need && (!workspace || off(workspace, 16) || workspace_bytes < need)) {
        set_last_error("%s: workspace missing, misaligned or too small", fn);
        return SPC_BAD_ARG;
    }
    const int64_t c = LoraNarrow::width(q.in_features), o = LoraNarrow::width(q.out_features);
    const LoraPlan f = lora_plan(dtype, n, q.n_items, c, o, q.rank);
    p.x = x;
    p.xs = x_stride;
    p.down = q.down;
    p.up = q.up;
    p.scale = q.scale;
    p.base = base;
    p.bs = base_stride;
    p.y = y;
    p.hidden = hidden;
    p.part = static_cast<float*>(workspace);
    p.c = (int)c;
    p.o = (int)o;
    p.r = (int)q.rank;
    p.k_per = f.k_per;
    p.splits = f.splits;
    p.col_per = f.col_per;
    p.seed = q.seed;
    p.factor = drop_factor(p.drop);
    auto launch = [&](int mode, int64_t blocks) {
        const dim3 grid((unsigned)f.tiles, (unsigned)blocks);
        return dtype == SPC_BF16  ? lora_forward_bf16(s, p, mode, f.mt, grid)
               : dtype == SPC_F16 ? lora_forward_f16(s, p, mode, f.mt, grid)
                                  : lora_forward_f32(s, p, mode, f.mt, grid);
    };
    LoraNarrow narrow(dtype, p.part + (f.mode == kLoraShrink ? lora_round_up((size_t)f.splits * n * q.rank) : 0));
    narrow.forward(&p, q.n_adapters, q.rank, q.in_features, q.out_features);
    hipError_t err = lora_copy(s, dtype, narrow.in);
    if (err == hipSuccess && f.mode == kLoraFused) {
        err = launch(kLoraFused, f.col_blocks);
    } else if (err == hipSuccess) {
        err = launch(kLoraShrink, f.splits);
        if (err == hipSuccess) err = launch(kLoraExpand, f.col_blocks);
    }
    if (err == hipSuccess) err = lora_copy(s, dtype, narrow.out);
    return err == hipSuccess ? SPC_OK : hip_status(err, "spc_lora launch");
}

int spc_lora_backward(spc_stream_t stream, int dtype, const void* dy, int64_t dy_stride, const void* x,
                      int64_t x_stride, const float* hidden, int64_t n, const spc_lora_params* params,
                      const void* dx_base, int64_t dx_base_stride, void* dx, void* ddown, void* dup,
                      void* workspace, size_t workspace_bytes) {
    const char* fn = "spc_lora_backward";
    hipStream_t s = static_cast<hipStream_t>(stream);
    LoraBackArgs p{};
    const int st = lora_args(fn, dtype, x, x_stride, n, params, &p.it, &p.drop);
    if (st != SPC_OK) return st;
    const spc_lora_params& q = *params;
    const int64_t e = float_size(dtype);
    auto off = [](const void* a, int64_t by) { return (uintptr_t)a % by != 0; };
    if ((n > 0 && (!dy || (dup && !hidden))) || off(dy, e) || off(hidden, 4) || off(dx_base, e) || off(dx, e) ||
        off(ddown, e) || off(dup, e) || dy_stride < 0 || dx_base_stride < 0) {
        set_last_error("%s: null or misaligned pointer, or a negative stride", fn);
        return SPC_BAD_ARG;
    }
    if (!dx && !ddown && !dup) return SPC_OK;
    const size_t need = spc_lora_workspace_bytes(dtype, n, q.n_items, q.n_adapters, q.in_features, q.out_features, q.rank, 1);
    if (need && (!workspace || off(workspace, 16) || workspace_bytes < need)) {
        set_last_error("%s: workspace missing, misaligned or too small", fn);
        return SPC_BAD_ARG;
    }
    const int64_t c = LoraNarrow::width(q.in_features), o = LoraNarrow::width(q.out_features);
    const LoraBackPlan b = lora_back_plan(dtype, n, q.n_items, q.n_adapters, c, o, q.rank);
    float* ws = static_cast<float*>(workspace);
    p.dy = dy;
    p.dys = dy_stride;
    p.x = x;
    p.xs = x_stride;
    p.hidden = hidden;
    p.down = q.down;
    p.up = q.up;
    p.scale = q.scale;
    p.base = dx_base;
    p.bs = dx_base_stride;
    p.dx = dx;
    p.u = dx || ddown ? ws : nullptr;
    p.u_parts = b.few ? b.shares : (int)b.blocks_o;
    p.pu = dup ? ws + lora_round_up(b.u) : nullptr;
    p.pd = ddown ? ws + lora_round_up(b.u) + lora_round_up(b.pu) : nullptr;
    p.c = (int)c;
    p.o = (int)o;
    p.r = (int)q.rank;
    p.seed = q.seed;
    p.factor = drop_factor(p.drop);
    LoraNarrow narrow(dtype, ws + lora_round_up(b.u) + lora_round_up(b.pu) + lora_round_up(b.pd));
    narrow.backward(&p, &ddown, &dup, q.n_adapters, q.rank, q.in_features, q.out_features);
    hipError_t err = lora_copy(s, dtype, narrow.in);
    if (err == hipSuccess && b.few) err = lora_few_backward(s, dtype, p, b.o_per, ddown, dup);
    if (err == hipSuccess && !b.few) {
        const int rt = lora_rank_tiles(q.rank);
        auto carry = [&](float* part, void* dst, int64_t held, int64_t slot) {
            return dtype == SPC_F32 ? static_cast<float*>(dst) : part + lora_round_up((size_t)(held * slot));
        };
        LoraSum d = {p.pd, ddown, carry(p.pd, ddown, b.held_c, b.slot_c), b.slot_c, 0, 0, b.chunks_c, p.c, 1, b.rows_c};
        LoraSum u = {p.pu, dup, carry(p.pu, dup, b.held_o, b.slot_o), b.slot_o, 0, 0, b.chunks_o, p.o, 0, b.rows_o};
        auto sum = [&](const LoraSum& first, const LoraSum& second) {
            auto launch = [&](auto g) {
                constexpr int G = g.value;
                const dim3 grid((unsigned)std::min<int64_t>(std::max(first.slot, second.slot) / (1024 / G) * q.n_adapters, 1 << 20),
                                second.dst ? 2 : 1);
                if (dtype == SPC_BF16) lora_sum_kernel<SPC_BF16, G><<<grid, kLoraThreads, 0, s>>>(p.it, first, second, p.r, rt);
                else if (dtype == SPC_F16) lora_sum_kernel<SPC_F16, G><<<grid, kLoraThreads, 0, s>>>(p.it, first, second, p.r, rt);
                else lora_sum_kernel<SPC_F32, G><<<grid, kLoraThreads, 0, s>>>(p.it, first, second, p.r, rt);
            };
            // Few slots an adapter are wide work, many are long (us of the whole call, four groups
            // of slots / sixteen: 40 x 8192 to 8192 rank 64 34 / 51, 200 of four items 50 / 77, 40 x
            // 16,384 to 16,384 rank 32 34 / 51, 30,000 x 64 to 64 rank 16 27 / 23).
            if (std::max(b.chunks_o, b.chunks_c) <= 32 * q.n_adapters) launch(std::integral_constant<int, 4>{});
            else launch(std::integral_constant<int, 16>{});
            return hipGetLastError();
        };
        // A pass over the rows, as many chunks at a time as its slots hold (without sums as
        // many as a launch may have, 2^32 threads); the sums of a pass of several parts follow
        // each of them.
        auto pass = [&](bool out, LoraSum* z) {
            const int64_t held = z->dst ? (out ? b.held_o : b.held_c) : z->all, blocks = out ? b.blocks_o : b.blocks_c;
            const int64_t most = std::min<int64_t>(held, std::max<int64_t>(1, (1 << 23) / blocks));
            for (z->first = 0; z->first < z->all && err == hipSuccess; z->first += z->chunks) {
                z->chunks = std::min(most, z->all - z->first);
                p.chunk0 = (int)z->first;
                p.rows_per = z->rows_per;
                p.blocks = (int)blocks;
                const dim3 grid((unsigned)(blocks * z->chunks));
                if (out)
                    err = dtype == SPC_BF16  ? lora_back_out_bf16(s, p, grid)
                          : dtype == SPC_F16 ? lora_back_out_f16(s, p, grid)
                                             : lora_back_out_f32(s, p, grid);
                else
                    err = dtype == SPC_BF16  ? lora_back_in_bf16(s, p, grid)
                          : dtype == SPC_F16 ? lora_back_in_f16(s, p, grid)
                                             : lora_back_in_f32(s, p, grid);
                if (err == hipSuccess && z->dst && z->chunks < z->all) err = sum(*z, LoraSum{});
            }
            z->first = 0;
        };
        if (p.u || dup) pass(true, &u);
        if (err == hipSuccess && p.u && p.u_parts > lora_shares(lora_rank_tiles(p.r), lora_row_waves(dtype, p.r, p.c))) {
            const int64_t all = n * p.r, blocks = std::min<int64_t>(ceil_div(all, kLoraThreads), 1 << 14);
            lora_add_u_kernel<<<(unsigned)blocks, kLoraThreads, 0, s>>>(p.u, all, p.u_parts);
            err = hipGetLastError();
            p.u_parts = 1;
        }
        if (p.u) pass(false, &d);
        // (of passes in one part together)
        if (d.chunks < d.all) d.dst = nullptr;
        if (u.chunks < u.all) u.dst = nullptr;
        if (err == hipSuccess && (d.dst || u.dst)) err = d.dst ? sum(d, u) : sum(u, d);
    }
    if (err == hipSuccess) err = lora_copy(s, dtype, narrow.out);
    return err == hipSuccess ? SPC_OK : hip_status(err, "spc_lora_backward launch");
}

}  // extern "C"

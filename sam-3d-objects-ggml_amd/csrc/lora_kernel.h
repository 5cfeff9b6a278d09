// lora_kernel.h -- the kernels of the low-rank adapters (spc_lora) and their
// gradients (spc_lora_backward).  With a the adapter of a row's item, s_a its
// scale and d the dropout of the rows (rows8.h),
//
//   h = d(x) down_a^T,  y = base + s_a h up_a^T
//   u = s_a dy up_a,    dx = dx_base + d(u down_a)
//   ddown_a = sum over a's rows of u^T d(x),  dup_a = s_a sum of dy^T h
//
// Up to rank 32 it is bound by the rows' bytes (few rows: the adapters'), so every pass
// reads its rows once and the products run on the matrix instructions, which
// are far from their limit (rank 16: some 50 operations a byte at most).  BF16,
// inputs that change: y of 62,710 x 1024, rank 16, with a base 79 us (4.8 TB/s; a
// large copy 5.15); its gradients' pass over dy 38 us (132 MB and 24 of u and sums,
// 4.1 TB/s), over x 100 by itself (401 MB, 4.0 TB/s; the dropout's mask is 8 of them), the
// sums 9; the call 133.
// Larger ranks cost the adapters' way through L2 for each tile of rows and, in the gradients,
// where a block holds 128 columns (64 of F32), u's shares, their sum and the hidden rows by
// every block: more than the rows themselves.  30,000 x 1024 with a base, kernels alone, rank 16
// / 64 / 128: 41 / 57 / 101 us, gradients 71 / 146 / 223 (floors 36, 48 to 51); rank 100 F16 134
// and 315; F32 rank 128 258 and 504 (72 and 99).  Rows of 16-bit elements at odd addresses
// take twice the time (1023 to 1021: 79, 110).
//
// 16-bit rows meet 16-bit weights exactly (F32 sums).  h and u stay F32, and
// meet 16-bit operands as three bf16 parts of eight bits each, whose sum is the
// value itself (below 2^-110 but for what lies under 2^-133, bf16's last bit; two
// parts, 2^-16 of the value, turned outputs' roundings over); f16 operands of those
// products are two bf16 parts, exactly too, so that no range but F32's bounds h
// and u.  F32 rows run on F32 matrix instructions.
#pragma once

#include "rows8.h"

namespace spc {

constexpr int64_t kLoraMaxRank = 128, kLoraMaxItems = 65535, kLoraMaxAdapters = 65535;
constexpr int64_t kLoraMaxWidth = 1 << 24, kLoraMaxRows = 1 << 27;
constexpr int kLoraThreads = 256;

// Where the items' rows and adapters are.  Without offsets segment i is item i's
// rows, `per` of them; with them segment 0 is the rows before the first item,
// segment i + 1 item i's, the last the rows behind the items.
struct LoraItems {
    const int64_t* off;    // [items + 1] or null
    const int32_t* which;  // [items] or null: adapter 0
    int64_t items, adapters, n, per;

    __device__ __forceinline__ int64_t segments() const { return off ? items + 2 : items; }
    __device__ __forceinline__ int64_t begin(int64_t v) const {
        return !off ? v * per : v == 0 ? 0 : min(max(off[v - 1], (int64_t)0), n);
    }
    __device__ __forceinline__ int64_t end(int64_t v) const {
        return !off ? (v + 1) * per : v == items + 1 ? n : min(max(off[v], (int64_t)0), n);
    }
    // the segment's adapter, -1 for none
    __device__ __forceinline__ int64_t adapter(int64_t v) const {
        if (off) {
            if (v == 0 || v > items) return -1;
            --v;
        }
        const int64_t a = which ? which[v] : 0;
        return a >= 0 && a < adapters ? a : -1;
    }
    // The last segment v with begin(v) / rows + per v <= t, its rows and adapter (64 probes
    // at a time, by a whole wave; inside the segments' range whatever the offsets hold).
    // What the last probes' lanes need is read in one go: a wait of its own for each of
    // them is a good part of what few rows take.
    struct Found {
        int64_t v, begin, end, adapter;
    };
    __device__ __forceinline__ Found find(int64_t t, int rows, int64_t per) const {
        auto quotient = [&](int64_t b) { return (int64_t)((uint32_t)b / (uint32_t)rows); };
        const int lane = threadIdx.x & 63;
        int64_t lo = 0, size = segments();
        while (size > 64) {
            const int64_t step = (size + 63) / 64, at = lane * step;
            const bool ok = at < size && quotient(begin(lo + at)) + per * (lo + at) <= t;
            const int64_t past = max(__popcll(__ballot(ok)), 1) - 1;
            lo += past * step;
            size = min(step, size - past * step);
        }
        const int64_t v = lo + min((int64_t)lane, size - 1);
        const int64_t b = begin(v), e = end(v);
        const int a = (int)adapter(v);
        const bool ok = lane < size && quotient(b) + per * v <= t;
        const int k = max(__popcll(__ballot(ok)), 1) - 1;
        auto pick = [&](int64_t x) {
            return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), k) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane((int)x, k));
        };
        return {lo + k, pick(b), pick(e), __builtin_amdgcn_readlane(a, k)};
    }
};

struct LoraArgs {
    LoraItems it;
    const void* x;
    int64_t xs;
    const void* down;
    const void* up;
    const float* scale;
    const void* base;
    int64_t bs;
    void* y;
    float* hidden;
    float* part;  // [splits][n][r]
    int c, o, r;  // in_features, out_features, rank
    int k_per, splits, col_per;
    const int64_t* seed;
    uint32_t drop;
    float factor;
};

struct LoraBackArgs {
    LoraItems it;
    const void* dy;
    int64_t dys;
    const void* x;
    int64_t xs;
    const float* hidden;
    const void* down;
    const void* up;
    const float* scale;
    const void* base;  // dx_base
    int64_t bs;
    void* dx;
    float* u;          // [u_parts][n][r]
    int u_parts;
    float* pd;         // slots of ddown (lora_slot), null: not wanted
    float* pu;         // of dup
    int c, o, r;
    int rows_per, blocks;  // rows of a chunk, blocks along columns
    int chunk0;            // the launch's first chunk, whose slot is the first
    const int64_t* seed;
    uint32_t drop;
    float factor;
};

// Launches, one for each of the rows' dtypes (lora_bf16.hip, ...).  mt: row tiles
// of 16 in a block's tile, 1 or kLoraRowTiles, of ranks 33 to 64 twice as many too.
enum { kLoraFused, kLoraShrink, kLoraExpand };
#define LORA_LAUNCHERS(D)                                                                             \
    hipError_t lora_forward_##D(hipStream_t s, const LoraArgs& p, int mode, int mt, dim3 grid);       \
    hipError_t lora_back_out_##D(hipStream_t s, const LoraBackArgs& p, dim3 grid);                    \
    hipError_t lora_back_in_##D(hipStream_t s, const LoraBackArgs& p, dim3 grid);
LORA_LAUNCHERS(bf16)
LORA_LAUNCHERS(f16)
LORA_LAUNCHERS(f32)
#undef LORA_LAUNCHERS

// Copies of rows (lora_narrow.hip): `width` elements of each, then zeros up to `fill`
// (rows x fill < 2^31).
struct LoraCopy {
    const void* src;
    void* dst;
    int64_t rows, src_stride, dst_stride;
    int width, fill;
};
struct LoraCopies {
    LoraCopy job[5];
    int jobs;
};
hipError_t lora_copy(hipStream_t s, int dt, const LoraCopies& q);

// ranks in tiles of 16: 1, 2, 4 or 8
inline int lora_rank_tiles(int64_t r) { return r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : 8; }
constexpr int kLoraRowTiles = 2;
// waves of a block along the ranks in the backward kernels (the others along columns)
inline int lora_rank_waves(int64_t r) { return r <= 16 ? 1 : r <= 32 ? 2 : 4; }
// columns of one such wave
inline int lora_wave_cols(int dt) { return dt == SPC_F32 ? 64 : 128; }
// and the waves along columns: half of them where the last block of all would use no
// more, one for rows no wider than its own, the others along rows (us of the gradients, so /
// all along columns, rank 16 bf16: 200,000 x 64 to 64 54 / 112, 53,333 x 576 68 / 75, 40,000 x
// 768 64 / 66, 27,927 x 1100 74 / 78; where the last block would use more, all along columns
// and half of them: 34,133 x 900 84 / 88, 21,818 x 1408 76 / 75)
inline int lora_col_waves(int dt, int64_t r, int64_t width) {
    const int64_t tiles = (width + lora_wave_cols(dt) - 1) / lora_wave_cols(dt);
    int w = 4 / lora_rank_waves(r);
    if (w == 4 && (tiles - 1) % 4 < 2) w = 2;
    return tiles == 1 ? 1 : w;
}
inline int lora_row_waves(int dt, int64_t r, int64_t width) {
    return 4 / lora_rank_waves(r) / lora_col_waves(dt, r, width);
}

// The gradients of few rows (lora_few.hip); u in u_parts shares of o_per outputs.
hipError_t lora_few_backward(hipStream_t s, int dt, const LoraBackArgs& p, int o_per, void* ddown, void* dup);

// ---------------------------------------------------------------------------
// operands
// ---------------------------------------------------------------------------
template <int DT>
struct LoraNum {
    using S = typename RowElem<DT>::S;
    static constexpr int V = 16 / (int)sizeof(S);  // elements of 16 bytes
    static constexpr int STEP = 4 * V;             // summed elements of a matrix step
    static constexpr int PARTS = DT == SPC_F16 ? 2 : 1;   // of a weight or row that meets F32 values
};

// V elements of a row (c >= V of them, at any address) from `col` on, in two steps:
// 16 bytes that lie inside the row, without a branch, and, only in blocks that hold
// a row's end, what moves them into place and clears what is past it.  (With a
// branch at each load the backward kernels spilled the masks of all of them.)
typedef float floatx4_rows __attribute__((ext_vector_type(4), aligned(4)));  // (at any float)
template <typename S>
__device__ __forceinline__ u32x4 lora_shift(u32x4 w, int by) {
    constexpr int V = 16 / (int)sizeof(S);
    asm volatile("" : "+v"(by));  // (or its comparisons' masks are kept through the loops)
    if constexpr (V == 8)
        w = by & 1 ? u32x4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16} : w;
    w = by & (V / 4) ? u32x4{w[1], w[2], w[3], 0} : w;
    w = by & (V / 2) ? u32x4{w[2], w[3], 0, 0} : w;
    return by >= V ? u32x4{0, 0, 0, 0} : w;
}
template <typename S>
__device__ __forceinline__ u32x4 lora_fetch(const S* row, int col, int c) {
    return *reinterpret_cast<const u32x4_rows*>(row + min(col, c - 16 / (int)sizeof(S)));
}
// The same of rows that a call reads once, past the caches. With inputs that change from call to call it measured 32.4 us
// against 35.1 at 11,774 x 2048 to 1024 of rank 32, BF16, and 134.8 against 139 for the gradients of 62,710 x 1024 of rank 16.
// The same 96 MB over and over, which then stay in the memory's own cache, are faster kept: 29 us against 32.3.
template <typename S>
__device__ __forceinline__ u32x4 lora_stream(const S* row, int col, int c) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_rows*>(row + min(col, c - 16 / (int)sizeof(S))));
}
template <typename S>
__device__ __forceinline__ u32x4 lora_edge(u32x4 w, int col, int c) {
    return lora_shift<S>(w, max(col - (c - 16 / (int)sizeof(S)), 0));
}
template <typename S>
__device__ __forceinline__ u32x4 lora_load(const S* row, int col, int c) {
    return lora_edge<S>(lora_fetch(row, col, c), col, c);
}
// The same of a short row, r elements at `at` of an array of `all` >= V: the 16
// bytes lie inside the array, and what is not the row's is cleared.
template <typename S>
__device__ __forceinline__ u32x4 lora_fetch_short(const S* array, int64_t at, int64_t all) {
    return *reinterpret_cast<const u32x4_rows*>(array + min(at, all - 16 / (int)sizeof(S)));
}
template <typename S>
__device__ __forceinline__ u32x4 lora_edge_short(u32x4 w, int64_t at, int64_t all, int left) {
    constexpr int V = 16 / (int)sizeof(S);
    w = lora_shift<S>(w, (int)max(at - (all - V), (int64_t)0));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if constexpr (V == 4) w[q] = q < left ? w[q] : 0;
        else w[q] = 2 * q + 1 < left ? w[q] : 2 * q < left ? w[q] & 0xffff : 0;
    }
    return w;
}

// Stores V elements at q, `left` of which are the row's.
template <typename S>
__device__ __forceinline__ void lora_store(S* q, u32x4 w, int left) {
    constexpr int V = 16 / (int)sizeof(S);
    if (left >= V) {
        *reinterpret_cast<u32x4_rows*>(q) = w;
    } else {
        for (int e = 0; e < left; ++e) {
            if constexpr (V == 4) {
                q[e] = w[0];
                w = u32x4{w[1], w[2], w[3], 0};
            } else {
                q[e] = (uint16_t)w[0];
                w = u32x4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
            }
        }
    }
}

template <int DT>
__device__ __forceinline__ float lora_value(u32x4 w, int e) {
    if constexpr (DT == SPC_F32) return __uint_as_float(w[e]);
    else if constexpr (DT == SPC_BF16)
        return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    else return f16_bits_to_f32((uint16_t)(w[e / 2] >> (16 * (e & 1))));
}

// one element
template <int DT>
__device__ __forceinline__ float lora_get(const void* p, int64_t i) {
    if constexpr (DT == SPC_F32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == SPC_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void lora_put(void* p, int64_t i, float v) {
    if constexpr (DT == SPC_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = DT == SPC_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}

template <int DT>
__device__ __forceinline__ u32x4 lora_round(const float (&v)[LoraNum<DT>::V]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == SPC_F32) w[i] = __float_as_uint(v[i]);
        else w[i] = round_pair<DT>(v[2 * i], v[2 * i + 1]);
    }
    return w;
}

// 16 x 16 products over STEP summed elements: row operand a (lane % 16 the
// result's row), column operand b (lane % 16 its column), elements V (lane / 16)
// on of the step; the result's rows 4 (lane / 16) .. + 3 of column lane % 16.
template <int DT>
__device__ __forceinline__ floatx4 lora_mma(u32x4 a, u32x4 b, floatx4 c) {
    if constexpr (DT == SPC_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
    } else if constexpr (DT == SPC_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
        return c;
    }
}

// The upper halves of two values, a's below: their leading eight bits as bf16.
__device__ __forceinline__ uint32_t lora_cut(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
// What those leave, exactly.  (An infinity leaves NaN, and one that meets a part of zero
// makes it: LoraRanks and lora_flush_plain put right what that would spoil.)
__device__ __forceinline__ float lora_rest(float a) { return a - __uint_as_float(__float_as_uint(a) & 0xffff0000u); }

// F32 values h and u as column operand: 16-bit rows three bf16 parts, which hold all
// 24 bits.
struct LoraSplit {
    u32x4 hi, mid, lo;
};
__device__ __forceinline__ LoraSplit lora_split8(const float (&v)[8]) {
    LoraSplit s;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float a = v[2 * q], b = v[2 * q + 1], ra = lora_rest(a), rb = lora_rest(b);
        s.hi[q] = lora_cut(a, b);
        s.mid[q] = lora_cut(ra, rb);
        s.lo[q] = lora_cut(lora_rest(ra), lora_rest(rb));
    }
    return s;
}

// A 16-bit operand's bf16 parts (f16: two, exactly).
template <int DT>
struct LoraParts {
    u32x4 p[LoraNum<DT>::PARTS];
    __device__ __forceinline__ explicit LoraParts(u32x4 w) {
        if constexpr (DT == SPC_F16) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float a = lora_value<DT>(w, 2 * q), b = lora_value<DT>(w, 2 * q + 1);
                p[0][q] = lora_cut(a, b);
                p[1][q] = lora_cut(lora_rest(a), lora_rest(b));
            }
        } else {
            p[0] = w;
        }
    }
    LoraParts() = default;
};

// 16-bit operand times F32 values, the small products first.
template <int DT>
__device__ __forceinline__ floatx4 lora_mma_split(const LoraParts<DT>& a, const LoraSplit& b, floatx4 c) {
    if constexpr (DT == SPC_F16) {
        c = lora_mma<SPC_BF16>(a.p[1], b.lo, c);
        c = lora_mma<SPC_BF16>(a.p[1], b.mid, c);
        c = lora_mma<SPC_BF16>(a.p[1], b.hi, c);
    }
    c = lora_mma<SPC_BF16>(a.p[0], b.lo, c);
    c = lora_mma<SPC_BF16>(a.p[0], b.mid, c);
    return lora_mma<SPC_BF16>(a.p[0], b.hi, c);
}

// Dropout of V elements of a row from column `col` on: the group's mask (words of
// halves), and the elements with zeros where dropped.
__device__ __forceinline__ u32x4 lora_ones(DropKey key, uint32_t drop, int64_t row, int col, int c) {
    return drop_ones(philox7(key, (uint64_t)(row * ((c + 7) / 8) + col / 8)), drop);
}
// Column `col` of its group: kept.
__device__ __forceinline__ bool lora_keeps(u32x4 ones, int col) {
    const uint32_t q = col & 4 ? (col & 2 ? ones[3] : ones[2]) : (col & 2 ? ones[1] : ones[0]);
    return q >> (16 * (col & 1)) & 1;
}
template <int DT>
__device__ __forceinline__ u32x4 lora_masked(u32x4 w, u32x4 ones, int col) {
    if constexpr (DT == SPC_F32) {
        const bool second = col & 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = drop_word(w[e], second ? ones[2 + e / 2] : ones[e / 2], 16 * (e & 1));
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = drop_pair(w[q], ones[q]);
    }
    return w;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// The F32 operand (hidden rows; ranks are the summed index) of a row tile: steps
// of V lane-groups of ranks.  Rank up to 16 under 16-bit rows: lanes 0..31 hold the
// second parts of ranks 8 (lane / 16 % 2) on, lanes 32..63 the third, so that one
// matrix instruction takes both, and another the first beside zeros.
// The first parts have a sum of their own.  Where a value or a weight is infinite it is
// what the formula has, and the sum of the rest may be NaN, of a part that is zero or of an
// infinity's: then it stands alone.
template <int DT, int RT>
struct LoraRanks {
    static constexpr bool F = DT == SPC_F32, ONE = !F && RT == 1;
    static constexpr int V = LoraNum<DT>::V;
    static constexpr int STEPS = F ? RT : RT == 1 ? 1 : RT / 2;
    // first rank of lane group g in step s
    __device__ static __forceinline__ int rank(int s, int g) { return ONE ? 8 * (g & 1) : 4 * V * s + V * g; }

    // row operand: the weights' parts
    struct W {
        LoraParts<DT> w[STEPS];
        u32x4 first;  // (ONE: of the first parts, zeros in lanes 32..63)
        // from 16 bytes of a column's ranks a step
        __device__ __forceinline__ void set(const u32x4 (&raw)[STEPS], int g) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) w[s] = LoraParts<DT>(raw[s]);
            if constexpr (ONE) first = g < 2 ? w[0].p[0] : u32x4{0, 0, 0, 0};
        }
        // q: the same in LDS, zeros past the rank
        __device__ __forceinline__ void load_lds(const typename LoraNum<DT>::S* q, int g) {
            u32x4 raw[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) raw[s] = *reinterpret_cast<const u32x4*>(q + rank(s, g));
            set(raw, g);
        }
    };
    // column operand
    struct H {
        u32x4 hi[STEPS], mid[F ? 1 : STEPS], lo[F || ONE ? 1 : STEPS];
        // q: the row's F32 values in LDS, zeros past the rank
        __device__ __forceinline__ void load(const float* q, int g) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const float* f = q + rank(s, g);
                if constexpr (F) {
                    hi[s] = *reinterpret_cast<const u32x4*>(f);
                } else {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = f[e];
                    const LoraSplit t = lora_split8(v);
                    if constexpr (ONE) {
                        hi[s] = g < 2 ? t.hi : u32x4{0, 0, 0, 0};
                        mid[s] = g < 2 ? t.mid : t.lo;
                    } else {
                        hi[s] = t.hi;
                        mid[s] = t.mid;
                        lo[s] = t.lo;
                    }
                }
            }
        }
    };
    __device__ static __forceinline__ floatx4 mma(const W& w, const H& h) {
        floatx4 c = {0, 0, 0, 0}, rest = {0, 0, 0, 0};
        if constexpr (F) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) c = lora_mma<SPC_F32>(w.w[s].p[0], h.hi[s], c);
            return c;
        } else if constexpr (ONE) {
            if constexpr (DT == SPC_F16) {
                rest = lora_mma<SPC_BF16>(w.w[0].p[1], h.mid[0], rest);
                rest = lora_mma<SPC_BF16>(w.w[0].p[1], h.hi[0], rest);
            }
            rest = lora_mma<SPC_BF16>(w.w[0].p[0], h.mid[0], rest);
            c = lora_mma<SPC_BF16>(w.first, h.hi[0], c);
        } else {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                if constexpr (DT == SPC_F16) {
                    rest = lora_mma<SPC_BF16>(w.w[s].p[1], h.lo[s], rest);
                    rest = lora_mma<SPC_BF16>(w.w[s].p[1], h.mid[s], rest);
                    rest = lora_mma<SPC_BF16>(w.w[s].p[1], h.hi[s], rest);
                }
                rest = lora_mma<SPC_BF16>(w.w[s].p[0], h.lo[s], rest);
                rest = lora_mma<SPC_BF16>(w.w[s].p[0], h.mid[s], rest);
                c = lora_mma<SPC_BF16>(w.w[s].p[0], h.hi[s], c);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float z = c[e] + rest[e];
            c[e] = z == z ? z : c[e];
        }
        return c;
    }
};

// Column of a 16-column tile's row operand index m, tile t of the group at `col`:
// 16-bit rows take two tiles at once, interleaved so that a lane's results are
// eight consecutive columns V (lane / 16) on, as one 16-byte store wants them.
template <int DT>
__device__ __forceinline__ int lora_col(int col, int t, int m) {
    if constexpr (DT == SPC_F32) return col + m;
    else return col + 8 * (m >> 2) + 4 * t + (m & 3);
}

// Lanes 8 apart exchange one of two words: lora_mma's layout of two steps of columns
// (V columns from V (lane / 16) on of row lane % 16, the first step's in a, the second's
// in b) becomes eight lanes a row, rows 0 to 7 in a and 8 to 15 in b, and back.
__device__ __forceinline__ void lora_turn_pair(u32x4& a, u32x4& b) {
    const bool high = threadIdx.x & 8;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t mine = high ? a[q] : b[q];
        const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)mine, 0x128, 0xf, 0xf, true);  // lane ^ 8
        a[q] = high ? other : a[q];
        b[q] = high ? b[q] : other;
    }
}

// Stores a tile of 16 rows x 2 STEP columns whose results lie as lora_mma leaves
// them, rows below m of it: a lane has V columns from V (lane / 16) on of row lane %
// 16, of the first step in a and of the second in b.  Eight lanes a row take 128
// bytes of it in one store, after lanes 8 apart have exchanged one of the two
// (rows of 1024, read and written: 64 bytes of a row in a store 102 us, 128 76).
// Whole lines go past the caches, parts of lines meet there first (us, past / through:
// 62,710 rows of 1024 BF16 78.3 / 81.3; 30,000 of 1016 42 / 38, of 1022 48 / 41, of
// 1008 38 / 35).
template <typename S>
__device__ __forceinline__ void lora_store_pair(S* at, int64_t stride, u32x4 a, u32x4 b, int m) {
    constexpr int V = 16 / (int)sizeof(S);
    const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4;
    lora_turn_pair(a, b);
    S* q = at + (n16 & 7) * stride + V * g + (n16 & 8 ? 4 * V : 0);
    u32x4_rows *first = reinterpret_cast<u32x4_rows*>(q), *second = reinterpret_cast<u32x4_rows*>(q + 8 * stride);
    if (stride % (128 / (int)sizeof(S)) == 0) {
        if ((n16 & 7) < m) __builtin_nontemporal_store(a, first);
        if ((n16 & 7) + 8 < m) __builtin_nontemporal_store(b, second);
    } else {
        if ((n16 & 7) < m) *first = a;
        if ((n16 & 7) + 8 < m) *second = b;
    }
}

// Such a tile's elements, rows past m as the last (lora_turn_pair for lora_mma's layout).
template <typename S>
__device__ __forceinline__ void lora_fetch_pair(u32x4& first, u32x4& second, const S* at, int64_t stride, int m) {
    constexpr int V = 16 / (int)sizeof(S);
    const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4, row = n16 & 7;
    const S* q = at + V * g + (n16 & 8 ? 4 * V : 0);
    first = __builtin_nontemporal_load(reinterpret_cast<const u32x4_rows*>(q + min(row, m - 1) * stride));
    second = __builtin_nontemporal_load(reinterpret_cast<const u32x4_rows*>(q + min(row + 8, m - 1) * stride));
}
struct LoraTile {
    int64_t row0, a;
    int m;  // rows
};

constexpr int lora_pitch(int rp) { return rp + 4; }

// Sums of the block's four waves over columns [k0, k1) of rows: red[wave][row]
// [rank] in LDS.  Rows past the tile's and ranks past r hold what a valid one
// does (they are not read).
template <int DT, int RT, int MT, bool DROP>
__device__ __forceinline__ void lora_shrink(const LoraArgs& p, const LoraTile& t, int k0, int k1, float* red) {
    using N = LoraNum<DT>;
    using S = typename N::S;
    // (steps in flight: few rows are bound by the latency of their loads)
    constexpr int V = N::V, UN = RT <= 2 ? 4 : 2;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n16 = lane & 15, g = lane >> 4;
    const S* xr[MT];
    const S* wr[RT];
    int64_t row[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        row[i] = t.row0 + min(16 * i + n16, t.m - 1);
        xr[i] = static_cast<const S*>(p.x) + row[i] * p.xs;
    }
#pragma unroll
    for (int j = 0; j < RT; ++j)
        wr[j] = static_cast<const S*>(p.down) + (t.a * p.r + min(16 * j + n16, p.r - 1)) * p.c;
    floatx4 acc[MT][RT] = {};
    const DropKey key = DROP ? drop_key(p.seed) : DropKey{};
    for (int k = k0 + w * UN * N::STEP; k < k1; k += 4 * UN * N::STEP) {
        u32x4 xv[UN][MT], wv[UN][RT];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int col = k + u * N::STEP + V * g;
#pragma unroll
            for (int i = 0; i < MT; ++i) xv[u][i] = lora_fetch(xr[i], col, k1);
#pragma unroll
            for (int j = 0; j < RT; ++j) wv[u][j] = lora_fetch(wr[j], col, k1);
        }
        if (k + UN * N::STEP > k1) {
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int col = k + u * N::STEP + V * g;
#pragma unroll
                for (int i = 0; i < MT; ++i) xv[u][i] = lora_edge<S>(xv[u][i], col, k1);
#pragma unroll
                for (int j = 0; j < RT; ++j) wv[u][j] = lora_edge<S>(wv[u][j], col, k1);
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (DROP) {
                const int col = k + u * N::STEP + V * g;
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    xv[u][i] = lora_masked<DT>(xv[u][i], lora_ones(key, p.drop, row[i], col, p.c), col);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[i][j] = lora_mma<DT>(wv[u][j], xv[u][i], acc[i][j]);
        }
    }
    constexpr int P = lora_pitch(16 * RT);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j)
            *reinterpret_cast<floatx4*>(red + (w * 16 * MT + 16 * i + n16) * P + 16 * j + 4 * g) = acc[i][j];
}

// y's columns [c0, c1) of the tile's rows from their hidden rows in LDS.
template <int DT, int RT, int MT>
__device__ __forceinline__ void lora_expand(const LoraArgs& p, const LoraTile& t, int c0, int c1, const float* hid) {
    using N = LoraNum<DT>;
    using S = typename N::S;
    using K = LoraRanks<DT, RT>;
    constexpr int V = N::V, T = V / 4, P = lora_pitch(16 * RT);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n16 = lane & 15, g = lane >> 4;
    typename K::H h[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) h[i].load(hid + (16 * i + n16) * P, g);
    const float s = p.scale ? p.scale[t.a] : 1.0f;
    const S* up = static_cast<const S*>(p.up);
    const int64_t all = p.it.adapters * p.o * p.r;
    // two steps of columns at a time
    for (int cb = c0 + w * 2 * N::STEP; cb < c1; cb += 8 * N::STEP) {
        u32x4 wr[2][T][K::STEPS], b[2][MT];
        const bool edge = cb + 2 * N::STEP > p.o;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int q = 0; q < T; ++q) {
                const int64_t at = (t.a * p.o + min(lora_col<DT>(cb + x * N::STEP, q, n16), p.o - 1)) * p.r;
#pragma unroll
                for (int k = 0; k < K::STEPS; ++k) wr[x][q][k] = lora_fetch_short(up, at + K::rank(k, g), all);
            }
        }
        if (p.base) {
            const S* base = static_cast<const S*>(p.base) + t.row0 * p.bs;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (!edge) {
                    lora_fetch_pair(b[0][i], b[1][i], base + min(16 * i, t.m - 1) * p.bs + cb, p.bs, max(t.m - 16 * i, 1));
                } else {
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        b[x][i] = lora_fetch(base + min(16 * i + n16, t.m - 1) * p.bs, cb + x * N::STEP + V * g, p.o);
                }
            }
        }
        if (p.r < 16 * RT)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int q = 0; q < T; ++q) {
                    const int64_t at = (t.a * p.o + min(lora_col<DT>(cb + x * N::STEP, q, n16), p.o - 1)) * p.r;
#pragma unroll
                    for (int k = 0; k < K::STEPS; ++k)
                        wr[x][q][k] = lora_edge_short<S>(wr[x][q][k], at + K::rank(k, g), all, p.r - K::rank(k, g));
                }
        if (p.base)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (!edge) {
                    lora_turn_pair(b[0][i], b[1][i]);
                } else {
#pragma unroll
                    for (int x = 0; x < 2; ++x) b[x][i] = lora_edge<S>(b[x][i], cb + x * N::STEP + V * g, p.o);
                }
            }
        u32x4 out[2][MT];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            typename K::W wt[T];
#pragma unroll
            for (int q = 0; q < T; ++q) wt[q].set(wr[x][q], g);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float v[V];
#pragma unroll
                for (int q = 0; q < T; ++q) {
                    const floatx4 z = K::mma(wt[q], h[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * q + e] = s * z[e];
                }
                if (p.base)
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] += lora_value<DT>(b[x][i], e);
                out[x][i] = lora_round<DT>(v);
            }
        }
        S* y = static_cast<S*>(p.y) + t.row0 * p.o + cb;
        if (!edge) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
                lora_store_pair(y + (int64_t)16 * i * p.o, p.o, out[0][i], out[1][i], t.m - 16 * i);
        } else {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const int at = x * N::STEP + V * g;
                    if (16 * i + n16 < t.m) lora_store(y + (int64_t)(16 * i + n16) * p.o + at, out[x][i], p.o - cb - at);
                }
        }
    }
}

// Columns [c0, c1) of rows without an adapter: the base, or zeros.
template <int DT>
__device__ __forceinline__ void lora_pass(void* y, int64_t ys, const void* base, int64_t bs, int64_t row0, int m, int c0,
                                          int c1) {
    using S = typename LoraNum<DT>::S;
    constexpr int V = LoraNum<DT>::V;
    const int groups = (c1 - c0 + V - 1) / V;
    for (int i = threadIdx.x; i < m * groups; i += kLoraThreads) {
        const int64_t row = row0 + i / groups;
        const int col = c0 + i % groups * V;
        u32x4 w = {0, 0, 0, 0};
        if (base) w = lora_load(static_cast<const S*>(base) + row * bs, col, c1);
        lora_store(static_cast<S*>(y) + row * ys + col, w, c1 - col);
    }
}

// Blocks a CU: two, or as many more as fit; one for F32 rows and the largest ranks, whose
// registers for two cost more than the second gives (30,000 x 1024 rank 128, one / two:
// 235 / 256 us; BF16's two take 84).
constexpr int lora_forward_blocks(int dt, int rt, int mt) { return dt == SPC_F32 && rt == 8 && mt > 1 ? 1 : 2; }

// A block takes a tile of 16 MT rows of one segment (tile numbers begin at
// begin / rows + segment, so that no segment's meet another's whatever their
// lengths) and, by MODE, forms their hidden rows and from them `col_per` columns
// of y (kLoraFused), writes its hidden sums over `k_per` columns of x
// (kLoraShrink), or adds those and forms y (kLoraExpand).
//
// Where all tiles run at once, a tile's way through both products is what there is to
// wait for: 11,774 x 2048 to 1024, rank 32 BF16 33 us for 98 MB, one of them the
// dropout's mask; one row of 1024 to 2048 4.9 us in a graph, where an empty kernel is
// some 2.5.
template <int DT, int RT, int MT, int MODE, bool DROP>
__global__ __launch_bounds__(kLoraThreads, lora_forward_blocks(DT, RT, MT)) void lora_forward_kernel(LoraArgs p) {
    constexpr int R = 16 * MT, P = lora_pitch(16 * RT);
    __shared__ __attribute__((aligned(16))) float red[4 * R * P];
    float* hid = red;  // (the sums' own places)
    const LoraItems& it = p.it;
    const LoraItems::Found seg = it.find(blockIdx.x, R, 1);
    const int64_t row0 = seg.begin + (blockIdx.x - seg.begin / R - seg.v) * R;
    if (row0 >= seg.end || row0 < 0) return;
    const LoraTile t = {row0, seg.adapter, (int)min((int64_t)R, seg.end - row0)};
    const int c0 = MODE == kLoraShrink ? 0 : blockIdx.y * p.col_per;
    const int c1 = min(c0 + p.col_per, p.o);
    if (t.a < 0) {
        if (MODE != kLoraShrink) lora_pass<DT>(p.y, p.o, p.base, p.bs, row0, t.m, c0, c1);
        if (MODE != kLoraShrink && p.hidden && blockIdx.y == 0)
            for (int i = threadIdx.x; i < t.m * p.r; i += kLoraThreads) p.hidden[row0 * p.r + i] = 0.0f;
        return;
    }
    if constexpr (MODE != kLoraExpand) {
        const int k0 = MODE == kLoraShrink ? blockIdx.y * p.k_per : 0;
        const int k1 = MODE == kLoraShrink ? min(k0 + p.k_per, p.c) : p.c;
        lora_shrink<DT, RT, MT, DROP>(p, t, k0, k1, red);
    } else {
        // a wave takes every fourth share, so that few rows wait for few of them in turn, 16
        // bytes a lane (a value a lane, 40 rows of F32 rank 128 to 2368 71 us, so 32)
        const int w = threadIdx.x >> 6, all = t.m * p.r;
        for (int i = 4 * (threadIdx.x & 63); i < all; i += 256) {
            const int from = max(min(i, all - 4), 0);  // (a hidden row alone may hold fewer)
            const float* q = p.part + row0 * p.r + from;
            floatx4 s = {0, 0, 0, 0};
            if (all >= 4) {
#pragma unroll 8
                for (int k = w; k < p.splits; k += 4)
                    s += *reinterpret_cast<const floatx4_rows*>(q + (int64_t)k * it.n * p.r);
            } else {
                for (int k = w; k < p.splits; k += 4)
                    for (int e = 0; e < all; ++e) s[e] += q[(int64_t)k * it.n * p.r + e];
            }
            int m = from / p.r, j = from - m * p.r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (from + e < all) red[(w * R + m) * P + j] = s[e];
                if (++j == p.r) {
                    j = 0;
                    ++m;
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * 16 * RT; i += kLoraThreads) {
        const int m = i / (16 * RT), j = i % (16 * RT);
        float s = 0.0f;
        if (m < t.m && j < p.r) {
            const float* f = red + m * P + j;
            s = (f[0] + f[R * P]) + (f[2 * R * P] + f[3 * R * P]);
            if (DROP) s *= p.factor;
            if constexpr (MODE == kLoraShrink) p.part[((int64_t)blockIdx.y * it.n + row0 + m) * p.r + j] = s;
            else if (p.hidden && blockIdx.y == 0) p.hidden[(row0 + m) * p.r + j] = s;
        }
        if constexpr (MODE != kLoraShrink) hid[m * P + j] = s;
    }
    if constexpr (MODE != kLoraShrink) {
        __syncthreads();
        // (f16 tiles of 64 rows by halves: their parts and the weights' spill together, 30,000 x
        // 1024 rank 64 66 us so, 75 at once; bf16's fit, rank 33 68 and 64)
        constexpr int E = MT == 4 && DT == SPC_F16 ? 2 : MT;
        for (int i = 0; i < MT; i += E)
            if (16 * i < t.m)
                lora_expand<DT, RT, E>(p, LoraTile{t.row0 + 16 * i, t.a, min(t.m - 16 * i, 16 * E)}, c0, c1, hid + 16 * i * P);
    }
}

// (Tiles of more than 16 rows are of so many rows that they go in one kernel.)
template <int DT, int RT, int MT>
void lora_forward_mode(hipStream_t s, const LoraArgs& p, int mode, dim3 grid) {
    if constexpr (MT == 1) {
        if (mode == kLoraExpand) {
            lora_forward_kernel<DT, RT, MT, kLoraExpand, false><<<grid, kLoraThreads, 0, s>>>(p);
            return;
        }
        if (mode == kLoraShrink) {
            if (p.drop) lora_forward_kernel<DT, RT, MT, kLoraShrink, true><<<grid, kLoraThreads, 0, s>>>(p);
            else lora_forward_kernel<DT, RT, MT, kLoraShrink, false><<<grid, kLoraThreads, 0, s>>>(p);
            return;
        }
    }
    if (p.drop) lora_forward_kernel<DT, RT, MT, kLoraFused, true><<<grid, kLoraThreads, 0, s>>>(p);
    else lora_forward_kernel<DT, RT, MT, kLoraFused, false><<<grid, kLoraThreads, 0, s>>>(p);
}

template <int DT>
hipError_t lora_forward(hipStream_t s, const LoraArgs& p, int mode, int mt, dim3 grid) {
    const int rt = lora_rank_tiles(p.r);
    constexpr int M = kLoraRowTiles;
    if (rt == 1) mt == 1 ? lora_forward_mode<DT, 1, 1>(s, p, mode, grid) : lora_forward_mode<DT, 1, M>(s, p, mode, grid);
    else if (rt == 2) mt == 1 ? lora_forward_mode<DT, 2, 1>(s, p, mode, grid) : lora_forward_mode<DT, 2, M>(s, p, mode, grid);
    else if (rt == 4 && mt == 2 * M) lora_forward_mode<DT, 4, 2 * M>(s, p, mode, grid);
    else if (rt == 4) mt == 1 ? lora_forward_mode<DT, 4, 1>(s, p, mode, grid) : lora_forward_mode<DT, 4, M>(s, p, mode, grid);
    else mt == 1 ? lora_forward_mode<DT, 8, 1>(s, p, mode, grid) : lora_forward_mode<DT, 8, M>(s, p, mode, grid);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// Both kernels take chunks of rows_per rows by blocks of columns: a wave holds
// 32 rows x 16 V columns of them at a time, lane l rows 8 (l / 16) .. + 7 of columns
// V (l % 16) on (16 bytes a row).  That is the row operand of the weights'
// gradients (columns by summed rows; 16-bit elements are exchanged between the
// lane's registers to bring a column's eight rows together), whose sums stay in
// registers until the chunk, whose rows are of one segment, ends.  WC waves stand
// along the columns, WR along the ranks (16 RW each) and WG along the rows, a tile of
// 32 each: those of the same columns and rows load, and mask, a share of the rows each
// and pass them on through LDS, those along the rows add their sums there at the end.
constexpr int kLoraRows = 32;

// NR of a lane's eight rows, from j0 on.
template <int DT, int NR>
struct LoraRows {
    u32x4 v[NR];
    // Rows row0 + 8 g on, from `col` on (lora_fetch; rows past `end` are its last).
    __device__ __forceinline__ void load(const void* base, int64_t stride, int64_t row0, int64_t end, int j0, int col,
                                         int c) {
        using S = typename LoraNum<DT>::S;
        if (row0 >= end) return;
        const int first = (threadIdx.x & 63) / 16 * 8 + j0;
        if (row0 + kLoraRows <= end) {
            const S* q = static_cast<const S*>(base) + (row0 + first) * stride;
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                v[j] = lora_stream(q, col, c);
                q += stride;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NR; ++j)
                v[j] = lora_stream(static_cast<const S*>(base) + min(row0 + first + j, end - 1) * stride, col, c);
        }
    }
    // Zeros for what is past the end of the rows, and, at the row's end, of the columns.
    __device__ __forceinline__ void trim(int64_t row0, int64_t end, int j0, bool edge, int col, int c) {
        using S = typename LoraNum<DT>::S;
        if (row0 + kLoraRows > end) {
            const int rows = (int)(end - row0) - ((threadIdx.x & 63) / 16 * 8 + j0);
#pragma unroll
            for (int j = 0; j < NR; ++j)
                if (j >= rows) v[j] = u32x4{0, 0, 0, 0};
        }
        if (edge)
#pragma unroll
            for (int j = 0; j < NR; ++j) v[j] = lora_edge<S>(v[j], col, c);
    }
    // A tile of rows `pitch` apart in LDS.
    template <typename S>
    __device__ __forceinline__ void put(S* tile, int pitch, int j0) const {
        const int lane = threadIdx.x & 63;
        S* q = tile + (8 * (lane >> 4) + j0) * pitch + LoraNum<DT>::V * (lane & 15);
#pragma unroll
        for (int j = 0; j < NR; ++j) *reinterpret_cast<u32x4*>(q + j * pitch) = v[j];
    }
    template <typename S>
    __device__ __forceinline__ void get(const S* tile, int pitch) {
        const int lane = threadIdx.x & 63;
        const S* q = tile + 8 * (lane >> 4) * pitch + LoraNum<DT>::V * (lane & 15);
#pragma unroll
        for (int j = 0; j < NR; ++j) v[j] = *reinterpret_cast<const u32x4*>(q + j * pitch);
    }
    // column e's eight rows (16-bit elements)
    __device__ __forceinline__ u32x4 column(int e) const {
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            w[q] = __builtin_amdgcn_perm(v[2 * q + 1][e / 2], v[2 * q][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
        return w;
    }
};

// acc[e][j] += rows of column e times F32 values b[j][row] (rank tile j).
template <int DT, int RW>
__device__ __forceinline__ void lora_outer(const LoraRows<DT, 8>& raw, const float (&b)[RW][8],
                                           floatx4 (&acc)[LoraNum<DT>::V][RW]) {
    if constexpr (DT == SPC_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < RW; ++j)
                    acc[e][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(raw.v[i][e]), b[j][i], acc[e][j],
                                                                     0, 0, 0);
    } else {
        LoraSplit s[RW];
#pragma unroll
        for (int j = 0; j < RW; ++j) s[j] = lora_split8(b[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const LoraParts<DT> w(raw.column(e));
#pragma unroll
            for (int j = 0; j < RW; ++j) acc[e][j] = lora_mma_split<DT>(w, s[j], acc[e][j]);
        }
    }
}

// A slot of the weights' gradients holds its sums as the waves' registers do: for
// each tile of 16 V columns, rank tile and e, a lane's four (columns V (4 (lane / 16)
// + i) + e, rank lane % 16), so that a wave writes and the sum over the slots reads
// whole lines (by rank and column, four bytes a lane and line, the writes alone
// were 20 us of 62,710 x 1024).
constexpr int64_t lora_slot(int64_t c, int cw, int rt) { return (c + cw - 1) / cw * cw * 16 * rt; }

template <int DT, int RW>
__device__ __forceinline__ void lora_flush(const floatx4 (&acc)[LoraNum<DT>::V][RW], float* slot, int tile, int rt, int rank_tile,
                                           float f) {
    constexpr int V = LoraNum<DT>::V;
    float* q = slot + ((int64_t)tile * rt + rank_tile) * V * 256 + 4 * (threadIdx.x & 63);
#pragma unroll
    for (int j = 0; j < RW; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) *reinterpret_cast<floatx4*>(q + (j * V + e) * 256) = f * acc[e][j];
}

// Sums of 16-bit rows that lora_flush wrote as NaN are formed again without parts, to be
// the infinity that the formula has, or NaN after all: term(row, column, rank) is what the
// chunk's rows [r0, r1) add up.
template <int DT, int RW, typename Term>
__device__ __forceinline__ void lora_flush_plain(const floatx4 (&acc)[LoraNum<DT>::V][RW], float* slot, int tile, int rt,
                                                 int rank_tile, float f, int64_t r0, int64_t r1, int c, int r, Term term) {
    constexpr int V = LoraNum<DT>::V;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < V; ++e)
#pragma unroll
        for (int j = 0; j < RW; ++j)
            nan |= __builtin_isunordered(acc[e][j][0], acc[e][j][1]) | __builtin_isunordered(acc[e][j][2], acc[e][j][3]);
    if (DT == SPC_F32 || !__any(nan)) return;
    const int lane = threadIdx.x & 63;
    float* q = slot + ((int64_t)tile * rt + rank_tile) * V * 256 + 4 * lane;
    for (int k = 0; k < V * RW; ++k) {
        floatx4 z = *reinterpret_cast<const floatx4*>(q + k * 256);
        const int rank = 16 * (rank_tile + k / V) + (lane & 15);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 16 * V * tile + V * (4 * (lane >> 4) + i) + k % V;
            if (z[i] == z[i] || col >= c || rank >= r) continue;
            float s = 0.0f;
            for (int64_t row = r0; row < r1 && s == s; ++row) s += term(row, col, rank);
            z[i] = f * s;
        }
        *reinterpret_cast<floatx4*>(q + k * 256) = z;
    }
}

// The sums of the waves along the rows (WAVES of each) added to the first ones', in
// their order; ls: 64 V RW floatx4 for each of the others, which nobody else uses.
template <int WAVES, int WG, int V, int RW>
__device__ __forceinline__ void lora_gather(floatx4 (&acc)[V][RW], floatx4* ls) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (w >= WAVES)
#pragma unroll
        for (int e = 0; e < V; ++e)
#pragma unroll
            for (int j = 0; j < RW; ++j) ls[((w - WAVES) * V * RW + e * RW + j) * 64 + lane] = acc[e][j];
    lds_barrier();
    if (w < WAVES)
#pragma unroll
        for (int q = 0; q < WG - 1; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int j = 0; j < RW; ++j) acc[e][j] += ls[((q * WAVES + w) * V * RW + e * RW + j) * 64 + lane];
}

__device__ __forceinline__ void lora_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// The first row of chunk number t of the segment that find(t, rows, 1) gave: a segment's
// chunks of `rows` rows begin at number begin / rows + segment, so that no segment's meet
// another's whatever their lengths.
__device__ __forceinline__ int64_t lora_chunk_row(const LoraItems::Found& seg, int64_t t, int rows) {
    return seg.begin + (t - (uint32_t)seg.begin / (uint32_t)rows - seg.v) * rows;
}

// The pass over dy: u of the block's columns (one of u_parts shares of the sum),
// and the sums of dup.  u sums along a row, so its operand is read back from the
// tile in LDS, and the waves' shares meet there too; the adapter's columns lie in
// LDS by rank.
template <int DT, int RW, int WR, int WC>
__global__ __launch_bounds__(kLoraThreads, 2) void lora_back_out_kernel(LoraBackArgs p) {
    using N = LoraNum<DT>;
    using S = typename N::S;
    constexpr int V = N::V, CW = 16 * V, CB = WC * CW, RP = 16 * RW * WR, P = lora_pitch(16 * RW);
    constexpr int TP = CW + V, WP = CB + V;  // pitches of a tile and of the weights
    constexpr int NR = 8 / WR;               // rows a lane loads
    constexpr int WG = 4 / (WR * WC), ROWS = WG * kLoraRows;
    __shared__ __attribute__((aligned(16))) S tile[WC * WG][kLoraRows * TP];
    __shared__ __attribute__((aligned(16))) S wl[RP * WP];
    __shared__ __attribute__((aligned(16))) float red[2][4][kLoraRows * P];
    const LoraItems& it = p.it;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wc = w % WC, wr = w / WC % WR, first = WG == 1 ? 0 : w / (WC * WR) * kLoraRows, rank0 = 16 * RW * wr, j0 = NR * wr;
    const int slot_at = blockIdx.x / p.blocks, chunk = p.chunk0 + slot_at, block = blockIdx.x % p.blocks;
    const int block0 = block * CB, col0 = block0 + wc * CW;
    const bool edge = block0 + CB > p.o;
    static_assert(sizeof(tile) >= (WG - 1) * WC * WR * 64 * V * RW * 16, "the sums meet there");
    floatx4 acc[V][RW] = {};
    int turn = 0;
    const LoraItems::Found seg = it.find(chunk, p.rows_per, 1);
    const int64_t a = seg.adapter, r0 = lora_chunk_row(seg, chunk, p.rows_per), r1 = min(r0 + p.rows_per, seg.end);
    if (r0 < seg.begin || r0 >= r1 || a < 0) return;
    const float s = p.scale ? p.scale[a] : 1.0f;
    // dy and the hidden rows (a wave's ranks) two tiles ahead: with u's way through LDS a
    // tile takes longer than a load (one tile ahead 40 us of 62,710 x 1024)
    LoraRows<DT, NR> even, odd;
    float heven[RW][8], hodd[RW][8];
    auto load_h = [&](int64_t row0, float (&h)[RW][8]) {
        if (!p.pu || row0 >= r1) return;
        const int n16 = lane & 15, g = lane >> 4;
        const bool full = row0 + kLoraRows <= r1;
#pragma unroll
        for (int j = 0; j < RW; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t row = row0 + 8 * g + i;
                h[j][i] = p.hidden[(full ? row : min(row, r1 - 1)) * p.r + min(rank0 + 16 * j + n16, p.r - 1)];
            }
    };
    load_h(r0 + first, heven);
    even.load(p.dy, p.dys, r0 + first, r1, j0, col0 + V * (lane & 15), p.o);
    if (p.u) {
        const S* up = static_cast<const S*>(p.up);
        const int64_t all = it.adapters * p.o * p.r;
        for (int i = threadIdx.x; i < CB * (RP / V); i += kLoraThreads) {
            const int k = i % CB, j = i / CB * V, col = block0 + k;
            const int64_t at = (a * p.o + min(col, p.o - 1)) * p.r + j;
            const u32x4 q = lora_edge_short<S>(lora_fetch_short(up, at, all), at, all, col < p.o ? p.r - j : 0);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (V == 4) wl[(j + e) * WP + k] = q[e];
                else wl[(j + e) * WP + k] = (S)(q[e / 2] >> (16 * (e & 1)));
            }
        }
        lds_barrier();
    }
    load_h(r0 + ROWS + first, hodd);
    odd.load(p.dy, p.dys, r0 + ROWS + first, r1, j0, col0 + V * (lane & 15), p.o);
    auto step = [&](int64_t block_row, LoraRows<DT, NR>& rows, float (&h)[RW][8]) {
        const int64_t row0 = block_row + first;  // the wave's
        // (what follows from the lane is formed anew each time: kept through the loops it
        // would not fit the registers)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int n16 = ln & 15, g = ln >> 4, mine = col0 + V * n16;
        const S* t = tile[w / (WC * WR) * WC + wc];
        LoraRows<DT, 8> raw;
        rows.trim(row0, r1, j0, edge, mine, p.o);
        if (p.u || WR > 1) rows.put(const_cast<S*>(t), TP, j0);
        if constexpr (WR == 1) {
            raw = rows;
            lora_wave_sync();
        } else {
            lds_barrier();
        }
        rows.load(p.dy, p.dys, row0 + 2 * ROWS, r1, j0, mine, p.o);
        if constexpr (WR > 1) raw.get(t, TP);
        if (p.u) {
            floatx4 u[2][RW] = {};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                u32x4 wt[RW];
#pragma unroll
                for (int j = 0; j < RW; ++j)
                    wt[j] = *reinterpret_cast<const u32x4*>(wl + (rank0 + 16 * j + n16) * WP + wc * CW + q * N::STEP +
                                                            V * g);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const u32x4 d = *reinterpret_cast<const u32x4*>(t + (16 * i + n16) * TP + q * N::STEP + V * g);
#pragma unroll
                    for (int j = 0; j < RW; ++j) u[i][j] = lora_mma<DT>(wt[j], d, u[i][j]);
                }
            }
            float* f = red[turn][w];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < RW; ++j)
                    *reinterpret_cast<floatx4*>(f + (16 * i + n16) * P + 16 * j + 4 * g) = u[i][j];
        }
        // (also: the tile has been read; red is not written again before the next one)
        if (p.u || WR > 1) lds_barrier();
        if (p.u) {
            // (the waves of the same rows and ranks stand together)
            for (int i = threadIdx.x; i < ROWS * RP; i += kLoraThreads) {
                const int m = i / RP, j = i % RP;
                float z = 0.0f;
#pragma unroll
                for (int q = 0; q < WC; ++q)
                    z += red[turn][(m / kLoraRows * WR + j / (16 * RW)) * WC + q][m % kLoraRows * P + j % (16 * RW)];
                if (block_row + m < r1 && j < p.r)
                    p.u[((int64_t)block * it.n + block_row + m) * p.r + j] = s * z;
            }
            turn ^= 1;
        }
        if (p.pu) {
            if (row0 + kLoraRows > r1)
#pragma unroll
                for (int j = 0; j < RW; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (row0 + 8 * g + i >= r1) h[j][i] = 0.0f;
            lora_outer<DT, RW>(raw, h, acc);
            load_h(row0 + 2 * ROWS, h);
        }
    };
    for (int64_t row0 = r0; row0 < r1; row0 += 2 * ROWS) {
        step(row0, even, heven);
        if (row0 + ROWS < r1) step(row0 + ROWS, odd, hodd);
    }
    if (WG > 1 && p.pu) {
        lds_barrier();
        lora_gather<WC * WR, WG>(acc, reinterpret_cast<floatx4*>(tile));
    }
    if (p.pu && col0 < p.o && first == 0) {
        float* slot = p.pu + slot_at * lora_slot(p.o, CW, RW * WR);
        lora_flush<DT, RW>(acc, slot, col0 / CW, RW * WR, RW * wr, s);
        lora_flush_plain<DT, RW>(acc, slot, col0 / CW, RW * WR, RW * wr, s, r0, r1, p.o, p.r,
                                 [&](int64_t row, int col, int rank) {
                                     return lora_get<DT>(p.dy, row * p.dys + col) * p.hidden[row * p.r + rank];
                                 });
    }
}

// Shares of u that the pass over x adds (registers); of more, their sum comes first.
constexpr int lora_shares(int rt, int wg) { return wg > 2 || rt == 8 ? 1 : wg == 2 || rt > 1 ? 2 : 4; }

// The pass over x: dx of the block's columns and the sums of ddown.  The
// adapter's columns lie in LDS by column.
template <int DT, int RW, int WR, int WC, bool DROP>
__global__ __launch_bounds__(kLoraThreads, 2) void lora_back_in_kernel(LoraBackArgs p) {
    using N = LoraNum<DT>;
    using S = typename N::S;
    constexpr int RT = RW * WR;
    using K = LoraRanks<DT, RT>;
    constexpr int V = N::V, CW = 16 * V, CB = WC * CW, RP = 16 * RT, P = lora_pitch(RP), T = V / 4;
    constexpr int TP = CW + V, WP = RP + V;  // pitches of a tile and of the weights
    constexpr int NR = 8 / WR;               // rows a lane loads
    constexpr int WG = 4 / (WR * WC), ROWS = WG * kLoraRows;
    constexpr int BUF = RT == 8 ? 1 : 2;     // (room for two blocks a CU)
    // of the 4 steps of columns x 2 halves of rows of dx, a wave forms QN x NI
    constexpr int QN = WR == 1 ? 4 : 2, NI = WR == 4 ? 1 : 2;
    constexpr int G = CW / 8;                // groups of eight columns
    constexpr int NU = ROWS * RP / kLoraThreads;  // values of u a thread
    constexpr int SH = lora_shares(RT, WG);       // and the shares of each
    __shared__ __attribute__((aligned(16))) float ub[BUF][ROWS * P];
    __shared__ __attribute__((aligned(16))) S wl[CB * WP];
    __shared__ __attribute__((aligned(16))) S tile[WR > 1 ? BUF : 1][WR > 1 ? WC * WG : 1][WR > 1 ? kLoraRows * TP : 8];
    __shared__ uint8_t kept[DROP ? BUF : 1][DROP ? WC * WG : 1][kLoraRows * G];
    __shared__ floatx4 sums[WG > 1 ? (WG - 1) * WC * WR * V * RW * 64 : 1];
    const LoraItems& it = p.it;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wc = w % WC, wr = w / WC % WR, wg = WG == 1 ? 0 : w / (WC * WR), rank0 = 16 * RW * wr, j0 = NR * wr;
    const int q0 = WR == 1 ? 0 : WR == 2 ? 2 * wr : wr / 2 * 2, i0 = WR == 4 ? wr & 1 : 0;
    const int slot_at = blockIdx.x / p.blocks, chunk = p.chunk0 + slot_at, block0 = blockIdx.x % p.blocks * CB, col0 = block0 + wc * CW;
    const bool edge = block0 + CB > p.c;
    const DropKey key = DROP ? drop_key(p.seed) : DropKey{};
    floatx4 acc[V][RW] = {};
    int turn = 0;
    const LoraItems::Found seg = it.find(chunk, p.rows_per, 1);
    const int64_t a = seg.adapter, r0 = lora_chunk_row(seg, chunk, p.rows_per), r1 = min(r0 + p.rows_per, seg.end);
    if (r0 < seg.begin || r0 >= r1) return;
    if (a < 0) {
        if (p.dx && block0 < p.c)
            for (int64_t row = r0; row < r1; row += kLoraRows)
                lora_pass<DT>(p.dx, p.c, p.base, p.bs, row, (int)min((int64_t)kLoraRows, r1 - row), block0,
                              min(block0 + CB, p.c));
        return;
    }
    LoraRows<DT, NR> rows = {};
    u32x4 base[NI][QN] = {};
    float un[SH][NU];
    // the tiles' rows of u (its shares), and the wave's of dx_base
    auto load_u = [&](int64_t row0) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int at = threadIdx.x + i * kLoraThreads, m = at / RP, j = at % RP;
            const bool on = row0 + m < r1 && j < p.r;
            const float* q = p.u + (row0 + m) * p.r + j;
#pragma unroll
            for (int k = 0; k < SH; ++k) un[k][i] = on && k < p.u_parts ? q[k * it.n * p.r] : 0.0f;
        }
    };
    auto load_base = [&](int64_t row0, int n16, int g) {
        const int m = (int)min(r1 - row0, (int64_t)kLoraRows);
        const S* from = static_cast<const S*>(p.base) + row0 * p.bs;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int q = 0; q < QN; q += 2) {
                const int col = col0 + (q0 + q) * N::STEP, first = 16 * (i0 + i);
                if (!edge) {
                    lora_fetch_pair(base[i][q], base[i][q + 1], from + min(first, m - 1) * p.bs + col, p.bs,
                                    max(m - first, 1));
                } else {
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        base[i][q + x] = lora_fetch(from + min(first + n16, m - 1) * p.bs, col + x * N::STEP + V * g, p.c);
                }
            }
    };
    load_u(r0);
    if (p.pd) rows.load(p.x, p.xs, r0 + wg * kLoraRows, r1, j0, col0 + V * (lane & 15), p.c);
    if (p.dx) {
        const S* down = static_cast<const S*>(p.down) + a * p.c * p.r;
        for (int i = threadIdx.x; i < RP * (CB / V); i += kLoraThreads) {
            const int j = i % RP, k = i / RP * V, col = block0 + k;
            const u32x4 w = lora_load(down + (int64_t)min(j, p.r - 1) * p.c, col, p.c);
            const u32x4 q = j < p.r ? w : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (V == 4) wl[(k + e) * WP + j] = q[e];
                else wl[(k + e) * WP + j] = (S)(q[e / 2] >> (16 * (e & 1)));
            }
        }
    }
    for (int64_t block_row = r0; block_row < r1; block_row += ROWS) {
        const int64_t row0 = block_row + wg * kLoraRows;  // the wave's
        // (what follows from the lane is formed anew each time: kept through the loops it
        // would not fit the registers)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int n16 = ln & 15, g = ln >> 4, mine = col0 + V * n16;
        float* f = ub[turn];
        S* t = tile[WR > 1 ? turn : 0][WR > 1 ? wg * WC + wc : 0];
        uint8_t* keep = kept[DROP ? turn : 0][DROP ? wg * WC + wc : 0];
        turn = BUF == 2 ? turn ^ 1 : 0;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int at = threadIdx.x + i * kLoraThreads, m = at / RP, j = at % RP;
            float z = un[0][i];
            if constexpr (SH >= 2) z += un[1][i];
            if constexpr (SH == 4) z += un[2][i] + un[3][i];
            f[m * P + j] = z;
        }
        f += wg * kLoraRows * P;
        // (loads return in order: u, wanted first, before dx_base and the next rows)
        load_u(block_row + ROWS);
        if (p.dx && p.base && (WG == 1 || row0 < r1)) load_base(row0, n16, g);
        LoraRows<DT, 8> raw;
        LoraRows<DT, NR> now = rows;
        if (p.pd) {
            rows.load(p.x, p.xs, row0 + ROWS, r1, j0, mine, p.c);
            now.trim(row0, r1, j0, edge, mine, p.c);
        }
        if (DROP) {
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const u32x4 ones = lora_ones(key, p.drop, row0 + 8 * g + j0 + i, mine, p.c);
                now.v[i] = lora_masked<DT>(now.v[i], ones, mine);
                if (V == 8 || !(n16 & 1)) keep[(8 * g + j0 + i) * G + n16 * V / 8] = (uint8_t)drop_bits(ones);
            }
        }
        if constexpr (WR == 1) raw = now;
        else if (p.pd) now.put(t, TP, j0);
        lds_barrier();
        if (p.pd) {
            if constexpr (WR > 1) raw.get(t, TP);
            float b[RW][8];
#pragma unroll
            for (int j = 0; j < RW; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) b[j][i] = f[(8 * g + i) * P + rank0 + 16 * j + n16];
            lora_outer<DT, RW>(raw, b, acc);
        }
        if (p.dx && (WG == 1 || row0 < r1)) {
            if (p.base)
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int q = 0; q < QN; q += 2) {
                        if (!edge) {
                            lora_turn_pair(base[i][q], base[i][q + 1]);
                        } else {
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                                base[i][q + x] =
                                    lora_edge<S>(base[i][q + x], col0 + (q0 + q + x) * N::STEP + V * g, p.c);
                        }
                    }
            typename K::H h[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) h[i].load(f + (16 * (i0 + i) + n16) * P, g);
            const int m = (int)min(r1 - row0, (int64_t)kLoraRows);
            S* d = static_cast<S*>(p.dx) + row0 * p.c + col0 + q0 * N::STEP;
#pragma unroll
            for (int q = 0; q < QN; q += 2) {
                u32x4 out[NI][2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int at = (q0 + q + x) * N::STEP;
                    typename K::W wt[T];
#pragma unroll
                    for (int k = 0; k < T; ++k) wt[k].load_lds(wl + lora_col<DT>(wc * CW + at, k, n16) * WP, g);
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        float z[V];
#pragma unroll
                        for (int k = 0; k < T; ++k) {
                            const floatx4 d = K::mma(wt[k], h[i]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) z[4 * k + e] = d[e];
                        }
                        if (DROP) {
                            const uint32_t bits = keep[(16 * (i0 + i) + n16) * G + (at + V * g) / 8] >>
                                                  (V == 8 ? 0 : 2 * (g & 1));
#pragma unroll
                            for (int e = 0; e < V; ++e)
                                z[e] = p.factor * __uint_as_float(drop_word(__float_as_uint(z[e]), bits, drop_bit(e)));
                        }
                        if (p.base)
#pragma unroll
                            for (int e = 0; e < V; ++e) z[e] += lora_value<DT>(base[i][q + x], e);
                        out[i][x] = lora_round<DT>(z);
                    }
                }
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    S* to = d + (int64_t)16 * (i0 + i) * p.c + q * N::STEP;
                    const int left = m - 16 * (i0 + i);
                    if (!edge) {
                        lora_store_pair(to, p.c, out[i][0], out[i][1], left);
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int at = x * N::STEP + V * g;
                            if (n16 < left)
                                lora_store(to + n16 * (int64_t)p.c + at, out[i][x], p.c - col0 - (q0 + q) * N::STEP - at);
                        }
                    }
                }
            }
        }
        if (BUF == 1) lds_barrier();
    }
    if (WG > 1 && p.pd) lora_gather<WC * WR, WG>(acc, sums);
    if (p.pd && col0 < p.c && wg == 0) {
        float* slot = p.pd + slot_at * lora_slot(p.c, CW, RT);
        const float f = DROP ? p.factor : 1.0f;
        lora_flush<DT, RW>(acc, slot, col0 / CW, RT, RW * wr, f);
        lora_flush_plain<DT, RW>(acc, slot, col0 / CW, RT, RW * wr, f, r0, r1, p.c, p.r,
                                 [&](int64_t row, int col, int rank) {
                                     float u = 0.0f, x = lora_get<DT>(p.x, row * p.xs + col);
                                     for (int k = 0; k < p.u_parts; ++k) u += p.u[(k * it.n + row) * p.r + rank];
                                     if (DROP && !lora_keeps(lora_ones(key, p.drop, row, col, p.c), col)) x = 0.0f;
                                     return u * x;
                                 });
    }
}

template <int DT>
hipError_t lora_back_out(hipStream_t s, const LoraBackArgs& p, dim3 grid) {
    const int rt = lora_rank_tiles(p.r), wc = lora_col_waves(DT, p.r, p.o);
    if (rt == 1 && wc == 4) lora_back_out_kernel<DT, 1, 1, 4><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 1 && wc == 2) lora_back_out_kernel<DT, 1, 1, 2><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 1) lora_back_out_kernel<DT, 1, 1, 1><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 2 && wc == 2) lora_back_out_kernel<DT, 1, 2, 2><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 2) lora_back_out_kernel<DT, 1, 2, 1><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 4) lora_back_out_kernel<DT, 1, 4, 1><<<grid, kLoraThreads, 0, s>>>(p);
    else lora_back_out_kernel<DT, 2, 4, 1><<<grid, kLoraThreads, 0, s>>>(p);
    return hipGetLastError();
}

template <int DT, bool DROP>
void lora_back_in_rank(hipStream_t s, const LoraBackArgs& p, dim3 grid) {
    const int rt = lora_rank_tiles(p.r), wc = lora_col_waves(DT, p.r, p.c);
    if (rt == 1 && wc == 4) lora_back_in_kernel<DT, 1, 1, 4, DROP><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 1 && wc == 2) lora_back_in_kernel<DT, 1, 1, 2, DROP><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 1) lora_back_in_kernel<DT, 1, 1, 1, DROP><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 2 && wc == 2) lora_back_in_kernel<DT, 1, 2, 2, DROP><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 2) lora_back_in_kernel<DT, 1, 2, 1, DROP><<<grid, kLoraThreads, 0, s>>>(p);
    else if (rt == 4) lora_back_in_kernel<DT, 1, 4, 1, DROP><<<grid, kLoraThreads, 0, s>>>(p);
    else lora_back_in_kernel<DT, 2, 4, 1, DROP><<<grid, kLoraThreads, 0, s>>>(p);
}

template <int DT>
hipError_t lora_back_in(hipStream_t s, const LoraBackArgs& p, dim3 grid) {
    if (p.drop) lora_back_in_rank<DT, true>(s, p, grid);
    else lora_back_in_rank<DT, false>(s, p, grid);
    return hipGetLastError();
}

}  // namespace spc

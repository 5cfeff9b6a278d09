// linear_q4.hip -- products of a few rows with Q4_0 weights: y = x W^T + bias
// (spc_linear_q4_0) and the rows' gradient dx = dy W (spc_linear_q4_0_input_grad).
//
// A Q4_0 block is 32 weights along the input features: an f16 scale d and 32
// four-bit q, w = d (q - 8).  The weights' bytes bound both products, so they
// are read once, as they are, and expanded in registers for the matrix
// instructions, which take 16 rows at the price of one:
//
//   16 + q is the bf16 pattern 0x4180 | q << 3 (f16: 0x4c00 | q << 6), exactly,
//   so two weights cost one shift and one and-or;
//   sum x (q - 8) = sum x (16 + q) + sum x (-24), and the second sum is one
//   more matrix instruction on a constant, shared by all columns.
//
// Forward, one 16x16x32 product covers exactly one block of every column; its
// F32 result times d is added to the F32 accumulator, so no weight is ever
// rounded.  F32 rows run as three bf16 parts that add up to them exactly.
// For the gradient the scale varies along the summed index.  F32 rows are
// multiplied by it first (F32) and run as three bf16 parts; for 16-bit rows the
// weights are, as f16(d (q - 8)).
//
// The weights are laid out once (spc_linear_q4_0_pack) in the order the lanes
// want them: for 16 columns and 128 summed features a lane's 16 bytes are its
// eight weights of four instructions, so a wave's load is one 1 KB run.
#include <algorithm>

#include "common.h"

namespace spc {

namespace {

constexpr int kQ4Cols = 16;    // columns of a tile
constexpr int kQ4Group = 128;  // summed features of a tile
constexpr int kQ4TileBytes = kQ4Cols * kQ4Group / 2;

// Nibble of element e (0..7) in a packed word: pairs (2p, 2p + 1) 16 bits
// apart, so that one shift aligns both halves of operand register p.
__host__ __device__ inline int q4_shift(int e) { return 4 * (e / 2) + 16 * (e & 1); }

struct Q4Layout {
    int64_t cols, sum;          // columns of the product, summed features
    int64_t col_tiles, groups;  // in tiles of 16 and groups of 128
    int64_t quant_bytes, scale_bytes;
};

// Forward operand: columns are the output features, scales f16
// [tile][group][16][4].  Transposed (gradient): columns are the input features,
// scales f16 [input block][groups * 128] along the summed output features.
inline Q4Layout q4_layout(int64_t out, int64_t in, bool transpose) {
    Q4Layout l;
    l.cols = transpose ? in : out;
    l.sum = transpose ? out : in;
    l.col_tiles = ceil_div(l.cols, kQ4Cols);
    l.groups = ceil_div(l.sum, kQ4Group);
    l.quant_bytes = l.col_tiles * l.groups * kQ4TileBytes;
    l.scale_bytes = transpose ? in / 32 * l.groups * kQ4Group * 2
                              : l.col_tiles * l.groups * kQ4Cols * 4 * 2;
    return l;
}

__device__ __forceinline__ int q4_at(const uint8_t* blocks, int64_t in, int64_t o, int64_t k) {
    const uint8_t* b = blocks + (o * (in / 32) + k / 32) * 18 + 2;
    const int e = (int)(k % 32);
    return e < 16 ? b[e] & 15 : b[e - 16] >> 4;
}

__device__ __forceinline__ uint16_t q4_scale_bits(const uint8_t* blocks, int64_t in, int64_t o,
                                                  int64_t k) {
    const uint8_t* b = blocks + (o * (in / 32) + k / 32) * 18;
    return (uint16_t)(b[0] | (b[1] << 8));
}

// One thread a packed word, then one a scale.  Padding: q 8 and scale 0.
__global__ __launch_bounds__(256) void q4_pack_kernel(const uint8_t* __restrict__ blocks, int64_t out,
                                                      int64_t in, Q4Layout l, int transpose,
                                                      uint32_t* __restrict__ quants,
                                                      uint16_t* __restrict__ scales) {
    const int64_t words = l.quant_bytes / 4, total = words + l.scale_bytes / 2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        if (i < words) {
            const int j = (int)(i & 3), lane = (int)(i >> 2 & 63);
            const int64_t tile = i >> 8;
            const int64_t col = tile / l.groups * kQ4Cols + lane % 16;
            const int64_t s0 = tile % l.groups * kQ4Group + 32 * j + 8 * (lane / 16);
            uint32_t w = 0;
            for (int e = 0; e < 8; ++e) {
                int q = 8;
                if (col < l.cols && s0 + e < l.sum)
                    q = transpose ? q4_at(blocks, in, s0 + e, col) : q4_at(blocks, in, col, s0 + e);
                w |= (uint32_t)q << q4_shift(e);
            }
            quants[i] = w;
        } else {
            const int64_t t = i - words;
            uint16_t d = 0;
            if (transpose) {
                const int64_t o = t % (l.groups * kQ4Group), kb = t / (l.groups * kQ4Group);
                if (o < out) d = q4_scale_bits(blocks, in, o, 32 * kb);
            } else {
                const int64_t tile = t >> 6, o = tile / l.groups * kQ4Cols + (t >> 2 & 15);
                const int64_t k = tile % l.groups * kQ4Group + 32 * (t & 3);
                if (o < out && k < in) d = q4_scale_bits(blocks, in, o, k);
            }
            scales[t] = d;
        }
    }
}

// Q4_0 of F32 weights, one thread a block: d = (the value of largest
// magnitude, the first such) / -8 rounded to f16, q = floor(w / d + 8.5) in
// 0..15 with the rounded d.
__global__ __launch_bounds__(256) void q4_quantize_kernel(const float* __restrict__ w, int64_t nblocks,
                                                          uint8_t* __restrict__ blocks) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= nblocks) return;
    float v[32];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const floatx4 q = *reinterpret_cast<const floatx4*>(w + 32 * i + 4 * j);
        v[4 * j] = q.x; v[4 * j + 1] = q.y; v[4 * j + 2] = q.z; v[4 * j + 3] = q.w;
    }
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j)
        if (fabsf(v[j]) > fabsf(top)) top = v[j];
    const uint16_t d = f32_to_f16_bits(top * -0.125f);
    const float df = f16_bits_to_f32(d);
    const float inv = df != 0.0f ? 1.0f / df : 0.0f;
    uint8_t* b = blocks + 18 * i;
    b[0] = (uint8_t)d;
    b[1] = (uint8_t)(d >> 8);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int lo = (int)fminf(fmaxf(floorf(v[j] * inv + 8.5f), 0.0f), 15.0f);
        const int hi = (int)fminf(fmaxf(floorf(v[j + 16] * inv + 8.5f), 0.0f), 15.0f);
        b[2 + j] = (uint8_t)(lo | (hi << 4));
    }
}

// ---- operands -------------------------------------------------------------
// The patterns' fixed bits: one of the two in a vector register, since an
// instruction reads one scalar operand, and the and-or is one instruction then.
template <bool F16>
__device__ __forceinline__ uint32_t q4_one() {
    uint32_t v = F16 ? 0x4c004c00u : 0x41804180u;
    asm("" : "+v"(v));
    return v;
}
template <bool F16>
__device__ __forceinline__ u32x4 q4_expand(uint32_t w, uint32_t one) {
    if constexpr (F16) {
        constexpr uint32_t m = 0x03c003c0u;
        return u32x4{((w << 6) & m) | one, ((w << 2) & m) | one, ((w >> 2) & m) | one,
                     ((w >> 6) & m) | one};
    } else {
        constexpr uint32_t m = 0x00780078u;
        return u32x4{((w << 3) & m) | one, ((w >> 1) & m) | one, ((w >> 5) & m) | one,
                     ((w >> 9) & m) | one};
    }
}

template <bool F16>
__device__ __forceinline__ floatx4 q4_mfma(u32x4 a, u32x4 b, floatx4 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool F16>
__device__ __forceinline__ u32x4 q4_minus_24() {
    constexpr uint32_t v = F16 ? 0xce00ce00u : 0xc1c0c1c0u;
    return u32x4{v, v, v, v};
}

// The high halves of two F32 words as a bf16 pair (a cut, not a rounding).
__device__ __forceinline__ uint32_t q4_high_pair(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float q4_rest(float v) {
    return v - __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}

// Eight F32 values as three bf16 operands that add up to them: cuts of eight
// bits each, and the last one's rest is nothing.
__device__ __forceinline__ void q4_split(const float (&v)[8], u32x4 (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            p[s][i] = q4_high_pair(a, b);
            a = q4_rest(a);
            b = q4_rest(b);
        }
    }
}

// Eight consecutive elements of a row as loaded.
template <int DT>
struct Q4Row {
    u32x4 w[DT == SPC_F32 ? 2 : 1];
};
// The lane's elements of one group: for each of its four instructions j eight,
// from 128 g + 32 j + 8 (lane / 16) on, of a row of `sum` elements at `row`.
// WIDE: 16-byte loads without a branch; in a last, partial group those past the
// end become the row's last eight, which meet weights of scale 0.
template <int DT, bool WIDE>
__device__ __forceinline__ void q4_load_rows(Q4Row<DT> (&r)[4], const char* row, int g, int sum) {
    constexpr int NW = DT == SPC_F32 ? 2 : 1, ES = DT == SPC_F32 ? 4 : 2;
    const int k0 = 8 * ((threadIdx.x & 63) / 16);
    if constexpr (WIDE) {
        const char* p = row + (int64_t)g * kQ4Group * ES;
        if ((g + 1) * kQ4Group <= sum) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < NW; ++i)
                    r[j].w[i] = *reinterpret_cast<const u32x4*>(p + (k0 + 32 * j) * ES + 16 * i);
        } else {
            const int last = sum - 8 - g * kQ4Group;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < NW; ++i)
                    r[j].w[i] = *reinterpret_cast<const u32x4*>(p + min(k0 + 32 * j, last) * ES + 16 * i);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int i = 0; i < NW; ++i) r[j].w[i] = u32x4{0, 0, 0, 0};
            const int64_t k = (int64_t)g * kQ4Group + 32 * j + k0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (k + e >= sum) break;
                if constexpr (DT == SPC_F32)
                    r[j].w[e / 4][e % 4] = reinterpret_cast<const uint32_t*>(row)[k + e];
                else
                    r[j].w[0][e / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(row)[k + e]
                                        << (16 * (e & 1));
            }
        }
    }
}
__device__ __forceinline__ void q4_row_floats(const Q4Row<SPC_F32>& r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r.w[e / 4][e % 4]);
}

struct Q4Args {
    const void* x;       // rows [m, sum], x_stride elements apart
    int64_t x_stride;
    int64_t m, cols, col_tiles;
    int sum, groups;     // summed features, in groups of 128
    const uint32_t* quants;
    const uint16_t* scales;
    const void* bias;    // [cols] or null
    int bias_dtype;
    const float* factor; // [m]: x is f16 rows times these
    bool wide;           // rows take 16-byte loads
    void* y;             // [m, cols]
};

template <int DT>
__device__ __forceinline__ void q4_store(void* y, int64_t at, float v) {
    if constexpr (DT == SPC_F32) static_cast<float*>(y)[at] = v;
    else if constexpr (DT == SPC_BF16) static_cast<uint16_t*>(y)[at] = f32_to_bf16_bits(v);
    else static_cast<uint16_t*>(y)[at] = f32_to_f16_bits(v);
}

// Adds the W waves' accumulators and stores: tiles [MT][NT] of 16 rows x 16
// columns; lane l of a tile holds column l % 16, rows 4 (l / 16) + i.
template <int DT, int MT, int NT, int W>
__device__ __forceinline__ void q4_finish(const Q4Args& p, floatx4 (&acc)[MT][NT], int64_t row0,
                                          int64_t col0, floatx4* lds) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    constexpr int TILES = MT * NT;
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) lds[(wave * TILES + a * NT + b) * 64 + lane] = acc[a][b];
    __syncthreads();
    for (int t = wave; t < TILES; t += W) {
        const int a = t / NT, b = t % NT;
        floatx4 v = lds[t * 64 + lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v += lds[(w * TILES + t) * 64 + lane];
        const int64_t col = col0 + 16 * b + lane % 16;
        if (col >= p.cols) continue;
        float bias = 0.0f;
        if (p.bias)
            bias = p.bias_dtype == SPC_F32 ? static_cast<const float*>(p.bias)[col]
                   : p.bias_dtype == SPC_BF16
                       ? bf16_bits_to_f32(static_cast<const uint16_t*>(p.bias)[col])
                       : f16_bits_to_f32(static_cast<const uint16_t*>(p.bias)[col]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = row0 + 16 * a + 4 * (lane / 16) + i;
            if (row < p.m) q4_store<DT>(p.y, row * p.cols + col, v[i] + bias);
        }
    }
}

// A block's W waves take the groups of 128 summed features in turn, each with
// its next step of weights and rows under way: f(step) for every step of this
// wave.  (Two or three steps under way measured slower: 8192 -> 16,384, one
// bf16 row, 16.2 / 17.3 us with one / two; the waves hide each other's loads.)
template <int W, typename Step, typename Load, typename F>
__device__ __forceinline__ void q4_pipeline(int groups, Load&& load, F&& f) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Step next;
    if (wave < groups) load(next, wave);
    for (int g = wave; g < groups; g += W) {
        const Step now = next;
        if (g + W < groups) load(next, g + W);
        f(now);
    }
}

// The lane's rows: row0 + 16 a + lane % 16, those past the last repeat it
// (their results are not stored).
template <int DT, int MT>
__device__ __forceinline__ void q4_rows(const Q4Args& p, int64_t row0, const char* (&row)[MT]) {
#pragma unroll
    for (int a = 0; a < MT; ++a)
        row[a] = static_cast<const char*>(p.x) +
                 min(row0 + 16 * a + (threadIdx.x & 15), p.m - 1) * p.x_stride * (DT == SPC_F32 ? 4 : 2);
}

// y = x W^T: a block's W waves share 16 NT columns and 16 MT rows.
template <int DT, int MT, int NT, int W, bool WIDE>
__global__ __launch_bounds__(64 * W) void q4_forward_kernel(Q4Args p) {
    constexpr bool F16 = DT == SPC_F16;
    constexpr int PARTS = DT == SPC_F32 ? 3 : 1;
    __shared__ floatx4 lds[W * MT * NT * 64];
    const uint32_t lane = threadIdx.x & 63;
    const int64_t tile0 = (int64_t)blockIdx.x * NT, row0 = (int64_t)blockIdx.y * 16 * MT;
    struct Step {
        u32x4 q[NT];
        u32x2 d[NT];
        Q4Row<DT> x[MT][4];
    };
    const char* row[MT];
    q4_rows<DT, MT>(p, row0, row);
    auto load = [&](Step& s, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const int64_t t = min(tile0 + b, p.col_tiles - 1) * p.groups + g;
            s.q[b] = (reinterpret_cast<const u32x4*>(p.quants) + t * 64)[lane];
            s.d[b] = (reinterpret_cast<const u32x2*>(p.scales) + t * 16)[lane % 16];
        }
#pragma unroll
        for (int a = 0; a < MT; ++a) q4_load_rows<DT, WIDE>(s.x[a], row[a], g, p.sum);
    };
    floatx4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0, 0, 0, 0};
    const uint32_t one = q4_one<F16>();
    q4_pipeline<W, Step>(p.groups, load, [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 xp[MT][PARTS];
            floatx4 off[MT];
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                if constexpr (PARTS == 1) {
                    xp[a][0] = s.x[a][j].w[0];
                } else {
                    float v[8];
                    q4_row_floats(s.x[a][j], v);
                    q4_split(v, xp[a]);
                }
                off[a] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int q = 0; q < PARTS; ++q) off[a] = q4_mfma<F16>(xp[a][q], q4_minus_24<F16>(), off[a]);
            }
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const u32x4 w = q4_expand<F16>(s.q[b][j], one);
                const float d = f16_bits_to_f32((uint16_t)(s.d[b][j / 2] >> (16 * (j & 1))));
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    floatx4 t = off[a];
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) t = q4_mfma<F16>(xp[a][q], w, t);
                    acc[a][b] += t * d;
                }
            }
        }
    });
    q4_finish<DT, MT, NT, W>(p, acc, row0, tile0 * 16, lds);
}

// Eight scales for each of a group's four instructions, from 128 in one load:
// lane i of the wave's 16-lane row r holds scales 8 (i + r) .. + 7, so what the
// row needs for instruction j (from 32 j + 8 r on) is in its lane 4 j.  Four
// loads instead, 16 lanes to an address, cost the vector memory path as much as
// 4 KB (64 cycles a step; it bound one row: 4096 -> 16,384 16.6 us, XX).
__device__ __forceinline__ u32x4 q4_load_scales(const uint16_t* d) {
    const uint32_t lane = threadIdx.x & 63;
    return reinterpret_cast<const u32x4*>(d)[(lane + lane / 16) & 15];
}
template <int J>
__device__ __forceinline__ u32x4 q4_scales(u32x4 d) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int v = (int)d[i];
        r[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, v, 0x150 + 4 * J, 0xf, 0xf, true);
    }
    return r;
}
__device__ __forceinline__ u32x4 q4_scales(u32x4 d, int j) {  // j unrolled
    return j == 0 ? q4_scales<0>(d) : j == 1 ? q4_scales<1>(d) : j == 2 ? q4_scales<2>(d) : q4_scales<3>(d);
}

// dx = dy W of F32 rows: 16 NT input features (NT 1 or 2: within one block of
// scales) and 16 MT rows a block.
template <int MT, int NT, int W, bool WIDE>
__global__ __launch_bounds__(64 * W) void q4_grad_kernel(Q4Args p) {
    constexpr int DT = SPC_F32;
    __shared__ floatx4 lds[W * MT * NT * 64];
    const uint32_t lane = threadIdx.x & 63;
    const int64_t tile0 = (int64_t)blockIdx.x * NT, row0 = (int64_t)blockIdx.y * 16 * MT;
    struct Step {
        u32x4 q[NT];
        u32x4 d;     // scales along the summed features
        Q4Row<DT> x[MT][4];
    };
    const char* row[MT];
    q4_rows<DT, MT>(p, row0, row);
    const uint16_t* scales = p.scales + tile0 / 2 * p.groups * kQ4Group;
    auto load = [&](Step& s, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < NT; ++b)
            s.q[b] = (reinterpret_cast<const u32x4*>(p.quants) + ((tile0 + b) * p.groups + g) * 64)[lane];
        s.d = q4_load_scales(scales + (int64_t)g * kQ4Group);
#pragma unroll
        for (int a = 0; a < MT; ++a) q4_load_rows<DT, WIDE>(s.x[a], row[a], g, p.sum);
    };
    floatx4 acc[MT][NT], off[MT];
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        off[a] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0, 0, 0, 0};
    }
    const uint32_t one = q4_one<false>();
    q4_pipeline<W, Step>(p.groups, load, [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 w[NT];
#pragma unroll
            for (int b = 0; b < NT; ++b) w[b] = q4_expand<false>(s.q[b][j], one);
            const u32x4 d = q4_scales(s.d, j);
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                float v[8];
                q4_row_floats(s.x[a][j], v);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] *= f16_bits_to_f32((uint16_t)(d[e / 2] >> (16 * (e & 1))));
                u32x4 xp[3];
                q4_split(v, xp);
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    off[a] = q4_mfma<false>(xp[q], q4_minus_24<false>(), off[a]);
#pragma unroll
                    for (int b = 0; b < NT; ++b) acc[a][b] = q4_mfma<false>(xp[q], w[b], acc[a][b]);
                }
            }
        }
    });
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] += off[a];
    q4_finish<DT, MT, NT, W>(p, acc, row0, tile0 * 16, lds);
}

// ---- the gradient of 16-bit rows -------------------------------------------
// Multiplying the rows by a scale that differs for every 32 columns costs six
// instructions an element and block of columns, and their split into two parts
// three matrix instructions a tile, which bound 16-bit rows
// (16 rows, 4096 -> 16,384: 23 us of a floor of 8).  Here the weights take the
// scale, f16(d (q - 8)), rounded to 11 bits -- at most 2^-11 of a weight, an
// eighth of a bf16 output's own rounding and as much as an f16 output's -- and
// the rows enter as f16 whatever their columns: f16 rows as they are, bf16 rows
// with their exponents moved into f16's range by a power of two that each wave
// chooses for each row from what it has seen of it (exact for values down to
// 2^-27 of the row's largest; of smaller ones less than 2^-28 of it is lost).

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The eight weights of a word times their eight scales.
__device__ __forceinline__ u32x4 q4_expand_scaled(uint32_t w, u32x4 d, uint32_t one) {
    const u32x4 q = q4_expand<true>(w, one);  // 16 + q
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // (copies: a bit cast of a vector's element takes the vector's first)
        const uint32_t qi = q[i], di = d[i];
        const f16x2 t = (__builtin_bit_cast(f16x2, qi) - (f16x2)(_Float16)24.0f) *
                        __builtin_bit_cast(f16x2, di);
        r[i] = __builtin_bit_cast(uint32_t, t);
    }
    return r;
}

// A row's exponent bias: what is taken off its bf16 exponents to make f16's.
// The row's largest value seen so far has f16 exponent 28 when the bias is
// set, so it may grow by 2^2 before the bias has to move.
struct Q4Bias {
    uint32_t top = 0;  // largest magnitude seen, bf16 bits
    int bias = 0;

    // Takes a group's elements in (all lanes of a row agree); true if the bias
    // moves, by `*by`.
    __device__ __forceinline__ bool see(const Q4Row<SPC_BF16> (&r)[4], int* by) {
        u16x2 m = {0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, r[j].w[0][i] & 0x7fff7fffu));
        uint32_t t = max((uint32_t)m.x, (uint32_t)m.y);
        // over the four lanes of a row
        const auto s = __builtin_amdgcn_permlane16_swap(t, t, false, false);
        t = max(s[0], s[1]);
        const auto u = __builtin_amdgcn_permlane32_swap(t, t, false, false);
        t = max(u[0], u[1]);
        const uint32_t had = top;
        top = max(top, t);
        const int e = (int)(top >> 7);
        const bool move = e - bias > 30 || (had == 0 && top != 0);
        const int to = move ? max(e - 28, 0) : bias;
        *by = to - bias;
        bias = to;
        return move;
    }
    // bf16 -> f16 with the bias taken off; what falls below f16's range is 0
    // (or, in the last binade, loses its leading bit).
    __device__ __forceinline__ u32x4 f16(u32x4 v) const {
        const u16x2 off = (u16x2)(uint16_t)(bias << 7);
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u16x2 mag = __builtin_elementwise_sub_sat(
                __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu), off);
            r[i] = __builtin_bit_cast(uint32_t, mag << 3) | (v[i] & 0x80008000u);
        }
        return r;
    }
    // What a sum of the moved values is to be multiplied by; NaN for a row
    // with an infinity or NaN.
    __device__ __forceinline__ float factor() const {
        return top >= 0x7f80u ? __builtin_nanf("") : ldexpf(1.0f, bias - 112);
    }
};

// bf16 rows to f16 rows ahead of the product, for products so large that
// moving the exponents in every column's wave costs more than a kernel: a
// block a row, the bias from the whole row (largest value to f16 exponent 28),
// its factor beside it.  Rows of `ld` elements, those past n zero.
constexpr int kQ4RowThreads = 1024;
__global__ __launch_bounds__(kQ4RowThreads) void q4_rows_kernel(const uint16_t* __restrict__ x,
                                                                int64_t x_stride, int n, int ld,
                                                                uint16_t* __restrict__ y,
                                                                float* __restrict__ factor) {
    __shared__ uint32_t ws[kQ4RowThreads / 64];
    const uint16_t* row = x + (int64_t)blockIdx.x * x_stride;
    uint32_t top = 0;
    for (int i = threadIdx.x; i < n; i += kQ4RowThreads) top = max(top, (uint32_t)row[i] & 0x7fffu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQ4RowThreads / 64; ++w) top = max(top, ws[w]);
    Q4Bias b;
    b.top = top;
    b.bias = max((int)(top >> 7) - 28, 0);
    if (threadIdx.x == 0) factor[blockIdx.x] = b.factor();
    for (int i = 8 * threadIdx.x; i < ld; i += 8 * kQ4RowThreads) {
        u32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i + e < n) v[e / 2] |= (uint32_t)row[i + e] << (16 * (e & 1));
        *reinterpret_cast<u32x4*>(y + (int64_t)blockIdx.x * ld + i) = b.f16(v);
    }
}

// dx = dy W of 16-bit rows: 16 NT input features and 16 MT rows a block.  MOVED:
// rows of q4_rows_kernel (OT the output's type).
template <int OT, bool MOVED, int MT, int NT, int W, bool WIDE>
__global__ __launch_bounds__(64 * W) void q4_grad16_kernel(Q4Args p) {
    constexpr int DT = MOVED ? SPC_F16 : OT;
    constexpr int KB = (NT + 1) / 2;  // blocks of scales
    __shared__ floatx4 lds[W * MT * NT * 64];
    const uint32_t lane = threadIdx.x & 63;
    const int64_t tile0 = (int64_t)blockIdx.x * NT, row0 = (int64_t)blockIdx.y * 16 * MT;
    struct Step {
        u32x4 q[NT];
        u32x4 d[KB];  // scales along the summed features
        Q4Row<DT> x[MT][4];
    };
    const char* row[MT];
    q4_rows<DT, MT>(p, row0, row);
    const int64_t last = p.col_tiles - 1;
    auto load = [&](Step& s, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < NT; ++b)
            s.q[b] = (reinterpret_cast<const u32x4*>(p.quants) +
                      (min(tile0 + b, last) * p.groups + g) * 64)[lane];
#pragma unroll
        for (int k = 0; k < KB; ++k)
            s.d[k] = q4_load_scales(p.scales + (min(tile0 + 2 * k, last) / 2 * p.groups + g) * kQ4Group);
#pragma unroll
        for (int a = 0; a < MT; ++a) q4_load_rows<DT, WIDE>(s.x[a], row[a], g, p.sum);
    };
    floatx4 acc[MT][NT];
    Q4Bias bias[MT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0, 0, 0, 0};
    // the accumulator rows' factors: row 4 (lane / 16) + i is lane row's % 16
    auto scale_rows = [&](int a, float f) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float fi = __shfl(f, 4 * (lane / 16) + i);
#pragma unroll
            for (int b = 0; b < NT; ++b) acc[a][b][i] *= fi;
        }
    };
    const uint32_t one = q4_one<true>();
    q4_pipeline<W, Step>(p.groups, load, [&](const Step& s) __attribute__((always_inline)) {
        if constexpr (DT == SPC_BF16) {
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                int by;
                const bool move = bias[a].see(s.x[a], &by);
                if (__any(move)) scale_rows(a, ldexpf(1.0f, -by));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 x[MT];
#pragma unroll
            for (int a = 0; a < MT; ++a)
                x[a] = DT == SPC_BF16 ? bias[a].f16(s.x[a][j].w[0]) : s.x[a][j].w[0];
            u32x4 d[KB];
#pragma unroll
            for (int k = 0; k < KB; ++k) d[k] = q4_scales(s.d[k], j);
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const u32x4 w = q4_expand_scaled(s.q[b][j], d[b / 2], one);
#pragma unroll
                for (int a = 0; a < MT; ++a) acc[a][b] = q4_mfma<true>(x[a], w, acc[a][b]);
            }
        }
    });
    if constexpr (MOVED || DT == SPC_BF16) {
#pragma unroll
        for (int a = 0; a < MT; ++a) {
            float f;
            if constexpr (MOVED) f = p.factor[min(row0 + 16 * a + lane % 16, p.m - 1)];
            else f = bias[a].factor();
            scale_rows(a, f);
        }
    }
    q4_finish<OT, MT, NT, W>(p, acc, row0, tile0 * 16, lds);
}

template <int DT, int MT, int NT, int W>
void q4_forward_launch(hipStream_t s, const Q4Args& p) {
    const dim3 grid((unsigned)ceil_div(p.col_tiles, NT), (unsigned)ceil_div(p.m, 16 * MT));
    if (p.wide) q4_forward_kernel<DT, MT, NT, W, true><<<grid, 64 * W, 0, s>>>(p);
    else q4_forward_kernel<DT, MT, NT, W, false><<<grid, 64 * W, 0, s>>>(p);
}

template <int DT, int MT, int NT, int W>
void q4_grad_launch(hipStream_t s, const Q4Args& p) {
    const dim3 grid((unsigned)ceil_div(p.col_tiles, NT), (unsigned)ceil_div(p.m, 16 * MT));
    if constexpr (DT == SPC_F32) {
        if (p.wide) q4_grad_kernel<MT, NT, W, true><<<grid, 64 * W, 0, s>>>(p);
        else q4_grad_kernel<MT, NT, W, false><<<grid, 64 * W, 0, s>>>(p);
    } else {
        if (DT == SPC_BF16 && p.factor)
            q4_grad16_kernel<DT, DT == SPC_BF16, MT, NT, W, true><<<grid, 64 * W, 0, s>>>(p);
        else if (p.wide) q4_grad16_kernel<DT, false, MT, NT, W, true><<<grid, 64 * W, 0, s>>>(p);
        else q4_grad16_kernel<DT, false, MT, NT, W, false><<<grid, 64 * W, 0, s>>>(p);
    }
}

template <int DT>
hipError_t q4_forward(hipStream_t s, const Q4Args& p) {
    // F32 rows hold three operands each: two row tiles at most
    // More column tiles a wave read the rows (and split F32 ones) less often, as
    // long as 256 blocks are left for the CUs.  us with 1 / 2 / 4 tiles: 8192 ->
    // 16,384, one bf16 row 16.2 / 15.0 / 15.7, eight 25.6 / 18.0 / 16.3, sixteen
    // 36.0 / 22.3 / 17.5, two F32 rows 36.7 / 28.3 / 22.6; 4096 -> 8192, one
    // 6.8 / 6.4 / 8.7, sixteen 11.8 / 8.5 / 9.9; 4096 -> 4096, one 4.6 / 5.4 / 7.8.
    if (p.m <= 16) {
        if (p.col_tiles >= 1024 && (p.m > 4 || DT == SPC_F32)) q4_forward_launch<DT, 1, 4, 8>(s, p);
        else if (p.col_tiles >= 512) q4_forward_launch<DT, 1, 2, 8>(s, p);
        else q4_forward_launch<DT, 1, 1, 8>(s, p);
    } else if (p.m <= 32 || DT == SPC_F32) {
        q4_forward_launch<DT, 2, 1, 8>(s, p);
    } else if constexpr (DT != SPC_F32) {
        q4_forward_launch<DT, 4, 1, 8>(s, p);
    }
    return hipGetLastError();
}

// bf16 rows moved to f16 ahead of the product (q4_rows_kernel): from XX column
// tiles times groups on.
inline bool q4_moves_rows(int dtype, const Q4Layout& l) {
    return dtype == SPC_BF16 && l.col_tiles * l.groups >= 16384;
}

template <int DT>
hipError_t q4_grad(hipStream_t s, Q4Args p, void* workspace) {
    if (workspace) {
        const int ld = (p.sum + 7) / 8 * 8;
        float* factor = static_cast<float*>(workspace);
        uint16_t* rows = reinterpret_cast<uint16_t*>(factor + (p.m + 3) / 4 * 4);
        q4_rows_kernel<<<(unsigned)p.m, kQ4RowThreads, 0, s>>>(static_cast<const uint16_t*>(p.x),
                                                               p.x_stride, p.sum, ld, rows, factor);
        p.x = rows;
        p.x_stride = p.sum = ld;
        p.factor = factor;
    }
    if (p.m <= 16) {
        if (p.col_tiles >= 512) q4_grad_launch<DT, 1, 2, 8>(s, p);
        else q4_grad_launch<DT, 1, 1, 8>(s, p);
    } else {
        q4_grad_launch<DT, 2, 2, 8>(s, p);
    }
    return hipGetLastError();
}

int q4_shape(const char* fn, int64_t out, int64_t in) {
    if (out < 1 || in < 32 || in % 32 || out > INT32_MAX - 127 || in > INT32_MAX - 127) {
        set_last_error("%s: unsupported shape out_features=%lld in_features=%lld (a multiple of 32)",
                       fn, (long long)out, (long long)in);
        return SPC_BAD_SHAPE;
    }
    return SPC_OK;
}

// Checks a product's arguments and fills the kernel's.
int q4_args(const char* fn, int dtype, const void* x, int64_t x_stride, int64_t m, const void* packed,
            int64_t out, int64_t in, bool transpose, void* y, Q4Args* p) {
    const int st = q4_shape(fn, out, in);
    if (st != SPC_OK) return st;
    if (m < 0 || m > (int64_t)65535 * 16 || x_stride < 0) {
        set_last_error("%s: unsupported rows m=%lld (0 to %d)", fn, (long long)m, 65535 * 16);
        return SPC_BAD_SHAPE;
    }
    if (dtype != SPC_F32 && dtype != SPC_F16 && dtype != SPC_BF16) {
        set_last_error("%s: unknown dtype %d", fn, dtype);
        return SPC_BAD_ARG;
    }
    const int64_t e = dtype == SPC_F32 ? 4 : 2;
    if (m > 0 && (!x || !y || !packed || (uintptr_t)x % e || (uintptr_t)y % e || (uintptr_t)packed % 16)) {
        set_last_error("%s: null or misaligned pointer (packed weights 16-byte aligned)", fn);
        return SPC_BAD_ARG;
    }
    const Q4Layout l = q4_layout(out, in, transpose);
    *p = Q4Args{};
    p->x = x;
    p->x_stride = x_stride;
    p->m = m;
    p->sum = (int)l.sum;
    p->cols = l.cols;
    p->groups = (int)l.groups;
    p->col_tiles = l.col_tiles;
    p->quants = static_cast<const uint32_t*>(packed);
    p->scales = reinterpret_cast<const uint16_t*>(static_cast<const char*>(packed) + l.quant_bytes);
    p->wide = (uintptr_t)x % 16 == 0 && x_stride * e % 16 == 0 && l.sum % 8 == 0;
    p->y = y;
    return SPC_OK;
}

}  // namespace

}  // namespace spc

using namespace spc;

extern "C" {

int spc_q4_0_quantize(spc_stream_t stream, const float* w, int64_t n, uint8_t* blocks) {
    if (n < 0 || n % 32 || (n > 0 && (!w || !blocks || (uintptr_t)w % 16))) {
        set_last_error("spc_q4_0_quantize: n must be a multiple of 32, w 16-byte aligned");
        return SPC_BAD_ARG;
    }
    if (n == 0) return SPC_OK;
    q4_quantize_kernel<<<(unsigned)ceil_div(n / 32, 256), 256, 0, static_cast<hipStream_t>(stream)>>>(
        w, n / 32, blocks);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPC_OK : hip_status(e, "spc_q4_0_quantize launch");
}

size_t spc_linear_q4_0_packed_bytes(int64_t out_features, int64_t in_features, int transpose) {
    if (out_features < 1 || in_features < 32 || in_features % 32 || out_features > INT32_MAX - 127 ||
        in_features > INT32_MAX - 127)
        return 0;
    const Q4Layout l = q4_layout(out_features, in_features, transpose != 0);
    return (size_t)(l.quant_bytes + l.scale_bytes);
}

int spc_linear_q4_0_pack(spc_stream_t stream, const uint8_t* blocks, int64_t out_features,
                         int64_t in_features, int transpose, void* packed) {
    const int st = q4_shape("spc_linear_q4_0_pack", out_features, in_features);
    if (st != SPC_OK) return st;
    if (!blocks || !packed || (uintptr_t)packed % 16) {
        set_last_error("spc_linear_q4_0_pack: null pointer, or packed not 16-byte aligned");
        return SPC_BAD_ARG;
    }
    const Q4Layout l = q4_layout(out_features, in_features, transpose != 0);
    const int64_t items = l.quant_bytes / 4 + l.scale_bytes / 2;
    q4_pack_kernel<<<(unsigned)std::min<int64_t>(ceil_div(items, 256), 1 << 16), 256, 0,
                     static_cast<hipStream_t>(stream)>>>(
        blocks, out_features, in_features, l, transpose != 0, static_cast<uint32_t*>(packed),
        reinterpret_cast<uint16_t*>(static_cast<char*>(packed) + l.quant_bytes));
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPC_OK : hip_status(e, "spc_linear_q4_0_pack launch");
}

int spc_linear_q4_0(spc_stream_t stream, int dtype, const void* x, int64_t x_stride, int64_t m,
                    const void* packed, int64_t out_features, int64_t in_features, const void* bias,
                    int bias_dtype, void* y) {
    const char* fn = "spc_linear_q4_0";
    Q4Args p;
    const int st = q4_args(fn, dtype, x, x_stride, m, packed, out_features, in_features, false, y, &p);
    if (st != SPC_OK) return st;
    if (bias && ((bias_dtype != SPC_F32 && bias_dtype != SPC_F16 && bias_dtype != SPC_BF16) ||
                 (uintptr_t)bias % (bias_dtype == SPC_F32 ? 4 : 2))) {
        set_last_error("%s: unknown bias dtype or misaligned bias", fn);
        return SPC_BAD_ARG;
    }
    if (m == 0) return SPC_OK;
    p.bias = bias;
    p.bias_dtype = bias_dtype;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = dtype == SPC_BF16  ? q4_forward<SPC_BF16>(s, p)
                         : dtype == SPC_F16 ? q4_forward<SPC_F16>(s, p)
                                            : q4_forward<SPC_F32>(s, p);
    return e == hipSuccess ? SPC_OK : hip_status(e, "spc_linear_q4_0 launch");
}

size_t spc_linear_q4_0_input_grad_workspace_bytes(int dtype, int64_t m, int64_t out_features,
                                                  int64_t in_features) {
    if (m < 1 || m > (int64_t)65535 * 16 ||
        spc_linear_q4_0_packed_bytes(out_features, in_features, 1) == 0)
        return 0;
    if (!q4_moves_rows(dtype, q4_layout(out_features, in_features, true))) return 0;
    return (size_t)((m + 3) / 4 * 16 + m * ((out_features + 7) / 8 * 16));
}

int spc_linear_q4_0_input_grad(spc_stream_t stream, int dtype, const void* dy, int64_t dy_stride,
                               int64_t m, const void* packed, int64_t out_features,
                               int64_t in_features, void* dx, void* workspace,
                               size_t workspace_bytes) {
    const char* fn = "spc_linear_q4_0_input_grad";
    Q4Args p;
    const int st = q4_args(fn, dtype, dy, dy_stride, m, packed, out_features, in_features, true, dx, &p);
    if (st != SPC_OK) return st;
    if (m == 0) return SPC_OK;
    const size_t need =
        spc_linear_q4_0_input_grad_workspace_bytes(dtype, m, out_features, in_features);
    if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)) {
        set_last_error("%s: workspace missing, misaligned (16 bytes) or too small", fn);
        return SPC_BAD_ARG;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    void* ws = need ? workspace : nullptr;
    const hipError_t e = dtype == SPC_BF16  ? q4_grad<SPC_BF16>(s, p, ws)
                         : dtype == SPC_F16 ? q4_grad<SPC_F16>(s, p, ws)
                                            : q4_grad<SPC_F32>(s, p, ws);
    return e == hipSuccess ? SPC_OK : hip_status(e, "spc_linear_q4_0_input_grad launch");
}

}  // extern "C"

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
// For the gradient the scale varies along the summed index: the rows are
// multiplied by it first (F32) and run as two bf16 parts (16 bits; a relative
// error of at most 2^-15), three for F32 rows.
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
template <bool F16>
__device__ __forceinline__ u32x4 q4_expand(uint32_t w) {
    if constexpr (F16) {
        constexpr uint32_t m = 0x03c003c0u, b = 0x4c004c00u;
        return u32x4{((w << 6) & m) | b, ((w << 2) & m) | b, ((w >> 2) & m) | b, ((w >> 6) & m) | b};
    } else {
        constexpr uint32_t m = 0x00780078u, b = 0x41804180u;
        return u32x4{((w << 3) & m) | b, ((w >> 1) & m) | b, ((w >> 5) & m) | b, ((w >> 9) & m) | b};
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

// Eight F32 values as PARTS bf16 operands that add up to them: the cut to
// bf16, the cut rest, and the rest's rest (3 parts: exact; 2: the rest
// rounded, at most 2^-15 relative).
template <int PARTS>
__device__ __forceinline__ void q4_split(float (&v)[8], u32x4 (&p)[PARTS]) {
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (PARTS == 2 && s == 1)
                p[s][i] = (uint32_t)f32_to_bf16_bits(v[2 * i]) |
                          ((uint32_t)f32_to_bf16_bits(v[2 * i + 1]) << 16);
            else
                p[s][i] = q4_high_pair(v[2 * i], v[2 * i + 1]);
            if (s + 1 < PARTS) {
                v[2 * i] = q4_rest(v[2 * i]);
                v[2 * i + 1] = q4_rest(v[2 * i + 1]);
            }
        }
    }
}

// Eight consecutive elements of a row as loaded.
template <int DT>
struct Q4Row {
    u32x4 w[DT == SPC_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Q4Row<DT> q4_load_row(const void* base, int64_t at, int64_t left, bool wide) {
    Q4Row<DT> r;
    constexpr int NW = DT == SPC_F32 ? 2 : 1, PER = DT == SPC_F32 ? 4 : 8;
#pragma unroll
    for (int i = 0; i < NW; ++i) r.w[i] = u32x4{0, 0, 0, 0};
    if (left <= 0) return r;
    if (wide && left >= 8) {
#pragma unroll
        for (int i = 0; i < NW; ++i)
            r.w[i] = *reinterpret_cast<const u32x4*>(static_cast<const char*>(base) +
                                                     (at + PER * i) * (16 / PER));
        return r;
    }
    // rows that are not 16-byte aligned, or the last elements of one
    if constexpr (DT == SPC_F32) {
        const uint32_t* p = static_cast<const uint32_t*>(base) + at;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) r.w[e / 4][e % 4] = p[e];
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(base) + at;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) r.w[0][e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void q4_row_floats(const Q4Row<DT>& r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (DT == SPC_F32) {
            v[e] = __uint_as_float(r.w[e / 4][e % 4]);
        } else {
            const uint32_t w = r.w[0][e / 2];
            if constexpr (DT == SPC_BF16) v[e] = __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
            else v[e] = f16_bits_to_f32((uint16_t)(e & 1 ? w >> 16 : w));
        }
    }
}

struct Q4Args {
    const void* x;       // rows [m, sum], x_stride elements apart
    int64_t x_stride;
    int64_t m, sum, cols;
    int64_t groups, col_tiles;
    const uint32_t* quants;
    const uint16_t* scales;
    const void* bias;    // [cols] or null
    int bias_dtype;
    int wide;            // 16-byte loads of the rows
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

// y = x W^T: a block's W waves share 16 NT columns and 16 MT rows and take the
// groups of 128 input features in turn.
template <int DT, int MT, int NT, int W>
__global__ __launch_bounds__(64 * W) void q4_forward_kernel(Q4Args p) {
    constexpr bool F16 = DT == SPC_F16;
    constexpr int PARTS = DT == SPC_F32 ? 3 : 1;
    __shared__ floatx4 lds[W * MT * NT * 64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t tile0 = (int64_t)blockIdx.x * NT, row0 = (int64_t)blockIdx.y * 16 * MT;
    struct Step {
        u32x4 q[NT];
        u32x2 d[NT];
        Q4Row<DT> x[MT][4];
    };
    auto load = [&](int64_t g) __attribute__((always_inline)) {
        Step s;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            s.q[b] = u32x4{0, 0, 0, 0};
            s.d[b] = u32x2{0, 0};
            if (g < p.groups && tile0 + b < p.col_tiles) {
                const int64_t t = (tile0 + b) * p.groups + g;
                s.q[b] = reinterpret_cast<const u32x4*>(p.quants)[t * 64 + lane];
                s.d[b] = reinterpret_cast<const u32x2*>(p.scales)[t * 16 + lane % 16];
            }
        }
#pragma unroll
        for (int a = 0; a < MT; ++a) {
            const int64_t row = row0 + 16 * a + lane % 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t k = g * kQ4Group + 32 * j + 8 * (lane / 16);
                s.x[a][j] = q4_load_row<DT>(p.x, row * p.x_stride + k, row < p.m ? p.sum - k : 0, p.wide);
            }
        }
        return s;
    };
    floatx4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0, 0, 0, 0};
    Step next = load(wave);
    for (int64_t g = wave; g < p.groups; g += W) {
        const Step s = next;
        next = load(g + W);
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
                    q4_row_floats<DT>(s.x[a][j], v);
                    q4_split<PARTS>(v, xp[a]);
                }
                off[a] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int q = 0; q < PARTS; ++q) off[a] = q4_mfma<F16>(xp[a][q], q4_minus_24<F16>(), off[a]);
            }
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const u32x4 w = q4_expand<F16>(s.q[b][j]);
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
    }
    q4_finish<DT, MT, NT, W>(p, acc, row0, tile0 * 16, lds);
}

// dx = dy W: 32 input features (two tiles, one block of scales) and 16 MT rows
// a block, the groups of 128 output features in turn over its W waves.
template <int DT, int MT, int W>
__global__ __launch_bounds__(64 * W) void q4_grad_kernel(Q4Args p) {
    constexpr int PARTS = DT == SPC_F32 ? 3 : 2, NT = 2;
    __shared__ floatx4 lds[W * MT * NT * 64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t tile0 = (int64_t)blockIdx.x * NT, row0 = (int64_t)blockIdx.y * 16 * MT;
    struct Step {
        u32x4 q[NT];
        u32x4 d[4];  // eight scales along the summed features
        Q4Row<DT> x[MT][4];
    };
    auto load = [&](int64_t g) __attribute__((always_inline)) {
        Step s;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            s.q[b] = u32x4{0, 0, 0, 0};
            if (g < p.groups)
                s.q[b] = reinterpret_cast<const u32x4*>(p.quants)[((tile0 + b) * p.groups + g) * 64 + lane];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t o = g * kQ4Group + 32 * j + 8 * (lane / 16);
            s.d[j] = u32x4{0, 0, 0, 0};
            if (g < p.groups)
                s.d[j] = *reinterpret_cast<const u32x4*>(p.scales + blockIdx.x * p.groups * kQ4Group + o);
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                const int64_t row = row0 + 16 * a + lane % 16;
                s.x[a][j] = q4_load_row<DT>(p.x, row * p.x_stride + o, row < p.m ? p.sum - o : 0, p.wide);
            }
        }
        return s;
    };
    floatx4 acc[MT][NT], off[MT];
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        off[a] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0, 0, 0, 0};
    }
    Step next = load(wave);
    for (int64_t g = wave; g < p.groups; g += W) {
        const Step s = next;
        next = load(g + W);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float d[8];
            Q4Row<SPC_F16> dr;
            dr.w[0] = s.d[j];
            q4_row_floats<SPC_F16>(dr, d);
            u32x4 w[NT];
#pragma unroll
            for (int b = 0; b < NT; ++b) w[b] = q4_expand<false>(s.q[b][j]);
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                float v[8];
                q4_row_floats<DT>(s.x[a][j], v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= d[e];
                u32x4 xp[PARTS];
                q4_split<PARTS>(v, xp);
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    off[a] = q4_mfma<false>(xp[q], q4_minus_24<false>(), off[a]);
#pragma unroll
                    for (int b = 0; b < NT; ++b) acc[a][b] = q4_mfma<false>(xp[q], w[b], acc[a][b]);
                }
            }
        }
    }
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] += off[a];
    q4_finish<DT, MT, NT, W>(p, acc, row0, tile0 * 16, lds);
}

template <int DT>
hipError_t q4_forward(hipStream_t s, const Q4Args& p) {
    // F32 rows hold three operands each: two row tiles at most
    const int64_t mt = std::min<int64_t>(ceil_div(p.m, 16), DT == SPC_F32 ? 2 : 4);
#define SPC_Q4(MT, NT, W)                                                                        \
    q4_forward_kernel<DT, MT, NT, W><<<dim3((unsigned)ceil_div(p.col_tiles, NT),                  \
                                            (unsigned)ceil_div(p.m, 16 * MT)), 64 * W, 0, s>>>(p)
    if (mt == 1) {
        SPC_Q4(1, 1, 8);
    } else if (mt == 2) {
        SPC_Q4(2, 1, 8);
    } else {
        if constexpr (DT != SPC_F32) SPC_Q4(4, 1, 8);
    }
#undef SPC_Q4
    return hipGetLastError();
}

template <int DT>
hipError_t q4_grad(hipStream_t s, const Q4Args& p) {
#define SPC_Q4(MT, W)                                                                              \
    q4_grad_kernel<DT, MT, W><<<dim3((unsigned)(p.col_tiles / 2), (unsigned)ceil_div(p.m, 16 * MT)), \
                                64 * W, 0, s>>>(p)
    if (p.m <= 16) SPC_Q4(1, 8);
    else SPC_Q4(2, 8);
#undef SPC_Q4
    return hipGetLastError();
}

int q4_shape(const char* fn, int64_t out, int64_t in) {
    if (out < 1 || in < 32 || in % 32 || out > INT32_MAX || in > INT32_MAX) {
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
    p->sum = l.sum;
    p->cols = l.cols;
    p->groups = l.groups;
    p->col_tiles = l.col_tiles;
    p->quants = static_cast<const uint32_t*>(packed);
    p->scales = reinterpret_cast<const uint16_t*>(static_cast<const char*>(packed) + l.quant_bytes);
    p->wide = (uintptr_t)x % 16 == 0 && x_stride * e % 16 == 0;
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
    if (out_features < 1 || in_features < 32 || in_features % 32 || out_features > INT32_MAX ||
        in_features > INT32_MAX)
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

int spc_linear_q4_0_input_grad(spc_stream_t stream, int dtype, const void* dy, int64_t dy_stride,
                               int64_t m, const void* packed, int64_t out_features,
                               int64_t in_features, void* dx) {
    Q4Args p;
    const int st = q4_args("spc_linear_q4_0_input_grad", dtype, dy, dy_stride, m, packed, out_features,
                           in_features, true, dx, &p);
    if (st != SPC_OK) return st;
    if (m == 0) return SPC_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = dtype == SPC_BF16  ? q4_grad<SPC_BF16>(s, p)
                         : dtype == SPC_F16 ? q4_grad<SPC_F16>(s, p)
                                            : q4_grad<SPC_F32>(s, p);
    return e == hipSuccess ? SPC_OK : hip_status(e, "spc_linear_q4_0_input_grad launch");
}

}  // extern "C"

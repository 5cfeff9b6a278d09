// linear_q4.hip -- products of a few rows with Q4_0 weights: y = x W^T + bias
// (spc_linear_q4_0) and the rows' gradient dx = dy W (spc_linear_q4_0_input_grad).
//
// A Q4_0 block is 32 weights along the input features: an f16 scale d and 32
// four-bit q, w = d (q - 8).  The weights' bytes bound both products, so they
// are read once, as they are, and expanded in registers for the matrix
// instructions, which take 16 rows at the price of one:
//
//   f16: 16 + q is the pattern 0x4c00 | q << 6, exactly, so two weights are one
//   shift, one and-or and one subtraction of 24;
//   bf16: (q - 8) / 16 by the conversion of four-bit integers.
//
// ((q - 8) itself, not 16 + q beside a sum of -24 x, though that saves an
// instruction: a row's large value that meets zero weights would leave its own
// rounding in every column, or overflow.)
//
// Forward, one 16x16x32 product covers exactly one block of every column; its
// F32 result times d is added to the F32 accumulator, so no weight is ever
// rounded.  F32 rows run as three bf16 parts that add up to them exactly.
// For the gradient the scale varies along the summed index.  F32 rows are
// multiplied by it first (F32) and run as three bf16 parts; for 16-bit rows the
// weights are, as one or two operands.
//
// The weights are laid out once (spc_linear_q4_0_pack) in the order the lanes
// want them: for 16 columns and 128 summed features a lane's 16 bytes are its
// eight weights of four instructions, so a wave's load is one 1 KB run.
//
// Times below are a kernel's in a captured graph, rows times weights as in ->
// out.  The two of a choice were measured side by side; those of the loads'
// order (16 bf16 rows through LDS, steps under way) on weights as 16 + q.
#include <algorithm>

#include "common.h"

namespace spc {

// (gfx950 loads 16 bytes from any address)
typedef u32x4 u32x4_any __attribute__((aligned(2)));

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
// The f16 pattern's fixed bits: one of the two in a vector register, since an
// instruction reads one scalar operand, and the and-or is one instruction then.
__device__ __forceinline__ uint32_t q4_one() {
    uint32_t v = 0x4c004c00u;
    asm("" : "+v"(v));
    return v;
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// (q - 8) of a word's weights as f16.
__device__ __forceinline__ u32x4 q4_expand_f16(uint32_t w, uint32_t one) {
    constexpr uint32_t m = 0x03c003c0u;
    u32x4 r = {((w << 6) & m) | one, ((w << 2) & m) | one, ((w >> 2) & m) | one, ((w >> 6) & m) | one};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t ri = r[i];  // (a copy: a bit cast of a vector's element takes the vector's first)
        r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, ri) - (f16x2)(_Float16)24.0f);
    }
    return r;
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

// (q - 8) / 16 of a word's weights as bf16: the conversion of four-bit
// integers, whose results end in zeros, so the cut to bf16 is exact.  It takes
// a byte's low half, so every other nibble costs no shift of its own (compiled
// from shifts: 144 instructions for 64 weights, 112 so).
template <int BYTE>
__device__ __forceinline__ float q4_signed(uint32_t w) {
    float f;
    if constexpr (BYTE == 0) f = __builtin_amdgcn_cvt_off_f32_i4(w);
    if constexpr (BYTE == 1)
        asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(w));
    if constexpr (BYTE == 2)
        asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(w));
    if constexpr (BYTE == 3)
        asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(w));
    return f;
}
__device__ __forceinline__ u32x4 q4_expand_signed(uint32_t w) {
    w ^= 0x88888888u;  // q - 8 as four bits of two's complement
    const uint32_t odd = w >> 4;
    auto pair = [](float a, float b) __attribute__((always_inline)) {
        return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    };
    return u32x4{pair(q4_signed<0>(w), q4_signed<2>(w)), pair(q4_signed<0>(odd), q4_signed<2>(odd)),
                 pair(q4_signed<1>(w), q4_signed<3>(w)), pair(q4_signed<1>(odd), q4_signed<3>(odd))};
}

// The high halves of two F32 words as a bf16 pair (a cut, not a rounding).
__device__ __forceinline__ uint32_t q4_high_pair(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ float q4_rest(float v) {
    return v - __uint_as_float(__float_as_uint(v) & 0xffff0000u);
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
    void* y;             // [m, cols]
};

template <int DT>
__device__ __forceinline__ void q4_store(void* y, int64_t at, float v) {
    if constexpr (DT == SPC_F32) static_cast<float*>(y)[at] = v;
    else if constexpr (DT == SPC_BF16) static_cast<uint16_t*>(y)[at] = f32_to_bf16_bits(v);
    else static_cast<uint16_t*>(y)[at] = f32_to_f16_bits(v);
}

// ---- rows -------------------------------------------------------------------
// A step's rows: 128 summed features of ROWS rows, 16 bytes a lane and load, a
// row in consecutive lanes (LANES of them; PER elements each), kept by a wave
// for itself: loaded ahead, turned into operands once an element, written to
// its part of LDS and read back as the matrix instructions want them (lane l:
// row l % 16, features 32 j + 8 (l / 16) ..+ 7).  Loaded in that order
// instead, four neighbouring lanes are in four rows, a load is 64 accesses of
// the cache, and sixteen rows cost three times the weights (16 bf16 rows,
// 16,384 -> 4096: 19.7 us, 13.2 through LDS); few rows are few loads, and their
// conversion is done for ROWS rows, not for sixteen.
template <int DT, int ROWS>
struct Q4Rows {
    static constexpr int ES = DT == SPC_F32 ? 4 : 2, PER = 16 / ES, LANES = kQ4Group / PER;
    static constexpr int NI = ROWS * LANES / 64;         // loads a lane
    static constexpr int STRIDE = kQ4Group * 2 + 16;     // bytes of an operand row in LDS
    static constexpr int MT = (ROWS + 15) / 16;          // 16-row tiles
    const char* row[NI];

    __device__ __forceinline__ static int lane() { return threadIdx.x & 63; }
    __device__ __forceinline__ static int chunk() { return lane() % LANES; }
    // the row (of ROWS) of load i
    __device__ __forceinline__ static int in_tile(int i) { return i * (64 / LANES) + lane() / LANES; }

    // Rows past the last repeat it; their results are not stored.
    __device__ __forceinline__ Q4Rows(const void* x, int64_t x_stride, int64_t row0, int64_t m) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            row[i] = static_cast<const char*>(x) +
                     (min(row0 + in_tile(i), m - 1) * x_stride + chunk() * PER) * ES;
    }
    // Zeros past the end of a row of `sum` elements.
    __device__ __forceinline__ void load(u32x4 (&v)[NI], int g, int sum) const {
        const int64_t at = (int64_t)g * kQ4Group * ES;
        if ((g + 1) * kQ4Group <= sum) {
#pragma unroll
            for (int i = 0; i < NI; ++i) v[i] = *reinterpret_cast<const u32x4_any*>(row[i] + at);
        } else {
            const int left = sum - g * kQ4Group - chunk() * PER;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                v[i] = u32x4{0, 0, 0, 0};
                if (left >= PER) {
                    v[i] = *reinterpret_cast<const u32x4_any*>(row[i] + at);
                } else if (left > 0) {
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        if (e >= left) break;
                        if constexpr (DT == SPC_F32)
                            v[i][e] = reinterpret_cast<const uint32_t*>(row[i] + at)[e];
                        else
                            v[i][e / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(row[i] + at)[e]
                                           << (16 * (e & 1));
                    }
                }
            }
        }
    }
    // One 16-bit operand: the loads as they are.
    __device__ __forceinline__ static void put(char* lds, int i, u32x4 v) {
        *reinterpret_cast<u32x4*>(lds + in_tile(i) * STRIDE + chunk() * 16) = v;
    }
    // Four F32 values as three bf16 operands that add up to them: cuts of eight
    // bits each, and the last one's rest is nothing.
    __device__ __forceinline__ static void put_parts(char* lds, int i, float (&f)[4]) {
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            *reinterpret_cast<u32x2*>(lds + (s * ROWS + in_tile(i)) * STRIDE + chunk() * 8) =
                u32x2{q4_high_pair(f[0], f[1]), q4_high_pair(f[2], f[3])};
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = q4_rest(f[e]);
        }
    }
    // Operand `part` of row tile a for instruction j (fewer than 16 rows repeat).
    __device__ __forceinline__ static u32x4 get(const char* lds, int part, int a, int j) {
        const int r = ROWS >= 16 ? 16 * a + lane() % 16 : lane() % ROWS;
        return *reinterpret_cast<const u32x4*>(lds + (part * ROWS + r) * STRIDE +
                                               (4 * j + lane() / 16) * 16);
    }
};

// A wave's own LDS, written and read back by different lanes of it: its LDS
// operations complete in order, so only the compiler has to keep theirs.
__device__ __forceinline__ void q4_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Adds the W waves' accumulators and stores: tiles [MT][NT] of 16 rows x 16
// columns; lane l of a tile holds column l % 16, rows 4 (l / 16) + i.  Of a block
// of fewer than 16 rows the tile's others repeat them.  lds is the block's,
// whatever it held.
template <int DT, int ROWS, int MT, int NT, int W>
__device__ __forceinline__ void q4_finish(const Q4Args& p, floatx4 (&acc)[MT][NT], int64_t row0,
                                          int64_t col0, floatx4* lds) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    constexpr int TILES = MT * NT;
    const int64_t end = min(p.m, row0 + ROWS);
    __syncthreads();
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
            if (row < end) q4_store<DT>(p.y, row * p.cols + col, v[i] + bias);
        }
    }
}

// Bytes of a block's LDS: the waves' rows (and, for the gradient, scales and
// row factors), then the accumulators.
constexpr size_t q4_lds(size_t wave_bytes, int tiles, int w) {
    return wave_bytes * w > (size_t)tiles * w * 1024 ? wave_bytes * w : (size_t)tiles * w * 1024;
}

// A block's W waves take the groups of 128 summed features in turn, each with
// its next step of weights and rows under way: f(step) for every step of this
// wave.  (Two or three steps under way measured slower: 8192 -> 16,384, one
// bf16 row, 16.2 / 17.3 us with one / two; two buffers in turn instead of a move
// 14.8 / 15.4: the waves hide each other's loads.)
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

// y = x W^T: a block's W waves share 16 NT columns and ROWS rows.
template <int DT, int ROWS, int NT, int W>
__global__ __launch_bounds__(64 * W) void q4_forward_kernel(Q4Args p) {
    constexpr bool F16 = DT == SPC_F16;
    constexpr int PARTS = DT == SPC_F32 ? 3 : 1;
    typedef Q4Rows<DT, ROWS> R;
    constexpr int MT = R::MT;
    constexpr size_t WAVE = PARTS * ROWS * R::STRIDE;
    __shared__ __attribute__((aligned(16))) char lds[q4_lds(WAVE, MT * NT, W)];
    const uint32_t lane = threadIdx.x & 63;
    char* mine = lds + (threadIdx.x >> 6) * WAVE;
    const int64_t tile0 = (int64_t)blockIdx.x * NT, row0 = (int64_t)blockIdx.y * ROWS;
    struct Step {
        u32x4 q[NT];
        u32x2 d[NT];
        u32x4 x[R::NI];
    };
    const R rows(p.x, p.x_stride, row0, p.m);
    auto load = [&](Step& s, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            // (tiles past the last repeat it; their results are not stored)
            const int64_t t = min(tile0 + b, p.col_tiles - 1) * p.groups + g;
            s.q[b] = (reinterpret_cast<const u32x4*>(p.quants) + t * 64)[lane];
            s.d[b] = (reinterpret_cast<const u32x2*>(p.scales) + t * 16)[lane % 16];
        }
        rows.load(s.x, g, p.sum);
    };
    floatx4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0, 0, 0, 0};
    const uint32_t one = q4_one();
    q4_pipeline<W, Step>(p.groups, load, [&](const Step& s) __attribute__((always_inline)) {
        q4_wave_sync();
#pragma unroll
        for (int i = 0; i < R::NI; ++i) {
            if constexpr (PARTS == 1) {
                R::put(mine, i, s.x[i]);
            } else {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(s.x[i][e]);
                R::put_parts(mine, i, f);
            }
        }
        q4_wave_sync();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 xp[MT][PARTS];
            floatx4 off[MT];
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                off[a] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int q = 0; q < PARTS; ++q) xp[a][q] = R::get(mine, q, a, j);
                // (nothing, or NaN where the row has an infinity or NaN)
                if constexpr (PARTS == 1) off[a] = q4_mfma<F16>(xp[a][0], u32x4{0, 0, 0, 0}, off[a]);
            }
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const float d = f16_bits_to_f32((uint16_t)(s.d[b][j / 2] >> (16 * (j & 1))));
                u32x4 w;
                if constexpr (F16) w = q4_expand_f16(s.q[b][j], one);
                else w = q4_expand_signed(s.q[b][j]);
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
    if constexpr (!F16) {
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int b = 0; b < NT; ++b) acc[a][b] *= 16.0f;
    }
    q4_finish<DT, ROWS, MT, NT, W>(p, acc, row0, tile0 * 16, reinterpret_cast<floatx4*>(lds));
}

// dx = dy W of F32 rows: 16 NT input features (NT 1 or 2: within one block of
// scales) and ROWS rows a block.  dy times the scale (F32) enters as three parts.
template <int ROWS, int NT, int W>
__global__ __launch_bounds__(64 * W) void q4_grad_kernel(Q4Args p) {
    typedef Q4Rows<SPC_F32, ROWS> R;
    constexpr int MT = R::MT;
    constexpr size_t WAVE = 3 * ROWS * R::STRIDE;
    __shared__ __attribute__((aligned(16))) char lds[q4_lds(WAVE, MT * NT, W)];
    const uint32_t lane = threadIdx.x & 63;
    char* mine = lds + (threadIdx.x >> 6) * WAVE;
    const int64_t tile0 = (int64_t)blockIdx.x * NT, row0 = (int64_t)blockIdx.y * ROWS;
    struct Step {
        u32x4 q[NT];
        u32x2 d;  // the scales of this lane's four summed features
        u32x4 x[R::NI];
    };
    const R rows(p.x, p.x_stride, row0, p.m);
    const uint16_t* scales = p.scales + tile0 / 2 * p.groups * kQ4Group;
    auto load = [&](Step& s, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < NT; ++b)
            s.q[b] = (reinterpret_cast<const u32x4*>(p.quants) + ((tile0 + b) * p.groups + g) * 64)[lane];
        s.d = reinterpret_cast<const u32x2*>(scales + (int64_t)g * kQ4Group)[lane % 32];
        rows.load(s.x, g, p.sum);
    };
    floatx4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = floatx4{0, 0, 0, 0};
    q4_pipeline<W, Step>(p.groups, load, [&](const Step& s) __attribute__((always_inline)) {
        q4_wave_sync();
#pragma unroll
        for (int i = 0; i < R::NI; ++i) {
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                f[e] = __uint_as_float(s.x[i][e]) *
                       f16_bits_to_f32((uint16_t)(s.d[e / 2] >> (16 * (e & 1))));
            R::put_parts(mine, i, f);
        }
        q4_wave_sync();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 w[NT];
#pragma unroll
            for (int b = 0; b < NT; ++b) w[b] = q4_expand_signed(s.q[b][j]);
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    const u32x4 xp = R::get(mine, q, a, j);
#pragma unroll
                    for (int b = 0; b < NT; ++b) acc[a][b] = q4_mfma<false>(xp, w[b], acc[a][b]);
                }
        }
    });
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] *= 16.0f;
    q4_finish<SPC_F32, ROWS, MT, NT, W>(p, acc, row0, tile0 * 16, reinterpret_cast<floatx4*>(lds));
}

// ---- the gradient of 16-bit rows -------------------------------------------
// Multiplying the rows by a scale that differs for every 32 columns costs six
// instructions an element and block of columns, and their split into parts
// three matrix instructions a tile, which bound 16-bit rows (16 rows, 4096 ->
// 16,384: 23 us of a floor of 8).  Here the weights take the scale, f16(d (q -
// 8)), and the rows enter as f16 whatever their columns.
//
// f16 rows enter as they are, and so that no weight's rounding adds to the
// output's own, what f16(d (q - 8)) leaves over is a second operand: a multiple
// of d's last bit below 2^-11 of the weight, so an f16 too (outputs off by
// 2.1e-4 of their size with it, 2.7e-4 without, as much as the plain form's).
// Under bf16 rows it stays out: at most 2^-11 of a weight, an eighth of a bf16
// output's rounding.
//
// bf16 rows have a range that f16 has not, and a value may not vanish under its
// row's largest: where the large ones meet zero weights it is the result.  Two ways:
// - raw: the rows as they are, f16(d (q - 8)) as two bf16 operands, cut and the
//   three bits below the cut: exact for every bf16, for twelve instructions a
//   pair of weights where one operand takes four;
// - moved: the rows' exponents moved into f16's range by a power of two that each
//   wave chooses for each row from what it has seen of it, eleven instructions a
//   pair of row elements; a row's step with a value that does not fit (below
//   2^-27 of its largest) goes raw.
// The first falls on a block's 16 NT columns, the second on its ROWS rows, so
// rows are moved where they are few (us raw / moved: one row, 16,384 -> 8192
// 28.2 / 17.5, eight, 1024 -> 8192 9.4 / 7.8, sixteen by two tiles, 16,384 ->
// 8192 31.3 / 30.2, by one, 4096 -> 16,384 21.2 / 22.7, thirty, 16,384 -> 4096
// 22.4 / 27.0).

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The eight weights of a word times their eight scales, rounded, and (PARTS 2)
// what the rounding left over.
// BF16: the rounded weight as two bf16 operands.
template <bool BF16, int PARTS>
__device__ __forceinline__ void q4_expand_scaled(uint32_t w, u32x4 d, uint32_t one, u32x4 (&r)[PARTS]) {
    const u32x4 q = q4_expand_f16(w, one);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t qi = q[i], di = d[i];
        const f16x2 v = __builtin_bit_cast(f16x2, qi);
        const f16x2 s = __builtin_bit_cast(f16x2, di);
        const f16x2 t = v * s;
        if constexpr (BF16) {
            const float a = (float)t.x, b = (float)t.y;
            r[0][i] = q4_high_pair(a, b);
            r[1][i] = q4_high_pair(q4_rest(a), q4_rest(b));
        } else {
            r[0][i] = __builtin_bit_cast(uint32_t, t);
            if constexpr (PARTS == 2)
                r[1][i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(v, s, -t));
        }
    }
}

// A row's exponent bias: what is taken off its bf16 exponents to make f16's.
// The row's largest value seen so far has f16 exponent 28 when the bias is
// set, so it may grow by 2^2 before the bias has to move.  A step only looks
// for values past that in its lane; the row's maximum is formed when one is
// found.
struct Q4Bias {
    u16x2 seen = {0, 0};   // the lane's largest magnitudes, bf16 bits
    u16x2 limit = {0, 0};  // largest that fits; 0 until the row has one but 0
    u16x2 least = {0, 0};  // smallest but 0 that fits, less one
    int bias = 0;

    // Takes a step's elements in; true if one does not fit.
    __device__ __forceinline__ bool see(u32x4 v) {
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
        seen = __builtin_elementwise_max(seen, m);
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(m, limit)) != 0;
    }
    // Whether an element but 0 is too small to fit.
    __device__ __forceinline__ bool small(u32x4 v) const {
        u16x2 m = {0xffff, 0xffff};
#pragma unroll
        for (int i = 0; i < 4; ++i)  // (zeros become the largest)
            m = __builtin_elementwise_min(
                m, (u16x2)(__builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu) - (u16x2){1, 1}));
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(least, m)) != 0;
    }
    // The largest magnitude the row's 16 lanes have seen.
    __device__ __forceinline__ int top() const {
        int t = max((int)seen.x, (int)seen.y);
        t = max(t, __builtin_amdgcn_update_dpp(0, t, 0xB1, 0xf, 0xf, true));    // lane ^ 1
        t = max(t, __builtin_amdgcn_update_dpp(0, t, 0x4E, 0xf, 0xf, true));    // lane ^ 2
        t = max(t, __builtin_amdgcn_update_dpp(0, t, 0x141, 0xf, 0xf, true));   // mirror in 8
        return max(t, __builtin_amdgcn_update_dpp(0, t, 0x140, 0xf, 0xf, true));  // in 16
    }
    // Whether the row needs another bias; moves it.
    __device__ __forceinline__ bool must_move() const {
        const int t = top();
        return t >> 7 > bias + 30 || (limit.x == 0 && t != 0);
    }
    __device__ __forceinline__ void move() {
        const int t = top();
        if (must_move()) bias = max((t >> 7) - 28, 0);
        if (t != 0) limit = (u16x2)(uint16_t)(((bias + 31) << 7) - 1);
        // (without a bias subnormals are f16's)
        least = (u16x2)(uint16_t)(bias ? ((bias + 1) << 7) - 1 : 0);
    }
    // bf16 -> f16 with the bias taken off, for elements that fit.
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
        return top() >= 0x7f80 ? __builtin_nanf("") : ldexpf(1.0f, bias - 112);
    }
};

// dx = dy W of 16-bit rows: 16 NT input features (NT 1 or 2: within one block
// of scales) and ROWS rows a block.
template <int DT, int ROWS, int NT, int W>
__global__ __launch_bounds__(64 * W) void q4_grad16_kernel(Q4Args p) {
    typedef Q4Rows<DT, ROWS> R;
    constexpr bool MOVED = DT == SPC_BF16 && ROWS < 16 * NT;
    constexpr int MT = R::MT, NI = R::NI;
    constexpr size_t SCALES = ROWS * R::STRIDE, FACTORS = SCALES + kQ4Group * 2;
    constexpr size_t WAVE = FACTORS + (ROWS * 4 + 15) / 16 * 16;
    __shared__ __attribute__((aligned(16))) char lds[q4_lds(WAVE, MT * NT, W)];
    const uint32_t lane = threadIdx.x & 63;
    char* mine = lds + (threadIdx.x >> 6) * WAVE;
    u32x4* scales = reinterpret_cast<u32x4*>(mine + SCALES);  // [16]
    const int64_t tile0 = (int64_t)blockIdx.x * NT, row0 = (int64_t)blockIdx.y * ROWS;
    struct Step {
        u32x4 q[NT];
        u32x4 d;  // scales 8 (lane % 16) .. + 7 along the summed features
        u32x4 x[NI];
    };
    const R rows(p.x, p.x_stride, row0, p.m);
    const uint16_t* all_scales = p.scales + tile0 / 2 * p.groups * kQ4Group;
    auto load = [&](Step& s, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < NT; ++b)
            s.q[b] = (reinterpret_cast<const u32x4*>(p.quants) + ((tile0 + b) * p.groups + g) * 64)[lane];
        s.d = reinterpret_cast<const u32x4*>(all_scales + (int64_t)g * kQ4Group)[lane % 16];
        rows.load(s.x, g, p.sum);
    };
    // (moved rows: acc in units of the biases, raw in ones)
    floatx4 acc[MT][NT], raw[MT][NT];
    Q4Bias bias[NI];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = raw[a][b] = floatx4{0, 0, 0, 0};
    // adds acc's rows, of those loads' rows that f(i) says, times their factors to
    // raw, and starts them again
    auto flush = [&](auto&& f) __attribute__((always_inline)) {
        float* fs = reinterpret_cast<float*>(mine + FACTORS);
        q4_wave_sync();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const float v = f(i) ? bias[i].factor() : 0.0f;  // (a factor is never 0)
            if (R::chunk() == 0) fs[R::in_tile(i)] = v;
        }
        q4_wave_sync();
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = fs[(16 * a + 4 * (lane / 16) + i) % ROWS];
#pragma unroll
                for (int b = 0; b < NT; ++b) {
                    raw[a][b][i] = v != 0.0f ? raw[a][b][i] + acc[a][b][i] * v : raw[a][b][i];
                    acc[a][b][i] = v != 0.0f ? 0.0f : acc[a][b][i];
                }
            }
    };
    const uint32_t one = q4_one();
    // a step's products of the rows in LDS, as f16 or bf16, added to `to`
    auto products = [&](const Step& s, auto bf16, floatx4 (&to)[MT][NT]) __attribute__((always_inline)) {
        constexpr bool BF16 = decltype(bf16)::value;
        constexpr int PARTS = BF16 || DT == SPC_F16 ? 2 : 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 x[MT];
#pragma unroll
            for (int a = 0; a < MT; ++a) x[a] = R::get(mine, 0, a, j);
            const u32x4 d = scales[4 * j + lane / 16];
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                u32x4 w[PARTS];
                q4_expand_scaled<BF16, PARTS>(s.q[b][j], d, one, w);
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) to[a][b] = q4_mfma<!BF16>(x[a], w[q], to[a][b]);
            }
        }
    };
    q4_pipeline<W, Step>(p.groups, load, [&](const Step& s) __attribute__((always_inline)) {
        bool small[NI] = {}, any_small = false;
        if constexpr (MOVED) {
            bool over = false;
#pragma unroll
            for (int i = 0; i < NI; ++i) over |= bias[i].see(s.x[i]);
            if (__any(over)) {
                // (into raw: moved with the biases, what is there could vanish)
                flush([&](int i) { return bias[i].must_move(); });
#pragma unroll
                for (int i = 0; i < NI; ++i) bias[i].move();
            }
            // a row's 16 lanes decide for it alone, so its result is its own
            static_assert(R::LANES == 16, "a row's lanes");
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const uint64_t m = __ballot(bias[i].small(s.x[i]));
                small[i] = (m >> (lane & 48) & 0xffff) != 0;
                any_small |= m != 0;
            }
        }
        const u32x4 zero = {0, 0, 0, 0};
        q4_wave_sync();
#pragma unroll
        for (int i = 0; i < NI; ++i)
            R::put(mine, i, !MOVED ? s.x[i] : small[i] ? zero : bias[i].f16(s.x[i]));
        if (lane < 16) scales[lane] = s.d;
        q4_wave_sync();
        products(s, std::bool_constant<DT == SPC_BF16 && !MOVED>{}, acc);
        if (MOVED && any_small) {
            q4_wave_sync();
#pragma unroll
            for (int i = 0; i < NI; ++i) R::put(mine, i, small[i] ? s.x[i] : zero);
            q4_wave_sync();
            products(s, std::true_type{}, raw);
        }
    });
    if constexpr (MOVED) flush([](int) { return true; });
    q4_finish<DT, ROWS, MT, NT, W>(p, MOVED ? raw : acc, row0, tile0 * 16, reinterpret_cast<floatx4*>(lds));
}

template <int DT, int ROWS, int NT, int W>
void q4_forward_launch(hipStream_t s, const Q4Args& p) {
    const dim3 grid((unsigned)ceil_div(p.col_tiles, NT), (unsigned)ceil_div(p.m, ROWS));
    q4_forward_kernel<DT, ROWS, NT, W><<<grid, 64 * W, 0, s>>>(p);
}

template <int DT, int ROWS, int NT, int W>
void q4_grad_launch(hipStream_t s, const Q4Args& p) {
    const dim3 grid((unsigned)(p.col_tiles / NT), (unsigned)ceil_div(p.m, ROWS));
    if constexpr (DT == SPC_F32) q4_grad_kernel<ROWS, NT, W><<<grid, 64 * W, 0, s>>>(p);
    else q4_grad16_kernel<DT, ROWS, NT, W><<<grid, 64 * W, 0, s>>>(p);
}

// f(ROWS) with the fewest rows a block that hold m or leave a CU to every block, at
// most 32 (F32, whose three operands take as much LDS as that: 16): beyond a few
// rows a block's time is its rows' conversion, while other CUs would stand
// idle.  us with the fewest that hold m / that spread: forward, thirty bf16 rows
// 8192 -> 1024 11.4 / 7.2, 1024 -> 1024 4.4 / 3.8, sixteen F32 rows 4096 -> 1024
// 9.2 / 6.1; gradient, thirty bf16 rows of 1024 -> 16,384 24.8 / 16.2, sixteen 18.0 /
// 12.6.  Past a block to a CU it loses (sixteen bf16 rows, 8192 -> 4096 9.3 / 11.1,
// gradient of 4096 -> 16,384 19.6 / 22.4), but half the most rows hardly do (thirty
// bf16 rows, 4096 -> 4096 8.6 / 7.9, gradient of 4096 -> 8192 15.3 / 16.0; sixteen
// F32 rows, gradient of 4096 -> 4096 10.2 / 8.9).
template <int DT, typename F>
void q4_row_tile(const Q4Args& p, F&& f) {
    auto fits = [&](int rows) {
        const int blocks = rows < (DT == SPC_F32 ? 8 : 16) ? 256 : 512;
        return p.m <= rows || p.col_tiles * ceil_div(p.m, rows) <= blocks;
    };
    if (fits(4)) f(std::integral_constant<int, 4>{});
    else if (fits(8)) f(std::integral_constant<int, 8>{});
    else if (fits(16) || DT == SPC_F32) f(std::integral_constant<int, 16>{});
    else if constexpr (DT != SPC_F32) f(std::integral_constant<int, 32>{});
}

// Two column tiles a wave where that leaves a block for every CU: each reads
// (and converts) the rows half as often.  us with one / two: 8192 -> 16,384, one
// bf16 row 20.3 / 16.7, eight 23.0 / 18.3, sixteen 23.6 / 20.2, two F32 rows
// 27.8 / 21.6; 4096 -> 4096 (256 tiles), one 4.9 / 6.1, forty 13.9 / 10.5; the
// gradient of 8192 -> 16,384, one 22.8 / 19.5, sixteen 35.8 / 27.9, of 4096 ->
// 16,384 (256 tiles), sixteen 19.7 / 26.5.
template <int ROWS>
inline bool q4_two_tiles(const Q4Args& p) {
    return p.col_tiles * ceil_div(p.m, ROWS) >= 512;
}

// Sixteen waves a block instead of eight for one tile of 8192 summed features or
// more: hardly a CU has a second block to hide the loads' latency.  us with
// eight / sixteen: one bf16 row, 8192 -> 1024 6.4 / 6.0, 16,384 -> 4096 11.6 / 10.6,
// eight F32 rows, 8192 -> 1024 8.8 / 8.3; sixteen bf16 rows, 8192 -> 4096 9.3 both,
// 16,384 -> 4096 15.0 / 13.9, the gradient of 4096 to 8192 12.8 / 12.4, 10,240 14.4 /
// 13.9, 12,288 16.4 / 15.8, 14,336 18.3 / 17.7, 16,384 20.6 / 19.6; shorter sums the
// same or slower (2048 -> 1024 3.65 / 3.74).  More rows have no registers left
// (thirty, spilled, lost four times their time).
template <int DT, int ROWS>
constexpr int kQ4MoreWaves = ROWS <= (DT == SPC_F32 ? 8 : 16) ? 16 : 8;
inline bool q4_long_sum(const Q4Args& p) { return p.groups >= 64; }

template <int DT>
hipError_t q4_forward(hipStream_t s, const Q4Args& p) {
    q4_row_tile<DT>(p, [&](auto rows) {
        constexpr int ROWS = decltype(rows)::value, W = kQ4MoreWaves<DT, ROWS>;
        if (q4_two_tiles<ROWS>(p)) q4_forward_launch<DT, ROWS, 2, 8>(s, p);
        else if (q4_long_sum(p)) q4_forward_launch<DT, ROWS, 1, W>(s, p);
        else q4_forward_launch<DT, ROWS, 1, 8>(s, p);
    });
    return hipGetLastError();
}

template <int DT>
hipError_t q4_grad(hipStream_t s, const Q4Args& p) {
    q4_row_tile<DT>(p, [&](auto rows) {
        constexpr int ROWS = decltype(rows)::value, W = kQ4MoreWaves<DT, ROWS>;
        if (q4_two_tiles<ROWS>(p)) q4_grad_launch<DT, ROWS, 2, 8>(s, p);
        else if (q4_long_sum(p)) q4_grad_launch<DT, ROWS, 1, W>(s, p);
        else q4_grad_launch<DT, ROWS, 1, 8>(s, p);
    });
    return hipGetLastError();
}

// ---- the bias' gradient -----------------------------------------------------
// Sums of the rows' columns, F32 in a fixed order: 32 columns and 512 rows a
// block, 16 rows a thread (eight under way), then the lanes of a wave, then the
// waves through LDS; more than 512 rows by the same kernel again over the
// blocks' sums.  (Queued calls, us, 16-bit rows, beside a library's cast, sum
// and cast: 16 x 2048 6.9 / 14.5, 5,000 x 130 11.3 / 17, 62,710 x 1024 65 / 126.
// The sum was the one step of the pass that could record a memory node into a
// captured graph.)
constexpr int kQ4SumCols = 32, kQ4SumThreads = 1024, kQ4SumRows = 512;
// Blocks along the columns, each taking every such many-th 32: a launch holds
// below 2^32 threads.
constexpr int64_t kQ4SumBlocks = 1 << 21;

__device__ __forceinline__ float q4_element(const void* p, int dt, int64_t i) {
    if (dt == SPC_F32) return static_cast<const float*>(p)[i];
    const uint16_t b = static_cast<const uint16_t*>(p)[i];
    return dt == SPC_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

__global__ __launch_bounds__(kQ4SumThreads) void q4_column_sums_kernel(const void* x, int dtype,
                                                                       int64_t stride, int64_t m,
                                                                       int64_t rows_per, int64_t cols,
                                                                       void* out, int out_dtype) {
    constexpr int C = kQ4SumCols, L = kQ4SumThreads / C, W = kQ4SumThreads / 64, DEEP = 8;
    __shared__ float ls[W][C];
    const int cl = threadIdx.x % C, l = threadIdx.x / C;
    const int64_t lo = (int64_t)blockIdx.y * rows_per, hi = min(m, lo + rows_per);
    for (int64_t c0 = (int64_t)blockIdx.x * C; c0 < cols; c0 += (int64_t)gridDim.x * C) {
        const int64_t col = c0 + cl;
        float s = 0.0f;
        if (col < cols)
            for (int64_t r = lo + l; r < hi; r += DEEP * L) {
                float v[DEEP];
#pragma unroll
                for (int i = 0; i < DEEP; ++i) {
                    const int64_t at = r + i * L;
                    v[i] = q4_element(x, dtype, min(at, hi - 1) * stride + col);
                    if (at >= hi) v[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < DEEP; ++i) s += v[i];
            }
        s += __shfl_xor(s, C);
        if ((threadIdx.x & 63) < C) ls[threadIdx.x >> 6][cl] = s;
        __syncthreads();
        if (l == 0 && col < cols) {
            s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += ls[w][cl];
            const int64_t at = (int64_t)blockIdx.y * cols + col;
            if (out_dtype == SPC_F32) q4_store<SPC_F32>(out, at, s);
            else if (out_dtype == SPC_BF16) q4_store<SPC_BF16>(out, at, s);
            else q4_store<SPC_F16>(out, at, s);
        }
        __syncthreads();  // (before the sums of the next columns)
    }
}

// Blocks along the rows: at most a y-dimension's, of more rows where that is few.
inline int64_t q4_sum_rows(int64_t m) { return std::max<int64_t>(kQ4SumRows, ceil_div(m, kQ4SumRows)); }

inline bool q4_float_dtype(int dt) { return dt == SPC_F32 || dt == SPC_F16 || dt == SPC_BF16; }

// Up to 2^27 features: a launch holds below 2^32 threads, the products' 512 for
// 16 or 32 columns.
constexpr int64_t kQ4MaxFeatures = 1 << 27;
constexpr int64_t kQ4MaxRows = 65535 * 16;  // a launch's y dimension, 16 rows a block

bool q4_known(int64_t out, int64_t in) {
    return out >= 1 && in >= 32 && in % 32 == 0 && out <= kQ4MaxFeatures && in <= kQ4MaxFeatures;
}

int q4_shape(const char* fn, int64_t out, int64_t in) {
    if (!q4_known(out, in)) {
        set_last_error("%s: unsupported shape out_features=%lld in_features=%lld (a multiple of 32, "
                       "both up to 2^27)", fn, (long long)out, (long long)in);
        return SPC_BAD_SHAPE;
    }
    return SPC_OK;
}

// Checks a product's arguments and fills the kernel's.
int q4_args(const char* fn, int dtype, const void* x, int64_t x_stride, int64_t m, const void* packed,
            int64_t out, int64_t in, bool transpose, void* y, Q4Args* p) {
    const int st = q4_shape(fn, out, in);
    if (st != SPC_OK) return st;
    if (m < 0 || m > kQ4MaxRows || x_stride < 0) {
        set_last_error("%s: unsupported rows m=%lld (0 to %lld)", fn, (long long)m,
                       (long long)kQ4MaxRows);
        return SPC_BAD_SHAPE;
    }
    if (!q4_float_dtype(dtype)) {
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
    if (!q4_known(out_features, in_features)) return 0;
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
    if (bias && (!q4_float_dtype(bias_dtype) ||
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

size_t spc_linear_q4_0_bias_grad_workspace_bytes(int64_t m, int64_t out_features) {
    if (m < 0 || m > kQ4MaxRows || out_features < 1 || out_features > kQ4MaxFeatures) return 0;
    return m <= kQ4SumRows ? 0 : (size_t)(ceil_div(m, q4_sum_rows(m)) * out_features * 4);
}

int spc_linear_q4_0_bias_grad(spc_stream_t stream, int dtype, const void* dy, int64_t dy_stride,
                              int64_t m, int64_t out_features, int bias_dtype, void* dbias,
                              void* workspace, size_t workspace_bytes) {
    const char* fn = "spc_linear_q4_0_bias_grad";
    if (m < 0 || m > kQ4MaxRows || dy_stride < 0 || out_features < 1 || out_features > kQ4MaxFeatures) {
        set_last_error("%s: unsupported shape m=%lld out_features=%lld", fn, (long long)m,
                       (long long)out_features);
        return SPC_BAD_SHAPE;
    }
    const size_t need = spc_linear_q4_0_bias_grad_workspace_bytes(m, out_features);
    if (!q4_float_dtype(dtype) || !q4_float_dtype(bias_dtype) || (m > 0 && !dy) || !dbias ||
        (uintptr_t)dy % (dtype == SPC_F32 ? 4 : 2) || (uintptr_t)dbias % (bias_dtype == SPC_F32 ? 4 : 2) ||
        workspace_bytes < need || (need && (!workspace || (uintptr_t)workspace % 4))) {
        set_last_error("%s: unknown dtype, null or misaligned pointer, or workspace too small", fn);
        return SPC_BAD_ARG;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned cb = (unsigned)std::min(ceil_div(out_features, kQ4SumCols), kQ4SumBlocks);
    if (need) {
        const int64_t per = q4_sum_rows(m), parts = ceil_div(m, per);
        q4_column_sums_kernel<<<dim3(cb, (unsigned)parts), kQ4SumThreads, 0, s>>>(
            dy, dtype, dy_stride, m, per, out_features, workspace, SPC_F32);
        q4_column_sums_kernel<<<cb, kQ4SumThreads, 0, s>>>(workspace, SPC_F32, out_features, parts, parts,
                                                           out_features, dbias, bias_dtype);
    } else {
        q4_column_sums_kernel<<<cb, kQ4SumThreads, 0, s>>>(dy, dtype, dy_stride, m, std::max<int64_t>(m, 1),
                                                           out_features, dbias, bias_dtype);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SPC_OK : hip_status(e, "spc_linear_q4_0_bias_grad launch");
}

}  // extern "C"

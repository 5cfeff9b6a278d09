// rows8.h -- feature rows in groups of eight columns, and the counter-based
// random numbers of such a group (dropout and the adapters' products share the
// mask).
#pragma once

#include "common.h"

namespace spc {

// (gfx950 loads and stores 16 bytes at any address)
typedef u32x4 u32x4_rows __attribute__((aligned(2)));

inline bool float_dtype(int dt) { return dt == SPC_F32 || dt == SPC_F16 || dt == SPC_BF16; }
inline int64_t float_size(int dt) { return dt == SPC_F32 ? 4 : 2; }

template <int DT>
struct RowElem {
    using S = uint16_t;
    static constexpr int W = 1;  // 16-byte words of eight elements
};
template <>
struct RowElem<SPC_F32> {
    using S = uint32_t;
    static constexpr int W = 2;
};

// Dropout's random numbers.  Element (row, col) of rows of c takes 16 bits of
// Philox4x32 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3",
// 2011) with seven rounds, the fewest that the paper's authors found to pass
// BigCrush (ten, the usual number, is a margin that a mask does not need),
// keyed by seed[0], on the counter (k, seed[1]), k = row ceil(c / 8) + col / 8:
// one call serves the eight columns of a group.  The element is kept iff its
// bits are at least `drop` = p 65536, to the nearest whole number; sixteen bits
// move p by at most 2^-17, and the factor 65536 / (65536 - drop) goes with the
// probability that is used, so the expectation is the value itself.
constexpr int kDropOne = 65536;

struct DropKey {
    uint32_t k0, k1, s0, s1;
};

__device__ __forceinline__ DropKey drop_key(const int64_t* seed) {
    const uint64_t k = (uint64_t)seed[0], s = (uint64_t)seed[1];
    return {(uint32_t)k, (uint32_t)(k >> 32), (uint32_t)s, (uint32_t)(s >> 32)};
}

__device__ __forceinline__ u32x4 philox7(DropKey key, uint64_t k) {
    uint32_t a = (uint32_t)k, b = (uint32_t)(k >> 32), c = key.s0, d = key.s1;
    uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        const uint64_t u = (uint64_t)0xD2511F53u * a, v = (uint64_t)0xCD9E8D57u * c;
        a = (uint32_t)(v >> 32) ^ b ^ k0;
        b = (uint32_t)v;
        c = (uint32_t)(u >> 32) ^ d ^ k1;
        d = (uint32_t)u;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{a, b, c, d};
}

// The group's columns 2 q and 2 q + 1 as the halves of word q: 1 where kept (drop
// from 1 to 65536; u >= drop as a saturating difference, both halves at once).
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x4 drop_ones(u32x4 words, uint32_t drop) {
    const u16x2 d = {(uint16_t)(drop - 1), (uint16_t)(drop - 1)};
    uint32_t one = 0x00010001u;
    asm("" : "+s"(one));  // (known, the halves would be compared one by one)
    u32x4 r;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t w = words[q];  // (a bit cast of a vector's element itself takes element 0)
        r[q] = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(
                                                __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, w), d),
                                                __builtin_bit_cast(u16x2, one)));
    }
    return r;
}
// The same as eight bits, column e at drop_bit(e).
__device__ __forceinline__ uint32_t drop_bits(u32x4 ones) {
    const uint32_t c = ones[0] | ones[1] << 1 | ones[2] << 2 | ones[3] << 3;
    return (c | c >> 12) & 0xff;
}
__device__ constexpr int drop_bit(int e) { return (e >> 1) + 4 * (e & 1); }
// Word q's two elements of 16 bits, zeros where dropped; and one of 32.
__device__ __forceinline__ uint32_t drop_pair(uint32_t w, uint32_t ones) {
    const u16x2 zero = {0, 0};
    return w & __builtin_bit_cast(uint32_t, (u16x2)(zero - __builtin_bit_cast(u16x2, ones)));
}
__device__ __forceinline__ uint32_t drop_word(uint32_t w, uint32_t bits, int bit) {
    return w & (uint32_t)((int32_t)(bits << (31 - bit)) >> 31);
}

// p as a whole number of 65536ths (p in [0, 1]), and the kept values' factor.
inline uint32_t drop_threshold(double p) { return (uint32_t)(p * kDropOne + 0.5); }
inline float drop_factor(uint32_t drop) {
    return drop < (uint32_t)kDropOne ? (float)(65536.0 / (65536.0 - drop)) : 0.0f;
}

// Two values rounded to 16 bits, to the nearest, ties to even.
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <int DT>
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
    const floatx2 v = {a, b};
    if constexpr (DT == SPC_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// Eight elements as they are stored.
template <int DT>
struct Row8 {
    static constexpr int W = RowElem<DT>::W;
    using S = typename RowElem<DT>::S;
    u32x4 w[W];

    // `left` of them (> 0) are the row's, the rest read as zeros.
    __device__ __forceinline__ void load(const S* p, int64_t left) {
        if (left >= 8) {
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = reinterpret_cast<const u32x4_rows*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 7; ++e) {
                if (e >= left) continue;
                if constexpr (DT == SPC_F32) w[e / 4][e % 4] = p[e];
                else w[0][e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
            }
        }
    }
    __device__ __forceinline__ void store(S* p, int64_t left) const {
        if (left >= 8) {
#pragma unroll
            for (int i = 0; i < W; ++i) reinterpret_cast<u32x4_rows*>(p)[i] = w[i];
        } else {
#pragma unroll
            for (int e = 0; e < 7; ++e) {
                if (e >= left) continue;
                if constexpr (DT == SPC_F32) p[e] = w[e / 4][e % 4];
                else p[e] = (uint16_t)(w[0][e / 2] >> (16 * (e & 1)));
            }
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (DT == SPC_F32) {
            return __uint_as_float(w[e / 4][e % 4]);
        } else if constexpr (DT == SPC_BF16) {
            return __uint_as_float(e & 1 ? w[0][e / 2] & 0xffff0000u : w[0][e / 2] << 16);
        } else {
            return f16_bits_to_f32((uint16_t)(w[0][e / 2] >> (16 * (e & 1))));
        }
    }
    // zeros where the group's columns are dropped
    __device__ __forceinline__ void mask(u32x4 ones) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (DT == SPC_F32) {
                w[q / 2][2 * (q & 1)] = drop_word(w[q / 2][2 * (q & 1)], ones[q], 0);
                w[q / 2][2 * (q & 1) + 1] = drop_word(w[q / 2][2 * (q & 1) + 1], ones[q], 16);
            } else {
                w[0][q] = drop_pair(w[0][q], ones[q]);
            }
        }
    }
    // rounds to the nearest, ties to even
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (DT == SPC_F32) {
                w[q / 2][2 * (q & 1)] = __float_as_uint(v[2 * q]);
                w[q / 2][2 * (q & 1) + 1] = __float_as_uint(v[2 * q + 1]);
            } else {
                w[0][q] = round_pair<DT>(v[2 * q], v[2 * q + 1]);
            }
        }
    }
};

}  // namespace spc

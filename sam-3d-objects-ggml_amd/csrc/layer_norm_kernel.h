// layer_norm_kernel.h -- the row layer norm of any width up to 8192 and its
// gradient (spc_layer_norm, spc_layer_norm_backward), one pass over the rows
// each.  With a and k the row's coefficients,
//
//   h = (x - mean) r, r = 1 / sqrt(var + eps), z = h a + k, y = z or silu(z)
//   a = gamma (1 + scale_b), k = beta (1 + scale_b) + shift_b
//
// and, for the gradient, dz = dy silu'(z), g = dz a,
//
//   dx = r (g - mean_c(g) - h mean_c(g h))
//   A_b = sum over item b's rows of dz h, B_b = sum of dz
//
// from which the parameters' gradients follow (ln_finalize_kernel): the row
// pass forms two sums a channel and item, whatever is asked for.
//
// A team of T lanes (a part of a wave, a wave, or the block's four) holds a
// row in registers, so the statistics are those of the values themselves
// (mean first, then squares of the differences) and x is read once.  A block
// takes `rows_per` consecutive rows, so the coefficients are loaded once for
// many rows and the two sums stay in registers until the chunk or the item
// ends; a team loads its next row before it works on the present one.
#pragma once

#include "common.h"

namespace spc {

constexpr int kLnThreads = 256;
constexpr int kLnMaxC = 8192;

struct LnArgs {
    const void* x;
    int64_t x_stride;
    const void* dy;
    int64_t dy_stride;
    int64_t n;
    int c;
    const void* gamma;  // p_dtype [c] or null
    const void* beta;
    int p_dtype;
    const void* scale;  // m_dtype, rows of c `m_stride` apart, or null
    const void* shift;
    int64_t m_stride;
    int m_dtype;
    const int64_t* off;  // [nb + 1] or null: one item of all rows
    int64_t nb;
    float eps;
    int silu;
    int rows_per;
    void* y;             // y, or dx (null: only the sums)
    float* stats;        // [n, 2] mean, r: written (or null), or read
    float* part;         // [chunks + items][2][c], or null
};

// U elements of 16 bytes (U = all of them), 4 or 2.
template <int DT>
struct LnElem {
    static constexpr int V = DT == SPC_F32 ? 4 : 8;  // elements in 16 bytes
    using S = uint16_t;
    __device__ static float lo(uint32_t w) {
        return DT == SPC_BF16 ? __uint_as_float(w << 16) : f16_bits_to_f32((uint16_t)w);
    }
    __device__ static float hi(uint32_t w) {
        return DT == SPC_BF16 ? __uint_as_float(w & 0xffff0000u) : f16_bits_to_f32((uint16_t)(w >> 16));
    }
    __device__ static uint32_t bits(float f) {
        return DT == SPC_BF16 ? f32_to_bf16_bits(f) : f32_to_f16_bits(f);
    }
};
template <>
struct LnElem<SPC_F32> {
    static constexpr int V = 4;
    using S = float;
};

// A row's elements as they were loaded (16 bytes a vector, NV of them).
template <int NV>
struct LnRaw {
    u32x4 v[NV];
};

// Where a team's lane holds element e of its vector k: units of U elements
// lie next to each other across the lanes, so every load and store of a team
// is one contiguous run (U = V: 16-byte words; rows whose width or address
// they do not divide: 4- or 2-byte units).
template <int T, int V, int U>
__device__ __forceinline__ int ln_channel(int lane, int k, int e) {
    return (lane + T * ((k * V + e) / U)) * U + e % U;
}

template <int DT, int T, int NV, int U>
__device__ __forceinline__ LnRaw<NV> ln_load(const void* base, int64_t at, int c, int lane, bool on) {
    constexpr int V = LnElem<DT>::V;
    LnRaw<NV> r;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        r.v[k] = u32x4{0, 0, 0, 0};
        if constexpr (U == V) {
            const int ch = ln_channel<T, V, U>(lane, k, 0);
            if (on && ch < c)
                r.v[k] = *reinterpret_cast<const u32x4*>(
                    static_cast<const typename LnElem<DT>::S*>(base) + at + ch);
        } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if constexpr (DT == SPC_F32 || U == 2) {
                    const int ch = ln_channel<T, V, U>(lane, k, w * V / 4);
                    if (on && ch < c)
                        r.v[k][w] = *reinterpret_cast<const uint32_t*>(
                            static_cast<const typename LnElem<DT>::S*>(base) + at + ch);
                } else {
                    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
                    const int c0 = ln_channel<T, V, U>(lane, k, 2 * w);
                    const int c1 = ln_channel<T, V, U>(lane, k, 2 * w + 1);
                    const uint32_t a = on && c0 < c ? p[c0] : 0u;
                    const uint32_t b = on && c1 < c ? p[c1] : 0u;
                    r.v[k][w] = a | (b << 16);
                }
            }
        }
    }
    return r;
}

template <int DT, int NV>
__device__ __forceinline__ float ln_get(const LnRaw<NV>& r, int k, int e) {
    if constexpr (DT == SPC_F32) return __uint_as_float(r.v[k][e]);
    else return e & 1 ? LnElem<DT>::hi(r.v[k][e / 2]) : LnElem<DT>::lo(r.v[k][e / 2]);
}

template <int DT, int T, int NV, int U>
__device__ __forceinline__ void ln_store(void* base, int64_t at, int c, int lane,
                                         const float (&o)[NV][LnElem<DT>::V]) {
    constexpr int V = LnElem<DT>::V;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        u32x4 q;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if constexpr (DT == SPC_F32) q[w] = __float_as_uint(o[k][w]);
            else q[w] = LnElem<DT>::bits(o[k][2 * w]) | (LnElem<DT>::bits(o[k][2 * w + 1]) << 16);
        }
        auto* p = static_cast<typename LnElem<DT>::S*>(base) + at;
        if constexpr (U == V) {
            const int ch = ln_channel<T, V, U>(lane, k, 0);
            if (ch < c) __builtin_nontemporal_store(q, reinterpret_cast<u32x4*>(p + ch));
        } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if constexpr (DT == SPC_F32 || U == 2) {
                    const int ch = ln_channel<T, V, U>(lane, k, w * V / 4);
                    if (ch < c) *reinterpret_cast<uint32_t*>(p + ch) = q[w];
                } else {
                    const int c0 = ln_channel<T, V, U>(lane, k, 2 * w);
                    const int c1 = ln_channel<T, V, U>(lane, k, 2 * w + 1);
                    if (c0 < c) p[c0] = (uint16_t)q[w];
                    if (c1 < c) p[c1] = (uint16_t)(q[w] >> 16);
                }
            }
        }
    }
}

// Element i of a parameter stored as dtype dt.
__device__ __forceinline__ float ln_param(const void* p, int dt, int64_t i) {
    if (dt == SPC_F32) return static_cast<const float*>(p)[i];
    const uint16_t b = static_cast<const uint16_t*>(p)[i];
    return dt == SPC_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// The lane's coefficients for item b.
template <int T, int NV, int V, int U>
__device__ __forceinline__ void ln_coefficients(const LnArgs& p, int64_t b, int lane,
                                                float (&a)[NV][V], float (&k0)[NV][V]) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int ch = ln_channel<T, V, U>(lane, k, e);
            float g = 1.0f, t = 0.0f;
            if (ch < p.c) {
                if (p.gamma) g = ln_param(p.gamma, p.p_dtype, ch);
                if (p.beta) t = ln_param(p.beta, p.p_dtype, ch);
                if (p.scale) {
                    const float s = 1.0f + ln_param(p.scale, p.m_dtype, b * p.m_stride + ch);
                    g *= s;
                    t = t * s + ln_param(p.shift, p.m_dtype, b * p.m_stride + ch);
                }
            }
            a[k][e] = g;
            k0[k][e] = t;
        }
}

// Sum over the T lanes of a team (T = 256: over the block's four waves too,
// through one of two LDS slots in turn, so one barrier a sum is enough: a
// thread that writes a slot again has passed the barrier behind which every
// thread read it).  Every step adds a lane's value and its partner's, so all
// lanes end with the same bits.  Lane exchanges are DPP moves and permlane
// swaps within the register file; the same steps as LDS permutes were what
// bound narrow rows.
template <int T>
__device__ __forceinline__ float wave_part_sum(float v) {
    constexpr int W = T > 64 ? 64 : T;
    auto dpp = [](float u, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(u), decltype(ctrl)::value,
                                                          0xf, 0xf, true));
    };
    if constexpr (W >= 2) v += dpp(v, std::integral_constant<int, 0xB1>{});    // lane ^ 1
    if constexpr (W >= 4) v += dpp(v, std::integral_constant<int, 0x4E>{});    // lane ^ 2
    if constexpr (W >= 8) v += dpp(v, std::integral_constant<int, 0x141>{});   // mirror in 8
    if constexpr (W >= 16) v += dpp(v, std::integral_constant<int, 0x140>{});  // mirror in 16
    if constexpr (W >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                        false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if constexpr (W >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                        false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return v;
}

struct LnBlockSum {
    float (*slot)[2][4];  // LDS [2 slots][2 values][4 waves]
    int turn = 0;
    template <int T>
    __device__ __forceinline__ float sum(float v) {
        v = wave_part_sum<T>(v);
        if constexpr (T > 64) {
            float(*s)[4] = slot[turn];
            if ((threadIdx.x & 63) == 0) s[0][threadIdx.x >> 6] = v;
            __syncthreads();
            v = (s[0][0] + s[0][1]) + (s[0][2] + s[0][3]);
            turn ^= 1;
        }
        return v;
    }
    template <int T>
    __device__ __forceinline__ void sum2(float& v, float& u) {
        v = wave_part_sum<T>(v);
        u = wave_part_sum<T>(u);
        if constexpr (T > 64) {
            float(*s)[4] = slot[turn];
            if ((threadIdx.x & 63) == 0) {
                s[0][threadIdx.x >> 6] = v;
                s[1][threadIdx.x >> 6] = u;
            }
            __syncthreads();
            v = (s[0][0] + s[0][1]) + (s[0][2] + s[0][3]);
            u = (s[1][0] + s[1][1]) + (s[1][2] + s[1][3]);
            turn ^= 1;
        }
    }
};

// sigmoid(z); F32 rows take the correctly scaled exponential, 16-bit rows the
// hardware's (its error grows as |z| 2^-24, far below half their last bit).
template <int DT>
__device__ __forceinline__ float ln_sigmoid(float z) {
    const float e = DT == SPC_F32 ? expf(-z) : __expf(-z);
    return __builtin_amdgcn_rcpf(1.0f + e);
}

// Last item i in [0, nb) with off[i] <= row (0 if there is none).
__device__ __forceinline__ int64_t ln_item(const int64_t* off, int64_t nb, int64_t row) {
    int64_t lo = 0, hi = nb;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (off[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Zeros for the rows [lo, hi), which belong to no item.
template <int DT, int T, int NV, int U>
__device__ __forceinline__ void ln_zero_rows(const LnArgs& p, int64_t lo, int64_t hi, int lane) {
    constexpr int TPB = kLnThreads / T;
    const float z[NV][LnElem<DT>::V] = {};
    for (int64_t row = lo + threadIdx.x / T; row < hi; row += TPB) {
        if (p.y) ln_store<DT, T, NV, U>(p.y, row * p.c, p.c, lane, z);
    }
}

template <int DT, int T, int NV, int U>
__global__ __launch_bounds__(kLnThreads) void ln_forward_kernel(LnArgs p) {
    constexpr int V = LnElem<DT>::V, TPB = kLnThreads / T;
    __shared__ float slots[2][2][4];
    LnBlockSum team{slots};
    const int lane = threadIdx.x % T;
    const int64_t lo = (int64_t)blockIdx.x * p.rows_per;
    const int64_t hi = min(p.n, lo + p.rows_per);
    const float inv_c = 1.0f / (float)p.c;
    int64_t item = 0, first = lo;
    if (p.off) {
        item = ln_item(p.off, p.nb, lo);
        first = min(max(p.off[0], lo), hi);
        ln_zero_rows<DT, T, NV, U>(p, lo, first, lane);
    }
    for (; first < hi && item < p.nb; ++item) {
        const int64_t last = p.off ? min(hi, p.off[item + 1]) : hi;
        if (last <= first) continue;
        float a[NV][V], k0[NV][V];
        ln_coefficients<T, NV, V, U>(p, item, lane, a, k0);
        int64_t row = first + threadIdx.x / T;
        LnRaw<NV> next = ln_load<DT, T, NV, U>(p.x, row * p.x_stride, p.c, lane, row < last);
        for (int64_t base = first; base < last; base += TPB, row += TPB) {
            const LnRaw<NV> cur = next;
            next = ln_load<DT, T, NV, U>(p.x, (row + TPB) * p.x_stride, p.c, lane, row + TPB < last);
            float v[NV][V];
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) s += v[k][e] = ln_get<DT>(cur, k, e);
            const float mean = team.template sum<T>(s) * inv_c;
            s = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    v[k][e] -= mean;
                    if (ln_channel<T, V, U>(lane, k, e) < p.c) s += v[k][e] * v[k][e];
                }
            const float r = 1.0f / sqrtf(team.template sum<T>(s) * inv_c + p.eps);
            if (row < last) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) v[k][e] = v[k][e] * r * a[k][e] + k0[k][e];
                if (p.silu) {
#pragma unroll
                    for (int k = 0; k < NV; ++k)
#pragma unroll
                        for (int e = 0; e < V; ++e) v[k][e] *= ln_sigmoid<DT>(v[k][e]);
                }
                ln_store<DT, T, NV, U>(p.y, row * p.c, p.c, lane, v);
                if (p.stats && lane == 0) {
                    p.stats[2 * row] = mean;
                    p.stats[2 * row + 1] = r;
                }
            }
        }
        first = last;
    }
    if (p.off) ln_zero_rows<DT, T, NV, U>(p, first, hi, lane);
}

// Adds a segment's sums over the block's teams and writes them to the slot of
// (chunk, item): chunk + item, since along the rows either index grows from
// one segment to the next, so the slots are distinct and at most chunks +
// items.  Lanes of one wave first, then the waves through LDS, in a fixed
// order.
template <int T, int NV, int V, int U>
__device__ __forceinline__ void ln_flush(const LnArgs& p, int64_t slot, int lane, float* lds,
                                         float (&sum)[NV][V], int which) {
    float* out = p.part + (slot * 2 + which) * p.c;
    if constexpr (T <= 64) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
#pragma unroll
                for (int o = T; o < 64; o <<= 1) sum[k][e] += __shfl_xor(sum[k][e], o);
            }
        constexpr int W = T * NV * V;  // channels a team covers
        __syncthreads();
        if ((threadIdx.x & 63) < T) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    lds[(threadIdx.x >> 6) * W + ln_channel<T, V, U>(lane, k, e)] = sum[k][e];
        }
        __syncthreads();
        for (int ch = threadIdx.x; ch < p.c; ch += kLnThreads)
            out[ch] = (lds[ch] + lds[W + ch]) + (lds[2 * W + ch] + lds[3 * W + ch]);
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int ch = ln_channel<T, V, U>(lane, k, e);
                if (ch < p.c) out[ch] = sum[k][e];
            }
    }
}

// SUMS: the parameters' sums too.
template <int DT, int T, int NV, int U, bool SUMS>
__global__ __launch_bounds__(kLnThreads) void ln_backward_kernel(LnArgs p) {
    constexpr int V = LnElem<DT>::V, TPB = kLnThreads / T;
    __shared__ float slots[2][2][4];
    __shared__ float lds[SUMS && T <= 64 ? 4 * T * NV * V : 1];
    LnBlockSum team{slots};
    const int lane = threadIdx.x % T;
    const int64_t lo = (int64_t)blockIdx.x * p.rows_per;
    const int64_t hi = min(p.n, lo + p.rows_per);
    const float inv_c = 1.0f / (float)p.c;
    int64_t item = 0, first = lo;
    if (p.off) {
        item = ln_item(p.off, p.nb, lo);
        first = min(max(p.off[0], lo), hi);
        ln_zero_rows<DT, T, NV, U>(p, lo, first, lane);
    }
    for (; first < hi && item < p.nb; ++item) {
        const int64_t last = p.off ? min(hi, p.off[item + 1]) : hi;
        if (last <= first) continue;
        float a[NV][V], k0[NV][V];
        ln_coefficients<T, NV, V, U>(p, item, lane, a, k0);
        float sa[SUMS ? NV : 1][V], sb[SUMS ? NV : 1][V];
        if constexpr (SUMS) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) sa[k][e] = sb[k][e] = 0.0f;
        }
        int64_t row = first + threadIdx.x / T;
        bool on = row < last;
        LnRaw<NV> nx = ln_load<DT, T, NV, U>(p.x, row * p.x_stride, p.c, lane, on);
        LnRaw<NV> ny = ln_load<DT, T, NV, U>(p.dy, row * p.dy_stride, p.c, lane, on);
        float nm = on ? p.stats[2 * row] : 0.0f, nr = on ? p.stats[2 * row + 1] : 0.0f;
        for (int64_t base = first; base < last; base += TPB, row += TPB) {
            const LnRaw<NV> cx = nx, cy = ny;
            const float mean = nm, r = nr;
            const bool now = on;
            on = row + TPB < last;
            nx = ln_load<DT, T, NV, U>(p.x, (row + TPB) * p.x_stride, p.c, lane, on);
            ny = ln_load<DT, T, NV, U>(p.dy, (row + TPB) * p.dy_stride, p.c, lane, on);
            nm = on ? p.stats[2 * (row + TPB)] : 0.0f;
            nr = on ? p.stats[2 * (row + TPB) + 1] : 0.0f;
            float h[NV][V], g[NV][V];
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    // lanes past the width: dy = 0 there, so no sum takes them
                    h[k][e] = (ln_get<DT>(cx, k, e) - mean) * r;
                    g[k][e] = ln_get<DT>(cy, k, e);
                }
            if (p.silu) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float z = h[k][e] * a[k][e] + k0[k][e];
                        const float sg = ln_sigmoid<DT>(z);
                        g[k][e] *= sg * (1.0f + z * (1.0f - sg));
                    }
            }
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if constexpr (SUMS) {
                        sa[k][e] += g[k][e] * h[k][e];
                        sb[k][e] += g[k][e];
                    }
                    g[k][e] *= a[k][e];
                    s1 += g[k][e];
                    s2 += g[k][e] * h[k][e];
                }
            if (p.y) {
                team.template sum2<T>(s1, s2);
                s1 *= inv_c;
                s2 *= inv_c;
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) g[k][e] = r * (g[k][e] - s1 - h[k][e] * s2);
                if (now) ln_store<DT, T, NV, U>(p.y, row * p.c, p.c, lane, g);
            }
        }
        if constexpr (SUMS) {
            ln_flush<T, NV, V, U>(p, blockIdx.x + item, lane, lds, sa, 0);
            ln_flush<T, NV, V, U>(p, blockIdx.x + item, lane, lds, sb, 1);
        }
        first = last;
    }
    if (p.off) ln_zero_rows<DT, T, NV, U>(p, first, hi, lane);
}

// Team width and vectors a lane for c channels: f(T, NV).  A wave takes up to
// 16 elements a lane, wider rows the whole block.
template <int DT, int U, typename F>
hipError_t ln_dispatch(int c, F&& f) {
    constexpr int V = LnElem<DT>::V;
    const int nvec = (c + V - 1) / V;
#define SPC_LN(T, NV) return f(std::integral_constant<int, T>{}, std::integral_constant<int, NV>{})
    if constexpr (U == V) {
        if (nvec <= 4) SPC_LN(4, 1);
        if (nvec <= 8) SPC_LN(8, 1);
    }
    if (nvec <= 16) SPC_LN(16, 1);
    if (nvec <= 32) SPC_LN(32, 1);
    if (nvec <= 64) SPC_LN(64, 1);
    if (nvec <= 128) SPC_LN(64, 2);
    if constexpr (DT == SPC_F32) {
        if (nvec <= 256) SPC_LN(64, 4);
        if (nvec <= 512) SPC_LN(256, 2);
        if (nvec <= 1024) SPC_LN(256, 4);
        SPC_LN(256, 8);
    } else {
        if (nvec <= 256) SPC_LN(256, 1);
        if (nvec <= 512) SPC_LN(256, 2);
        SPC_LN(256, 4);
    }
#undef SPC_LN
}

// Elements a load takes: 16 bytes where the width, the strides and every
// address allow, else 4 bytes, else one element.
inline int ln_unit(const LnArgs& p, int esize, bool backward) {
    auto fits = [&](int64_t bytes) {
        auto ok = [&](const void* q) { return (uintptr_t)q % bytes == 0; };
        const int64_t u = bytes / esize;
        return u >= 1 && p.c % u == 0 && p.x_stride % u == 0 && ok(p.x) && ok(p.y) &&
               (!backward || (p.dy_stride % u == 0 && ok(p.dy)));
    };
    return fits(16) ? 16 / esize : fits(4) ? 4 / esize : 1;
}

template <int DT, int U>
hipError_t ln_forward_u(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_dispatch<DT, U>(p.c, [&](auto t, auto nv) {
        ln_forward_kernel<DT, decltype(t)::value, decltype(nv)::value, U>
            <<<blocks, kLnThreads, 0, s>>>(p);
        return hipGetLastError();
    });
}

template <int DT, int U>
hipError_t ln_backward_u(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_dispatch<DT, U>(p.c, [&](auto t, auto nv) {
        constexpr int T = decltype(t)::value, NV = decltype(nv)::value;
        if (p.part) ln_backward_kernel<DT, T, NV, U, true><<<blocks, kLnThreads, 0, s>>>(p);
        else ln_backward_kernel<DT, T, NV, U, false><<<blocks, kLnThreads, 0, s>>>(p);
        return hipGetLastError();
    });
}

template <int DT>
hipError_t ln_forward(hipStream_t s, const LnArgs& p, unsigned blocks) {
    constexpr int V = LnElem<DT>::V;
    const int u = ln_unit(p, 16 / V, false);
    if (u == V) return ln_forward_u<DT, V>(s, p, blocks);
    if constexpr (DT != SPC_F32)
        if (u == 2) return ln_forward_u<DT, 2>(s, p, blocks);
    return ln_forward_u<DT, 1>(s, p, blocks);
}

template <int DT>
hipError_t ln_backward(hipStream_t s, const LnArgs& p, unsigned blocks) {
    constexpr int V = LnElem<DT>::V;
    const int u = ln_unit(p, 16 / V, true);
    if (u == V) return ln_backward_u<DT, V>(s, p, blocks);
    if constexpr (DT != SPC_F32)
        if (u == 2) return ln_backward_u<DT, 2>(s, p, blocks);
    return ln_backward_u<DT, 1>(s, p, blocks);
}

// One file a dtype (layer_norm_bf16.hip, layer_norm_f16.hip, layer_norm_f32.hip).
hipError_t ln_forward_bf16(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_forward_f16(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_forward_f32(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_backward_bf16(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_backward_f16(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_backward_f32(hipStream_t s, const LnArgs& p, unsigned blocks);

// Rows a block's four waves work on at once.
inline int ln_teams(int dtype, int c) {
    const int v = dtype == SPC_F32 ? 4 : 8;
    const int nvec = (c + v - 1) / v;
    int t = 4;
    while (t < nvec && t < 64) t <<= 1;
    const int wave_max = dtype == SPC_F32 ? 256 : 128;
    return nvec > wave_max ? 1 : kLnThreads / t;
}

}  // namespace spc

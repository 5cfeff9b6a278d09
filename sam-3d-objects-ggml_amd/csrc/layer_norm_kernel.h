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
    const void* gamma;  // p_dtype (F32 or the rows') [c] or null
    const void* beta;
    int p_dtype;
    const void* scale;  // m_dtype (F32 or the rows'), rows of c `m_stride` apart, or null
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
    // instead of `part`, where there is one chunk and one item: A and B as the
    // parameters' gradients themselves
    void* grad_a;
    void* grad_b;
    int grad_dtype;
};

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
    using S = uint32_t;
};

// Element e of a lane's vector k is channel (lane + T k) V + e: the team's
// vectors lie side by side, so its loads and stores are one contiguous run.
// Rows need only their elements' alignment (gfx950 loads 16 bytes from any
// address); a width that is no multiple of V leaves one lane of the team with
// a part of a vector, `tail` = c % V elements, which it takes in pairs (TAIL).
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(2)));

template <typename S, int V>
__device__ __forceinline__ void ln_load_tail(u32x4 (&w)[V * (int)sizeof(S) / 16], const S* q, int tail) {
#pragma unroll
    for (int e = 0; e < V; e += 4 / (int)sizeof(S)) {
        constexpr int P = 4 / (int)sizeof(S);  // elements a word
        uint32_t v = 0;
        if (e + P <= tail) v = *reinterpret_cast<const u32_any*>(q + e);
        else if (e < tail) v = *reinterpret_cast<const uint16_t*>(q + e);
        w[e / P / 4][e / P % 4] = v;
    }
}

// V elements of size S, `left` of them (> 0) inside the width.
template <typename S, int V, bool TAIL>
__device__ __forceinline__ void ln_load_vector(u32x4 (&w)[V * (int)sizeof(S) / 16], const S* q, int left,
                                               int tail) {
    if (!TAIL || left >= V) {
#pragma unroll
        for (int i = 0; i < V * (int)sizeof(S) / 16; ++i)
            w[i] = *reinterpret_cast<const u32x4_any*>(q + i * (16 / (int)sizeof(S)));
    } else {
        ln_load_tail<S, V>(w, q, tail);
    }
}

// A row's elements as they were loaded (16 bytes a vector, NV of them).
template <int NV>
struct LnRaw {
    u32x4 v[NV][1];
};

template <int DT, int T, int NV, bool TAIL>
__device__ __forceinline__ LnRaw<NV> ln_load(const void* base, int64_t at, int c, int lane, bool on) {
    constexpr int V = LnElem<DT>::V;
    using S = typename LnElem<DT>::S;
    const S* row = static_cast<const S*>(base) + at;
    LnRaw<NV> r;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int ch = (lane + T * k) * V;
        r.v[k][0] = u32x4{0, 0, 0, 0};
        if (on && ch < c) ln_load_vector<S, V, TAIL>(r.v[k], row + ch, c - ch, c % V);
    }
    return r;
}

template <int DT, int NV>
__device__ __forceinline__ float ln_get(const LnRaw<NV>& r, int k, int e) {
    if constexpr (DT == SPC_F32) return __uint_as_float(r.v[k][0][e]);
    else return e & 1 ? LnElem<DT>::hi(r.v[k][0][e / 2]) : LnElem<DT>::lo(r.v[k][0][e / 2]);
}

template <int DT, int T, int NV, bool TAIL>
__device__ __forceinline__ void ln_store(void* base, int64_t at, int c, int lane,
                                         const float (&o)[NV][LnElem<DT>::V]) {
    constexpr int V = LnElem<DT>::V, P = DT == SPC_F32 ? 1 : 2;
    using S = typename LnElem<DT>::S;
    S* row = static_cast<S*>(base) + at;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        u32x4 q;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if constexpr (DT == SPC_F32) q[w] = __float_as_uint(o[k][w]);
            else q[w] = LnElem<DT>::bits(o[k][2 * w]) | (LnElem<DT>::bits(o[k][2 * w + 1]) << 16);
        }
        const int ch = (lane + T * k) * V;
        if (TAIL ? ch + V <= c : ch < c) {
            __builtin_nontemporal_store(q, reinterpret_cast<u32x4_any*>(row + ch));
        } else if (TAIL && ch < c) {
            const int tail = c % V;
#pragma unroll
            for (int e = 0; e < V; e += P) {
                if (e + P <= tail) *reinterpret_cast<u32_any*>(row + ch + e) = q[e / P];
                else if (e < tail) row[ch + e] = (S)q[e / P];
            }
        }
    }
}

// Element i of a parameter stored as F32, or as the rows are.
__device__ __forceinline__ float ln_param(const void* p, int dt, int64_t i) {
    if (dt == SPC_F32) return static_cast<const float*>(p)[i];
    const uint16_t b = static_cast<const uint16_t*>(p)[i];
    return dt == SPC_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// A lane's share of a parameter as loaded.  Loading and converting are apart
// so that every load of a block's coefficients is under way before the first
// is waited for: converted where they were loaded, each element's load was a
// latency of its own (one row of 1,024, modulated: 7.2 us, 3.4 apart; 62,710
// rows x 128 bf16 with SiLU: 19.3 and 8.8).
template <int DT, int T, int NV, bool TAIL>
struct LnParam {
    static constexpr int V = LnElem<DT>::V;
    using S = typename LnElem<DT>::S;
    u32x4 w[NV][V / 4];  // F32: V words; as the rows: 16 bytes

    __device__ __forceinline__ void load(const void* p, bool f32, int64_t at, int c, int lane) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int ch = (lane + T * k) * V;
            if (ch < c) {
                // (unsigned: a scalar base and a 32-bit offset)
                if (DT == SPC_F32 || f32)
                    ln_load_vector<uint32_t, V, TAIL>(w[k], static_cast<const uint32_t*>(p) + at + (uint32_t)ch,
                                                      c - ch, c % V);
                else
                    ln_load_vector<S, V, TAIL>(reinterpret_cast<u32x4(&)[1]>(w[k]),
                                               static_cast<const S*>(p) + at + (uint32_t)ch, c - ch, c % V);
            }
        }
    }
    // f(k, e, value) for every element
    template <typename F>
    __device__ __forceinline__ void each(bool f32, F&& f) const {
        if (DT == SPC_F32 || f32) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) f(k, e, __uint_as_float(w[k][e / 4][e % 4]));
        } else if constexpr (DT != SPC_F32) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    f(k, e, e & 1 ? LnElem<DT>::hi(w[k][0][e / 2]) : LnElem<DT>::lo(w[k][0][e / 2]));
        }
    }
};

// The lane's coefficients for item b (past the width: finite).
template <int DT, int T, int NV, bool TAIL>
__device__ __forceinline__ void ln_coefficients(const LnArgs& p, int64_t b, int lane,
                                                float (&a)[NV][LnElem<DT>::V],
                                                float (&k0)[NV][LnElem<DT>::V]) {
    constexpr int V = LnElem<DT>::V;
    const bool pf = p.p_dtype == SPC_F32, mf = p.m_dtype == SPC_F32;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            a[k][e] = 1.0f;
            k0[k][e] = 0.0f;
        }
    {
        LnParam<DT, T, NV, TAIL> g{}, t{};
        if (p.gamma) g.load(p.gamma, pf, 0, p.c, lane);
        if (p.beta) t.load(p.beta, pf, 0, p.c, lane);
        if (p.gamma) g.each(pf, [&](int k, int e, float v) { a[k][e] = v; });
        if (p.beta) t.each(pf, [&](int k, int e, float v) { k0[k][e] = v; });
    }
    if (p.scale) {
        LnParam<DT, T, NV, TAIL> s{}, h{};
        s.load(p.scale, mf, b * p.m_stride, p.c, lane);
        h.load(p.shift, mf, b * p.m_stride, p.c, lane);
        s.each(mf, [&](int k, int e, float v) {
            a[k][e] *= 1.0f + v;
            k0[k][e] *= 1.0f + v;
        });
        h.each(mf, [&](int k, int e, float v) { k0[k][e] += v; });
    }
}

// Sum over the T lanes of a team (T > 64: over its waves too, through one of
// two LDS slots in turn, so one barrier a sum is enough: a thread that writes a
// slot again has passed the barrier behind which every thread read it).  Every
// step adds a lane's value and its partner's, so all lanes end with the same
// bits.  Lane exchanges are DPP moves and permlane swaps within the register
// file.
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

struct LnTeamSum {
    float (*slot)[2][4];  // LDS [2 slots][2 values][4 waves]
    int turn = 0;
    // the team's waves' values of one slot row
    template <int T>
    __device__ __forceinline__ float waves(const float* s) const {
        if constexpr (T == 128) {
            const int w = threadIdx.x >> 6 & 2;
            return s[w] + s[w + 1];
        } else {
            return (s[0] + s[1]) + (s[2] + s[3]);
        }
    }
    template <int T>
    __device__ __forceinline__ float sum(float v) {
        v = wave_part_sum<T>(v);
        if constexpr (T > 64) {
            if ((threadIdx.x & 63) == 0) slot[turn][0][threadIdx.x >> 6] = v;
            __syncthreads();
            v = waves<T>(slot[turn][0]);
            turn ^= 1;
        }
        return v;
    }
    template <int T>
    __device__ __forceinline__ void sum2(float& v, float& u) {
        v = wave_part_sum<T>(v);
        u = wave_part_sum<T>(u);
        if constexpr (T > 64) {
            if ((threadIdx.x & 63) == 0) {
                slot[turn][0][threadIdx.x >> 6] = v;
                slot[turn][1][threadIdx.x >> 6] = u;
            }
            __syncthreads();
            v = waves<T>(slot[turn][0]);
            u = waves<T>(slot[turn][1]);
            turn ^= 1;
        }
    }
};

// 1 / sqrt(v) by the hardware's instruction (one unit in the last place);
// it takes subnormals for zero, so tiny values are scaled by a power of 4.
__device__ __forceinline__ float ln_rsqrt(float v) {
    const bool tiny = v < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(tiny ? v * 0x1p100f : v);
    return tiny ? r * 0x1p50f : r;
}

// sigmoid(z); F32 rows take the correctly scaled exponential, 16-bit rows the
// hardware's (its error grows as |z| 2^-24, far below half their last bit).  A
// sigmoid below 2^-126 is zero (z < -87.3: |silu| below 1.1e-36).
template <int DT>
__device__ __forceinline__ float ln_sigmoid(float z) {
    const float e = DT == SPC_F32 ? expf(-z) : __expf(-z);
    return __builtin_amdgcn_rcpf(1.0f + e);
}

// The items' row offsets: up to 63 items in one load a wave, a lane each, so
// that finding a block's first item and its bounds costs one latency; more by
// a binary search.
struct LnItems {
    const int64_t* off;
    int64_t nb;
    int64_t mine = 0;
    __device__ __forceinline__ LnItems(const int64_t* o, int64_t n) : off(o), nb(n) {
        if (off && nb < 64) mine = off[min((int64_t)(threadIdx.x & 63), nb)];
    }
    __device__ __forceinline__ int64_t at(int64_t i) const {
        if (nb >= 64) return off[i];
        const int l = (int)i;
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)mine, l);
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)mine >> 32), l);
        return (int64_t)(((uint64_t)hi << 32) | lo);
    }
    // Last item i in [0, nb) with off[i] <= row (0 if there is none).
    __device__ __forceinline__ int64_t find(int64_t row) const {
        if (nb < 64) {
            const uint64_t m = __ballot((int64_t)(threadIdx.x & 63) < nb && mine <= row);
            return m ? 63 - __builtin_clzll(m) : 0;
        }
        int64_t lo = 0, hi = nb;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (off[mid] <= row) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};

// Adds the squares of the lane's values inside the width.
template <int DT, int T, int NV, bool TAIL>
__device__ __forceinline__ void ln_squares(const float (&v)[NV][LnElem<DT>::V], int c, int lane,
                                           float& s) {
    constexpr int V = LnElem<DT>::V;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int left = c - (lane + T * k) * V;
        float q = 0.0f;
        if (!TAIL) {
#pragma unroll
            for (int e = 0; e < V; ++e) q += v[k][e] * v[k][e];
            s += left > 0 ? q : 0.0f;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) s += e < left ? v[k][e] * v[k][e] : 0.0f;
        }
    }
}

// Zeros for the chunk's rows that belong to no item: [lo, first) and [end, hi)
// (of the forward pass their statistics too).
template <int DT, int T, int NV, bool TAIL>
__device__ __forceinline__ void ln_zero_rows(const LnArgs& p, int64_t lo, int64_t first, int64_t end,
                                             int64_t hi, int lane, float* stats) {
    constexpr int TPB = kLnThreads / T;
    if (lo == first && end >= hi) return;
    const float z[NV][LnElem<DT>::V] = {};
    for (int64_t row = lo + threadIdx.x / T; row < hi; row += TPB) {
        if (row >= first && row < end) continue;
        if (p.y) ln_store<DT, T, NV, TAIL>(p.y, row * p.c, p.c, lane, z);
        if (stats && lane == 0) stats[2 * row] = stats[2 * row + 1] = 0.0f;
    }
}

template <int DT, int T, int NV, bool TAIL, bool SILU>
__global__ __launch_bounds__(kLnThreads) void ln_forward_kernel(LnArgs p) {
    constexpr int V = LnElem<DT>::V, TPB = kLnThreads / T;
    __shared__ float slots[2][2][4];
    LnTeamSum team{slots};
    const int lane = threadIdx.x % T;
    const int64_t lo = (int64_t)blockIdx.x * p.rows_per;
    const int64_t hi = min(p.n, lo + p.rows_per);
    const float inv_c = 1.0f / (float)p.c;
    const LnItems items(p.off, p.nb);
    // the chunk's first rows: under way before the offsets are known
    int64_t row = lo + threadIdx.x / T;
    LnRaw<NV> next = ln_load<DT, T, NV, TAIL>(p.x, row * p.x_stride, p.c, lane, row < hi);
    int64_t item = 0, first = lo, loaded = lo;
    if (p.off) {
        item = items.find(lo);
        first = min(max(items.at(0), lo), hi);
    }
    const int64_t begin = first;
    for (; first < hi && item < p.nb; ++item) {
        const int64_t last = p.off ? min(hi, items.at(item + 1)) : hi;
        if (last <= first) continue;
        row = first + threadIdx.x / T;
        if (first != loaded)
            next = ln_load<DT, T, NV, TAIL>(p.x, row * p.x_stride, p.c, lane, row < last);
        loaded = -1;
        float a[NV][V], k0[NV][V];
        ln_coefficients<DT, T, NV, TAIL>(p, item, lane, a, k0);
        for (int64_t base = first; base < last; base += TPB, row += TPB) {
            const LnRaw<NV> cur = next;
            next = ln_load<DT, T, NV, TAIL>(p.x, (row + TPB) * p.x_stride, p.c, lane, row + TPB < last);
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
                for (int e = 0; e < V; ++e) v[k][e] -= mean;
            ln_squares<DT, T, NV, TAIL>(v, p.c, lane, s);
            const float r = ln_rsqrt(team.template sum<T>(s) * inv_c + p.eps);
            if (row < last) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) v[k][e] = v[k][e] * r * a[k][e] + k0[k][e];
                if constexpr (SILU) {
#pragma unroll
                    for (int k = 0; k < NV; ++k)
#pragma unroll
                        for (int e = 0; e < V; ++e) v[k][e] *= ln_sigmoid<DT>(v[k][e]);
                }
                ln_store<DT, T, NV, TAIL>(p.y, row * p.c, p.c, lane, v);
                if (p.stats && lane == 0) {
                    p.stats[2 * row] = mean;
                    p.stats[2 * row + 1] = r;
                }
            }
        }
        first = last;
    }
    if (p.off) ln_zero_rows<DT, T, NV, TAIL>(p, lo, begin, first, hi, lane, p.stats);
}

__device__ __forceinline__ void ln_put(void* p, int dt, int64_t i, float v) {
    if (dt == SPC_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = dt == SPC_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}

// Adds a segment's sums over the block's teams and writes them to the slot of
// (chunk, item): chunk + item, since along the rows either index grows from
// one segment to the next, so the slots are distinct and at most chunks +
// items.  Lanes of one wave first, then the waves through LDS, in a fixed
// order.
template <int T, int NV, int V>
__device__ __forceinline__ void ln_flush(const LnArgs& p, int64_t slot, int lane, float* lds,
                                         float (&sum)[NV][V], int which) {
    float* out = p.part + (slot * 2 + which) * p.c;
    void* grad = which ? p.grad_b : p.grad_a;
    auto put = [&](int ch, float v) __attribute__((always_inline)) {
        if (p.part) out[ch] = v;
        else if (grad) ln_put(grad, p.grad_dtype, ch, v);
    };
    if constexpr (T < 256) {
        constexpr int W = T * NV * V;              // channels a team covers
        constexpr int COPIES = T > 64 ? 2 : 4;     // teams left once a wave's are added
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
#pragma unroll
                for (int o = T; o < 64; o <<= 1) sum[k][e] += __shfl_xor(sum[k][e], o);
            }
        __syncthreads();
        if (T >= 64 || (threadIdx.x & 63) < T) {
            float* mine = lds + threadIdx.x / (T > 64 ? T : 64) * W;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) mine[(lane + T * k) * V + e] = sum[k][e];
        }
        __syncthreads();
        for (int ch = threadIdx.x; ch < p.c; ch += kLnThreads) {
            float v = lds[ch] + lds[W + ch];
            if constexpr (COPIES == 4) v += lds[2 * W + ch] + lds[3 * W + ch];
            put(ch, v);
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int ch = (lane + T * k) * V + e;
                if (ch < p.c) put(ch, sum[k][e]);
            }
    }
}

// SUMS: the parameters' sums too.
template <int DT, int T, int NV, bool TAIL, bool SILU, bool SUMS>
__global__ __launch_bounds__(kLnThreads) void ln_backward_kernel(LnArgs p) {
    constexpr int V = LnElem<DT>::V, TPB = kLnThreads / T;
    __shared__ float slots[2][2][4];
    __shared__ float lds[SUMS && T < 256 ? (T > 64 ? 2 : 4) * T * NV * V : 1];
    LnTeamSum team{slots};
    const int lane = threadIdx.x % T;
    const int64_t lo = (int64_t)blockIdx.x * p.rows_per;
    const int64_t hi = min(p.n, lo + p.rows_per);
    const float inv_c = 1.0f / (float)p.c;
    const LnItems items(p.off, p.nb);
    LnRaw<NV> nx, ny;
    float nm, nr;
    auto fetch = [&](int64_t r, bool in) __attribute__((always_inline)) {
        nx = ln_load<DT, T, NV, TAIL>(p.x, r * p.x_stride, p.c, lane, in);
        ny = ln_load<DT, T, NV, TAIL>(p.dy, r * p.dy_stride, p.c, lane, in);
        nm = in ? p.stats[2 * r] : 0.0f;
        nr = in ? p.stats[2 * r + 1] : 0.0f;
    };
    // the chunk's first rows: under way before the offsets are known
    int64_t row = lo + threadIdx.x / T;
    fetch(row, row < hi);
    int64_t item = 0, first = lo, loaded = lo;
    if (p.off) {
        item = items.find(lo);
        first = min(max(items.at(0), lo), hi);
    }
    const int64_t begin = first;
    for (; first < hi && item < p.nb; ++item) {
        const int64_t last = p.off ? min(hi, items.at(item + 1)) : hi;
        if (last <= first) continue;
        row = first + threadIdx.x / T;
        bool on = row < last;
        // (an item that ends inside the chunk must not sum the next one's rows)
        if (first != loaded || last < hi) fetch(row, on);
        loaded = -1;
        float a[NV][V], k0[NV][V];
        ln_coefficients<DT, T, NV, TAIL>(p, item, lane, a, k0);
        float sa[SUMS ? NV : 1][V], sb[SUMS ? NV : 1][V];
        if constexpr (SUMS) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) sa[k][e] = sb[k][e] = 0.0f;
        }
        for (int64_t base = first; base < last; base += TPB, row += TPB) {
            const LnRaw<NV> cx = nx, cy = ny;
            const float mean = nm, r = nr;
            const bool now = on;
            on = row + TPB < last;
            fetch(row + TPB, on);
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
            if constexpr (SILU) {
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
                if (now) ln_store<DT, T, NV, TAIL>(p.y, row * p.c, p.c, lane, g);
            }
        }
        if constexpr (SUMS) {
            ln_flush<T, NV, V>(p, blockIdx.x + item, lane, lds, sa, 0);
            ln_flush<T, NV, V>(p, blockIdx.x + item, lane, lds, sb, 1);
        }
        first = last;
    }
    if (p.off) ln_zero_rows<DT, T, NV, TAIL>(p, lo, begin, first, hi, lane, nullptr);
}

// Lanes of a team and vectors a lane for c channels: f(T, NV).  As many rows to
// a wave as fit, then up to 32 elements a lane (forward) before a row is shared
// by waves, which costs a barrier a sum (2,048 channels bf16, 31,355 rows: 62 us
// by four waves a row, 48 by one).  The gradient holds twice the registers a
// channel, so half the elements a lane.
template <int DT, bool BACKWARD, typename F>
hipError_t ln_dispatch(int c, F&& f) {
    constexpr int V = LnElem<DT>::V, Q = DT == SPC_F32 ? 2 : 1;
    const int nvec = (c + V - 1) / V;
#define SPC_LN(T, NV) return f(std::integral_constant<int, T>{}, std::integral_constant<int, NV>{})
    if (nvec <= 4) SPC_LN(4, 1);
    if (nvec <= 8) SPC_LN(8, 1);
    if (nvec <= 16) SPC_LN(16, 1);
    if (nvec <= 32) SPC_LN(32, 1);
    if (nvec <= 64) SPC_LN(64, 1);
    if (nvec <= 96 && DT != SPC_F32) SPC_LN(32, 3);
    if (nvec <= 128) SPC_LN(64, 2);
    if constexpr (DT == SPC_F32) {
        if (nvec <= 192) SPC_LN(64, 3);
        if (nvec <= 256) SPC_LN(64, 4);
    }
    if constexpr (!BACKWARD) {
        if (nvec <= 192 * Q) SPC_LN(64, 3 * Q);
        if (nvec <= 256 * Q) SPC_LN(64, 4 * Q);
    } else {
        if (nvec <= 256 * Q) SPC_LN(128, 2 * Q);
    }
    if (nvec <= 512 * Q) SPC_LN(256, 2 * Q);
    SPC_LN(256, 4 * Q);
#undef SPC_LN
}

// Rows a block works on at once.
inline int ln_teams(int dtype, int c, bool backward) {
    auto f = [](auto t, auto) { return (hipError_t)(kLnThreads / decltype(t)::value); };
    if (dtype == SPC_F32)
        return (int)(backward ? ln_dispatch<SPC_F32, true>(c, f) : ln_dispatch<SPC_F32, false>(c, f));
    return (int)(backward ? ln_dispatch<SPC_BF16, true>(c, f) : ln_dispatch<SPC_BF16, false>(c, f));
}

// f(TAIL, SILU) for p
template <int V, typename F>
void ln_flags(const LnArgs& p, F&& f) {
    if (p.c % V) {
        if (p.silu) f(std::true_type{}, std::true_type{});
        else f(std::true_type{}, std::false_type{});
    } else {
        if (p.silu) f(std::false_type{}, std::true_type{});
        else f(std::false_type{}, std::false_type{});
    }
}

template <int DT>
hipError_t ln_forward(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_dispatch<DT, false>(p.c, [&](auto t, auto nv) {
        constexpr int T = decltype(t)::value, NV = decltype(nv)::value;
        ln_flags<LnElem<DT>::V>(p, [&](auto tail, auto silu) {
            ln_forward_kernel<DT, T, NV, decltype(tail)::value, decltype(silu)::value>
                <<<blocks, kLnThreads, 0, s>>>(p);
        });
        return hipGetLastError();
    });
}

template <int DT>
hipError_t ln_backward(hipStream_t s, const LnArgs& p, unsigned blocks) {
    return ln_dispatch<DT, true>(p.c, [&](auto t, auto nv) {
        constexpr int T = decltype(t)::value, NV = decltype(nv)::value;
        ln_flags<LnElem<DT>::V>(p, [&](auto tail, auto silu) {
            constexpr bool TL = decltype(tail)::value, SI = decltype(silu)::value;
            if (p.part || p.grad_a || p.grad_b)
                ln_backward_kernel<DT, T, NV, TL, SI, true><<<blocks, kLnThreads, 0, s>>>(p);
            else ln_backward_kernel<DT, T, NV, TL, SI, false><<<blocks, kLnThreads, 0, s>>>(p);
        });
        return hipGetLastError();
    });
}

// One file a dtype (layer_norm_bf16.hip, layer_norm_f16.hip, layer_norm_f32.hip).
hipError_t ln_forward_bf16(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_forward_f16(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_forward_f32(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_backward_bf16(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_backward_f16(hipStream_t s, const LnArgs& p, unsigned blocks);
hipError_t ln_backward_f32(hipStream_t s, const LnArgs& p, unsigned blocks);

}  // namespace spc

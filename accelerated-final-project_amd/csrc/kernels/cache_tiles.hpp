// Building blocks of the kernels that read a key/value cache: pieces of rows
// of any alignment, and MFMA tiles of keys against query rows.
#pragma once

#include "kv_cache.hpp"
#include "split16.hpp"

namespace atn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// A row's scores lie in 4 lanes (L, L ^ 16, L ^ 32, L ^ 48): their maximum and sum.
__device__ __forceinline__ float row_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// the reference point of exponentials for a maximum m: nothing seen yet counts from 0
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// two values as bf16, rounded to nearest even
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 x = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}

// BYTES / sizeof(T) elements of a row whose `left` elements are valid
// (EXACT: all of them), zeros past those.  Rows need only element alignment.
template <typename T, int BYTES>
struct Words {
    uint32_t w[BYTES / 4];
};
template <bool EXACT, int BYTES, typename T>
__device__ __forceinline__ Words<T, BYTES> ld_words(const T* p, int left) {
    constexpr int N = BYTES / (int)sizeof(T);
    Words<T, BYTES> v;
    if (EXACT || left >= N) {
        __builtin_memcpy(&v, p, BYTES);
        return v;
    }
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) v.w[i] = 0;
    if (left > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i < left) {
                if constexpr (sizeof(T) == 4)
                    v.w[i] = __float_as_uint(p[i]);
                else
                    v.w[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
            }
        }
    }
    return v;
}

// Tiles of keys against tiles of queries, MFMA 16 x 16 with keys as rows and queries as columns:
// S^T = K Q^T leaves a lane the scores of query L % 16 for 4 consecutive keys, which are the
// operand of O^T = V^T P^T as they lie -- the product's key order only has to be the one V is
// loaded in.
//   bf16: 32 keys a block, 16x16x32.  K fragments are 16-byte pieces of rows as
//     they lie in memory.  A lane loads VL = 8 (or 4) dims of 8 keys, 16 lanes a
//     row, and pairs the keys' halves with one byte permute per operand word:
//     output tile c holds dims VL m + c, so a lane ends with whole runs of dims.
//   fp32: 16 keys a block, 16x16x4 in fp32 (exact products); V's operands are
//     the loaded words themselves.
// DP dims (head_d rounded up; EXACT: head_d itself), MT tiles of 16 query rows.
template <typename T, int DP, int MT, bool EXACT>
struct CacheTiles {
    static constexpr bool kBf = sizeof(T) == 2;
    static constexpr int KB = kBf ? 32 : 16;       // keys of a block
    static constexpr int SUB = KB / 16;            // score tiles of a block
    static constexpr int EL = 16 / (int)sizeof(T); // elements of a 16-byte piece
    static constexpr int KS = DP / (4 * EL);       // pieces of a key row per lane
    static constexpr int VD = kBf ? (DP % 128 == 0 ? 128 : 64) : 64;  // dims of a V step
    static constexpr int VS = DP / VD;             // V steps
    static constexpr int VL = VD / 16;             // dims of a lane's V piece
    static constexpr int VB = VL * (int)sizeof(T);
    static constexpr int KEYS = KB / 4;            // keys of a lane
    static constexpr int RUN = 4 * VL;             // consecutive dims of a lane per V step
    static constexpr int ROWS = 16 * MT;
    // registers: the output tile, K and V of a block, the scores and weights, addresses; with the
    // next block's K loaded ahead except where only that would not leave two waves a SIMD
    static constexpr int kRegs = DP / 4 * (MT + 1) + 20 * MT + 44;
    static constexpr int kWith = kRegs + DP / 4;
    static constexpr bool kAhead = kWith <= 250 || kRegs > 220;
    static constexpr int kOccupancy = kWith <= 124 ? 4 : kWith <= 164 ? 3 : kRegs <= 220 ? 2 : 1;
    static constexpr int LDO = DP + 4;             // row of the exchange, floats
    static constexpr int kQBytes = ROWS * DP * (int)sizeof(T);
    static constexpr int kXBytes = 2 * ROWS * LDO * 4;
    static constexpr int kLds = (kQBytes > kXBytes ? kQBytes : kXBytes) + 2 * ROWS * 16;

    using KPiece = Words<T, 16>;
    using VPiece = Words<T, VB>;

    struct Keys {
        KPiece p[SUB][KS];
    };
    struct Vals {
        VPiece p[KEYS][VS];
    };

    static __device__ __forceinline__ void load_k(Keys& k, const T* base, int64_t stride, int rows,
                                                  int D, int lane) {
        const int q = lane >> 4;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const int r = min(16 * s + (lane & 15), rows - 1);
            const T* p = base + r * stride + EL * q;
#pragma unroll
            for (int i = 0; i < KS; ++i)
                k.p[s][i] = ld_words<EXACT, 16>(p + 4 * EL * i, D - 4 * EL * i - EL * q);
        }
    }

    // key of a lane's j-th V row
    static __device__ __forceinline__ int key_of(int lane, int j) {
        return 16 * (j >> 2) + 4 * (lane >> 4) + (j & 3);
    }

    // (rows past the block's are zeros: a weight of 0 times whatever they hold must be 0)
    static __device__ __forceinline__ void load_v(Vals& v, const T* base, int64_t stride, int rows,
                                                  int D, int lane) {
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
            const int r = key_of(lane, j);
            const T* p = base + min(r, rows - 1) * stride + VL * (lane & 15);
#pragma unroll
            for (int i = 0; i < VS; ++i)
                v.p[j][i] = ld_words<EXACT, VB>(p + VD * i, D - VD * i - VL * (lane & 15));
        }
        if (rows < KB) {
#pragma unroll
            for (int j = 0; j < KEYS; ++j)
                if (key_of(lane, j) >= rows)
#pragma unroll
                    for (int i = 0; i < VS; ++i)
#pragma unroll
                        for (int w = 0; w < VB / 4; ++w) v.p[j][i].w[w] = 0;
        }
    }

    static __device__ __forceinline__ v4f dot(const KPiece& k, const KPiece& q, v4f c) {
        if constexpr (kBf) {
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k),
                                                           __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.w[e]),
                                                         __uint_as_float(q.w[e]), c, 0, 0, 0);
            return c;
        }
    }

    // bf16: O^T += V^T P^T with the weights' operands in registers
    static __device__ __forceinline__ void products(v4f (&o)[MT][VS][VL], const Vals& v,
                                                    const KPiece (&f)[MT]) {
#pragma unroll
        for (int i = 0; i < VS; ++i)
#pragma unroll
            for (int c = 0; c < VL; ++c) {
                KPiece a;
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    a.w[h] = __builtin_amdgcn_perm(v.p[2 * h + 1][i].w[c / 2],
                                                   v.p[2 * h][i].w[c / 2],
                                                   (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    o[t][i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, f[t]), o[t][i][c],
                        0, 0, 0);
            }
    }

    // O^T += V^T P^T with the weights in LDS, rows of ld elements: operands of the keys of load_v
    static __device__ __forceinline__ void accumulate_lds(v4f (&o)[MT][VS][VL], const Vals& v,
                                                          const T* p, int ld, int lane) {
        float w[MT][SUB][4];
        KPiece f[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const T* at = p + (16 * t + (lane & 15)) * ld + 4 * (lane >> 4);
            if constexpr (kBf) {
                const uint2 lo = *reinterpret_cast<const uint2*>(at);
                const uint2 hi = *reinterpret_cast<const uint2*>(at + 16);
                f[t].w[0] = lo.x, f[t].w[1] = lo.y, f[t].w[2] = hi.x, f[t].w[3] = hi.y;
            } else {
                const float4 x = *reinterpret_cast<const float4*>(at);
                w[t][0][0] = x.x, w[t][0][1] = x.y, w[t][0][2] = x.z, w[t][0][3] = x.w;
            }
        }
        if constexpr (kBf)
            products(o, v, f);
        else
            accumulate(o, v, w);
    }

    // O^T += V^T P^T for all tiles
    static __device__ __forceinline__ void accumulate(v4f (&o)[MT][VS][VL], const Vals& v,
                                                      const float (&p)[MT][SUB][4]) {
        if constexpr (kBf) {
            // the weights as bf16, half a step (2^-8 of their size) off at most: V's own
            // precision, and what lets one MFMA take both
            KPiece f[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    f[t].w[h] = pack2(p[t][h >> 1][2 * (h & 1)], p[t][h >> 1][2 * (h & 1) + 1]);
            products(o, v, f);
        } else {
#pragma unroll
            for (int i = 0; i < VS; ++i)
#pragma unroll
                for (int c = 0; c < VL; ++c)
#pragma unroll
                    for (int t = 0; t < MT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[t][i][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(v.p[e][i].w[c]), p[t][0][e], o[t][i][c], 0, 0, 0);
        }
    }
};

// Scores of 32 keys against 16 MT query rows over this wave's share of the dims (`waves` share
// them), from row pointers of each lane (at its piece of the rows).  EXACT: every step of 4
// pieces lies inside the rows.
template <typename T, int MT, bool EXACT, int WAVES>
__device__ __forceinline__ void wide_scores(v4f (&s)[MT][2], const T* const (&kp)[2],
                                            const T* const (&qp)[MT], int D, int wave, int q) {
    using N = CacheTiles<T, 64, MT, EXACT>;
    constexpr int EL = N::EL, STEP = 4 * EL, U = 4;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[t][u] = v4f{0.f, 0.f, 0.f, 0.f};
    const int per = ((D + STEP * U - 1) / (STEP * U) + WAVES - 1) / WAVES * STEP * U;
    const int d1 = min(D, (wave + 1) * per);
    for (int d = wave * per; d < d1; d += STEP * U) {
        typename N::KPiece k[U][2], f[U][MT];
#pragma unroll
        for (int e = 0; e < U; ++e) {
            const int at = d + STEP * e, left = D - at - EL * q;
#pragma unroll
            for (int u = 0; u < 2; ++u) k[e][u] = ld_words<EXACT, 16>(kp[u] + at, left);
#pragma unroll
            for (int t = 0; t < MT; ++t) f[e][t] = ld_words<EXACT, 16>(qp[t] + at, left);
        }
#pragma unroll
        for (int e = 0; e < U; ++e)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u) s[t][u] = N::dot(k[e][u], f[e][t], s[t][u]);
    }
}

}  // namespace atn

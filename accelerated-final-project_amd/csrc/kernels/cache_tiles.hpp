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

// the sum over a row of 16 lanes
__device__ __forceinline__ float row16_sum(float x) {
    x += dpp<kDppQuadXor1>(x);
    x += dpp<kDppQuadXor2>(x);
    x += dpp<kDppRowHalfMirror>(x);
    return x + dpp<kDppRowMirror>(x);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// the reference point of exponentials for a maximum m: nothing seen yet counts from 0
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// two values as bf16, rounded to nearest even
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 x = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}

// sum + the products of two pairs of bf16
__device__ __forceinline__ float dot2(uint32_t x, uint32_t y, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x),
                                           __builtin_bit_cast(bf16x2, y), sum, false);
}
// sum + both halves of a pair of bf16
__device__ __forceinline__ float add2(uint32_t w, float sum) { return dot2(w, 0x3f803f80u, sum); }

// BYTES of a row.  Rows need only element alignment (the hardware loads 16 bytes from any).
template <typename T, int BYTES>
struct Words {
    uint32_t w[BYTES / 4];
};
template <int BYTES, typename T>
__device__ __forceinline__ Words<T, BYTES> ld_words(const T* p) {
    Words<T, BYTES> v;
    __builtin_memcpy(&v, p, BYTES);
    return v;
}
// The first `left` elements, then zeros.
template <int BYTES, typename T>
__device__ __forceinline__ Words<T, BYTES> ld_some(const T* p, int left) {
    constexpr int N = BYTES / (int)sizeof(T);
    Words<T, BYTES> v;
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) v.w[i] = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i < left) {
            if constexpr (sizeof(T) == 4)
                v.w[i] = __float_as_uint(p[i]);
            else
                v.w[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
        }
    }
    return v;
}
// Zeros in the first z elements (any z).
template <int BYTES, typename T>
__device__ __forceinline__ void clear_first(Words<T, BYTES>& v, int z) {
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) {
        if constexpr (sizeof(T) == 4)
            v.w[i] = i < z ? 0u : v.w[i];
        else
            v.w[i] &= 2 * i >= z ? ~0u : 2 * i + 1 >= z ? 0xffff0000u : 0u;
    }
}

// x, as a value that the compiler knows nothing about: what follows is computed where it stands,
// not before a loop and kept in registers across it.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
// How the pieces of a row of D elements are read.  kExact: every piece lies in the row.
// kClamp (D holds a piece at least): a piece that would pass the row's end is read where the row
// ends.  In a score the elements that other pieces hold already are then cleared, in K and Q
// alike; as dims of an output they are computed twice, alike.  kElem: element by element.
constexpr int kExact = 0, kClamp = 1, kElem = 2;

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
// DP dims (more than head_d by less than 64), read as MODE says; MT tiles of 16 query rows.
template <typename T, int DP, int MT, int MODE>
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
    using KPiece = Words<T, 16>;
    using VPiece = Words<T, VB>;

    struct Keys {
        KPiece p[SUB][KS];
    };
    struct Vals {
        VPiece p[KEYS][VS];
    };

    // Rows are addressed as a uniform base and each lane's 32-bit byte offset: a block's rows lie
    // within 4 GiB.
    static __device__ __forceinline__ const T* at(const T* base, uint32_t off) {
        return reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + off);
    }

    // Piece i of a row of K or Q for the lanes of group q (`off`: of their piece 0)
    static __device__ __forceinline__ KPiece piece(const T* base, uint32_t off, int i, int q, int D) {
        const int d = 4 * EL * i + EL * q;
        if constexpr (MODE == kElem) {
            return ld_some<16>(at(base, off) + 4 * EL * i, D - d);
        } else if (MODE == kExact || 4 * EL * (i + 1) <= DP - 64) {
            return ld_words<16>(at(base, off) + 4 * EL * i);
        } else {
            const int past = max(0, opaque(d) - (D - EL));
            KPiece v = ld_words<16>(at(base, off + (4 * EL * i - past) * (int)sizeof(T)));
            clear_first(v, past);
            return v;
        }
    }

    // K of a block of `rows` rows from `base` on (the last one again in the places behind them)
    static __device__ __forceinline__ void load_k(Keys& k, const T* base, int64_t stride, int rows,
                                                  int D, int lane) {
        const uint32_t row = (uint32_t)stride * (uint32_t)sizeof(T);
        const uint32_t end = (uint32_t)(min(rows, KB) - 1) * row, mine = (lane & 15) * row;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const uint32_t off = min(mine + 16 * s * row, end) + 16 * (lane >> 4);
#pragma unroll
            for (int i = 0; i < KS; ++i) k.p[s][i] = piece(base, off, i, lane >> 4, D);
        }
    }

    // key of a lane's j-th V row
    static __device__ __forceinline__ int key_of(int lane, int j) {
        return 16 * (j >> 2) + 4 * (lane >> 4) + (j & 3);
    }
    // first dim of V's piece m (of 16) in step i, where the row ends at D
    static __device__ __forceinline__ int dim_of(int i, int m, int D) {
        const int d = VD * i + VL * m;
        return MODE == kClamp ? min(d, D - VL) : d;
    }
    // (the rows behind a block's enter with a weight of 0: whoever calls takes out what times 0 is
    // not 0)
    static __device__ __forceinline__ VPiece v_piece(const T* base, uint32_t off, int i, int D,
                                                     int lane) {
        const int d = dim_of(i, lane & 15, D);
        if constexpr (MODE == kElem) return ld_some<VB>(at(base, off) + d, D - d);
        // (dims before the base, where a row's last piece begins: the sum does not wrap)
        const int before = min(D - VL, 0);
        return ld_words<VB>(at(base + before, off + (uint32_t)((d - before) * (int)sizeof(T))));
    }
    static __device__ __forceinline__ void load_v(Vals& v, const T* base, int64_t stride, int rows,
                                                  int D, int lane) {
        const uint32_t row = (uint32_t)stride * (uint32_t)sizeof(T);
        const uint32_t end = (uint32_t)(min(rows, KB) - 1) * row, mine = key_of(lane, 0) * row;
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
            const uint32_t off = min(mine + key_of(0, j) * row, end);
#pragma unroll
            for (int i = 0; i < VS; ++i) v.p[j][i] = v_piece(base, off, i, D, lane);
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
                // (the permutes of all tiles ahead of the products would take 32 registers)
                if (c & 1) __builtin_amdgcn_sched_barrier(0);
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
        if constexpr (kBf) {
            products(o, v, f);
        } else {
            float none[MT];
            accumulate(o, v, w, none);
        }
    }

    // bf16: weights as the products' operands
    static __device__ __forceinline__ void round(KPiece (&f)[MT], const float (&p)[MT][SUB][4],
                                                 float (&used)[MT]) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                f[t].w[h] = pack2(p[t][h >> 1][2 * (h & 1)], p[t][h >> 1][2 * (h & 1) + 1]);
                used[t] = add2(f[t].w[h], used[t]);
            }
    }

    // O^T += V^T P^T for all tiles.  bf16: the weights enter as bf16 (V's own precision, and what
    // lets one MFMA take both), half a step (2^-8 of their size) off at most; `used` gathers
    // them as rounded, so that the output is their exact mean of V
    static __device__ __forceinline__ void accumulate(v4f (&o)[MT][VS][VL], const Vals& v,
                                                      const float (&p)[MT][SUB][4],
                                                      float (&used)[MT]) {
        if constexpr (kBf) {
            KPiece f[MT];
            round(f, p, used);
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

// Scores of 16 SUB keys against 16 MT query rows over wave `wave`'s share of the dims (of `waves`),
// from each lane's row pointers.  AHEAD: all loads of a step go out before its products (waves of
// several steps: left to itself the compiler keeps six in flight, and the memory idles, 100 MB
// in 37 against 27 us); else fewer registers and more waves (of one step: 18 against 15 us).
template <typename T, int MT, bool AHEAD, int SUB>
__device__ __forceinline__ void wide_scores(v4f (&s)[MT][SUB], const T* const (&kp)[SUB],
                                            const T* const (&qp)[MT], int D, int wave, int waves,
                                            int q) {
    using N = CacheTiles<T, 64, MT, kExact>;
    constexpr int EL = N::EL, STEP = 4 * EL, U = 4;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[t][u] = v4f{0.f, 0.f, 0.f, 0.f};
    const int per = ((D + STEP * U - 1) / (STEP * U) + waves - 1) / waves * STEP * U;
    const int d1 = min(D, (wave + 1) * per);
    int d = wave * per;
    for (; d + STEP * U <= d1; d += STEP * U) {
        typename N::KPiece k[U][SUB], f[U][MT];
#pragma unroll
        for (int e = 0; e < U; ++e) {
            const int at = d + STEP * e + EL * q;
#pragma unroll
            for (int u = 0; u < SUB; ++u) k[e][u] = ld_words<16>(kp[u] + at);
#pragma unroll
            for (int t = 0; t < MT; ++t) f[e][t] = ld_words<16>(qp[t] + at);
        }
        if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < U; ++e)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int u = 0; u < SUB; ++u) s[t][u] = N::dot(k[e][u], f[e][t], s[t][u]);
    }
    if (d < d1) {  // the row's end (kClamp's pieces)
#pragma unroll 1
        for (int e = 0; e < U; ++e) {
            const int want = d + STEP * e + EL * q, at = min(want, D - EL);
            typename N::KPiece x[SUB], y;
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                x[u] = ld_words<16>(kp[u] + at);
                clear_first(x[u], want - at);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                y = ld_words<16>(qp[t] + at);
                clear_first(y, want - at);
#pragma unroll
                for (int u = 0; u < SUB; ++u) s[t][u] = N::dot(x[u], y, s[t][u]);
            }
        }
    }
}

}  // namespace atn

// Attention of drafted tokens over a key/value cache: row (h, t) attends
// every cache row in use and the drafts that its mask names,
//   x_j = scale q . k_j,  m = max x,  l = sum exp(x - m),
//   out = sum exp(x - m) v / l,  lse = m + log l.
//
// The query rows of one kv head (its heads times the tokens) share the reads
// of K and V: tiles of 16 MT rows.  Scores are in units of log2 throughout.
#include <algorithm>

#include "kv_cache.hpp"
#include "split16.hpp"

namespace atn {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kStat = 3;  // floats of a row's statistics in a split
constexpr float kLn2 = 0.69314718055994531f;

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

// N = 16 / sizeof(T) elements of a row whose `left` elements are valid
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

// ---------------------------------------------------------------- head_d <= 256
// Every wave walks its own blocks of keys, alone: scores, running maximum and
// sum, and its own output tile in registers; nothing passes through LDS but Q
// and, at the end, the four waves' results.  MFMA tiles 16 x 16 with keys as
// rows and queries as columns: S^T = K Q^T leaves a lane the scores of query
// L % 16 for 4 consecutive keys, which are the operand of O^T = V^T P^T as
// they lie -- the product's key order only has to be the one V is loaded in.
//   bf16: 32 keys a block, 16x16x32.  K fragments are 16-byte pieces of rows as
//     they lie in memory.  A lane loads VL = 8 (or 4) dims of 8 keys, 16 lanes a
//     row, and pairs the keys' halves with one byte permute per operand word:
//     output tile c holds dims VL m + c, so a lane ends with whole runs of dims.
//   fp32: 16 keys a block, 16x16x4 in fp32 (exact products); V's operands are
//     the loaded words themselves.
template <typename T, int DP, int MT, bool EXACT>
struct Narrow {
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

    // O^T += V^T P^T for all tiles
    static __device__ __forceinline__ void accumulate(v4f (&o)[MT][VS][VL], const Vals& v,
                                                      const float (&p)[MT][SUB][4]) {
        if constexpr (kBf) {
            bf16x8 pf[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                Words<T, 16> w;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    // the weights as bf16, half a step (2^-9 of their size) off: V's own
                    // precision, and what lets one MFMA take both
                    const f32x2 x = {p[t][h >> 1][2 * (h & 1)], p[t][h >> 1][2 * (h & 1) + 1]};
                    w.w[h] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
                }
                pf[t] = __builtin_bit_cast(bf16x8, w);
            }
#pragma unroll
            for (int i = 0; i < VS; ++i)
#pragma unroll
                for (int c = 0; c < VL; ++c) {
                    Words<T, 16> a;
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        a.w[h] = __builtin_amdgcn_perm(v.p[2 * h + 1][i].w[c / 2],
                                                       v.p[2 * h][i].w[c / 2],
                                                       (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int t = 0; t < MT; ++t)
                        o[t][i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            __builtin_bit_cast(bf16x8, a), pf[t], o[t][i][c], 0, 0, 0);
                }
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

// Whether any lane's V holds an infinity or NaN, which are cleared.
template <typename T, typename V>
__device__ __forceinline__ bool clear_not_finite(V& v) {
    bool any = false;
    for (auto& row : v.p)
        for (auto& piece : row)
            for (auto& w : piece.w) {
                if constexpr (sizeof(T) == 4) {
                    const bool bad = (w & 0x7f800000u) == 0x7f800000u;
                    any |= bad;
                    w = bad ? 0u : w;
                } else {
                    const bool lo = (w & 0x7f80u) == 0x7f80u;
                    const bool hi = (w & 0x7f800000u) == 0x7f800000u;
                    any |= lo | hi;
                    w &= (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
                }
            }
    return __builtin_amdgcn_ballot_w64(any) != 0;
}

// What the infinities and NaNs that clear_not_finite() took out of the drafts' V add to dim d of
// token tok: every weight is above 0, so whatever it is, theirs is the value itself.
template <typename T>
__device__ __forceinline__ float not_finite_sum(const TreeArgs& a, int b, int g, int n, int tok,
                                                int d) {
    const T* v = (const T*)a.d.V + b * a.d.vs[0] + g * a.d.vs[1] + d;
    float sum = 0.f;
    for (int j = 0; j < n; ++j) {
        const float x = Elem<T>::ld(v + j * a.d.vs[2], 0);
        if (!(fabsf(x) < INFINITY) && sees(a.d, b, tok, j)) sum += x;
    }
    return sum;
}

// Keys [0, 32 n) of the cache, then the drafts in blocks of their own: where
// a split's blocks lie.
struct Blocks {
    int cache, all;    // blocks of the cache, and with the drafts'
    int first, last;   // this split's
};
template <int KB>
__device__ __forceinline__ Blocks blocks_of(const TreeArgs& a, int L, int n, int split) {
    Blocks x;
    x.cache = (L + KB - 1) / KB;
    x.all = x.cache + (a.d.K ? (n + KB - 1) / KB : 0);
    // whole turns of the workgroup's waves, so that every split but the last is full
    const int per = ((x.all + a.plan.nsplit - 1) / a.plan.nsplit + kWaves - 1) / kWaves * kWaves;
    x.first = min(split * per, x.all);
    x.last = min(x.first + per, x.all);
    return x;
}

template <typename T, int DP, int MT, bool EXACT>
__global__ __launch_bounds__(64 * kWaves, (Narrow<T, DP, MT, EXACT>::kOccupancy)) void
k_tree_narrow(TreeArgs a) {
    using N = Narrow<T, DP, MT, EXACT>;
    constexpr int KB = N::KB, SUB = N::SUB, KS = N::KS, VS = N::VS, VL = N::VL, RUN = N::RUN;
    __shared__ __align__(16) char lds[N::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    // workgroups go to the 8 XCDs in turn: the row tiles that read the same keys are 8 apart
    const int tiles = a.plan.row_tiles, nsplit = a.plan.nsplit;
    const int units = a.c.B * a.c.G * nsplit, full = units / 8 * 8 * tiles;
    int unit, tile;
    if ((int)blockIdx.x < full) {
        const int x = blockIdx.x % 8, y = blockIdx.x / 8;
        tile = y % tiles;
        unit = y / tiles * 8 + x;
    } else {
        const int y = blockIdx.x - full;
        tile = y % tiles;
        unit = units / 8 * 8 + y / tiles;
    }
    const int split = unit % nsplit, bg = unit / nsplit, g = bg % a.c.G, b = bg / a.c.G;
    const int L = rows_in_use(a.c, b), n = drafts_of(a.d, b), D = a.c.D;
    const int rep = a.d.H / a.c.G, R = rep * a.d.T;
    const Blocks blk = blocks_of<KB>(a, L, n, split);
    // (nothing for this split: the merge knows; a call of one split writes zeros)
    if (blk.first >= blk.last && nsplit > 1 && split > 0) return;

    // Q in the order of the fragments: piece (t, i) of lane L is piece i of row 16 t + L % 16
    auto* qs = reinterpret_cast<typename N::KPiece*>(lds);
    for (int e = threadIdx.x; e < MT * KS * 64; e += 64 * kWaves) {
        const int el = e & 63, i = (e >> 6) % KS, t = (e >> 6) / KS;
        const int row = tile * N::ROWS + 16 * t + (el & 15);
        typename N::KPiece z{};
        if (row < R && row % a.d.T < n) {
            const int d0 = 4 * N::EL * i + N::EL * (el >> 4);
            z = ld_words<EXACT, 16>((const T*)a.d.Q + b * a.d.qs[0] +
                                        (g * rep + row / a.d.T) * a.d.qs[1] +
                                        (row % a.d.T) * a.d.qs[2] + d0,
                                    D - d0);
        }
        qs[e] = z;
    }
    __syncthreads();

    const T* kc = (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1];
    const T* vc = (const T*)a.c.V + b * a.c.vs[0] + g * a.c.vs[1];
    const T* kd = (const T*)a.d.K + b * a.d.ks[0] + g * a.d.ks[1];
    const T* vd = (const T*)a.d.V + b * a.d.vs[0] + g * a.d.vs[1];

    v4f o[MT][VS][VL];
    float m[MT], l[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int i = 0; i < VS; ++i)
#pragma unroll
            for (int c = 0; c < VL; ++c) o[t][i][c] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    auto rows_of = [&](int i) {
        return i < blk.cache ? min(KB, L - i * KB) : min(KB, n - (i - blk.cache) * KB);
    };
    auto load_k = [&](typename N::Keys& k, int i) {
        const bool in = i < blk.cache;
        const int64_t s = in ? a.c.ks[2] : a.d.ks[2];
        N::load_k(k, (in ? kc : kd) + (int64_t)(in ? i : i - blk.cache) * KB * s, s, rows_of(i), D,
                  lane);
    };

    bool odd = false;
    typename N::Keys k;
    int i = blk.first + wave;
    if (N::kAhead && i < blk.last) load_k(k, i);
    for (; i < blk.last; i += kWaves) {
        const bool in = i < blk.cache;
        const int j0 = in ? i * KB : (i - blk.cache) * KB, rows = rows_of(i);
        if (!N::kAhead) load_k(k, i);
        typename N::Vals v;
        {
            const int64_t s = in ? a.c.vs[2] : a.d.vs[2];
            N::load_v(v, (in ? vc : vd) + (int64_t)j0 * s, s, rows, D, lane);
        }
        float p[MT][SUB][4];
        {
            v4f s[MT][SUB];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int u = 0; u < SUB; ++u) s[t][u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < KS; ++e)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const typename N::KPiece f = qs[(t * KS + e) * 64 + lane];
#pragma unroll
                    for (int u = 0; u < SUB; ++u) s[t][u] = N::dot(k.p[u][e], f, s[t][u]);
                }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[t][u][e] = s[t][u][e] * a.scale;
        }
        if (N::kAhead && i + kWaves < blk.last) load_k(k, i + kWaves);
        uint32_t see[MT];  // bit 16 u + 4 q + e: the row attends key 16 u + 4 q + e of the block
        const uint32_t valid = rows >= 32 ? ~0u : (1u << rows) - 1;
        if (!in || rows < KB) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                see[t] = valid;
                if (!in) {
                    const int row = tile * N::ROWS + 16 * t + col, tok = row % a.d.T;
                    if (a.d.mask) {
                        const uint32_t w =
                            row < R ? a.d.mask[((size_t)b * a.d.T + tok) * a.d.W + (j0 >> 5)] : 0u;
                        see[t] &= w >> (j0 & 31);
                    } else {
                        const int upto = tok - j0;  // keys 0 .. upto
                        see[t] &= upto < 0 ? 0u : upto >= 31 ? ~0u : (2u << upto) - 1;
                    }
                }
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((see[t] >> (16 * u + 4 * q + e)) & 1u)) p[t][u][e] = -INFINITY;
            }
        }
        // The running maximum moves only when a score passes it by more than 8 (weights up to
        // 2^8 lose nothing in fp32 or bf16), so the tile is rarely rescaled.
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float top = p[t][0][0];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, p[t][u][e]);
            if (__builtin_amdgcn_ballot_w64(top > m[t] + 8.f)) {
                const float m_new = fmaxf(m[t], row_max(top));
                const float alpha = exp2_(m[t] - base_of(m_new));
                m[t] = m_new;
                l[t] *= alpha;
#pragma unroll
                for (int x = 0; x < VS; ++x)
#pragma unroll
                    for (int c = 0; c < VL; ++c) o[t][x][c] *= alpha;
            }
            const float base = base_of(m[t]);
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[t][u][e] = exp2_(p[t][u][e] - base);
                    l[t] += p[t][u][e];
                }
        }
        // A draft that some rows attend and others do not: an infinity or NaN in its V belongs
        // to the first alone.  The product runs without it; not_finite_sum() adds it at the end.
        if (!in) odd |= clear_not_finite<T>(v);
        N::accumulate(o, v, p);
    }

    // the waves' tiles into wave 0: 2 and 3 hand theirs to 0 and 1, then 1 to 0
#pragma unroll
    for (int t = 0; t < MT; ++t) l[t] = row_sum(l[t]);
    float* xo = reinterpret_cast<float*>(lds);
    float4* xs = reinterpret_cast<float4*>(lds + N::kLds - 2 * N::ROWS * 16);
    for (int half = kWaves / 2; half > 0; half /= 2) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
            float* to = xo + (wave - half) * N::ROWS * N::LDO;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if (q == 0)
                    xs[(wave - half) * N::ROWS + 16 * t + col] =
                        make_float4(m[t], l[t], odd ? 1.f : 0.f, 0.f);
#pragma unroll
                for (int x = 0; x < VS; ++x)
#pragma unroll
                    for (int c = 0; c < VL; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            to[(16 * t + col) * N::LDO + N::VD * x + RUN * q + VL * e + c] =
                                o[t][x][c][e];
            }
        }
        __syncthreads();
        if (wave < half) {
            const float* from = xo + wave * N::ROWS * N::LDO;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float4 y = xs[wave * N::ROWS + 16 * t + col];
                const float m_new = fmaxf(m[t], y.x), base = base_of(m_new);
                const float fa = exp2_(m[t] - base), fb = exp2_(y.x - base);
                m[t] = m_new;
                l[t] = l[t] * fa + y.y * fb;
                odd |= y.z != 0.f;
#pragma unroll
                for (int x = 0; x < VS; ++x)
#pragma unroll
                    for (int c = 0; c < VL; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[t][x][c][e] = o[t][x][c][e] * fa +
                                            fb * from[(16 * t + col) * N::LDO + N::VD * x +
                                                      RUN * q + VL * e + c];
            }
        }
    }
    if (wave != 0) return;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = tile * N::ROWS + 16 * t + col;
        const int h = g * rep + row / a.d.T, tok = row % a.d.T;
        if (row >= R || tok >= n) continue;
        const size_t at = ((size_t)b * a.d.H + h) * a.d.T + tok;
        if (nsplit > 1) {
            float* to = a.part + (at * nsplit + split) * D;
            // behind the parts: maximum, sum and whether infinities or NaNs were left out
            float* st = a.part + (size_t)a.c.B * a.d.H * a.d.T * nsplit * D +
                        (at * nsplit + split) * kStat;
            if (q == 0) {
                st[0] = m[t];
                st[1] = l[t];
                st[2] = odd ? 1.f : 0.f;
            }
#pragma unroll
            for (int x = 0; x < VS; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < VL; ++c) {
                        const int d = N::VD * x + RUN * q + VL * e + c;
                        if (EXACT || d < D) to[d] = o[t][x][c][e];
                    }
        } else {
            T* to = (T*)a.out + b * a.os[0] + h * a.os[1] + tok * a.os[2];
            // (l == 0: nothing visible, or no score above -infinity)
            const float inv = l[t] == 0.f ? 0.f : 1.f / l[t];
            if (q == 0 && a.lse)
                a.lse[at] = l[t] == 0.f ? -INFINITY : (m[t] + log2f(l[t])) * kLn2;
#pragma unroll
            for (int x = 0; x < VS; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < VL; ++c) {
                        const int d = N::VD * x + RUN * q + VL * e + c;
                        if (EXACT || d < D) Elem<T>::st(to, d, o[t][x][c][e] * inv);
                    }
        }
    }
    if (nsplit == 1 && __builtin_amdgcn_ballot_w64(odd)) {
        __threadfence_block();  // (this wave's own stores, from other lanes)
        for (int r = 0; r < N::ROWS; ++r) {
            const int row = tile * N::ROWS + r, tok = row % a.d.T;
            if (row >= R || tok >= n) continue;
            T* to = (T*)a.out + b * a.os[0] + (g * rep + row / a.d.T) * a.os[1] + tok * a.os[2];
            for (int d = lane; d < D; d += 64) {
                const float x = not_finite_sum<T>(a, b, g, n, tok, d);
                if (x != 0.f) Elem<T>::st(to, d, Elem<T>::ld(to, d) + x);
            }
        }
    }
}

// ---------------------------------------------------------------- splits
// The splits of a row added up: one workgroup per (row, 256 dims).
template <typename T>
__global__ __launch_bounds__(256) void k_tree_merge(TreeArgs a, int kb) {
    const int D = a.c.D, chunks = (D + 255) / 256;
    const size_t at = blockIdx.x / chunks;
    const int d = (blockIdx.x % chunks) * 256 + threadIdx.x;
    const int tok = at % a.d.T, h = (at / a.d.T) % a.d.H, b = at / a.d.T / a.d.H;
    const int L = rows_in_use(a.c, b), n = drafts_of(a.d, b), nsplit = a.plan.nsplit;
    if (tok >= n) return;
    int used = 1;
    {
        const int all = (L + kb - 1) / kb + (a.d.K ? (n + kb - 1) / kb : 0);
        const int per = ((all + nsplit - 1) / nsplit + kWaves - 1) / kWaves * kWaves;
        if (all > 0) used = (all + per - 1) / per;
    }
    const float* st = a.part + (size_t)a.c.B * a.d.H * a.d.T * nsplit * D + at * nsplit * kStat;
    const float* part = a.part + at * nsplit * D;
    float M = -INFINITY, l = 0.f, acc = 0.f;
    bool odd = false;
    for (int s = 0; s < used; ++s) M = fmaxf(M, st[s * kStat]);
    const float base = base_of(M);
#pragma unroll 4
    for (int s = 0; s < used; ++s) {
        const float f = exp2_(st[s * kStat] - base);
        l += f * st[s * kStat + 1];
        odd |= st[s * kStat + 2] != 0.f;
        if (d < D) acc += f * part[(size_t)s * D + d];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (d < D) {
        float x = acc * inv;
        if (odd) x += not_finite_sum<T>(a, b, h / (a.d.H / a.c.G), n, tok, d);
        Elem<T>::st((T*)a.out + b * a.os[0] + h * a.os[1] + tok * a.os[2], d, x);
    }
    if (d == 0 && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (M + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------- head_d > 256
// One workgroup per row: keys in blocks of 256 (a wave per key, lanes over
// the dims), the running maximum and sum in fp32, the output's dims in
// registers (32 per thread at head_d 8192).
constexpr int kDimsPerThread = 32;

template <typename T>
__global__ __launch_bounds__(256) void k_tree_rows(TreeArgs a) {
    __shared__ float p[256];
    __shared__ float red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x % a.d.T, h = (blockIdx.x / a.d.T) % a.d.H;
    const int b = blockIdx.x / (a.d.T * a.d.H), g = h / (a.d.H / a.c.G);
    const int L = rows_in_use(a.c, b), n = drafts_of(a.d, b), D = a.c.D;
    if (t >= n) return;
    const T* q = (const T*)a.d.Q + b * a.d.qs[0] + h * a.d.qs[1] + t * a.d.qs[2];
    const T* kc = (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1];
    const T* vc = (const T*)a.c.V + b * a.c.vs[0] + g * a.c.vs[1];
    const T* kd = (const T*)a.d.K + b * a.d.ks[0] + g * a.d.ks[1];
    const T* vd = (const T*)a.d.V + b * a.d.vs[0] + g * a.d.vs[1];
    const int keys = L + (a.d.K ? n : 0);
    float m = -INFINITY, l = 0.f, acc[kDimsPerThread];
#pragma unroll
    for (int i = 0; i < kDimsPerThread; ++i) acc[i] = 0.f;
    for (int k0 = 0; k0 < keys; k0 += 256) {
        const int nk = min(256, keys - k0);
        for (int i = wave; i < nk; i += 4) {
            const int j = k0 + i;
            float s = -INFINITY;
            if (j < L || sees(a.d, b, t, j - L)) {
                const T* k = j < L ? kc + j * a.c.ks[2] : kd + (j - L) * a.d.ks[2];
                float x = 0.f;
                for (int d = lane; d < D; d += 64) x = fmaf(Elem<T>::ld(q, d), Elem<T>::ld(k, d), x);
                s = wave_sum(x) * a.scale;
            }
            if (lane == 0) p[i] = s;
        }
        __syncthreads();
        const float s = threadIdx.x < nk ? p[threadIdx.x] : -INFINITY;
        const float wm = wave_max(s);
        if (lane == 0) red[wave] = wm;
        __syncthreads();
        const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        // no key seen so far: nothing to scale, and no key of this block counts
        const float base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = m == -INFINITY ? 0.f : exp2f(m - base);
        const float e = exp2f(s - base);
        const float ws = wave_sum(e);
        __syncthreads();
        if (lane == 0) red[wave] = ws;
        if (threadIdx.x < nk) p[threadIdx.x] = e;
        __syncthreads();
        l = l * alpha + (red[0] + red[1]) + (red[2] + red[3]);
        m = m_new;
#pragma unroll
        for (int i = 0; i < kDimsPerThread; ++i) acc[i] *= alpha;
        for (int i = 0; i < nk; ++i) {
            const int j = k0 + i;
            if (j >= L && !sees(a.d, b, t, j - L)) continue;  // its V may be anything
            const T* v = j < L ? vc + j * a.c.vs[2] : vd + (j - L) * a.d.vs[2];
#pragma unroll
            for (int c = 0; c < kDimsPerThread; ++c) {
                const int d = threadIdx.x + 256 * c;
                if (d < D) acc[c] = fmaf(p[i], Elem<T>::ld(v, d), acc[c]);
            }
        }
        __syncthreads();
    }
    T* o = (T*)a.out + b * a.os[0] + h * a.os[1] + t * a.os[2];
    // (l == 0: nothing visible, or no score above -infinity)
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < kDimsPerThread; ++c) {
        const int d = threadIdx.x + 256 * c;
        if (d < D) Elem<T>::st(o, d, l == 0.f ? 0.f : acc[c] * inv);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[((size_t)b * a.d.H + h) * a.d.T + t] =
            l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int DP, int MT>
void go_narrow(const TreeArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)a.plan.workgroups);
    if (a.c.D == DP)
        hipLaunchKernelGGL((k_tree_narrow<T, DP, MT, true>), grid, dim3(64 * kWaves), 0, st, a);
    else
        hipLaunchKernelGGL((k_tree_narrow<T, DP, MT, false>), grid, dim3(64 * kWaves), 0, st, a);
}

template <typename T, int DP>
void go_rows(const TreeArgs& a, hipStream_t st) {
    if (a.plan.rows == 16) return go_narrow<T, DP, 1>(a, st);
    if (a.plan.rows == 32 || DP > 128 || sizeof(T) == 4) return go_narrow<T, DP, 2>(a, st);
    if constexpr (DP <= 128 && sizeof(T) == 2) go_narrow<T, DP, 4>(a, st);
}

template <typename T>
void go(const TreeArgs& a, hipStream_t st) {
    const int D = a.c.D;
    if (D > 256) {
        hipLaunchKernelGGL(k_tree_rows<T>, dim3((unsigned)a.plan.workgroups), dim3(256), 0, st, a);
        return;
    }
    if (D <= 64) go_rows<T, 64>(a, st);
    else if (D <= 128) go_rows<T, 128>(a, st);
    else if (D <= 192) go_rows<T, 192>(a, st);
    else go_rows<T, 256>(a, st);
    if (a.plan.nsplit > 1)
        hipLaunchKernelGGL(k_tree_merge<T>,
                           dim3((unsigned)((size_t)a.c.B * a.d.H * a.d.T * ((D + 255) / 256))),
                           dim3(256), 0, st, a, sizeof(T) == 2 ? 32 : 16);
}

}  // namespace

TreePlan tree_plan(int dtype, int B, int G, int H, int T, int D, int max_len, size_t scratch_cap) {
    TreePlan p{};
    if (D > 256) return TreePlan{1, 1, 1, 0, (int64_t)B * H * T};
    const int R = H / G * T;
    const int most = dtype == kDtypeBF16 && D <= 128 ? 64 : 32;
    p.rows = R <= 16 ? 16 : R <= 32 ? 32 : most;
    p.row_tiles = (R + p.rows - 1) / p.rows;
    const int kb = dtype == kDtypeBF16 ? 32 : 16;
    const int64_t units = (int64_t)B * G * p.row_tiles;
    // splits of at least two blocks a wave, and about three workgroups per CU
    const int64_t blocks = (max_len + kb - 1) / kb + (T + kb - 1) / kb;
    int64_t ns = std::min<int64_t>((768 + units - 1) / units, blocks / (2 * kWaves));
    const size_t per = (size_t)B * H * T * (D + kStat) * sizeof(float);
    if (ns > (int64_t)(scratch_cap / per)) ns = (int64_t)(scratch_cap / per);
    p.nsplit = (int)std::max<int64_t>(1, ns);
    p.scratch = p.nsplit > 1 ? per * p.nsplit : 0;
    p.workgroups = units * p.nsplit;
    return p;
}

hipError_t launch_tree_attention(int dtype, const TreeArgs& a, hipStream_t st) {
    if (dtype == kDtypeF32)
        go<float>(a, st);
    else
        go<uint16_t>(a, st);
    return hipGetLastError();
}

}  // namespace atn

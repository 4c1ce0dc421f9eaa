// Attention of drafted tokens over a key/value cache: row (h, t) attends
// every cache row in use and the drafts that its mask names,
//   x_j = scale q . k_j,  m = max x,  l = sum exp(x - m),
//   out = sum exp(x - m) v / l,  lse = m + log l.
//
// The query rows of one kv head (its heads times the tokens) share the reads
// of K and V: tiles of 16 MT rows.  Scores are in units of log2 throughout.
#include <algorithm>

#include "cache_tiles.hpp"

namespace atn {

namespace {

constexpr int kWaves = 4;
constexpr int kTreeNarrow = 256;  // head_d up to which a wave holds a row tile's output
constexpr float kLn2 = 0.69314718055994531f;

// ---------------------------------------------------------------- head_d <= 256
// Every wave walks its own blocks of keys, alone: scores, running maximum and
// sum, and its own output tile in registers (cache_tiles.hpp); nothing passes through LDS
// but Q and, at the end, the four waves' results.
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

// A row's results in a split: maximum and sum, then, behind all of these, the dims.
__device__ __forceinline__ float2* stats_of(const TreeArgs& a) {
    return reinterpret_cast<float2*>(a.part);
}
__device__ __forceinline__ float* parts_of(const TreeArgs& a) {
    return a.part + 2 * (size_t)a.plan.heads * (a.d.H / a.c.G) * a.d.T * a.plan.nsplit;
}

// not_finite_sum() added to dims [d0, d1) of a row where its result lies (a wave's work, after
// the wave has written it): the output, or the split's part.
template <typename T>
__device__ void add_not_finite(const TreeArgs& a, int bg, int row, int split, int n, int d0, int d1,
                               int lane) {
    const int g = bg % a.c.G, b = bg / a.c.G, rep = a.d.H / a.c.G;
    const int tok = row % a.d.T;
    if (row >= rep * a.d.T || tok >= n) return;
    T* out = (T*)a.out + b * a.os[0] + (g * rep + row / a.d.T) * a.os[1] + tok * a.os[2];
    float* part =
        parts_of(a) + (((size_t)(bg - a.bg0) * rep * a.d.T + row) * a.plan.nsplit + split) * a.c.D;
    for (int d = d0 + lane; d < d1; d += 64) {
        const float x = not_finite_sum<T>(a, b, g, n, tok, d);
        if (x == 0.f) continue;
        if (a.plan.nsplit > 1)
            part[d] += x;
        else
            Elem<T>::st(out, d, Elem<T>::ld(out, d) + x);
    }
}

// Blocks of a split: whole turns of a workgroup's waves, so that every split but the last is full.
__device__ __forceinline__ int split_blocks(int all, int nsplit) {
    return ((all + nsplit - 1) / nsplit + kWaves - 1) / kWaves * kWaves;
}

// The cache's keys in blocks, then the drafts in blocks of their own: where
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
    const int per = split_blocks(x.all, a.plan.nsplit);
    x.first = min(split * per, x.all);
    x.last = min(x.first + per, x.all);
    return x;
}

// Workgroup -> (unit of keys, tile of it): workgroups go to the 8 XCDs in turn, so the tiles
// that read the same keys are 8 apart and share an L2.
__device__ __forceinline__ void tile_of(int id, int units, int tiles, int* unit, int* tile) {
    const int full = units / 8 * 8 * tiles, whole = id < full;
    const int x = whole ? id % 8 : 0, y = whole ? id / 8 : id - full;
    *tile = y % tiles;
    *unit = whole ? y / tiles * 8 + x : units / 8 * 8 + y / tiles;
}

template <typename T, int DP, int MT, bool EXACT>
__global__ __launch_bounds__(64 * kWaves, (CacheTiles<T, DP, MT, EXACT>::kOccupancy)) void
k_tree_narrow(TreeArgs a) {
    using N = CacheTiles<T, DP, MT, EXACT>;
    constexpr int KB = N::KB, SUB = N::SUB, KS = N::KS, VS = N::VS, VL = N::VL, RUN = N::RUN;
    __shared__ __align__(16) char lds[N::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    const int tiles = a.plan.row_tiles, nsplit = a.plan.nsplit;
    int unit, tile;
    tile_of(blockIdx.x, a.bgs * nsplit, tiles, &unit, &tile);
    const int split = unit % nsplit, bg = a.bg0 + unit / nsplit, g = bg % a.c.G, b = bg / a.c.G;
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
        const size_t at = (size_t)(bg - a.bg0) * R + row;
        if (nsplit > 1) {
            float* to = parts_of(a) + (at * nsplit + split) * D;
            if (q == 0) stats_of(a)[at * nsplit + split] = make_float2(m[t], l[t]);
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
                a.lse[((size_t)b * a.d.H + h) * a.d.T + tok] = l[t] == 0.f ? -INFINITY : (m[t] + log2f(l[t])) * kLn2;
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
    if (__builtin_amdgcn_ballot_w64(odd)) {
        __threadfence_block();  // (this wave's own stores, from other lanes)
        for (int r = 0; r < N::ROWS; ++r)
            add_not_finite<T>(a, bg, tile * N::ROWS + r, split, n, 0, D, lane);
    }
}

// ---------------------------------------------------------------- head_d > 256
// No output tile fits a wave's registers, so two kernels with the scores between them:
// k_tree_scores writes x (rows of R floats, small beside K and V's rows of head_d), each
// workgroup's 8 waves sharing a tile's dims and adding up through LDS; k_tree_values is the
// softmax over them and the product with V, each wave 16 VL dims of the output.
// Keys lie in blocks of 32: the cache's, then the drafts'.
constexpr int kBlock = 32;
constexpr int kScoreWaves = 8;
constexpr int kValueKeys = 128;  // keys between barriers of k_tree_values

template <typename T, int MT, bool EXACT>
__global__ __launch_bounds__(64 * kScoreWaves) void k_tree_scores(TreeArgs a) {
    using N = CacheTiles<T, 64, MT, EXACT>;
    constexpr int EL = N::EL, SUB = kBlock / 16;
    __shared__ v4f red[kScoreWaves][MT * SUB * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    const int tiles = a.plan.row_tiles, most = a.plan.ld_scores / kBlock;
    int unit, tile;
    tile_of(blockIdx.x, a.bgs * most, tiles, &unit, &tile);
    const int i = unit % most, bgl = unit / most, bg = a.bg0 + bgl, g = bg % a.c.G, b = bg / a.c.G;
    const int L = rows_in_use(a.c, b), n = drafts_of(a.d, b), D = a.c.D;
    const int cache = (L + kBlock - 1) / kBlock;
    const int all = cache + (a.d.K ? (n + kBlock - 1) / kBlock : 0);
    if (i >= all) return;
    const bool in = i < cache;
    const int j0 = (in ? i : i - cache) * kBlock, rows = min(kBlock, (in ? L : n) - j0);
    const int rep = a.d.H / a.c.G, R = rep * a.d.T;
    const T* kp[SUB];
    const T* qp[MT];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
        const int64_t r = j0 + min(16 * u + col, rows - 1);
        kp[u] = (in ? (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1] + r * a.c.ks[2]
                    : (const T*)a.d.K + b * a.d.ks[0] + g * a.d.ks[1] + r * a.d.ks[2]) +
                EL * q;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {  // (rows past R: the last one's scores, which nobody reads)
        const int row = min((tile * MT + t) * 16 + col, R - 1);
        qp[t] = (const T*)a.d.Q + b * a.d.qs[0] + (g * rep + row / a.d.T) * a.d.qs[1] +
                (row % a.d.T) * a.d.qs[2] + EL * q;
    }
    v4f s[MT][SUB];
    wide_scores<T, MT, EXACT, kScoreWaves>(s, kp, qp, D, wave, q);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < SUB; ++u) red[wave][(t * SUB + u) * 64 + lane] = s[t][u];
    __syncthreads();
    // one thread per row and 4 keys
    if (threadIdx.x >= MT * SUB * 64) return;
    const int u = (threadIdx.x >> 6) % SUB, t = (threadIdx.x >> 6) / SUB;
    v4f x = red[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kScoreWaves; ++w) x += red[w][threadIdx.x];
    const int row = (tile * MT + t) * 16 + col, tok = row % a.d.T, k0 = 16 * u + 4 * q;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool on = k0 + e < rows && row < R && (in || sees(a.d, b, tok, j0 + k0 + e));
        y[e] = on ? x[e] * a.scale : -INFINITY;
    }
    float* to = a.scores + ((size_t)bgl * tiles * N::ROWS + row) * a.plan.ld_scores + i * kBlock + k0;
    *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
}

template <typename T, int MT, bool EXACT>
__global__ __launch_bounds__(64 * kWaves) void k_tree_values(TreeArgs a) {
    constexpr bool kBf = sizeof(T) == 2;
    // (a wave's dims: one V step of 128 in bf16, 64 in fp32)
    using N = CacheTiles<T, kBf ? 128 : 64, MT, EXACT>;
    constexpr int VL = N::VL, WD = N::VD, ROWS = N::ROWS, PK = N::KB;
    constexpr int LDP = kValueKeys + 16 / (int)sizeof(T);
    __shared__ __align__(16) T pl[2][ROWS * LDP];
    __shared__ float alpha[2][ROWS];
    __shared__ float2 fin[ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    const int D = a.c.D, groups = (D + WD * kWaves - 1) / (WD * kWaves);
    const int tiles = a.plan.row_tiles, nsplit = a.plan.nsplit;
    int unit, tile;
    tile_of(blockIdx.x, a.bgs * nsplit * groups, tiles, &unit, &tile);
    const int split = unit / groups % nsplit, bgl = unit / groups / nsplit, bg = a.bg0 + bgl;
    const int d0 = (unit % groups * kWaves + wave) * WD;
    const int g = bg % a.c.G, b = bg / a.c.G;
    const int L = rows_in_use(a.c, b), n = drafts_of(a.d, b);
    const int rep = a.d.H / a.c.G, R = rep * a.d.T;
    const int cache = (L + kBlock - 1) / kBlock;
    const int all = cache + (a.d.K ? (n + kBlock - 1) / kBlock : 0);
    const int per = split_blocks(all, nsplit);
    const int first = min(split * per, all), last = min(first + per, all);
    if (first >= last && split > 0) return;
    const T* vc = (const T*)a.c.V + b * a.c.vs[0] + g * a.c.vs[1] + d0;
    const T* vd = (const T*)a.d.V + b * a.d.vs[0] + g * a.d.vs[1] + d0;
    const float* sc = a.scores + ((size_t)bgl * tiles + tile) * ROWS * a.plan.ld_scores;

    // softmax: 16 threads a row, 8 keys each, one pass per 16 rows
    const int sr = threadIdx.x >> 4, sk = (threadIdx.x & 15) * 8;
    float m[MT], l[MT];
    v4f o[MT][1][VL];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int c = 0; c < VL; ++c) o[t][0][c] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    bool odd = false;
    int buf = 0;
    for (int i0 = first; i0 < last; i0 += kValueKeys / kBlock, buf ^= 1) {
        const int k1 = (last - i0) * kBlock;  // scores of this step
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float x[8];
            const float* from = sc + (size_t)(16 * t + sr) * a.plan.ld_scores + i0 * kBlock + sk;
            if (sk < k1) {
                const float4 u = *reinterpret_cast<const float4*>(from);
                const float4 w = *reinterpret_cast<const float4*>(from + 4);
                x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
                x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = -INFINITY;
            }
            float top = x[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
            top = fmaxf(top, dpp<kDppQuadXor1>(top));
            top = fmaxf(top, dpp<kDppQuadXor2>(top));
            top = fmaxf(top, dpp<kDppRowHalfMirror>(top));
            top = fmaxf(top, dpp<kDppRowMirror>(top));
            const float m_new = fmaxf(m[t], top), base = base_of(m_new);
            const float f = exp2_(m[t] - base);
            m[t] = m_new;
            l[t] *= f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = exp2_(x[e] - base);
                l[t] += x[e];
            }
            if ((threadIdx.x & 15) == 0) alpha[buf][16 * t + sr] = f;
            T* to = pl[buf] + (16 * t + sr) * LDP + sk;
            if constexpr (kBf) {
                // (weights as bf16: see CacheTiles::accumulate)
                uint4 w;
                w.x = pack2(x[0], x[1]), w.y = pack2(x[2], x[3]);
                w.z = pack2(x[4], x[5]), w.w = pack2(x[6], x[7]);
                *reinterpret_cast<uint4*>(to) = w;
            } else {
                *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
            }
        }
        // (two buffers: a wave past this barrier writes the other one, and comes to write this
        // one only after the next barrier, when every wave has read it)
        __syncthreads();
        if (d0 >= D) continue;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float f = alpha[buf][16 * t + col];
            if (__builtin_amdgcn_ballot_w64(f != 1.f)) {
#pragma unroll
                for (int c = 0; c < VL; ++c) o[t][0][c] *= f;
            }
        }
        for (int k = 0; k < kValueKeys && k < k1; k += PK) {
            const int i = i0 + k / kBlock, sub = k % kBlock;
            const bool in = i < cache;
            const int j0 = (in ? i : i - cache) * kBlock + sub;
            const int rows = min(PK, (in ? L : n) - j0);
            if (rows <= 0) continue;  // (fp32: the second half of a last block)
            typename N::Vals v;
            const int64_t s = in ? a.c.vs[2] : a.d.vs[2];
            N::load_v(v, (in ? vc : vd) + j0 * s, s, rows, D - d0, lane);
            if (!in) odd |= clear_not_finite<T>(v);
            N::accumulate_lds(o, v, pl[buf] + k, LDP, lane);
        }
    }
    // sums of the rows, for the waves that hold their outputs
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        float x = l[t];
        x += dpp<kDppQuadXor1>(x);
        x += dpp<kDppQuadXor2>(x);
        x += dpp<kDppRowHalfMirror>(x);
        x += dpp<kDppRowMirror>(x);
        if ((threadIdx.x & 15) == 0) fin[16 * t + sr] = make_float2(m[t], x);
    }
    __syncthreads();
    if (d0 >= D) return;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = tile * ROWS + 16 * t + col, tok = row % a.d.T, h = g * rep + row / a.d.T;
        if (row >= R || tok >= n) continue;
        const float2 z = fin[16 * t + col];
        const size_t at = (size_t)bgl * R + row;
        const bool teller = q == 0 && d0 == 0;
        if (nsplit > 1) {
            float* to = parts_of(a) + (at * nsplit + split) * D + d0;
            if (teller) stats_of(a)[at * nsplit + split] = z;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < VL; ++c) {
                    const int d = N::RUN * q + VL * e + c;
                    if (EXACT || d0 + d < D) to[d] = o[t][0][c][e];
                }
        } else {
            T* to = (T*)a.out + b * a.os[0] + h * a.os[1] + tok * a.os[2] + d0;
            const float inv = z.y == 0.f ? 0.f : 1.f / z.y;
            if (teller && a.lse)
                a.lse[((size_t)b * a.d.H + h) * a.d.T + tok] =
                    z.y == 0.f ? -INFINITY : (z.x + log2f(z.y)) * kLn2;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < VL; ++c) {
                    const int d = N::RUN * q + VL * e + c;
                    if (EXACT || d0 + d < D) Elem<T>::st(to, d, o[t][0][c][e] * inv);
                }
        }
    }
    if (odd) {
        __threadfence_block();
        for (int r = 0; r < ROWS; ++r)
            add_not_finite<T>(a, bg, tile * ROWS + r, split, n, d0, min(D, d0 + WD), lane);
    }
}

// ---------------------------------------------------------------- splits
// The splits of a row added up: one workgroup per (row, 256 dims).
template <typename T>
__global__ __launch_bounds__(256) void k_tree_merge(TreeArgs a, int kb) {
    const int D = a.c.D, chunks = (D + 255) / 256, rep = a.d.H / a.c.G, R = rep * a.d.T;
    const size_t at = blockIdx.x / chunks;
    const int d = (blockIdx.x % chunks) * 256 + threadIdx.x;
    const int row = at % R, bg = a.bg0 + (int)(at / R), g = bg % a.c.G, b = bg / a.c.G;
    const int tok = row % a.d.T, h = g * rep + row / a.d.T;
    const int L = rows_in_use(a.c, b), n = drafts_of(a.d, b), nsplit = a.plan.nsplit;
    if (tok >= n) return;
    const int all = (L + kb - 1) / kb + (a.d.K ? (n + kb - 1) / kb : 0);
    const int per = split_blocks(all, nsplit), used = all > 0 ? (all + per - 1) / per : 1;
    const float2* st = stats_of(a) + at * nsplit;
    const float* part = parts_of(a) + at * nsplit * D;
    float M = -INFINITY, l = 0.f, acc = 0.f;
    for (int s = 0; s < used; ++s) M = fmaxf(M, st[s].x);
    const float base = base_of(M);
#pragma unroll 4
    for (int s = 0; s < used; ++s) {
        const float f = exp2_(st[s].x - base);
        l += f * st[s].y;
        if (d < D) {
            const float x = part[(size_t)s * D + d];
            // (infinity times a weight too small for fp32 stays infinity)
            acc += f == 0.f && !(fabsf(x) < INFINITY) ? x : f * x;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (d < D) Elem<T>::st((T*)a.out + b * a.os[0] + h * a.os[1] + tok * a.os[2], d, acc * inv);
    if (d == 0 && a.lse)
        a.lse[((size_t)b * a.d.H + h) * a.d.T + tok] =
            l == 0.f ? -INFINITY : (M + log2f(l)) * kLn2;
}

template <typename T, int DP, int MT>
void go_narrow(const TreeArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.bgs * a.plan.row_tiles * a.plan.nsplit));
    if (a.c.D == DP)
        hipLaunchKernelGGL((k_tree_narrow<T, DP, MT, true>), grid, dim3(64 * kWaves), 0, st, a);
    else
        hipLaunchKernelGGL((k_tree_narrow<T, DP, MT, false>), grid, dim3(64 * kWaves), 0, st, a);
}

template <typename T, int DP>
void go_rows(const TreeArgs& a, hipStream_t st) {
    if (a.plan.rows == 16) return go_narrow<T, DP, 1>(a, st);
    if (a.plan.rows == 32) return go_narrow<T, DP, 2>(a, st);
    if constexpr (DP <= 128 && sizeof(T) == 2) go_narrow<T, DP, 4>(a, st);
}

template <typename T>
constexpr int kWideDims = (sizeof(T) == 2 ? 128 : 64) * kWaves;  // dims of a value workgroup

template <typename T, int MT, bool EXACT>
void go_wide(const TreeArgs& a, hipStream_t st) {
    const int tiles = a.bgs * a.plan.row_tiles;
    hipLaunchKernelGGL((k_tree_scores<T, MT, EXACT>),
                       dim3((unsigned)(tiles * (a.plan.ld_scores / kBlock))),
                       dim3(64 * kScoreWaves), 0, st, a);
    const int groups = (a.c.D + kWideDims<T> - 1) / kWideDims<T>;
    hipLaunchKernelGGL((k_tree_values<T, MT, EXACT>), dim3((unsigned)(tiles * a.plan.nsplit * groups)),
                       dim3(64 * kWaves), 0, st, a);
}

template <typename T, int MT>
void go_wide(const TreeArgs& a, hipStream_t st) {
    // (exact: a wave's steps over the dims all lie inside the row)
    if (a.c.D % 128 == 0) return go_wide<T, MT, true>(a, st);
    go_wide<T, MT, false>(a, st);
}

template <typename T>
void go(const TreeArgs& a, hipStream_t st) {
    const int D = a.c.D;
    if (D > kTreeNarrow) {
        if (a.plan.rows == 16) go_wide<T, 1>(a, st);
        else if (a.plan.rows == 32) go_wide<T, 2>(a, st);
        else go_wide<T, 4>(a, st);
    } else if (D <= 64) {
        go_rows<T, 64>(a, st);
    } else if (D <= 128) {
        go_rows<T, 128>(a, st);
    } else if (D <= 192) {
        go_rows<T, 192>(a, st);
    } else {
        go_rows<T, 256>(a, st);
    }
    if (a.plan.nsplit > 1) {
        const int kb = D > kTreeNarrow || sizeof(T) == 2 ? 32 : 16;
        hipLaunchKernelGGL(
            k_tree_merge<T>,
            dim3((unsigned)((size_t)a.bgs * (a.d.H / a.c.G) * a.d.T * ((D + 255) / 256))), dim3(256),
            0, st, a, kb);
    }
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

}  // namespace

TreePlan tree_plan(int dtype, int B, int G, int H, int T, int D, int max_len, bool draft_keys,
                   size_t scratch_cap) {
    TreePlan p{};
    const bool bf = dtype == kDtypeBF16, wide = D > kTreeNarrow;
    const int R = H / G * T;
    const int most = wide || (bf && D <= 128) ? 64 : 32;
    p.rows = R <= 16 ? 16 : R <= 32 ? 32 : most;
    p.row_tiles = ceil_div(R, p.rows);
    const int kb = wide || bf ? 32 : 16;
    const int64_t blocks = ceil_div(max_len, kb) + (draft_keys ? ceil_div(T, kb) : 0);
    // workgroups of a pair without splits
    const int groups = wide ? ceil_div(D, (bf ? 128 : 64) * kWaves) : 1;
    const int64_t units = (int64_t)B * G * p.row_tiles * groups;
    // splits of at least two blocks a wave (wide: two steps), and about three workgroups per CU
    int64_t ns = std::max<int64_t>(1, std::min<int64_t>((768 + units - 1) / units,
                                                        blocks / (2 * kWaves)));
    p.ld_scores = wide ? (int)std::max<int64_t>(blocks, 1) * kBlock : 0;
    const size_t sc = wide ? (size_t)p.row_tiles * p.rows * p.ld_scores : 0;  // floats of a pair
    const size_t part = (size_t)R * (D + 2);                                   // ... and split
    const size_t room = scratch_cap / sizeof(float);
    // fewer splits where the scratch does not hold them, then fewer pairs at a time
    auto need = [&](int64_t heads, int64_t n) { return heads * (sc + (n > 1 ? n * part : 0)); };
    const int64_t pairs = (int64_t)B * G;
    while (ns > 1 && need(pairs, ns) > room) --ns;
    p.nsplit = (int)ns;
    p.heads = (int)pairs;
    if (need(pairs, ns) > room) p.heads = (int)std::max<size_t>(1, room / std::max<size_t>(sc, 1));
    p.scores = sc * p.heads;
    p.scratch = need(p.heads, ns) * sizeof(float);
    const int64_t most_groups = wide ? std::max<int64_t>(groups * ns, p.ld_scores / kBlock) : ns;
    p.workgroups = std::max((int64_t)p.heads * p.row_tiles * most_groups,
                            (int64_t)p.heads * R * ceil_div(D, 256));
    return p;
}

hipError_t launch_tree_attention(int dtype, TreeArgs a, hipStream_t st) {
    const int pairs = a.c.B * a.c.G;
    for (a.bg0 = 0; a.bg0 < pairs; a.bg0 += a.plan.heads) {
        a.bgs = std::min(a.plan.heads, pairs - a.bg0);
        if (dtype == kDtypeF32)
            go<float>(a, st);
        else
            go<uint16_t>(a, st);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace atn

// Attention of drafted tokens over a key/value cache: row (h, t) attends
// every cache row in use and the drafts that its mask names,
//   x_j = scale q . k_j,  m = max x,  l = sum exp(x - m),
//   out = sum exp(x - m) v / l,  lse = m + log l.
//
// The query rows of one kv head (its heads times the tokens) share the reads
// of K and V: tiles of 16 MT rows.  Scores are in units of log2 throughout.
//
// The lengths are on the device, so the host only fixes how many workgroups there
// are.  The blocks of keys of all (sequence, kv head) pairs lie in one line; each
// workgroup takes an equal range of it, which may end one pair and begin the next.
// A pair inside one range is written at once; the parts of one that ranges cut
// lie in the scratch until k_tree_merge has added them up.
#include <algorithm>
#include <cfloat>

#include "cache_tiles.hpp"

namespace atn {

namespace {

constexpr int kTreeNarrow = 256;  // head_d up to which a wave holds a row tile's output
constexpr float kLn2 = 0.69314718055994531f;

// ---------------------------------------------------------------- the line of blocks
// Blocks of sequence b for each of its kv heads: the cache's, then the drafts'.  At least
// one, so that some workgroup writes the outputs of tokens that attend nothing.
__device__ __forceinline__ int blocks_of(const TreeArgs& a, int b, int kb) {
    const int L = rows_in_use(a.c, b), n = drafts_of(a.d, b);
    return max(1, (L + kb - 1) / kb + (a.d.K ? (n + kb - 1) / kb : 0));
}

// A pair takes as many places of the line as it has blocks, and kPad before them: beginning and
// ending a pair costs a workgroup about as much time as so many blocks, so ranges of many short
// pairs have fewer blocks (8 sequences of 1000 to 8176 rows of 128 bf16 dims: 46.2 us with 16, 47.4
// with 8).  Few pairs of few blocks, as wide heads have them, are left with ranges of padding
// alone: 5 of 25 for 4 pairs of 33 blocks.
constexpr int kPad = 16;

// The line: its length, and the places of a range (whole turns of `turn`, a power of two).  A wave's work, as
// are the others here; results are uniform.  n, upto: of sequence b0 + lane where the pass has
// at most 64, its pairs' places and the sum of all sequences' up to it.
struct Line {
    int total, per;
    int n, upto;
};
__device__ __forceinline__ Line line_of(const TreeArgs& a, int kb, int turn, int lane) {
    Line x;
    x.n = lane < a.bs ? blocks_of(a, a.b0 + lane, kb) + kPad : 0;
    x.upto = wave_scan(x.n * a.gs);
    x.total = __builtin_amdgcn_readlane(x.upto, 63);
#pragma unroll 1
    for (int i0 = 64; i0 < a.bs; i0 += 64) {
        const int n = i0 + lane < a.bs ? blocks_of(a, a.b0 + i0 + lane, kb) + kPad : 0;
        x.total += __builtin_amdgcn_readlane(wave_scan(n * a.gs), 63);
    }
    const unsigned ranges = a.plan.ranges;
    const int per = (x.total + ranges - 1) / ranges;
    x.per = max((per + turn - 1) & -turn, 2 * turn);
    return x;
}

// The sequence at place `at` of the line.
struct Place {
    int b, n, start;  // sequence, places of each of its pairs, place of the first
};
__device__ __forceinline__ Place place_at(const TreeArgs& a, const Line& line, int at, int kb,
                                          int lane) {
    int n = line.n, upto = line.upto;
#pragma unroll 1
    for (int i0 = 0;; i0 += 64) {
        const uint64_t done = __builtin_amdgcn_ballot_w64(upto <= at);
        if (done != ~0ull || i0 + 64 >= a.bs) {
            const int l = min(__builtin_popcountll(done), min(63, a.bs - 1 - i0));
            Place p;
            p.b = a.b0 + i0 + l;
            p.n = __builtin_amdgcn_readlane(n, l);
            p.start = __builtin_amdgcn_readlane(upto, l) - p.n * a.gs;
            return p;
        }
        const int before = __builtin_amdgcn_readlane(upto, 63), b = i0 + 64 + lane;
        n = b < a.bs ? blocks_of(a, a.b0 + b, kb) + kPad : 0;
        upto = before + wave_scan(n * a.gs);
    }
}
// Place of sequence b's first pair.
__device__ __forceinline__ int start_of(const TreeArgs& a, const Line& line, int b, int kb, int lane) {
    const int i = b - a.b0;
    if (i < 64)
        return __builtin_amdgcn_readlane(line.upto, i) - __builtin_amdgcn_readlane(line.n, i) * a.gs;
    int before = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < i; i0 += 64) {
        const int n = i0 + lane < i ? blocks_of(a, a.b0 + i0 + lane, kb) + kPad : 0;
        before += __builtin_amdgcn_readlane(wave_scan(n * a.gs), 63);
    }
    return before;
}

// One pair's blocks [first, last) of a range (none where the range ends before them), and where
// they go: `part` < 0: the output, else the range's part of that number.
struct Span {
    int b, g, first, last, part;
};
// The span of range r that begins at `at` (*next: the place after it).
__device__ __forceinline__ Span span_at(const TreeArgs& a, const Line& line, int r, int at, int end,
                                        int kb, int lane, int* next) {
    const Place p = place_at(a, line, at, kb, lane);
    Span s;
    const int off = at - p.start, pair = (unsigned)off / (unsigned)p.n, in = off - pair * p.n;
    const int out = min(p.n, in + end - at);
    s.b = p.b;
    s.g = a.g0 + pair;
    s.first = max(0, in - kPad);
    s.last = out - kPad;
    s.part = s.first == 0 && out == p.n ? -1 : 2 * r + (s.first == 0 ? 1 : 0);
    *next = at + out - in;
    return s;
}
// The whole of pair r, where ranges are pairs.
__device__ __forceinline__ Span span_whole(const TreeArgs& a, int r, int kb) {
    Span s;
    const int seq = (unsigned)r / (unsigned)a.gs;
    s.b = a.b0 + seq;
    s.g = a.g0 + r - seq * a.gs;
    s.first = 0;
    s.last = of_wave(blocks_of(a, s.b, kb));
    s.part = -1;
    return s;
}

// Parts: statistics of the rows (maximum, sum of the weights, their sum as they entered the
// product with V), then, behind all of them, the rows' dims.
__device__ __forceinline__ size_t part_row(const TreeArgs& a, int part, int row) {
    return (size_t)part * a.plan.row_tiles * a.plan.rows + row;
}
__device__ __forceinline__ float4* part_stats(const TreeArgs& a) {
    return reinterpret_cast<float4*>(a.part);
}
__device__ __forceinline__ float* part_dims(const TreeArgs& a) {
    return a.part + 4 * part_row(a, 2 * a.plan.ranges, 0);
}

// Workgroup -> (range, tile): workgroups go to the 8 XCDs in turn, so the tiles that read the
// same keys are 8 apart and share an L2.
__device__ __forceinline__ void tile_of(int id, int ranges, int tiles, int* range, int* tile) {
    if (tiles == 1) {
        *tile = 0;
        *range = id;
        return;
    }
    const int full = ranges / 8 * 8 * tiles, whole = id < full;
    const int x = whole ? id % 8 : 0, y = whole ? id / 8 : id - full;
    *tile = y % tiles;
    *range = whole ? y / tiles * 8 + x : ranges / 8 * 8 + y / tiles;
}

// The first `left` of 4 consecutive elements stored, any alignment.
__device__ __forceinline__ void store4(float* to, const float (&x)[4], int left) {
    if (left >= 4) {
        __builtin_memcpy(to, x, 16);
    } else {
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (c < left) to[c] = x[c];
    }
}
__device__ __forceinline__ void store4(uint16_t* to, const float (&x)[4], int left) {
    const uint32_t w[2] = {pack2(x[0], x[1]), pack2(x[2], x[3])};
    if (left >= 4) {
        __builtin_memcpy(to, w, 8);
    } else {
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (c < left) to[c] = (uint16_t)(w[c / 2] >> (16 * (c & 1)));
    }
}

// ---------------------------------------------------------------- infinities and NaNs
// An infinity or NaN in V belongs to the rows that attend its key, whatever their weights, and to
// no others.  Weights of 0 would spread and lose them: 0 times infinity is NaN.
//   A block that is not whole cache rows alone -- the cache's last rows, the drafts -- has such
// weights for places behind its rows and drafts that a row does not attend: the product runs on
// V without them (clear_not_finite).
//   Whole blocks are attended by every row, but a weight, or a factor that rescales a tile to a
// new maximum, may have vanished: the result is NaN then.
// Where V was cleared or a result is NaN, the values themselves are summed again and written
// over the results that they belong to (put_not_finite).
// Whether any lane's V holds an infinity or NaN, which are cleared.  (What finds them is short: a
// sum of products with 0, which is NaN then.)
template <typename T, typename V>
__device__ __forceinline__ bool clear_not_finite(V& v) {
    float sum = 0.f;
    for (auto& row : v.p)
        for (auto& piece : row)
            for (auto& w : piece.w)
                sum = sizeof(T) == 4 ? fmaf(__uint_as_float(w), 0.f, sum) : dot2(w, 0u, sum);
    if (!__builtin_amdgcn_ballot_w64(sum != sum)) return false;
    for (auto& row : v.p)
        for (auto& piece : row)
            for (auto& w : piece.w) {
                const bool hi = (w & 0x7f800000u) == 0x7f800000u;
                if constexpr (sizeof(T) == 4) {
                    w = hi ? 0u : w;
                } else {
                    const bool lo = (w & 0x7f80u) == 0x7f80u;
                    w &= (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
                }
            }
    return true;
}

// The infinities and NaNs of every step-th of the rows [from, to) of a column of V, summed.
template <typename T>
__device__ __forceinline__ float not_finite_rows(const T* v, int64_t stride, int from, int to,
                                                 int step) {
    float sum = 0.f;
#pragma unroll 4
    for (int r = from; r < to; r += step) {
        const float x = Elem<T>::ld(v + r * stride, 0);
        sum += fabsf(x) < INFINITY ? 0.f : x;
    }
    return sum;
}

// Those of a span's V written to dims [d0, d1) of a row's result, the output or a part (a wave's
// work, after the results are written).  whole: of dim d, those of the whole blocks, which every
// row attends; the cache's rows from `tail` on and the drafts come to it (all of them: the ranges
// that a pair is cut into may add them more than once, which changes no such sum).  z: the row's
// maximum and sums.
template <typename T, typename F>
__device__ __forceinline__ void put_row(const TreeArgs& a, const Span& s, int row, float4 z, int tail,
                                        int L, int n, int d0, int d1, int lane, F whole) {
    const int rep = a.d.rep, h = head_of(a.d, row), tok = row - h * a.d.T;
    if (row >= rep * a.d.T || tok >= n) return;
    // (a NaN score: no number in any dim; no score above -infinity: zeros, which is known here
    // where no range cut the pair)
    if (z.y != z.y || (s.part < 0 && z.z == 0.f)) return;
    T* out = (T*)a.out + s.b * a.os[0] + (s.g * rep + h) * a.os[1] + tok * a.os[2];
    const T* vc = (const T*)a.c.V + s.b * a.c.vs[0] + s.g * a.c.vs[1];
    const T* vd = (const T*)a.d.V + s.b * a.d.vs[0] + s.g * a.d.vs[1];
    for (int d = d0 + lane; d < d1; d += 64) {
        float sum = whole(d) + not_finite_rows(vc + d, a.c.vs[2], tail, L, 1);
        for (int j = 0; a.d.K && j < n; ++j) {
            const float x = Elem<T>::ld(vd + j * a.d.vs[2], d);
            if (!(fabsf(x) < INFINITY) && sees(a.d, s.b, tok, j)) sum += x;
        }
        if (fabsf(sum) < INFINITY) continue;
        if (s.part >= 0)
            part_dims(a)[part_row(a, s.part, row) * a.c.D + d] = sum;
        else
            Elem<T>::st(out, d, sum);
    }
}

// ... of a workgroup's tile of ROWS rows of at most 256 dims.  sums: WAVES * 256 floats of LDS.
template <typename T, int ROWS, int WAVES, int KB>
__device__ void put_not_finite(const TreeArgs& a, const Span& s, int tile, const float4* fin,
                               float* sums, int L, int n, int wave, int lane) {
    const int D = a.c.D, whole = L / KB;
    const T* v = (const T*)a.c.V + s.b * a.c.vs[0] + s.g * a.c.vs[1];
    for (int d = lane; d < D; d += 64)
        sums[wave * 256 + d] = not_finite_rows(v + d, a.c.vs[2], s.first * KB + wave,
                                               min(s.last, whole) * KB, WAVES);
    __syncthreads();
    auto of_blocks = [&](int d) {
        float sum = 0.f;
        for (int w = 0; w < WAVES; ++w) sum += sums[w * 256 + d];
        return sum;
    };
    for (int r = wave; r < ROWS; r += WAVES)
        put_row<T>(a, s, tile * ROWS + r, fin[r], whole * KB, L, n, 0, D, lane, of_blocks);
}

// ---------------------------------------------------------------- steps of a block
// Scores of what a row does not attend become -infinity, in a block that is not whole cache rows:
// its `rows` rows from j0 on of the cache (in), or of the drafts.
template <int MT, int SUB>
__device__ __forceinline__ void hide(const TreeArgs& a, float (&p)[MT][SUB][4], int t, int b, int row,
                                     bool in, int j0, int rows, int q) {
    uint32_t see = rows >= 32 ? ~0u : (1u << rows) - 1;  // bit j: the row attends key j
    if (!in) {
        const int tok = row - head_of(a.d, row) * a.d.T;
        if (a.d.mask) {
            see &= a.d.mask[((size_t)b * a.d.T + tok) * a.d.W + (j0 >> 5)] >> (j0 & 31);
        } else {
            const int upto = tok - j0;  // keys 0 .. upto
            see &= upto < 0 ? 0u : upto >= 31 ? ~0u : (2u << upto) - 1;
        }
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!((see >> (16 * u + 4 * q + e)) & 1u)) p[t][u][e] = -INFINITY;
}

// Scores into weights.  The running maximum moves only when a score passes it by more than 8
// (weights up to 2^8 lose nothing in fp32 or bf16), so the tile is rarely rescaled.
template <int MT, int SUB, int VS, int VL>
__device__ __forceinline__ void weights(float (&p)[MT][SUB][4], v4f (&o)[MT][VS][VL], float (&m)[MT],
                                        float (&l)[MT], float (&used)[MT], float scale) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        float top = p[t][0][0];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, p[t][u][e]);
        if (__builtin_amdgcn_ballot_w64(top * scale > m[t] + 8.f)) {
            const float m_new = fmaxf(m[t], row_max(top) * scale);
            const float f = exp2_(m[t] - base_of(m_new));
            m[t] = m_new;
            l[t] *= f;
            used[t] *= f;
#pragma unroll
            for (int x = 0; x < VS; ++x)
#pragma unroll
                for (int c = 0; c < VL; ++c) o[t][x][c] *= f;
        }
        const float base = base_of(m[t]);
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[t][u][e] = exp2_(fmaf(p[t][u][e], scale, -base));
                l[t] += p[t][u][e];
            }
    }
}

// The results of `parts` waves a row, scaled alike, in LDS (rows of LDO floats), summed and
// written: to the output, or the span's part.  fin: the rows' maxima and sums.  Returns whether
// a result of this thread is NaN where the row's scores are not.
template <typename T, int DP, int ROWS, int PARTS, int LDO, int VL, int MODE, int THREADS>
__device__ __forceinline__ bool write_rows(const TreeArgs& a, const Span& sp, int tile, int n,
                                           const float* xo, const float4* fin) {
    const int D = MODE == kExact ? DP : a.c.D, rep = a.d.rep, R = rep * a.d.T;
    bool nan = false;
    // (opaque: or what this computes is hoisted out of the loop over spans, into registers; not
    // unrolled: twice the code, fetched once a launch, takes longer than the loop)
#pragma unroll 1
    for (int e = opaque(threadIdx.x); e < ROWS * (DP / 4); e += THREADS) {
        const int r = e / (DP / 4), d = e % (DP / 4) * 4, row = tile * ROWS + r;
        const int h = head_of(a.d, row), tok = row - h * a.d.T;
        const float4 z = fin[r];
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < PARTS; ++w) {
            const float* from = xo + (w * ROWS + r) * LDO;
            if constexpr (MODE == kClamp) {
                // (a piece that the row's end cut holds the row's last dims)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int piece = (d + c) / VL * VL;
                    x[c] += from[min(d + c + max(0, piece - (D - VL)), DP - 1)];
                }
            } else {
                const float4 y = *reinterpret_cast<const float4*>(from + d);
                x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
            }
        }
        if (row >= R || tok >= n || d >= D) continue;
        nan |= (z.y == z.y) &
               (__builtin_isunordered(x[0], x[1]) | __builtin_isunordered(x[2], x[3]));
        if (sp.part >= 0) {
            const size_t to = part_row(a, sp.part, row);
            if (d == 0) part_stats(a)[to] = z;
            store4(part_dims(a) + to * D + d, x, MODE == kExact ? 4 : D - d);
        } else {
            // (0: nothing visible, or no score above -infinity)
            const float inv = 1.f / z.z;
            if (d == 0 && a.lse)
                a.lse[((size_t)sp.b * a.d.H + sp.g * rep + h) * a.d.T + tok] =
                    z.y == 0.f ? -INFINITY : (z.x + log2f(z.y)) * kLn2;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = z.z == 0.f ? 0.f : x[c] * inv;
            store4((T*)a.out + sp.b * a.os[0] + (sp.g * rep + h) * a.os[1] + tok * a.os[2] + d, x,
                   MODE == kExact ? 4 : D - d);
        }
    }
    return nan;
}

// ---------------------------------------------------------------- head_d <= 256
// Every wave walks its own blocks of keys, alone: scores, running maximum and
// sum, and its own output tile in registers (cache_tiles.hpp); nothing passes through LDS
// but Q and, at the end, the waves' results.  A launch starts with a cold instruction
// cache, so what runs once is kept short: one loop for whole and other blocks, results added up
// in a loop (one token over 300 rows: 9.5 us with 20.6 KB of code, 9.0 with 13.8, 7.1 with 9.2).
//   One token, 8 heads of 128 bf16 dims over 300 rows (8 waves, whole pairs): 7.1 us, most of it
//     the code's fetch and the chain length -> K -> V -> results.
//   64 query rows, 8 kv heads, 8 sequences of 1000 to 8176 rows of 128 bf16 dims: 46 us, 3.3 TB/s
//     of K and V (and 8 us of merge).  One token of 32 heads over 131000 rows, where the lengths
//     are alike and the products few, reads 4.9 TB/s.
//   fp32, 21 query rows, 80 dims, 3 sequences of 777 to 1991 rows: 15 us, latency.
template <typename T, int DP, int MT, int MODE, int WAVES>
struct Narrow : CacheTiles<T, DP, MT, MODE> {
    using N = CacheTiles<T, DP, MT, MODE>;
    // registers: the output tile, K and V of a block, the scores and weights, addresses; with the
    // next block's K loaded ahead except where only that would not leave two waves a SIMD
    static constexpr int kRegs = DP / 4 * (MT + 1) + 20 * MT + 44;
    static constexpr int kWith = kRegs + DP / 4;
    static constexpr bool kAhead = kWith <= 250 || kRegs > 220;
    static constexpr int kPerSimd = kWith <= 124 ? 4 : kWith <= 164 ? 3 : kRegs <= 220 ? 2 : 1;
    static constexpr int kMinWaves = WAVES == 8 ? 2 : kPerSimd;
    static constexpr int LDO = DP + 4;  // row of the waves' results, floats
    static constexpr int kQBytes = N::ROWS * DP * (int)sizeof(T);
    static constexpr int kXBytes = WAVES * N::ROWS * LDO * 4;
    static constexpr int kOut = kQBytes > kXBytes ? kQBytes : kXBytes;
    static constexpr int kLds = kOut + (WAVES + 1) * N::ROWS * 16;
    static constexpr int kQ = (MT * N::KS * 64 + 64 * WAVES - 1) / (64 * WAVES);  // pieces a thread
    static_assert(kLds <= 160 * 1024, "LDS");
    static_assert(kXBytes >= WAVES * 256 * 4, "put_not_finite's sums");
};

template <typename T, int DP, int MT, int MODE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (Narrow<T, DP, MT, MODE, WAVES>::kMinWaves)) void
k_tree_narrow(TreeArgs a) {
    using N = Narrow<T, DP, MT, MODE, WAVES>;
    constexpr int KB = N::KB, SUB = N::SUB, KS = N::KS, VS = N::VS, VL = N::VL;
    __shared__ __align__(16) char lds[N::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    int range, tile;
    tile_of(blockIdx.x, a.plan.ranges, a.plan.row_tiles, &range, &tile);
    const int D = MODE == kExact ? DP : a.c.D, rep = a.d.rep, R = rep * a.d.T;
    const float scale = fabsf(a.scale);

    // (8 waves are for pairs that one workgroup takes whole: see tree_plan)
    const bool split = WAVES != 8 && a.plan.split;
    int at = 0, end = 1;
    Line line{};
    if (split) {
        line = line_of(a, KB, a.plan.turn, lane);
        at = range * line.per;
        end = min(line.total, at + line.per);
    }
    while (at < end) {
        Span sp;
        if (split) {
            sp = span_at(a, line, range, at, end, KB, lane, &at);
            if (sp.last <= sp.first) continue;
        } else {
            sp = span_whole(a, range, KB);
            at = end;
        }
        const int b = sp.b, g = sp.g;

        const int L = of_wave(rows_in_use(a.c, b)), n = of_wave(drafts_of(a.d, b));
        const int cache = (L + KB - 1) / KB;  // its blocks; the drafts' follow
        const int whole = L / KB;
        const T* kc = (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1];
        const T* vc = (const T*)a.c.V + b * a.c.vs[0] + g * a.c.vs[1];
        const T* kd = (const T*)a.d.K + b * a.d.ks[0] + g * a.d.ks[1];
        const T* vd = (const T*)a.d.V + b * a.d.vs[0] + g * a.d.vs[1];
        // (a pair without keys has one block of none)
        const int last = L > 0 || (a.d.K && n > 0) ? sp.last : 0;
        auto load_k = [&](typename N::Keys& to, int i) {
            const bool in = i < cache;
            const int j0 = (in ? i : i - cache) * KB;
            const int64_t s = in ? a.c.ks[2] : a.d.ks[2];
            N::load_k(to, (in ? kc : kd) + j0 * s, s, (in ? L : n) - j0, D, lane);
        };
        auto load_v = [&](typename N::Vals& to, int i) {
            const bool in = i < cache;
            const int j0 = (in ? i : i - cache) * KB;
            const int64_t s = in ? a.c.vs[2] : a.d.vs[2];
            N::load_v(to, (in ? vc : vd) + j0 * s, s, (in ? L : n) - j0, D, lane);
        };

        // Q in the order of the fragments: piece (t, i) of lane L is piece i of row 16 t + L % 16.
        // (Rows of no token hold the last token's: nobody reads their results.)
        auto* qs = reinterpret_cast<typename N::KPiece*>(lds);
        typename N::Keys k;
        typename N::Vals v;
        int i = sp.first + wave;
        {
            typename N::KPiece z[N::kQ];
            const T* qb = (const T*)a.d.Q + b * a.d.qs[0] + g * rep * a.d.qs[1];
#pragma unroll
            for (int x = 0; x < N::kQ; ++x) {
                const int e = x * WAVES + wave, i = e % KS, t = min(e / KS, MT - 1);
                const int row = min(tile * N::ROWS + 16 * t + col, R - 1), h = head_of(a.d, row);
                z[x] = N::piece(qb + h * a.d.qs[1] + (row - h * a.d.T) * a.d.qs[2], 16 * q, i, q, D);
            }
            // (the first block's K and V right behind, before anything waits for Q)
            if (i < last) {
                load_k(k, i);
                load_v(v, i);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (a.scale < 0.f) {
#pragma unroll
                for (int x = 0; x < N::kQ; ++x)
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        z[x].w[w] ^= sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
            }
            __syncthreads();  // (the last span's results are out of LDS)
#pragma unroll
            for (int x = 0; x < N::kQ; ++x)
                if (x * WAVES + wave < MT * KS) qs[(x * WAVES + wave) * 64 + lane] = z[x];
        }
        __syncthreads();


        v4f o[MT][VS][VL];
        float m[MT], l[MT], used[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            m[t] = -INFINITY;
            l[t] = used[t] = 0.f;
#pragma unroll
            for (int i = 0; i < VS; ++i)
#pragma unroll
                for (int c = 0; c < VL; ++c) o[t][i][c] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        bool odd = false;
        for (; i < last; i += WAVES) {
            const bool in = i < cache;
            const int j0 = (in ? i : i - cache) * KB;
            __builtin_amdgcn_sched_barrier(0);
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
                        for (int e = 0; e < 4; ++e) p[t][u][e] = s[t][u][e];
            }
            if (N::kAhead && i + WAVES < last) load_k(k, i + WAVES);
            __builtin_amdgcn_sched_barrier(0);
            if (i >= whole) {
                odd |= clear_not_finite<T>(v);
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    hide<MT, SUB>(a, p, t, b, tile * N::ROWS + 16 * t + col, in, j0,
                                  (in ? L : n) - j0, q);
            }
            weights<MT, SUB, VS, VL>(p, o, m, l, used, scale);
            N::accumulate(o, v, p, used);
            __builtin_amdgcn_sched_barrier(0);
            if (i + WAVES < last) {
                if (!N::kAhead) load_k(k, i + WAVES);
                load_v(v, i + WAVES);
            }
        }

        // The waves' results added up: each scales its own to the maximum of all and leaves it in
        // LDS, where every thread sums a few dims over the waves and writes them.
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            l[t] = row_sum(l[t]);
            used[t] = sizeof(T) == 2 ? row_sum(used[t]) : l[t];
        }
        float* xo = reinterpret_cast<float*>(lds);
        float4* xs = reinterpret_cast<float4*>(lds + N::kOut);
        if (q == 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
                xs[wave * N::ROWS + 16 * t + col] = make_float4(m[t], l[t], used[t], odd ? 1.f : 0.f);
        }
        __syncthreads();  // (and Q is no longer read)
        float4* fin = xs + WAVES * N::ROWS;  // of each row: maximum, sums, whether anything is odd
        odd = false;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float top = m[t];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) top = fmaxf(top, xs[w * N::ROWS + 16 * t + col].x);
            const float base = base_of(top), f = exp2_(m[t] - base);
            if (wave == t % WAVES) {
                float4 z = make_float4(top, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float4 y = xs[w * N::ROWS + 16 * t + col];
                    const float e = exp2_(y.x - base);
                    z.y += y.y * e;
                    z.z += y.z * e;
                    odd |= y.w != 0.f;
                }
                if (q == 0) fin[16 * t + col] = z;
            }
            float* to = xo + (wave * N::ROWS + 16 * t + col) * N::LDO + N::RUN * q;
#pragma unroll
            for (int x = 0; x < VS; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < VL; c += 4)
                        *reinterpret_cast<float4*>(to + N::VD * x + VL * e + c) =
                            make_float4(o[t][x][c][e] * f, o[t][x][c + 1][e] * f,
                                        o[t][x][c + 2][e] * f, o[t][x][c + 3][e] * f);
        }
        __syncthreads();
        odd |= write_rows<T, DP, N::ROWS, WAVES, N::LDO, VL, MODE, 64 * WAVES>(a, sp, tile, n, xo,
                                                                               fin);
        // (behind the barrier, which waits for the workgroup's stores and reads of xo)
        if (__syncthreads_or(odd))
            put_not_finite<T, N::ROWS, WAVES, KB>(a, sp, tile, fin, xo, L, n, wave, lane);
    }
}

// ---------------------------------------------------------------- many query rows
// bf16, 65 to 128 dims, more than 64 query rows of a kv head.  K and V now serve several waves'
// rows, and products and softmax weigh as much as the reads: 8 waves a workgroup, each with 32
// rows in registers (two waves a SIMD, one's softmax beside the other's products), RG of them
// over different rows and KG = 8 / RG over different blocks.  A stage of NB blocks comes
// through LDS while the stage before is worked on: K in the order of its fragments, as
// k_tree_narrow's lanes load them for themselves; V in rows, from which gfx950's transposing read
// takes the operands of V^T (pairing them by permutes, as k_tree_narrow does, took 40 % of the
// time here, once for every wave).  256 query rows, 8 kv heads, 4 sequences of 32000 to 32704 rows
// of 128 dims: 192 to 205 us with the merge, 610 to 650 TFLOP/s; a library product of two matrices
// reaches 1240.  Without the exponentials 15 us less, without the loads 40.  33 to 64 rows in this form (2 by 4
// waves): 50.5 us against k_tree_narrow's 46.
template <int RG, int MODE>
struct Shared : CacheTiles<uint16_t, 128, 2, MODE> {
    using N = CacheTiles<uint16_t, 128, 2, MODE>;
    static constexpr int KG = 8 / RG, ROWS_WG = 32 * RG;
    static constexpr int SB = 2;                // blocks of a wave in a stage
    static constexpr int NB = KG * SB;          // ... of the stage
    static_assert(N::SUB * N::KS == 8 && N::KEYS == 8 && N::VS == 1,
                  "a K piece and 4 V rows of each block a wave");
    // a row of V: 32 bytes more than its 256, so that the 8 rows of half a wave's transposing
    // read lie in different banks
    static constexpr int LDV = 128 + 16;
    static constexpr int kKBytes = 8 * 1024, kBytes = kKBytes + 32 * LDV * 2;  // of a block
    static constexpr int LDO = 128 + 4;
    static constexpr int kStage = NB * kBytes;
    static constexpr int kXBytes = KG * ROWS_WG * LDO * 4;
    static constexpr int kOut = 2 * kStage > kXBytes ? 2 * kStage : kXBytes;
    static constexpr int kLds = kOut + (KG + 1) * ROWS_WG * 16;
    static_assert(kLds <= 160 * 1024, "LDS");
    static_assert(kXBytes >= 8 * 256 * 4, "put_not_finite's sums");
};

template <int RG, int MODE>
__global__ __launch_bounds__(512, 2) void k_tree_shared(TreeArgs a) {
    using N = Shared<RG, MODE>;
    using T = uint16_t;
    constexpr int MT = 2, KB = N::KB, SUB = N::SUB, KS = N::KS, VL = N::VL, KG = N::KG, NB = N::NB;
    constexpr int DP = 128;
    struct VT {
        typename N::KPiece p[1][VL];
    };
    __shared__ __align__(16) char lds[N::kLds];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15, rg = wave % RG, kg = wave / RG;
    int range, tile;
    tile_of(blockIdx.x, a.plan.ranges, a.plan.row_tiles, &range, &tile);
    const int D = MODE == kExact ? DP : a.c.D, rep = a.d.rep, R = rep * a.d.T;
    const float scale = fabsf(a.scale);

    int at = 0, end = 1;
    Line line{};
    if (a.plan.split) {
        line = line_of(a, KB, a.plan.turn, lane);
        at = range * line.per;
        end = min(line.total, at + line.per);
    }
    while (at < end) {
        Span sp;
        if (a.plan.split) {
            sp = span_at(a, line, range, at, end, KB, lane, &at);
            if (sp.last <= sp.first) continue;
        } else {
            sp = span_whole(a, range, KB);
            at = end;
        }
        const int b = sp.b, g = sp.g;
        const int L = of_wave(rows_in_use(a.c, b)), n = of_wave(drafts_of(a.d, b));
        const int cache = (L + KB - 1) / KB, whole = L / KB;
        // (a pair without keys has one block of none)
        const int last = L > 0 || (a.d.K && n > 0) ? sp.last : 0;
        const T* kc = (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1];
        const T* vc = (const T*)a.c.V + b * a.c.vs[0] + g * a.c.vs[1];
        const T* kd = (const T*)a.d.K + b * a.d.ks[0] + g * a.d.ks[1];
        const T* vd = (const T*)a.d.V + b * a.d.vs[0] + g * a.d.vs[1];

        // this wave's pieces of the stage at block i: of every block K piece (wave / KS, wave % KS)
        // and V's rows 4 wave .. 4 wave + 3 (past the last block, of it)
        typename N::KPiece z[2 * NB];
        const uint32_t mine_k = (16 * (wave / KS) + col) * (uint32_t)a.c.ks[2] * 2 + 16 * q;
        const uint32_t mine_v = (4 * wave + q) * (uint32_t)a.c.vs[2] * 2;
        auto load = [&](int i) {
            if (i + NB <= min(whole, last)) {
                const T* kb = kc + (int64_t)i * KB * a.c.ks[2];
                const T* vb = vc + (int64_t)i * KB * a.c.vs[2];
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    z[2 * x] = N::piece(kb, mine_k, wave % KS, q, D);
                    z[2 * x + 1] = N::v_piece(vb, mine_v, 0, D, lane);
                    kb += KB * a.c.ks[2];
                    vb += KB * a.c.vs[2];
                }
                return;
            }
#pragma unroll
            for (int x = 0; x < NB; ++x) {
                const int y = min(i + x, last - 1);
                const bool in = y < cache;
                const int j0 = (in ? y : y - cache) * KB, rows = min(KB, (in ? L : n) - j0);
                const int64_t ks = in ? a.c.ks[2] : a.d.ks[2], vs = in ? a.c.vs[2] : a.d.vs[2];
                const uint32_t kr = (uint32_t)ks * 2, vr = (uint32_t)vs * 2;
                z[2 * x] = N::piece((in ? kc : kd) + j0 * ks,
                                    min(16 * (wave / KS) + col, rows - 1) * kr + 16 * q, wave % KS, q,
                                    D);
                z[2 * x + 1] = N::v_piece((in ? vc : vd) + j0 * vs,
                                          min(4 * wave + q, rows - 1) * vr, 0, D, lane);
            }
        };
        auto put = [&](int buf) {
#pragma unroll
            for (int x = 0; x < NB; ++x) {
                char* block = lds + (buf * NB + x) * N::kBytes;
                reinterpret_cast<typename N::KPiece*>(block)[wave * 64 + lane] = z[2 * x];
                *reinterpret_cast<typename N::KPiece*>(block + N::kKBytes +
                                                       (4 * wave + q) * N::LDV * 2 + 16 * col) =
                    z[2 * x + 1];
            }
        };
        if (sp.first < last) load(sp.first);
        // Q: this wave's rows in registers (those of no token hold the last token's: nobody reads
        // their results)
        typename N::KPiece qf[MT][KS];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int row = min(tile * N::ROWS_WG + rg * 32 + 16 * t + col, R - 1);
            const int h = head_of(a.d, row);
            const T* qb = (const T*)a.d.Q + b * a.d.qs[0] + (g * rep + h) * a.d.qs[1] +
                          (row - h * a.d.T) * a.d.qs[2];
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                qf[t][i] = N::piece(qb, 16 * q, i, q, D);
                if (a.scale < 0.f)
#pragma unroll
                    for (int w = 0; w < 4; ++w) qf[t][i].w[w] ^= 0x80008000u;
            }
        }
        v4f o[MT][1][VL];
        float m[MT], l[MT], used[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            m[t] = -INFINITY;
            l[t] = used[t] = 0.f;
#pragma unroll
            for (int c = 0; c < VL; ++c) o[t][0][c] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        bool odd = false;
        __syncthreads();  // (the last span's results are out of LDS)
        if (sp.first < last) put(0);
        __syncthreads();
        int buf = 0;
        for (int i0 = sp.first; i0 < last; i0 += NB, buf ^= 1) {
            const bool more = i0 + NB < last;
            if (more) load(i0 + NB);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
            for (int y = kg; y < NB; y += KG) {
                const int i = i0 + y;
                if (i >= last) break;
                const char* block = lds + (buf * NB + y) * N::kBytes;
                const auto* mine = reinterpret_cast<const typename N::KPiece*>(block) + lane;
                v4f s[MT][SUB];
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int u = 0; u < SUB; ++u) s[t][u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < KS; ++e)
#pragma unroll
                    for (int u = 0; u < SUB; ++u) {
                        const typename N::KPiece k = mine[(u * KS + e) * 64];
#pragma unroll
                        for (int t = 0; t < MT; ++t) s[t][u] = N::dot(k, qf[t][e], s[t][u]);
                    }
                float p[MT][SUB][4];
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[t][u][e] = s[t][u][e];
                if (i >= whole) {
                    const bool in = i < cache;
                    const int j0 = (in ? i : i - cache) * KB, rows = (in ? L : n) - j0;
#pragma unroll
                    for (int t = 0; t < MT; ++t)
                        hide<MT, SUB>(a, p, t, b, tile * N::ROWS_WG + rg * 32 + 16 * t + col, in, j0,
                                      rows, q);
                }
                weights<MT, SUB, 1, VL>(p, o, m, l, used, scale);
                __builtin_amdgcn_sched_barrier(0);  // (V's registers are the scores' until here)
                // V^T: lane (m, q) takes dim 16 c + m of keys 4 q .. 4 q + 3 and 16 on
                VT v;
                {
                    const uint16_t* rows = reinterpret_cast<const uint16_t*>(block + N::kKBytes) +
                                           (4 * q + (col >> 2)) * N::LDV + 4 * (col & 3);
#pragma unroll
                    for (int c = 0; c < VL; ++c) {
                        const uint2 lo = lds_tr16(rows + 16 * c);
                        const uint2 hi = lds_tr16(rows + 16 * N::LDV + 16 * c);
                        v.p[0][c].w[0] = lo.x, v.p[0][c].w[1] = lo.y;
                        v.p[0][c].w[2] = hi.x, v.p[0][c].w[3] = hi.y;
                    }
                }
                if (i >= whole) odd |= clear_not_finite<T>(v);
                typename N::KPiece f[MT];  // (rounded: see CacheTiles::accumulate)
                N::round(f, p, used);
#pragma unroll
                for (int c = 0; c < VL; ++c)
#pragma unroll
                    for (int t = 0; t < MT; ++t) o[t][0][c] = N::dot(v.p[0][c], f[t], o[t][0][c]);
            }
            if (more) put(buf ^ 1);
            __syncthreads();
        }

        // the KG waves of a row tile added up, as in k_tree_narrow
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            l[t] = row_sum(l[t]);
            used[t] = row_sum(used[t]);
        }
        float* xo = reinterpret_cast<float*>(lds);
        float4* xs = reinterpret_cast<float4*>(lds + N::kOut);
        float4* fin = xs + KG * N::ROWS_WG;
        if (q == 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
                xs[kg * N::ROWS_WG + rg * 32 + 16 * t + col] =
                    make_float4(m[t], l[t], used[t], odd ? 1.f : 0.f);
        }
        __syncthreads();
        odd = false;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = rg * 32 + 16 * t + col;
            float top = m[t];
#pragma unroll
            for (int w = 0; w < KG; ++w) top = fmaxf(top, xs[w * N::ROWS_WG + r].x);
            const float base = base_of(top), f = exp2_(m[t] - base);
            if (kg == 0) {
                float4 y = make_float4(top, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < KG; ++w) {
                    const float4 x = xs[w * N::ROWS_WG + r];
                    const float e = exp2_(x.x - base);
                    y.y += x.y * e;
                    y.z += x.z * e;
                    odd |= x.w != 0.f;
                }
                if (q == 0) fin[r] = y;
            }
            float* to = xo + (kg * N::ROWS_WG + r) * N::LDO + 4 * q;
#pragma unroll
            for (int c = 0; c < VL; ++c)
                *reinterpret_cast<v4f*>(to + 16 * c) = o[t][0][c] * f;
        }
        __syncthreads();
        odd |= write_rows<T, DP, N::ROWS_WG, KG, N::LDO, VL, MODE, 512>(a, sp, tile, n, xo, fin);
        if (__syncthreads_or(odd))
            put_not_finite<T, N::ROWS_WG, 8, KB>(a, sp, tile, fin, xo, L, n, wave, lane);
    }
}

// ---------------------------------------------------------------- head_d > 256
// No output tile fits a wave's registers, so two kernels with the scores between them:
// k_tree_scores writes x (rows of R floats, small beside K and V's rows of head_d), each
// workgroup's 8 waves sharing a tile's dims, or its share of them, and adding up through LDS;
// k_tree_values is the softmax over them and the product with V, each wave 16 VL dims of the
// output.  Keys lie in blocks of 32: the cache's, then the drafts'.
//   fp32, 8 query rows of 2048 dims, 2 sequences of 1000 to 2040 rows, 4 kv heads: 27 and 24.5 us,
//     3.7 and 4.1 TB/s.
//   bf16, 10 query rows of 8192 dims, 1001 rows, 4 kv heads: 17 and 21.2 us, 3.8 and 3.1 TB/s; V by
//     400 workgroups of 25 ranges, 5 of which hold no keys.
//   A workgroup of scores that walks several blocks with Q in registers: no less time (fp32, 408
//     dims, 44 rows: 40 against 36 us).
constexpr int kBlock = 32;
constexpr int kScoreWaves = 8;
constexpr int kWaves = 4;        // of a value workgroup
constexpr int kValueKeys = 128;  // keys between barriers of k_tree_values

// Scores of a row: [shares][pairs of the pass][rows of the tiles][ld_scores], to be added over
// the shares of the dims.
__device__ __forceinline__ size_t score_row(const TreeArgs& a, int share, int pair, int row) {
    return ((size_t)(share * a.bs * a.gs + pair) * a.plan.row_tiles * a.plan.rows + row) *
           a.plan.ld_scores;
}

template <typename T, int MT>
__global__ __launch_bounds__(64 * kScoreWaves) void k_tree_scores(TreeArgs a) {
    constexpr int SUB = kBlock / 16;
    __shared__ v4f red[kScoreWaves][MT * SUB * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    const int tiles = a.plan.row_tiles, most = a.plan.ld_scores / kBlock;
    int unit, tile;
    tile_of(blockIdx.x, a.bs * a.gs * a.plan.shares * most, tiles, &unit, &tile);
    const int share = unit % a.plan.shares, i = unit / a.plan.shares % most;
    const int pair = unit / a.plan.shares / most, g = a.g0 + pair % a.gs, b = a.b0 + pair / a.gs;
    const int L = of_wave(rows_in_use(a.c, b)), n = of_wave(drafts_of(a.d, b)), D = a.c.D;
    const int cache = (L + kBlock - 1) / kBlock;
    const int all = cache + (a.d.K ? (n + kBlock - 1) / kBlock : 0);
    if (i >= all) return;
    const bool in = i < cache;
    const int j0 = (in ? i : i - cache) * kBlock, rows = min(kBlock, (in ? L : n) - j0);
    const int rep = a.d.rep, R = rep * a.d.T;
    const T* kp[SUB];
    const T* qp[MT];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
        const int64_t r = j0 + min(16 * u + col, rows - 1);
        kp[u] = in ? (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1] + r * a.c.ks[2]
                   : (const T*)a.d.K + b * a.d.ks[0] + g * a.d.ks[1] + r * a.d.ks[2];
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {  // (rows past R: the last one's scores, which nobody reads)
        const int row = min((tile * MT + t) * 16 + col, R - 1), h = head_of(a.d, row);
        qp[t] = (const T*)a.d.Q + b * a.d.qs[0] + (g * rep + h) * a.d.qs[1] +
                (row - h * a.d.T) * a.d.qs[2];
    }
    v4f s[MT][SUB];
    wide_scores<T, MT, true>(s, kp, qp, D, share * kScoreWaves + wave, a.plan.shares * kScoreWaves, q);
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
    const int row = (tile * MT + t) * 16 + col, tok = row - head_of(a.d, row) * a.d.T;
    const int k0 = 16 * u + 4 * q;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool on = k0 + e < rows && row < R && (in || sees(a.d, b, tok, j0 + k0 + e));
        y[e] = on ? x[e] * a.scale : -INFINITY;
    }
    float* to = a.scores + score_row(a, share, pair, row) + i * kBlock + k0;
    *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
}

template <typename T, int MT>
__global__ __launch_bounds__(64 * kWaves, MT == 1 ? 3 : 2) void k_tree_values(TreeArgs a) {
    constexpr bool kBf = sizeof(T) == 2;
    // (a wave's dims: one V step of 128 in bf16, 64 in fp32; where the row ends before, its last
    // ones; those before d0 are the wave's before)
    using N = CacheTiles<T, kBf ? 128 : 64, MT, kClamp>;
    constexpr int VL = N::VL, WD = N::VD, ROWS = N::ROWS, PK = N::KB, NB = kValueKeys / PK;
    constexpr int LDP = kValueKeys + 16 / (int)sizeof(T);
    __shared__ __align__(16) T pl[2][ROWS * LDP];
    __shared__ float alpha[2][ROWS];
    __shared__ float4 fin[ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15;
    const int D = a.c.D, groups = (D + WD * kWaves - 1) / (WD * kWaves);
    const int tiles = a.plan.row_tiles;
    int unit, tile;
    tile_of(blockIdx.x, a.plan.ranges * groups, tiles, &unit, &tile);
    const int range = unit / groups, d0 = (unit % groups * kWaves + wave) * WD;
    const int rep = a.d.rep, R = rep * a.d.T;
    const bool busy = d0 < D;
    // softmax: 16 threads a row, 8 keys each, one pass per 16 rows
    const int sr = threadIdx.x >> 4, sk = (threadIdx.x & 15) * 8;

    int at = 0, end = 1;
    Line line{};
    if (a.plan.split) {
        line = line_of(a, kBlock, a.plan.turn, lane);
        at = range * line.per;
        end = min(line.total, at + line.per);
    }
    while (at < end) {
        Span sp;
        if (a.plan.split) {
            sp = span_at(a, line, range, at, end, kBlock, lane, &at);
            if (sp.last <= sp.first) continue;
        } else {
            sp = span_whole(a, range, kBlock);
            at = end;
        }
        const int b = sp.b, g = sp.g;
        const int L = of_wave(rows_in_use(a.c, b)), n = of_wave(drafts_of(a.d, b));
        const int cache = (L + kBlock - 1) / kBlock;
        const bool none = L == 0 && (!a.d.K || n == 0);  // a pair without keys has no scores either
        const T* vc = (const T*)a.c.V + b * a.c.vs[0] + g * a.c.vs[1] + d0;
        const T* vd = (const T*)a.d.V + b * a.d.vs[0] + g * a.d.vs[1] + d0;
        const float* sc = a.scores + score_row(a, 0, (b - a.b0) * a.gs + g - a.g0, tile * ROWS);
        const size_t next_share = score_row(a, 1, 0, 0);
        float m[MT], l[MT], used[MT], x[MT][8];
        v4f o[MT][1][VL];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            m[t] = -INFINITY;
            l[t] = used[t] = 0.f;
#pragma unroll
            for (int c = 0; c < VL; ++c) o[t][0][c] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        bool odd = false;
        // scores of the step at block i
        auto load_x = [&](int i) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float* from = sc + (size_t)(16 * t + sr) * a.plan.ld_scores + i * kBlock + sk;
                v4f u = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, w = u;
                if (sk < (sp.last - i) * kBlock) {
                    u = *reinterpret_cast<const v4f*>(from);
                    w = *reinterpret_cast<const v4f*>(from + 4);
                    for (int y = 1; y < a.plan.shares; ++y) {
                        from += next_share;
                        u += *reinterpret_cast<const v4f*>(from);
                        w += *reinterpret_cast<const v4f*>(from + 4);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[t][e] = u[e], x[t][4 + e] = w[e];
            }
        };
        // V of the x-th PK keys of the span's blocks on (past its end: of the last ones)
        auto load_v = [&](typename N::Vals& to, int x) {
            const int i = min(sp.first + x / (kBlock / PK), sp.last - 1);
            const bool in = i < cache;
            // (a block's second half may have no rows: its first row again)
            const int j1 = (in ? i : i - cache) * kBlock, half = j1 + x % (kBlock / PK) * PK;
            const int j0 = half < (in ? L : n) ? half : j1;
            const int64_t s = in ? a.c.vs[2] : a.d.vs[2];
            N::load_v(to, (in ? vc : vd) + j0 * s, s, (in ? L : n) - j0, D - d0, lane);
        };
        // Two buffers of weights: a wave past a barrier writes the other one, and comes to write
        // this one only after the next barrier, when every wave has read it.
        constexpr int STEP = kValueKeys / kBlock;
        typename N::Vals v0, v1;
        __syncthreads();  // (the last span's)
        if (!none) load_x(sp.first);
        if (!none && busy) load_v(v0, 0);
        int buf = 0;
        for (int i = sp.first; !none && i < sp.last; i += STEP, buf ^= 1) {
            // scores into weights
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                float top = x[t][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) top = fmaxf(top, x[t][e]);
                top = fmaxf(top, dpp<kDppQuadXor1>(top));
                top = fmaxf(top, dpp<kDppQuadXor2>(top));
                top = fmaxf(top, dpp<kDppRowHalfMirror>(top));
                top = fmaxf(top, dpp<kDppRowMirror>(top));
                const float m_new = fmaxf(m[t], top), base = base_of(m_new);
                const float f = exp2_(m[t] - base);
                m[t] = m_new;
                l[t] *= f;
                used[t] *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[t][e] = exp2_(x[t][e] - base);
                    l[t] += x[t][e];
                }
                if ((threadIdx.x & 15) == 0) alpha[buf][16 * t + sr] = f;
                T* to = pl[buf] + (16 * t + sr) * LDP + sk;
                if constexpr (kBf) {  // (rounded: see CacheTiles::accumulate)
                    uint32_t w[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        w[h] = pack2(x[t][2 * h], x[t][2 * h + 1]);
                        used[t] = add2(w[h], used[t]);
                    }
                    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    *reinterpret_cast<float4*>(to) =
                        make_float4(x[t][0], x[t][1], x[t][2], x[t][3]);
                    *reinterpret_cast<float4*>(to + 4) =
                        make_float4(x[t][4], x[t][5], x[t][6], x[t][7]);
                }
            }
            if (i + STEP < sp.last) load_x(i + STEP);
            __syncthreads();
            if (!busy) continue;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float f = alpha[buf][16 * t + col];
                if (__builtin_amdgcn_ballot_w64(f != 1.f)) {
#pragma unroll
                    for (int c = 0; c < VL; ++c) o[t][0][c] *= f;
                }
            }
            // each PK keys' V on their way while the ones before are used
            auto use = [&](typename N::Vals& v, int k) {
                const int y = i + k / kBlock;
                const bool in = y < cache;
                const int j0 = (in ? y : y - cache) * kBlock + k % kBlock;
                if (y >= sp.last || j0 >= (in ? L : n)) return;
                if (!in || j0 + PK > L) odd |= clear_not_finite<T>(v);
                N::accumulate_lds(o, v, pl[buf] + k, LDP, lane);
            };
            const int x0 = (i - sp.first) * (kBlock / PK);
#pragma unroll 1
            for (int k = 0; k < NB; k += 2) {
                load_v(v1, x0 + k + 1);
                __builtin_amdgcn_sched_barrier(0);
                use(v0, k * PK);
                load_v(v0, x0 + k + 2);
                __builtin_amdgcn_sched_barrier(0);
                use(v1, (k + 1) * PK);
            }
        }
        // sums of the rows, for the waves that hold their outputs
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float y = row16_sum(l[t]), z = kBf ? row16_sum(used[t]) : y;
            if ((threadIdx.x & 15) == 0) fin[16 * t + sr] = make_float4(m[t], y, z, 0.f);
        }
        __syncthreads();
        if (!busy) continue;
        // (computed here: hoisted out of the loop over spans, these take the loop's registers)
        const int late = opaque(lane), lq = late >> 4, lc = late & 15;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int row = tile * ROWS + 16 * t + lc, h = head_of(a.d, row), tok = row - h * a.d.T;
            if (row >= R || tok >= n) continue;
            const float4 z = fin[16 * t + lc];
            const bool teller = lq == 0 && d0 == 0;
            const size_t part = part_row(a, max(sp.part, 0), row);
            const bool zero = sp.part < 0 && z.z == 0.f;
            const float inv = sp.part >= 0 ? 1.f : 1.f / z.z;
            float* dims = part_dims(a) + part * D + d0;
            T* to = (T*)a.out + b * a.os[0] + (g * rep + h) * a.os[1] + tok * a.os[2] + d0;
            bool nan = false;
            if (teller && sp.part >= 0) part_stats(a)[part] = z;
            if (teller && sp.part < 0 && a.lse)
                a.lse[((size_t)b * a.d.H + g * rep + h) * a.d.T + tok] =
                    z.y == 0.f ? -INFINITY : (z.x + log2f(z.y)) * kLn2;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = N::dim_of(0, 4 * lq + e, D - d0);
#pragma unroll
                for (int c = 0; c < VL; c += 4) {
                    float y[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] = zero ? 0.f : o[t][0][c + r][e] * inv;
                    nan |= __builtin_isunordered(y[0], y[1]) | __builtin_isunordered(y[2], y[3]);
                    if (d + c >= 0) {
                        if (sp.part >= 0)
                            store4(dims + d + c, y, 4);
                        else
                            store4(to + d + c, y, 4);
                    } else {  // (a row's last dims, fewer than a piece)
#pragma unroll
                        for (int r = 1; r < 4; ++r)
                            if (d + c + r >= 0) {
                                if (sp.part >= 0)
                                    dims[d + c + r] = y[r];
                                else
                                    Elem<T>::st(to, d + c + r, y[r]);
                            }
                    }
                }
            }
            odd |= nan & (z.y == z.y);
        }
        if (__builtin_amdgcn_ballot_w64(odd)) {
            __threadfence_block();  // (this wave's own stores, from other lanes)
            const int tail = L / PK * PK, d1 = min(D, d0 + WD);
            float whole[WD / 64];  // of dims d0 + lane and on
#pragma unroll
            for (int x = 0; x < WD / 64; ++x) {
                const int d = min(64 * x + late, d1 - d0 - 1);
                whole[x] = not_finite_rows(vc + d, a.c.vs[2], sp.first * kBlock,
                                           min(sp.last * kBlock, tail), 1);
            }
            for (int r = 0; r < ROWS; ++r)
                put_row<T>(a, sp, tile * ROWS + r, fin[r], tail, L, n, d0, d1, late,
                           [&](int d) { return whole[WD == 64 || d < d0 + 64 ? 0 : 1]; });
        }
    }
}

// ---------------------------------------------------------------- parts
// The parts of a row added up, in their order: WAVES waves a row (and 256 dims), each every
// WAVES-th part; 4 rows a workgroup where there are many rows.  Rows of one range alone are
// written already.  A launch's latency and a chain of four loads: 4.3 to 8 us; 13.5 where
// 8192 rows of 8 parts come back from memory.
template <typename T, int WAVES, int KB>
__global__ __launch_bounds__(256) void k_tree_merge(TreeArgs a) {
    __shared__ float acc[4][256];
    __shared__ float2 sums[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int D = a.c.D, rep = a.d.rep, d0 = blockIdx.z * 256;
    const int row = WAVES == 4 ? blockIdx.x : blockIdx.x * 4 + wave;
    if (row >= rep * a.d.T) return;
    const unsigned pair = blockIdx.y, seq = pair / (unsigned)a.gs;
    const int g = a.g0 + (int)(pair - seq * a.gs), b = a.b0 + (int)seq;
    const int h = head_of(a.d, row), tok = row - h * a.d.T;
    if (tok >= drafts_of(a.d, b)) return;
    const int blocks = of_wave(blocks_of(a, b, KB));
    const Line line = line_of(a, KB, a.plan.turn, lane);
    const int first = start_of(a, line, b, KB, lane) + (g - a.g0) * (blocks + kPad) + kPad;
    const int r0 = (unsigned)first / (unsigned)line.per;
    const int r1 = (unsigned)(first + blocks - 1) / (unsigned)line.per;
    if (r0 == r1) return;
    const float4* st = part_stats(a);
    // part i is range r0 + i's: its second where the pair begins, its first after that
    auto row_of = [&](int i) { return part_row(a, 2 * (r0 + i) + (i == 0 ? 1 : 0), row); };
    const int parts = r1 - r0 + 1;
    float M = -INFINITY;
    for (int i = lane; i < parts; i += 64) M = fmaxf(M, st[row_of(i)].x);
    M = wave_max(M);
    const float base = base_of(M);
    float l = 0.f, used = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = WAVES == 4 ? wave : 0; i < parts; i += WAVES) {
        const size_t at = row_of(i);
        const float4 z = st[at];
        const float f = exp2_(z.x - base);
        l += f * z.y;
        used += f * z.z;
        const float* from = part_dims(a) + at * D + d0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = lane + 64 * c;
            const float y = d0 + d < D ? from[d] : 0.f;
            // (what is not finite stays so where the factor has vanished)
            x[c] += f == 0.f && !(fabsf(y) < INFINITY) ? y : f * y;
        }
    }
    T* out = (T*)a.out + b * a.os[0] + (g * rep + h) * a.os[1] + tok * a.os[2] + d0;
    if constexpr (WAVES == 4) {
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[wave][lane + 64 * c] = x[c];
        if (lane == 0) sums[wave] = make_float2(l, used);
        __syncthreads();
        l = (sums[0].x + sums[1].x) + (sums[2].x + sums[3].x);
        used = (sums[0].y + sums[1].y) + (sums[2].y + sums[3].y);
        const int d = threadIdx.x;
        const float sum = (acc[0][d] + acc[1][d]) + (acc[2][d] + acc[3][d]);
        if (d0 + d < D) Elem<T>::st(out, d, used == 0.f ? 0.f : sum * (1.f / used));
    } else {
        const float inv = 1.f / used;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (d0 + lane + 64 * c < D)
                Elem<T>::st(out, lane + 64 * c, used == 0.f ? 0.f : x[c] * inv);
    }
    if (d0 == 0 && (WAVES == 4 ? threadIdx.x : lane) == 0 && a.lse)
        a.lse[((size_t)b * a.d.H + g * rep + h) * a.d.T + tok] =
            l == 0.f ? -INFINITY : (M + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------- launches
template <typename T, int DP, int MT, int MODE>
void go_narrow(const TreeArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.plan.ranges * a.plan.row_tiles));
    if constexpr (MT <= 2 && DP <= 128) {
        if (a.plan.waves == 8) {
            hipLaunchKernelGGL((k_tree_narrow<T, DP, MT, MODE, 8>), grid, dim3(512), 0, st, a);
            return;
        }
    }
    hipLaunchKernelGGL((k_tree_narrow<T, DP, MT, MODE, 4>), grid, dim3(256), 0, st, a);
}

template <typename T, int DP, int MODE>
void go_rows(const TreeArgs& a, hipStream_t st) {
    if (a.plan.rows == 16) return go_narrow<T, DP, 1, MODE>(a, st);
    if (a.plan.rows == 32) return go_narrow<T, DP, 2, MODE>(a, st);
    if constexpr (DP == 64 && sizeof(T) == 2) go_narrow<T, DP, 4, MODE>(a, st);
    if constexpr (DP == 128 && sizeof(T) == 2) {
        const dim3 grid((unsigned)(a.plan.ranges * a.plan.row_tiles));
        if (a.plan.rows == 128)
            hipLaunchKernelGGL((k_tree_shared<4, MODE>), grid, dim3(512), 0, st, a);
        else
            hipLaunchKernelGGL((k_tree_shared<8, MODE>), grid, dim3(512), 0, st, a);
    }
}

template <typename T, int DP>
void go_dims(const TreeArgs& a, hipStream_t st) {
    if (a.c.D == DP) return go_rows<T, DP, kExact>(a, st);
    if constexpr (DP == 64) {
        if (a.c.D < 16 / (int)sizeof(T)) return go_rows<T, DP, kElem>(a, st);
    }
    go_rows<T, DP, kClamp>(a, st);
}

// dims of a value workgroup
constexpr int wide_dims(bool bf) { return (bf ? 128 : 64) * kWaves; }

template <typename T, int MT>
void go_wide(const TreeArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(
        (k_tree_scores<T, MT>),
        dim3((unsigned)(a.bs * a.gs * a.plan.row_tiles * a.plan.shares *
                        (a.plan.ld_scores / kBlock))),
        dim3(64 * kScoreWaves), 0, st, a);
    const int wd = wide_dims(sizeof(T) == 2), groups = (a.c.D + wd - 1) / wd;
    hipLaunchKernelGGL((k_tree_values<T, MT>),
                       dim3((unsigned)(a.plan.ranges * groups * a.plan.row_tiles)),
                       dim3(64 * kWaves), 0, st, a);
}

template <typename T, int KB>
void go_merge(const TreeArgs& a, hipStream_t st) {
    const int R = a.d.rep * a.d.T, chunks = (a.c.D + 255) / 256;
    if ((int64_t)a.bs * a.gs * R * chunks >= 1024)
        hipLaunchKernelGGL((k_tree_merge<T, 1, KB>), dim3((R + 3) / 4, a.bs * a.gs, chunks),
                           dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_tree_merge<T, 4, KB>), dim3(R, a.bs * a.gs, chunks), dim3(256), 0, st,
                           a);
}

template <typename T>
void go(const TreeArgs& a, hipStream_t st) {
    const int D = a.c.D;
    if (D > kTreeNarrow) {
        if (a.plan.rows == 16) go_wide<T, 1>(a, st);
        else go_wide<T, 2>(a, st);
    } else if (D <= 64) {
        go_dims<T, 64>(a, st);
    } else if (D <= 128) {
        go_dims<T, 128>(a, st);
    } else if (D <= 192) {
        go_dims<T, 192>(a, st);
    } else {
        go_dims<T, 256>(a, st);
    }
    if (a.plan.split) {
        if constexpr (sizeof(T) == 4) {
            if (D <= kTreeNarrow) return go_merge<T, 16>(a, st);
        }
        go_merge<T, 32>(a, st);
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

TreePlan tree_plan(int dtype, int B, int G, int H, int T, int D, int max_len, bool draft_keys,
                   size_t scratch_cap) {
    TreePlan p{};
    const bool bf = dtype == kDtypeBF16, wide = D > kTreeNarrow;
    const int R = H / G * T;
    const bool shared = bf && D > 64 && D <= 128 && R > 64;
    p.rows = R <= 16 ? 16 : R <= 32 || !bf || D > 64 ? 32 : 64;
    if (shared) {  // the rows of a workgroup that leave the fewest places empty
        p.rows = ceil_div(R, 128) * 128 < ceil_div(R, 256) * 256 ? 128 : 256;
    }
    p.row_tiles = (int)ceil_div(R, p.rows);
    p.waves = 4;
    const int kb = wide || bf ? 32 : 16, mt = p.rows / 16;
    const int64_t blocks =  // of a pair, at most
        std::max<int64_t>(1, ceil_div(max_len, kb) + (draft_keys ? ceil_div(T, kb) : 0));
    const int64_t pairs = (int64_t)B * G, rows = (int64_t)p.row_tiles * p.rows;
    const int groups = wide ? (int)ceil_div(D, wide_dims(bf)) : 1;
    p.ld_scores = wide ? (int)blocks * kBlock : 0;
    // workgroups that the card holds at once (256 CUs; the kernels' registers)
    const int per_cu = wide ? (mt == 1 ? 3 : 2)
                            : std::max(1, (mt == 1 ? 4 : mt == 2 ? 3 : 2) - (D > 64) - (D > 128));
    const int64_t slots =
        std::max<int64_t>(1, 256 * (shared ? 1 : per_cu) / (p.row_tiles * groups));
    const int64_t turn = wide ? kValueKeys / kBlock : shared ? 512 / p.rows : p.waves;
    int64_t ranges = std::min(slots, ceil_div(pairs * (blocks + kPad), 2 * turn));
    // one workgroup of 8 waves a pair where that leaves a wave few blocks: no second launch
    const bool small = !wide && mt <= 2 && D <= 128 && blocks <= 32 && pairs * p.row_tiles <= 512;
    // (pairs of few turns of blocks take less time whole than the parts and their merge: bf16,
    // head_d 1024, 75 rows, 14 blocks 35 against 46 us; fp32, head_d 512, 24 rows, 16 blocks 44
    // against 40)
    p.split = !small && ranges > 1 && pairs < 4 * slots && blocks > 7 * turn / 2;
    if (small) p.waves = 8;
    p.turn = small ? p.waves : (int)turn;
    const size_t room = scratch_cap / sizeof(float);
    // score workgroups: two a CU, where the dims give each wave two steps still
    p.shares = 1;
    while (wide && pairs * p.row_tiles * blocks * p.shares < 512 && p.shares < 8 &&
           D >= 2 * p.shares * kScoreWaves * (bf ? 256 : 128))
        p.shares *= 2;
    const size_t sc = wide ? (size_t)rows * p.ld_scores * p.shares : 0;  // floats of a pair
    const size_t part = 2 * (size_t)rows * (D + 4);           // ... of a range
    int64_t in_pass = pairs;
    if (sc * pairs + (p.split ? part * ranges : 0) > room) {
        // fewer pairs a pass where the scratch does not hold their scores, fewer ranges where it
        // does not hold their parts
        const size_t for_parts = p.split ? std::min(room / 2, (size_t)ranges * part) : 0;
        if (sc > 0)
            in_pass = std::max<int64_t>(1, std::min<int64_t>(pairs, (room - for_parts) / sc));
        const size_t left = room > sc * in_pass ? room - sc * in_pass : 0;
        ranges = std::min<int64_t>(ranges, left / part);
        if (ranges < 2) p.split = 0;
    }
    p.seqs = in_pass >= G ? (int)(in_pass / G) : 1;
    p.kv = in_pass >= G ? G : (int)in_pass;
    in_pass = (int64_t)p.seqs * p.kv;
    p.ranges = (int)(p.split ? ranges : in_pass);
    p.scores = sc * in_pass;
    p.scratch = (p.scores + (p.split ? part * ranges : 0)) * sizeof(float);
    // (range starts pass the line's end by one range at most)
    p.line = p.split ? in_pass * (blocks + kPad) + 2 * turn * p.ranges : 0;
    p.workgroups = std::max((int64_t)p.ranges * p.row_tiles * groups,
                            in_pass * p.row_tiles * p.shares * (p.ld_scores / kBlock));
    return p;
}

hipError_t launch_tree_attention(int dtype, TreeArgs a, hipStream_t st) {
    for (a.b0 = 0; a.b0 < a.c.B; a.b0 += a.plan.seqs)
        for (a.g0 = 0; a.g0 < a.c.G; a.g0 += a.plan.kv) {
            a.bs = std::min(a.plan.seqs, a.c.B - a.b0);
            a.gs = std::min(a.plan.kv, a.c.G - a.g0);
            TreeArgs pass = a;
            if (!a.plan.split) pass.plan.ranges = a.bs * a.gs;
            if (dtype == kDtypeF32)
                go<float>(pass, st);
            else
                go<uint16_t>(pass, st);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    return hipSuccess;
}

}  // namespace atn

// Attention over a paged key/value cache: row (h, t) of sequence b attends the rows r <= len + t,
//   x_r = scale q . k_r,  m = max x,  l = sum exp(x - m),
//   out = sum exp(x - m) v / l,  lse = m + log l.
//
// Rows that a group of sequences begins with are read once for all of them, in a pass of its own:
// there the query rows of all members are rows of one product with K and V, as the heads of a kv
// head are.  The second pass is every sequence's rows from there on; k_paged_merge adds up what
// both have left.
//
// An item is a tile of query rows of one kv head of a segment (a sequence, or a group) over its
// blocks of keys.  Lengths and groups are on the device, so the host only fixes how many
// workgroups there are: the blocks of all items lie in one line, each workgroup takes an equal
// range of it, and what range r computes of the line's i-th item is part r + i (one of the two
// grows from each span to the next, so parts are distinct, and those of an item consecutive).
// Items that a single range holds and no group precedes are written at once.
#pragma once

#include <algorithm>
#include <cfloat>

#include "cache_tiles.hpp"
#include "paged.hpp"

namespace atn {

constexpr int kPagedNarrow = 256;  // head_d up to which a wave holds a row tile's output
constexpr int kPagedPad = 12;      // places of the line that beginning and ending an item count for
constexpr int kPagedWideBlock = 32;  // head_d above: keys of a block
constexpr int kPagedWideTurn = 4;    // ... blocks between barriers
constexpr int kPagedWideRows = 32;   // ... query rows of a workgroup of values, at most
constexpr int kPagedWideDims = 512;  // ... dims of a workgroup (bf16; fp32: half)

namespace {

constexpr float kLn2 = 0.69314718055994531f;

// ---------------------------------------------------------------- segments
struct Segment {
    int first, members;  // sequences
    int lo, hi;          // rows of keys, [lo, hi)
    int tiles;           // of query rows
    int len;             // rows before the new tokens (own pass)
};
__device__ __forceinline__ int tokens_of(const PagedArgs& a, int b) {
    return a.count ? min(max(a.count[b], 0), a.T) : a.T;
}
// The group in lane L of a wave (of the first 64): its sequences and rows.
struct Groups {
    int first, end, rows;
};
// (first and shared may hold anything: groups of a list that does not ascend, which might overlap and
// have more items than the host counted on, share nothing; nor do those with too little to save.)
__device__ __forceinline__ Groups group_at(const PagedArgs& a, int i) {
    Groups g;
    g.first = min(max(a.first[i], 0), a.c.B - 1);
    g.end = min(max(a.first[i + 1], 0), a.c.B);
    const int L = min(rows_in_use(a.c, g.first), a.c.rows), m = g.end - g.first;
    g.rows = min(max(a.shared[i], 0), L);
    if (!saves_reads(g.rows, m, a.es, a.rep, a.T)) g.rows = 0;
    if (a.starts && !a.starts[a.c.B].x) g.rows = 0;  // (does not ascend)
    return g;
}
__device__ __forceinline__ Groups groups_of(const PagedArgs& a, int lane) {
    Groups g{0, 0, 0};
    bool down = false;
    if (lane < a.groups && !a.starts) {
        g = group_at(a, lane);
        down = a.first[lane + 1] < a.first[lane];
    }
    if (__builtin_amdgcn_ballot_w64(down)) g.rows = 0;
    return g;
}
// Where sequence b's own rows begin, and its group or -1 (a wave's work; b may differ by lane).
__device__ __forceinline__ int2 start_of(const PagedArgs& a, const Groups& g, int b) {
    if (a.starts) return a.starts[b];
    int2 x = make_int2(0, -1);
    for (int i = 0; i < a.groups; ++i) {
        const int rows = __builtin_amdgcn_readlane(g.rows, i);
        if (rows > 0 && b >= __builtin_amdgcn_readlane(g.first, i) &&
            b < __builtin_amdgcn_readlane(g.end, i))
            x = make_int2(rows, i);
    }
    return x;
}
// (a wave's work; i may differ by lane, and be past the last)
template <int PRE>
__device__ __forceinline__ Segment segment(const PagedArgs& a, const Groups& gr, int i) {
    Segment s;
    if (PRE) {
        const int j = min(i, a.groups - 1);
        Groups g;
        if (a.starts)
            g = group_at(a, j);
        else
            g.first = __shfl(gr.first, j), g.end = __shfl(gr.end, j), g.rows = __shfl(gr.rows, j);
        s.first = g.first;
        s.members = g.end - g.first;
        s.lo = 0;
        s.hi = g.rows;
        s.tiles = s.hi > 0 ? (s.members * a.T * a.rep + a.plan.pre.rows - 1) / a.plan.pre.rows : 0;
        s.len = 0;
    } else {
        i = min(i, a.c.B - 1);
        const int n = tokens_of(a, i);
        s.first = i;
        s.members = 1;
        s.len = rows_in_use(a.c, i);
        s.lo = start_of(a, gr, i).x;
        s.hi = min(s.len + n, a.c.rows);
        s.tiles = (n * a.rep + a.plan.own.rows - 1) / a.plan.own.rows;
    }
    return s;
}
template <int PRE>
__host__ __device__ __forceinline__ const PagedPass& pass_of(const PagedArgs& a) {
    return PRE ? a.plan.pre : a.plan.own;
}
// Blocks of an item (one at least, so that tokens that attend nothing are written).
__device__ __forceinline__ int blocks_of(const Segment& s, int kb) {
    return max(1, (s.hi + kb - 1) / kb - s.lo / kb);
}

// ---------------------------------------------------------------- the line
// Its length and the places of a range; of segment `lane` (the first 64): places of an item, items,
// and the sums of places and items up to it.
struct Line {
    int total, per;
    int n, m, upto, items;
};
template <int PRE>
__device__ __forceinline__ void line_lane(const PagedArgs& a, const Groups& gr, int i, int count,
                                          int kb, int pad, int* n, int* m) {
    const Segment s = segment<PRE>(a, gr, i);
    *m = i < count ? s.tiles * a.gs : 0;
    *n = blocks_of(s, kb) + pad;
}
template <int PRE>
__device__ __forceinline__ Line line_of(const PagedArgs& a, const Groups& gr, int kb, int lane,
                                        int pad = kPagedPad) {
    const PagedPass& p = pass_of<PRE>(a);
    const int count = PRE ? a.groups : a.c.B;
    Line x;
    line_lane<PRE>(a, gr, lane, count, kb, pad, &x.n, &x.m);
    x.upto = wave_scan(x.n * x.m);
    x.items = wave_scan(x.m);
    x.total = __builtin_amdgcn_readlane(x.upto, 63);
#pragma unroll 1
    for (int i0 = 64; i0 < count; i0 += 64) {
        int n, m;
        line_lane<PRE>(a, gr, i0 + lane, count, kb, pad, &n, &m);
        x.total += __builtin_amdgcn_readlane(wave_scan(n * m), 63);
    }
    const int per = (x.total + p.ranges - 1) / p.ranges;
    x.per = max((per + p.turn - 1) & -p.turn, 2 * p.turn);
    return x;
}
// The segment at place `at`: its number, places of an item, first place, items before it.
struct Place {
    int seg, n, start, items;
};
template <int PRE>
__device__ __forceinline__ Place place_at(const PagedArgs& a, const Groups& gr, const Line& line, int at,
                                          int kb, int lane, int pad = kPagedPad) {
    const int count = PRE ? a.groups : a.c.B;
    int n = line.n, m = line.m, upto = line.upto, items = line.items;
#pragma unroll 1
    for (int i0 = 0;; i0 += 64) {
        const uint64_t done = __builtin_amdgcn_ballot_w64(upto <= at);
        if (done != ~0ull || i0 + 64 >= count) {
            const int l = min(__builtin_popcountll(done), min(63, count - 1 - i0));
            Place p;
            p.seg = i0 + l;
            p.n = __builtin_amdgcn_readlane(n, l);
            const int mm = __builtin_amdgcn_readlane(m, l);
            p.start = __builtin_amdgcn_readlane(upto, l) - p.n * mm;
            p.items = __builtin_amdgcn_readlane(items, l) - mm;
            return p;
        }
        const int before = __builtin_amdgcn_readlane(upto, 63);
        const int ibefore = __builtin_amdgcn_readlane(items, 63);
        line_lane<PRE>(a, gr, i0 + 64 + lane, count, kb, pad, &n, &m);
        upto = before + wave_scan(n * m);
        items = ibefore + wave_scan(m);
    }
}
// ... of segment i
template <int PRE>
__device__ __forceinline__ Place place_of(const PagedArgs& a, const Groups& gr, const Line& line, int i,
                                          int kb, int lane, int pad = kPagedPad) {
    const int count = PRE ? a.groups : a.c.B;
    int n = line.n, m = line.m, upto = line.upto, items = line.items, i0 = 0;
#pragma unroll 1
    for (; i >= i0 + 64; i0 += 64) {
        const int before = __builtin_amdgcn_readlane(upto, 63);
        const int ibefore = __builtin_amdgcn_readlane(items, 63);
        line_lane<PRE>(a, gr, i0 + 64 + lane, count, kb, pad, &n, &m);
        upto = before + wave_scan(n * m);
        items = ibefore + wave_scan(m);
    }
    Place p;
    p.seg = i;
    p.n = __builtin_amdgcn_readlane(n, i - i0);
    const int mm = __builtin_amdgcn_readlane(m, i - i0);
    p.start = __builtin_amdgcn_readlane(upto, i - i0) - p.n * mm;
    p.items = __builtin_amdgcn_readlane(items, i - i0) - mm;
    return p;
}

// A range's blocks [first, last) of one item (counted from row 0 of the cache), and where they go:
// part < 0: the output.
// blocks_before: of the line, before the item's.
struct Span {
    Segment s;
    int seg, g, tile, first, last, part;
    int blocks_before;
};
__device__ __forceinline__ int bounded(const PagedPass& p, int part) {
    // (the host counts with the most items that lengths and groups can make; the bound is for those that
    // change between the kernels of a call)
    return (int)min((int64_t)part, p.parts - 1);
}
// The last block that any row of the item's tile attends, and one more.
template <int PRE>
__device__ __forceinline__ int tile_end(const PagedArgs& a, const Segment& s, int tile, int kb) {
    if (PRE) return (s.hi + kb - 1) / kb;
    const int tok = over(tile * a.plan.own.rows + a.plan.own.rows - 1, a.by_rep);
    return (min(s.hi, s.len + tok + 1) + kb - 1) / kb;
}
template <int PRE>
__device__ __forceinline__ Span span_at(const PagedArgs& a, const Groups& gr, const Line& line, int r,
                                        int at, int end, int kb, int lane, int* next) {
    const Place p = place_at<PRE>(a, gr, line, at, kb, lane);
    Span x;
    x.seg = p.seg;
    x.s = segment<PRE>(a, gr, p.seg);
    x.s.lo = of_wave(x.s.lo), x.s.hi = of_wave(x.s.hi), x.s.len = of_wave(x.s.len);
    x.s.first = of_wave(x.s.first), x.s.members = of_wave(x.s.members), x.s.tiles = of_wave(x.s.tiles);
    const int off = at - p.start, item = (unsigned)off / (unsigned)p.n, in = off - item * p.n;
    const int g = (unsigned)item / (unsigned)max(1, x.s.tiles);
    const int out = min(p.n, in + end - at), b0 = x.s.lo / kb;
    x.g = a.g0 + min(g, a.gs - 1);
    x.tile = item - g * x.s.tiles;
    x.first = max(0, in - kPagedPad);
    x.last = out - kPagedPad;
    const bool alone = !PRE && x.s.lo == 0 && x.first == 0 && out == p.n;
    x.part = alone ? -1 : bounded(pass_of<PRE>(a), r + p.items + item);
    x.blocks_before = at - in - kPagedPad * (p.items + item);
    x.first += b0;
    x.last += b0;
    *next = at + out - in;
    return x;
}
// The whole of item `id`, where items are workgroups (own pass alone): the tiles with the most keys
// first.
__device__ __forceinline__ Span span_whole(const PagedArgs& a, const Groups& gr, int id, int kb) {
    Span x;
    const int items = a.c.B * a.gs, tile = a.plan.own.tiles - 1 - (unsigned)id / (unsigned)items;
    const int pair = id % (unsigned)items;
    x.seg = pair / (unsigned)a.gs;
    x.s = segment<0>(a, gr, x.seg);
    x.s.lo = of_wave(x.s.lo), x.s.hi = of_wave(x.s.hi), x.s.len = of_wave(x.s.len);
    x.s.tiles = of_wave(x.s.tiles);
    x.g = a.g0 + pair - x.seg * a.gs;
    x.tile = tile;
    x.first = x.s.lo / kb;
    x.last = tile < x.s.tiles ? x.first + blocks_of(x.s, kb) : x.first;
    x.part = x.s.lo == 0 ? -1 : bounded(a.plan.own, pair * a.plan.own.tiles + tile);
    return x;
}

// Sequence, head and token of a tile's row (b < 0: of no token).
struct Row {
    int b, h, tok;
};
template <int PRE>
__device__ __forceinline__ Row row_of(const PagedArgs& a, const Span& sp, int row) {
    const int flat = over(row, a.by_rep);
    Row x;
    x.h = sp.g * a.rep + row - flat * a.rep;
    if (PRE) {
        const int m = over(flat, a.by_t);
        x.tok = flat - m * a.T;
        x.b = m < sp.s.members ? sp.s.first + m : -1;
    } else {
        x.b = flat < a.T ? sp.s.first : -1;
        x.tok = flat;
    }
    if (x.b >= 0 && x.tok >= tokens_of(a, x.b)) x.b = -1;
    return x;
}
// ... where its queries lie (those of no token: some token's; nobody reads their results)
template <int PRE>
__device__ __forceinline__ int64_t q_at(const PagedArgs& a, const Span& sp, int row) {
    const int flat = over(row, a.by_rep), h = sp.g * a.rep + row - flat * a.rep;
    int b = sp.s.first, t = flat;
    if (PRE) {
        const int m = over(flat, a.by_t);
        t = flat - m * a.T;
        b += min(m, sp.s.members - 1);
    }
    return b * a.qs[0] + h * a.qs[1] + min(t, a.T - 1) * a.qs[2];
}
// Rows of keys that a row attends, from 0 on.
template <int PRE>
__device__ __forceinline__ int attended(const PagedArgs& a, const Span& sp, int row) {
    return PRE ? sp.s.hi : min(sp.s.hi, sp.s.len + over(row, a.by_rep) + 1);
}

// Parts: statistics of the rows (maximum, sum of the weights, their sum as they entered the product
// with V), then, behind all of them, the rows' dims.
template <int PRE>
__device__ __forceinline__ size_t part_row(const PagedArgs& a, int part, int row) {
    return (size_t)part * pass_of<PRE>(a).part_rows + row;
}
template <int PRE>
__device__ __forceinline__ float4* part_stats(const PagedArgs& a) {
    return reinterpret_cast<float4*>(PRE ? a.pre_part : a.own_part);
}
template <int PRE>
__device__ __forceinline__ float* part_dims(const PagedArgs& a) {
    return (PRE ? a.pre_part : a.own_part) + 4 * part_row<PRE>(a, (int)pass_of<PRE>(a).parts, 0);
}

// ---------------------------------------------------------------- steps of a block
// bit j: j < n
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }

// The keys that a row attends of the 32 (16) from j0 on, as a lane of group q holds them (bit 4 u +
// e): not those past the row's, before the item's, and of no page (`there`).
template <int SUB>
__device__ __forceinline__ uint32_t seen(int j0, int lo, int upto, uint32_t there, int q) {
    const uint32_t see = there & below(upto - j0) & ~below(lo - j0);
    uint32_t mine = 0;
#pragma unroll
    for (int u = 0; u < SUB; ++u) mine |= (see >> (16 * u + 4 * q) & 15u) << (4 * u);
    return mine;
}
// Scores of the others become -infinity.
template <int SUB>
__device__ __forceinline__ void hide(float (&p)[SUB][4], uint32_t mine) {
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!((mine >> (4 * u + e)) & 1u)) p[u][e] = -INFINITY;
}

// Scores into weights.  The running maximum moves only when a score passes it by more than 8
// (weights up to 2^8 lose nothing in fp32 or bf16), so the tile is rarely rescaled.
template <int SUB, int VS, int VL>
__device__ __forceinline__ void weights(float (&p)[SUB][4], v4f (&o)[VS][VL], float& m, float& l,
                                        float& used, float scale) {
    float top = p[0][0];
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, p[u][e]);
    if (__builtin_amdgcn_ballot_w64(top * scale > m + 8.f)) {
        const float m_new = fmaxf(m, row_max(top) * scale);
        const float f = exp2_(m - base_of(m_new));
        m = m_new;
        l *= f;
        used *= f;
#pragma unroll
        for (int x = 0; x < VS; ++x)
#pragma unroll
            for (int c = 0; c < VL; ++c) o[x][c] *= f;
    }
    const float base = base_of(m);
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[u][e] = exp2_(fmaf(p[u][e], scale, -base));
            l += p[u][e];
        }
}

// Whether any lane's V holds an infinity or NaN.  (A sum of products with 0 is NaN then.)
template <typename T, typename V>
__device__ __forceinline__ bool not_finite(const V& v) {
    float sum = 0.f;
    for (auto& row : v.p)
        for (auto& piece : row)
            for (auto& w : piece.w)
                sum = sizeof(T) == 4 ? fmaf(__uint_as_float(w), 0.f, sum) : dot2(w, 0u, sum);
    return __builtin_amdgcn_ballot_w64(sum != sum) != 0;
}
// A word of V with its infinities and NaNs as numbers, all else 0: +inf 1, -inf 64, NaN 4096.
template <typename T>
__device__ __forceinline__ uint32_t flags_of(uint32_t x) {
    if constexpr (sizeof(T) == 4) {
        const uint32_t f = x & 0x7fffffu ? 0x45800000u : x >> 31 ? 0x42800000u : 0x3f800000u;
        return (x & 0x7f800000u) == 0x7f800000u ? f : 0u;
    } else {
        const uint32_t lo = x & 0x7fu ? 0x4580u : x & 0x8000u ? 0x4280u : 0x3f80u;
        const uint32_t hi = x & 0x7f0000u ? 0x45800000u : x >> 31 ? 0x42800000u : 0x3f800000u;
        return ((x & 0x7f80u) == 0x7f80u ? lo : 0u) |
               ((x & 0x7f800000u) == 0x7f800000u ? hi : 0u);
    }
}
// What a sum of flags adds to an output.
__device__ __forceinline__ float spread_of(float sum) {
    const int k = (int)sum, pos = k & 63, neg = k >> 6 & 63;
    const float add = k >= 4096 || (pos && neg) ? __builtin_nanf("") : pos ? INFINITY : -INFINITY;
    return k ? add : 0.f;
}
// In a block with keys that some rows do not attend, an infinity or NaN in V times a weight of 0
// would reach them.  V is cleared of these, and they go to the rows that attend their keys by a
// product of their own, the flags' with weights 1: sums over at most 32 keys, exact, whose
// digits (of 64) say what to add.
template <typename T, typename N, int MT>
__device__ __forceinline__ void spread_not_finite(v4f (&o)[MT][N::VS][N::VL], typename N::Vals& v,
                                                  const uint32_t (&see)[MT]) {
#pragma unroll
    for (int i = 0; i < N::VS; ++i)
#pragma unroll
        for (int c = 0; c < N::VL; ++c) {
            v4f n[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) n[t] = v4f{0.f, 0.f, 0.f, 0.f};
            if constexpr (N::kBf) {
                typename N::KPiece f;
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    f.w[h] = flags_of<T>(__builtin_amdgcn_perm(
                        v.p[2 * h + 1][i].w[c / 2], v.p[2 * h][i].w[c / 2],
                        (c & 1) ? 0x07060302u : 0x05040100u));
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    typename N::KPiece one;
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        one.w[h] = (see[t] >> (2 * h) & 1u ? 0x3f80u : 0u) |
                                   (see[t] >> (2 * h + 1) & 1u ? 0x3f800000u : 0u);
                    n[t] = N::dot(f, one, n[t]);
                }
            } else {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        n[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                            __uint_as_float(flags_of<T>(v.p[e][i].w[c])),
                            see[t] >> e & 1u ? 1.f : 0.f, n[t], 0, 0, 0);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][i][c][e] += spread_of(n[t][e]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
    for (int j = 0; j < N::KEYS; ++j)
#pragma unroll
        for (int i = 0; i < N::VS; ++i)
#pragma unroll
            for (int w = 0; w < N::VB / 4; ++w) {
                const uint32_t f = flags_of<T>(v.p[j][i].w[w]);
                if constexpr (N::kBf)
                    v.p[j][i].w[w] &= (f & 0xffffu ? 0xffff0000u : ~0u) & (f >> 16 ? 0xffffu : ~0u);
                else
                    v.p[j][i].w[w] = f ? 0u : v.p[j][i].w[w];
            }
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
__device__ __forceinline__ float lse_of(float4 z) {
    return z.y == 0.f ? -INFINITY : (z.x + log2f(z.y)) * kLn2;
}

// ---------------------------------------------------------------- pages
// The pages of a wave's blocks i, i + STEP, ...: where a page holds whole runs of 16 rows (RUNS), a
// lane's load names the page of 16 keys, and 64 of them serve the next blocks; else lane l has that
// of a block's key l.  Loads of rows go through them: all rows of a page are there to be read,
// and where an entry names no page, or lies past the table, some page is.
template <int KB, int STEP, bool RUNS>
struct Pages {
    static constexpr int SUB = KB / 16, AHEAD = RUNS ? 64 / SUB : 1;
    int b, at;  // sequence; first block of `now`
    int now, next;
    __device__ __forceinline__ int fetch(const PagedView& c, int i, int lane) const {
        if (RUNS) return page_of(c, b, (i + lane / SUB * STEP) * KB + 16 * (lane % SUB));
        return page_of(c, b, i * KB + (lane & (KB - 1)));
    }
    __device__ __forceinline__ void begin(const PagedView& c, int seq, int i, int lane) {
        b = seq, at = i;
        now = fetch(c, i, lane);
        next = fetch(c, i + AHEAD * STEP, lane);
    }
    // moves on to block i
    __device__ __forceinline__ void go(const PagedView& c, int i, int lane) {
        if (i < at + AHEAD * STEP) return;
        at += AHEAD * STEP;
        now = next;
        next = fetch(c, at + AHEAD * STEP, lane);
    }
    __device__ __forceinline__ int run(int i, int s) const {
        return __builtin_amdgcn_readlane(now, (unsigned)(i - at) / (unsigned)STEP * SUB + s);
    }
    // bit j: key j of the block has a page
    __device__ __forceinline__ uint32_t there(const PagedView& c, int i) const {
        if (RUNS) {
            uint32_t x = 0;
#pragma unroll
            for (int s = 0; s < SUB; ++s) x |= is_page(c, run(i, s)) ? 0xffffu << (16 * s) : 0u;
            return x;
        }
        return (uint32_t)__builtin_amdgcn_ballot_w64(is_page(c, now)) & below(KB);
    }
    // Elements from a pool's start to the 16 keys s of the block
    __device__ __forceinline__ int64_t run_at(const PagedView& c, const int64_t (&st)[3], int i,
                                              int s) const {
        const int r = i * KB + 16 * s, in = r - over(r, c.by_page) * c.page_rows;
        const int page = run(i, s);
        return (is_page(c, page) ? page : 0) * st[0] + in * st[2];
    }
    // ... to its key `key`, another one in each lane
    __device__ __forceinline__ int64_t key_at(const PagedView& c, const int64_t (&st)[3], int i,
                                              int key) const {
        const int r = i * KB + key, page = __shfl(now, key);
        return (is_page(c, page) ? page : 0) * st[0] +
               (r - over(r, c.by_page) * c.page_rows) * st[2];
    }
    // pool: of the kv head
    template <typename N, typename T>
    __device__ __forceinline__ void load_k(typename N::Keys& k, const PagedView& c, const T* pool,
                                           int i, int D, int lane) const {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const T* base;
            uint32_t off = 16 * (lane >> 4);
            if (RUNS) {
                base = pool + run_at(c, c.ks, i, s);
                off += (lane & 15) * (uint32_t)c.ks[2] * (uint32_t)sizeof(T);
            } else {
                base = pool + key_at(c, c.ks, i, 16 * s + (lane & 15));
            }
#pragma unroll
            for (int e = 0; e < N::KS; ++e) k.p[s][e] = N::piece(base, off, e, lane >> 4, D);
        }
    }
    template <typename N, typename T>
    __device__ __forceinline__ void load_v(typename N::Vals& v, const PagedView& c, const T* pool,
                                           int i, int D, int lane) const {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const T* base = pool;
            if (RUNS) base += run_at(c, c.vs, i, s);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const T* row = RUNS ? base : pool + key_at(c, c.vs, i, N::key_of(lane, 4 * s + e));
                const uint32_t off =
                    RUNS ? (4 * (lane >> 4) + e) * (uint32_t)c.vs[2] * (uint32_t)sizeof(T) : 0;
#pragma unroll
                for (int x = 0; x < N::VS; ++x)
                    v.p[4 * s + e][x] = N::v_piece(row, off, x, D, lane);
            }
        }
    }
};

// The results of `parts` waves a row, scaled alike, in LDS (rows of LDO floats), summed and
// written: to the output, or the span's part.  fin: the rows' maxima and sums.
template <typename T, int PRE, int DP, int ROWS, int PARTS, int LDO, int VL, int MODE, int THREADS>
__device__ __forceinline__ void write_rows(const PagedArgs& a, const Span& sp, const float* xo,
                                           const float4* fin) {
    const int D = MODE == kExact ? DP : a.c.D;
    // (opaque: or what this computes is hoisted out of the loop over spans, into registers)
#pragma unroll 1
    for (int e = opaque(threadIdx.x); e < ROWS * (DP / 4); e += THREADS) {
        const int r = e / (DP / 4), d = e % (DP / 4) * 4;
        const Row to = row_of<PRE>(a, sp, sp.tile * ROWS + r);
        if (to.b < 0 || d >= D) continue;
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
        if (PRE || sp.part >= 0) {
            const size_t at = part_row<PRE>(a, sp.part, r);
            if (d == 0) part_stats<PRE>(a)[at] = z;
            store4(part_dims<PRE>(a) + at * D + d, x, MODE == kExact ? 4 : D - d);
        } else {
            // (0: nothing attended, or no score above -infinity)
            const float inv = 1.f / z.z;
            if (d == 0 && a.lse) a.lse[((size_t)to.b * a.H + to.h) * a.T + to.tok] = lse_of(z);
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = z.z == 0.f ? 0.f : x[c] * inv;
            store4((T*)a.out + to.b * a.os[0] + to.h * a.os[1] + to.tok * a.os[2] + d, x,
                   MODE == kExact ? 4 : D - d);
        }
    }
}

// A workgroup's spans, one after another: f(span).
template <int PRE, bool SCORES = false, typename F>
__device__ __forceinline__ void each_span(const PagedArgs& a, int id, int kb, int lane, F f) {
    const bool split = PRE || a.plan.own.split;
    int at = 0, end = 1;
    Line line{};
    const Groups gr = groups_of(a, lane);
    if (split) {
        line = line_of<PRE>(a, gr, kb, lane);
        at = id * line.per;
        end = min(line.total, at + line.per);
    }
    while (at < end) {
        Span sp;
        if (split) {
            sp = span_at<PRE>(a, gr, line, id, at, end, kb, lane, &at);
        } else {
            sp = span_whole(a, gr, id, kb);
            at = end;
            if (SCORES) {
                const Place p = place_of<0>(a, gr, line_of<0>(a, gr, kb, lane, 0), sp.seg, kb, lane, 0);
                sp.blocks_before = p.start + ((sp.g - a.g0) * sp.s.tiles + sp.tile) * p.n;
            }
        }
        if (sp.last > sp.first) f(sp);
    }
}

// ---------------------------------------------------------------- head_d <= 256
// Every wave walks its own blocks of keys, alone: scores, running maximum and sum, and its own
// output tile in registers (cache_tiles.hpp); nothing passes through LDS but Q and, at the
// end, the waves' results.  The read of K and V bounds it: one token of 32 over 8 heads, 128 bf16 dims,
// 8 sequences of 1000 to 32000 rows, 100 us, 5.4 TB/s; 32 sequences of 64 to 1024 rows under 8192
// shared ones, 45 us, 4.5 TB/s with the shared rows' four reads, three of which L2 answers.  Of short
// contexts latency: code, lengths, pages, K and V are a chain; few items have 8 waves each (300 rows
// 8.4 us, 9.0 with 4).
template <typename T, int DP, int MT, int MODE, int WAVES_>
struct PagedNarrow : CacheTiles<T, DP, MT, MODE> {
    using N = CacheTiles<T, DP, MT, MODE>;
    static constexpr int WAVES = WAVES_;
    // registers: the output tile, K and V of a block, the scores and weights, addresses; with the
    // next block's K loaded ahead except where only that would not leave two waves a SIMD
    static constexpr int kRegs = DP / 4 * (MT + 1) + 20 * MT + 44;
    static constexpr int kWith = kRegs + DP / 4;
    static constexpr bool kAhead = kWith <= 250 || kRegs > 220;
    static constexpr int kMinWaves = kWith <= 124 ? 4 : kWith <= 164 ? 3 : kRegs <= 220 ? 2 : 1;
    static constexpr int LDO = DP + 4;  // row of the waves' results, floats
    static constexpr int kQBytes = N::ROWS * DP * (int)sizeof(T);
    static constexpr int kXBytes = WAVES * N::ROWS * LDO * 4;
    static constexpr int kOut = kQBytes > kXBytes ? kQBytes : kXBytes;
    static constexpr int kLds = kOut + (WAVES + 1) * N::ROWS * 16;
    static constexpr int kQ = (MT * N::KS * 64 + 64 * WAVES - 1) / (64 * WAVES);  // pieces a thread
    static_assert(kLds <= 160 * 1024, "LDS");
};

template <typename T, int DP, int MT, int MODE, bool RUNS, int WAVES_, int PRE>
__device__ __forceinline__ void paged_narrow(const PagedArgs& a, int id, char* lds) {
    using N = PagedNarrow<T, DP, MT, MODE, WAVES_>;
    constexpr int KB = N::KB, SUB = N::SUB, KS = N::KS, VS = N::VS, VL = N::VL, WAVES = N::WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    const int D = MODE == kExact ? DP : a.c.D;
    const float scale = fabsf(a.scale);

    each_span<PRE>(a, id, KB, lane, [&](const Span& sp) {
        const T* kp = (const T*)a.c.K + sp.g * a.c.ks[1];
        const T* vp = (const T*)a.c.V + sp.g * a.c.vs[1];
        const int row0 = sp.tile * N::ROWS, lo = sp.s.lo;
        const int last = min(sp.last, tile_end<PRE>(a, sp.s, sp.tile, KB));
        // blocks [w0, w1) are attended whole by every row
        const int w0 = (lo + KB - 1) / KB;
        const int w1 = of_wave(attended<PRE>(a, sp, row0)) / KB;
        Pages<KB, WAVES, RUNS> pages;
        int i = sp.first + wave;
        pages.begin(a.c, sp.s.first, i, lane);
        typename N::Keys k;
        typename N::Vals v;
        uint32_t there = ~0u;
        // Q in the order of the fragments: piece (t, i) of lane L is piece i of row 16 t + L % 16.
        auto* qs = reinterpret_cast<typename N::KPiece*>(lds);
        {
            typename N::KPiece z[N::kQ];
#pragma unroll
            for (int x = 0; x < N::kQ; ++x) {
                const int e = x * WAVES + wave, s = e % KS, t = min(e / KS, MT - 1);
                z[x] = N::piece((const T*)a.Q + q_at<PRE>(a, sp, row0 + 16 * t + col), 16 * q, s, q, D);
            }
            // (the first block's K and V right behind, before anything waits for Q)
            if (i < last) {
                there = pages.there(a.c, i);
                pages.template load_k<N>(k, a.c, kp, i, D, lane);
                pages.template load_v<N>(v, a.c, vp, i, D, lane);
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
            for (int x = 0; x < VS; ++x)
#pragma unroll
                for (int c = 0; c < VL; ++c) o[t][x][c] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        for (; i < last; i += WAVES) {
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
            const bool more = i + WAVES < last;
            if (more) pages.go(a.c, i + WAVES, lane);
            if (N::kAhead && more) pages.template load_k<N>(k, a.c, kp, i + WAVES, D, lane);
            __builtin_amdgcn_sched_barrier(0);
            const bool part = i < w0 || i >= w1 || there != below(KB);
            uint32_t see[MT];
            if (part) {
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    see[t] = seen<SUB>(i * KB, lo, attended<PRE>(a, sp, row0 + 16 * t + col), there, q);
                    hide<SUB>(p[t], see[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
                weights<SUB, VS, VL>(p[t], o[t], m[t], l[t], used[t], scale);
            // (behind the weights, whose rescaling by 0 would make NaN of an infinity)
            if (part && not_finite<T>(v)) spread_not_finite<T, N, MT>(o, v, see);
            N::accumulate(o, v, p, used);
            __builtin_amdgcn_sched_barrier(0);
            if (more) {
                there = pages.there(a.c, i + WAVES);
                if (!N::kAhead) pages.template load_k<N>(k, a.c, kp, i + WAVES, D, lane);
                pages.template load_v<N>(v, a.c, vp, i + WAVES, D, lane);
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
                xs[wave * N::ROWS + 16 * t + col] = make_float4(m[t], l[t], used[t], 0.f);
        }
        __syncthreads();  // (and Q is no longer read)
        float4* fin = xs + WAVES * N::ROWS;  // of each row: maximum, sums
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
        write_rows<T, PRE, DP, N::ROWS, WAVES, N::LDO, VL, MODE, 64 * WAVES>(a, sp, xo, fin);
    });
}

// The first workgroups take the prefixes' ranges (where those are tiles of as many rows), the others
// the sequences' own.
template <typename T, int DP, int MT, int MODE, bool RUNS>
__global__ __launch_bounds__(256, (PagedNarrow<T, DP, MT, MODE, 4>::kMinWaves)) void k_paged_narrow(
    PagedArgs a) {
    __shared__ __align__(16) char lds[PagedNarrow<T, DP, MT, MODE, 4>::kLds];
    const int id = (int)blockIdx.x - a.plan.first;
    if (id < 0)
        paged_narrow<T, DP, MT, MODE, RUNS, 4, 1>(a, blockIdx.x, lds);
    else
        paged_narrow<T, DP, MT, MODE, RUNS, 4, 0>(a, id, lds);
}
// Few whole items: 8 waves each (paged_plan).
template <typename T, int DP, int MT, int MODE, bool RUNS>
__global__ __launch_bounds__(512, 2) void k_paged_few(PagedArgs a) {
    __shared__ __align__(16) char lds[PagedNarrow<T, DP, MT, MODE, 8>::kLds];
    paged_narrow<T, DP, MT, MODE, RUNS, 8, 0>(a, blockIdx.x, lds);
}

// ---------------------------------------------------------------- parts
// The parts of a row added up, in their order: the prefix's, then its own.  A workgroup takes `each`
// rows a wave (or, WAVES = 4, `each` rows, whose parts its waves share) of one pair, whose place in
// the lines it finds once.  A launch and a chain of loads (groups, lengths, statistics, dims): 8 us for
// 256 rows, 11 to 17 for 1024 to 2048 of 10 to 17 parts, 29 where 32768 rows of two parts come back
// from memory.  With each part's dims asked for behind its statistics it took 1 to 6 us more.  Rows of
// one range and no prefix are written already.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void k_paged_merge(PagedArgs a, int each) {
    __shared__ float acc[4][256];
    __shared__ float2 sums[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int D = a.c.D;
    const unsigned pair = blockIdx.y, seq = pair / (unsigned)a.gs;
    const int b = (int)seq, lg = (int)(pair - seq * a.gs);
    const Groups gr = groups_of(a, lane);
    const Segment s = segment<0>(a, gr, b);
    const int rows = tokens_of(a, b) * a.rep;
    const int row0 = (WAVES == 4 ? blockIdx.x : blockIdx.x * 4 + wave) * each;
    if (row0 >= rows) return;
    const int group = of_wave(start_of(a, gr, b).y);
    if (group < 0 && !a.plan.own.split) return;
    Line own_line{}, pre_line{};
    Place own_place{}, pre_place{};
    Segment shared{};
    if (a.plan.own.split) {
        own_line = line_of<0>(a, gr, a.plan.own.kb, lane);
        own_place = place_of<0>(a, gr, own_line, b, a.plan.own.kb, lane);
    }
    if (group >= 0) {
        shared = segment<1>(a, gr, group);
        pre_line = line_of<1>(a, gr, a.plan.pre.kb, lane);
        pre_place = place_of<1>(a, gr, pre_line, group, a.plan.pre.kb, lane);
    }
    // the parts of an item: the first, and how many
    auto parts_of = [](const Line& line, const Place& p, int item) {
        const int first = p.start + item * p.n + kPagedPad;
        const int r0 = (unsigned)first / (unsigned)line.per;
        const int r1 = (unsigned)(first + p.n - kPagedPad - 1) / (unsigned)line.per;
        return make_int2(r0 + p.items + item, r1 - r0 + 1);
    };
#pragma unroll 1
    for (int row = row0; row < min(rows, row0 + each); ++row) {
        const int tok = over(row, a.by_rep), h = (a.g0 + lg) * a.rep + row - tok * a.rep;
        const int tile = row / a.plan.own.rows, in_tile = row - tile * a.plan.own.rows;
        int2 own = make_int2((b * a.gs + lg) * a.plan.own.tiles + tile, 1), pre = make_int2(0, 0);
        if (a.plan.own.split) own = parts_of(own_line, own_place, lg * s.tiles + tile);
        int pre_in = 0;
        if (group >= 0) {
            const int prow = (b - shared.first) * a.T * a.rep + row, ptile = prow / a.plan.pre.rows;
            pre_in = prow - ptile * a.plan.pre.rows;
            pre = parts_of(pre_line, pre_place, lg * shared.tiles + ptile);
        } else if (own.y == 1) {
            continue;
        }
        const int parts = pre.y + own.y;
        auto stats_of = [&](int i) {
            return i < pre.y
                       ? part_stats<1>(a)[part_row<1>(a, bounded(a.plan.pre, pre.x + i), pre_in)]
                       : part_stats<0>(a)[part_row<0>(a, bounded(a.plan.own, own.x + i - pre.y), in_tile)];
        };
        // (4 parts' dims are asked for at once, the first ones beside the statistics)
        constexpr int AT_ONCE = 4;
        const int i_first = WAVES == 4 ? wave : 0;
        float y[AT_ONCE][4];
        auto load = [&](int i0, int d0) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int i = min(i0 + WAVES * u, parts - 1);
                const float* from =
                    d0 + (i < pre.y ? part_dims<1>(a) +
                                          part_row<1>(a, bounded(a.plan.pre, pre.x + i), pre_in) * D
                                    : part_dims<0>(a) + part_row<0>(a, bounded(a.plan.own, own.x + i - pre.y),
                                                                    in_tile) * D);
#pragma unroll
                for (int c = 0; c < 4; ++c) y[u][c] = d0 + lane + 64 * c < D ? from[lane + 64 * c] : 0.f;
            }
        };
        const float4 mine = stats_of(min(lane, parts - 1));
        load(i_first, 256 * blockIdx.z);
        float M = mine.x;
        for (int i = lane + 64; i < parts; i += 64) M = fmaxf(M, stats_of(i).x);
        M = wave_max(M);
        const float base = base_of(M);
        T* out = (T*)a.out + b * a.os[0] + h * a.os[1] + tok * a.os[2];
#pragma unroll 1
        for (int d0 = 256 * blockIdx.z; d0 < D; d0 += 256 * gridDim.z) {
            float l = 0.f, used = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int i0 = i_first; i0 < parts; i0 += WAVES * AT_ONCE) {
                if (i0 > i_first || d0 > (int)(256 * blockIdx.z)) load(i0, d0);
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    const int i = i0 + WAVES * u;
                    if (i >= parts) break;
                    float4 z;
                    if (i < 64) {
                        z.x = __shfl(mine.x, i), z.y = __shfl(mine.y, i), z.z = __shfl(mine.z, i);
                    } else {
                        z = stats_of(i);
                    }
                    const float f = exp2_(z.x - base);
                    l += f * z.y;
                    used += f * z.z;
                    // (what is not finite stays so where the factor has vanished)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        x[c] += f == 0.f && !(fabsf(y[u][c]) < INFINITY) ? y[u][c] : f * y[u][c];
                }
            }
            if constexpr (WAVES == 4) {
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[wave][lane + 64 * c] = x[c];
                if (lane == 0) sums[wave] = make_float2(l, used);
                __syncthreads();
                l = (sums[0].x + sums[1].x) + (sums[2].x + sums[3].x);
                used = (sums[0].y + sums[1].y) + (sums[2].y + sums[3].y);
                const int d = threadIdx.x;
                const float sum = (acc[0][d] + acc[1][d]) + (acc[2][d] + acc[3][d]);
                if (d0 + d < D) Elem<T>::st(out, d0 + d, used == 0.f ? 0.f : sum * (1.f / used));
                __syncthreads();  // (for the next dims)
            } else {
                const float inv = 1.f / used;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (d0 + lane + 64 * c < D)
                        Elem<T>::st(out, d0 + lane + 64 * c, used == 0.f ? 0.f : x[c] * inv);
            }
            if (d0 == 0 && (WAVES == 4 ? threadIdx.x : lane) == 0 && a.lse)
                a.lse[((size_t)b * a.H + h) * a.T + tok] =
                    l == 0.f ? -INFINITY : (M + log2f(l)) * kLn2;
        }
    }
}

// ---------------------------------------------------------------- launches
template <typename T, int DP, int MT, int MODE>
void go_pages(const PagedArgs& a, dim3 grid, hipStream_t st) {
    if (a.c.page_rows % 16 == 0)
        hipLaunchKernelGGL((k_paged_narrow<T, DP, MT, MODE, true>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_paged_narrow<T, DP, MT, MODE, false>), grid, dim3(256), 0, st, a);
}
template <typename T, int DP, int MT, int MODE>
void go_few(const PagedArgs& a, dim3 grid, hipStream_t st) {
    if (a.c.page_rows % 16 == 0)
        hipLaunchKernelGGL((k_paged_few<T, DP, MT, MODE, true>), grid, dim3(512), 0, st, a);
    else
        hipLaunchKernelGGL((k_paged_few<T, DP, MT, MODE, false>), grid, dim3(512), 0, st, a);
}
template <typename T, int DP, int MODE>
void go_rows(const PagedArgs& a, dim3 grid, hipStream_t st) {
    if (a.plan.own.few && a.plan.own.rows == 16) return go_few<T, DP, 1, MODE>(a, grid, st);
    if constexpr (DP <= 128) {  // (paged_plan: their results in LDS)
        if (a.plan.own.few) return go_few<T, DP, 2, MODE>(a, grid, st);
    }
    if (a.plan.own.rows == 16) return go_pages<T, DP, 1, MODE>(a, grid, st);
    if (a.plan.own.rows == 32) return go_pages<T, DP, 2, MODE>(a, grid, st);
    if constexpr (DP == 64 && sizeof(T) == 2) go_pages<T, DP, 4, MODE>(a, grid, st);
}
template <typename T, int DP>
void go_dims(const PagedArgs& a, dim3 grid, hipStream_t st) {
    if (a.c.D == DP) return go_rows<T, DP, kExact>(a, grid, st);
    if constexpr (DP == 64) {
        if (a.c.D < 16 / (int)sizeof(T)) return go_rows<T, DP, kElem>(a, grid, st);
    }
    go_rows<T, DP, kClamp>(a, grid, st);
}
template <typename T>
void go_narrow(const PagedArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.plan.first + a.plan.own.workgroups));
    const int D = a.c.D;
    if (D <= 64) return go_dims<T, 64>(a, grid, st);
    if (D <= 128) return go_dims<T, 128>(a, grid, st);
    if (D <= 192) return go_dims<T, 192>(a, grid, st);
    go_dims<T, 256>(a, grid, st);
}
template <typename T>
void go_merge(const PagedArgs& a, hipStream_t st) {
    const int R = a.rep * a.T, chunks = (a.c.D + 255) / 256;
    const int64_t pairs = (int64_t)a.c.B * a.gs, rows = pairs * R;
    // (several rows and runs of dims each where there are more than the card holds waves)
    const unsigned z = (unsigned)std::min<int64_t>(chunks, std::max<int64_t>(1, 4096 / rows));
    if (rows >= 4096 || rows * chunks >= 16384) {
        const int each = (int)std::max<int64_t>(1, std::min<int64_t>(16, rows / 16384));
        const dim3 grid((unsigned)((R + 4 * each - 1) / (4 * each)), (unsigned)pairs, z);
        hipLaunchKernelGGL((k_paged_merge<T, 1>), grid, dim3(256), 0, st, a, each);
    } else {
        const dim3 grid((unsigned)R, (unsigned)pairs, z);
        hipLaunchKernelGGL((k_paged_merge<T, 4>), grid, dim3(256), 0, st, a, 1);
    }
}

}  // namespace
}  // namespace atn

// Argument views and launchers of the decoding operators: attention of
// drafted tokens over a key/value cache (tree_attn.hip), and the cache's
// commit, weights, eviction and lengths (kv_cache.hip).  The launchers
// validate nothing (the C-ABI layer does) and are asynchronous on `st`.
//
// Lengths live on the device, so that a captured graph replays with whatever
// they hold; the kernels clamp them to what the tensors hold, and no index
// read from device memory reaches an address unchecked.
#pragma once

#include "launch.hpp"

namespace atn {

constexpr int kTreeMaxTokens = 256;  // drafted tokens of a call, entries of a path

// K and V of [batch][kv head][row][head_d], strides in elements.
struct CacheView {
    void* K;
    void* V;
    int64_t ks[3], vs[3];  // batch, head, row
    const int* len;        // [B] rows in use
    float* weight;         // [B][G][cap]
    int* pos;              // [B][G][cap]
    int* seen;             // [B]
    int B, G, cap, D;
    int rows;              // bound of len (the capacity, or less where the call says so)
};

// Drafted tokens: Q [batch][head][token][head_d], K and V [batch][kv head][token][head_d].
struct DraftView {
    const void* Q;
    const void* K;
    const void* V;
    int64_t qs[3], ks[3], vs[3];  // batch, head, token
    const int* count;             // [B] tokens of each sequence, or null: T
    const uint32_t* mask;         // [B][T][W], or null: a chain
    int H, T, W;                  // W = ceil(T / 32)
    int rep;                      // heads of a kv head
    uint32_t by_t;                // 2^32 / T rounded up (T > 1)
};

// A query row of a kv head (its heads, each with T tokens): head and token of `row`.
__device__ __forceinline__ int head_of(const DraftView& d, int row) {
    return d.T == 1 ? row : (int)__umulhi((uint32_t)row, d.by_t);
}

// The drafts of each sequence that became part of it.
struct PathView {
    const int* path;      // [B][n] drafts, or null: 0, 1, ...
    const int* accepted;  // [B] entries of it that count, or null: all
    int n;
};

// Sums of the lanes up to each.
__device__ __forceinline__ int wave_scan(int x) {
#define ATN_SCAN_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xF, false)
    ATN_SCAN_STEP(0x111, 0xF);  // row_shr:1, 2, 4, 8 within 16 lanes
    ATN_SCAN_STEP(0x112, 0xF);
    ATN_SCAN_STEP(0x114, 0xF);
    ATN_SCAN_STEP(0x118, 0xF);
    ATN_SCAN_STEP(0x142, 0xA);  // row_bcast:15 into rows 1 and 3
    ATN_SCAN_STEP(0x143, 0xC);  // row_bcast:31 into rows 2 and 3
#undef ATN_SCAN_STEP
    return x;
}

// Rows in use of a sequence, and its drafts; of_wave: of one that the whole wave shares (the
// compiler keeps what follows from it in scalar registers only if told).
__device__ __forceinline__ int of_wave(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int rows_in_use(const CacheView& c, int b) {
    return min(max(c.len[b], 0), c.rows);
}
__device__ __forceinline__ int drafts_of(const DraftView& d, int b) {
    return d.count ? min(max(d.count[b], 0), d.T) : d.T;
}
// Drafts of sequence b that become rows of its cache: the path's entries up
// to the first that names no draft, as many as the cache still holds.  Every
// lane of a full wave calls it and gets the count.
__device__ __forceinline__ int rows_accepted(const CacheView& c, const DraftView& d,
                                             const PathView& p, int b) {
    const int n = drafts_of(d, b);
    int a = p.accepted ? min(max(p.accepted[b], 0), p.n) : p.n;
    if (!p.path) {
        a = min(a, n);
    } else {
        for (int i0 = 0; i0 < a; i0 += 64) {
            const int i = i0 + (int)(threadIdx.x & 63);
            const int t = i < a ? p.path[(size_t)b * p.n + i] : 0;
            const uint64_t bad = __builtin_amdgcn_ballot_w64(i < a && (t < 0 || t >= n));
            if (bad) {
                a = i0 + __builtin_ctzll(bad);
                break;
            }
        }
    }
    return min(a, c.cap - min(max(c.len[b], 0), c.cap));
}
// ... where `width` lanes (a power of two, `lane` of them) each have a sequence of their own: more
// than i exactly where draft i becomes a row.
__device__ __forceinline__ int rows_accepted_by(const CacheView& c, const DraftView& d,
                                                const PathView& p, int b, int i, int lane,
                                                int width) {
    const int n = drafts_of(d, b);
    int a = p.accepted ? min(max(p.accepted[b], 0), p.n) : p.n;
    a = min(a, c.cap - min(max(c.len[b], 0), c.cap));
    if (!p.path) return min(a, n);
    if (i >= a) return a;
    const int shift = (int)(threadIdx.x & 63) - lane;
    const uint64_t group = width == 64 ? ~0ull : (1ull << width) - 1;
    for (int j0 = 0; j0 <= i; j0 += width) {
        const int j = j0 + lane, t = j <= i ? p.path[(size_t)b * p.n + j] : 0;
        const uint64_t bad = __builtin_amdgcn_ballot_w64(t < 0 || t >= n) >> shift & group;
        if (bad && j0 + __builtin_ctzll(bad) <= i) return j0 + __builtin_ctzll(bad);
    }
    return a;
}
__device__ __forceinline__ int path_at(const PathView& p, int b, int i) {
    return p.path ? p.path[(size_t)b * p.n + i] : i;
}

// How a call runs (tree_plan): in passes over `seqs` sequences by `kv` kv heads (all of both
// unless the scratch would pass its limit), the blocks of keys of a pass dealt to `ranges`
// equal ranges, or a range per (sequence, kv head) where split is 0.
struct TreePlan {
    int rows;        // query rows of a tile
    int row_tiles;   // tiles of the query rows of one kv head
    int waves;       // of a workgroup (head_d <= 256)
    int split, turn; // ranges in whole turns of so many blocks
    int ranges;
    int seqs, kv;
    int ld_scores;   // head_d > 256: row of the scores, floats
    int shares;      // ... workgroups that share the dims of a tile of scores
    size_t scores;   // floats of the scores of a pass
    size_t scratch;  // bytes
    int64_t line;        // places of the line of blocks, at most
    int64_t workgroups;  // of a grid of one dimension, at most
};

struct TreeArgs {
    CacheView c;
    DraftView d;
    void* out;
    int64_t os[3];  // batch, head, token
    float* lse;     // [B][H][T] or null
    float scale;    // times log2(e)
    TreePlan plan;
    float* scores;  // scratch: [shares][pairs of a pass][rows of the tiles][ld_scores]
    float* part;    // scratch: parts of rows (2 of each range and tile): statistics, dims
    int b0, bs, g0, gs;  // this pass
};

// Whether draft t of sequence b (of n drafts) attends draft j.
__device__ __forceinline__ bool sees(const DraftView& d, int b, int t, int j) {
    if (!d.mask) return j <= t;
    return (d.mask[((size_t)b * d.T + t) * d.W + (j >> 5)] >> (j & 31)) & 1u;
}

// The plan depends on no device, so that workspace queries hold for any.
TreePlan tree_plan(int dtype, int B, int G, int H, int T, int D, int max_len, bool draft_keys,
                   size_t scratch_cap);
hipError_t launch_tree_attention(int dtype, TreeArgs a, hipStream_t st);

hipError_t launch_cache_commit(int dtype, const CacheView& c, const DraftView& d,
                               const PathView& p, hipStream_t st);
hipError_t launch_cache_weigh(int dtype, const CacheView& c, const DraftView& d,
                              const PathView& p, const float* lse, const float* weight_in,
                              float scale, hipStream_t st);
hipError_t launch_cache_advance(const CacheView& c, int* len, const DraftView* d,
                                const PathView& p, int limit, hipStream_t st);
size_t evict_scratch(int B, int G, int cap, int budget);
hipError_t launch_cache_evict(int dtype, const CacheView& c, int budget, int recent,
                              int* scratch, hipStream_t st);

}  // namespace atn

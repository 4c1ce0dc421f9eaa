// Argument views and launchers of the operators on a paged key/value cache: rotation of tokens by
// their positions and the append of their keys and values (rotary.hip), attention over the pages
// (paged_attn.hip).  The launchers validate nothing (the C-ABI layer does) and are asynchronous on
// `st`.  Lengths, page tables and prefixes are device memory; no index read from them reaches an
// address unchecked.
#pragma once

#include "kv_cache.hpp"

namespace atn {

// x / d for 0 <= x < 2^31: with l = ceil(log2 d) and m = ceil(2^(31 + l) / d), m d - 2^(31 + l) < d
// <= 2^l, so x m / 2^(31 + l) passes x / d by less than 1 / d.
struct Divider {
    uint32_t m;
    int shift;  // l - 1; -1: d = 1
};
inline Divider divider(int d) {
    int l = 0;
    while ((1ll << l) < d) ++l;
    if (l == 0) return {0, -1};
    return {(uint32_t)(((1ull << (31 + l)) + d - 1) / d), l - 1};
}
__device__ __forceinline__ int over(int x, Divider d) {
    return d.shift < 0 ? x : (int)(__umulhi((uint32_t)x, d.m) >> d.shift);
}

// K and V of [page][kv head][row][head_d], strides in elements.
struct PagedView {
    void* K;
    void* V;
    int64_t ks[3], vs[3];  // page, head, row
    const int* table;      // [B][slots] pages of a sequence
    int* len;              // [B] rows in use
    int B, G, D;
    int pages, page_rows, slots;
    int cap;   // rows of a table
    int rows;  // bound of the rows attended (cap, or less where the call says so)
    Divider by_page;
};

__device__ __forceinline__ int rows_in_use(const PagedView& c, int b) {
    return min(max(c.len[b], 0), c.cap);
}
// The table's entry for row r of sequence b (the last one's past its end).
__device__ __forceinline__ int page_of(const PagedView& c, int b, int r) {
    return c.table[(size_t)b * c.slots + min(over(r, c.by_page), c.slots - 1)];
}
__device__ __forceinline__ bool is_page(const PagedView& c, int page) {
    return (unsigned)page < (unsigned)c.pages;
}

// ---------------------------------------------------------------- rotation
struct RotaryView {
    const float* freq;  // [rot / 2] radians a position
    int half;           // pairs (i, i + rot / 2)
    int rot;            // 0: nothing is rotated
    float amplitude;
    float sign;         // -1: the inverse rotation
};
// Rows [b][head][token] read from `in` and written to `out`, or, where paged, to rows len + token of
// the cache's K or V (`out` and os its pool and strides).
struct RowJob {
    const void* in;
    void* out;
    int64_t is[3], os[3];
    int heads, rotate, paged;
    Divider by_heads;
};
struct RotaryArgs {
    PagedView c;        // jobs that are paged: len, table
    RotaryView r;
    RowJob job[3];
    int jobs;
    const int* pos;     // [B][T], or null: the row number in the cache, or t without one
    const int* count;   // [B], or null: T
    int B, T, D;
    int with_cache;
    Divider by_t, by_pairs;  // by_pairs: rot / 2
};
hipError_t launch_rotary(int dtype, const RotaryArgs& a, hipStream_t st);
hipError_t launch_paged_advance(const PagedView& c, const int* count, int T, hipStream_t st);

// ---------------------------------------------------------------- attention
// One of the two passes: the rows that groups of sequences share, and each sequence's own.
struct PagedPass {
    int many;        // 1: k_paged_many
    int kb;          // keys of a block
    int rows;        // query rows of a tile
    int part_rows;   // rows of a tile that any item has
    int tiles;       // tiles of a segment, at most
    int ranges;      // the line of blocks in so many ranges, or
    int split;       // ... 0: an item a workgroup
    int few;         // whole items of 8 waves each
    int turn;
    int groups;      // workgroups that share an item's dims (head_d > 256)
    int64_t items;   // at most
    int64_t parts;   // results kept in the scratch, at most
    int64_t workgroups;
    int64_t line;    // places, at most
    int64_t scores;  // floats (head_d > 256)
};
struct PagedPlan {
    PagedPass own, pre;
    int first;       // workgroups of a launch's grid that take the prefixes
    int seqs, kv;    // sequences (all, where there are groups) and kv heads of a launch
    int whole16;     // rows are whole 16-byte pieces that lie so
    int wide;        // head_d > 256:
    int shares;      // ... workgroups that share the dims of a block's scores
    unsigned score_grid;
    size_t scratch;  // bytes
};
struct PagedArgs {
    PagedView c;
    const void* Q;
    int64_t qs[3], os[3];
    void* out;
    float* lse;
    const int* count;
    int H, T, rep, es;    // es: bytes of an element
    Divider by_rep, by_t;
    float scale;          // times log2(e)
    const int* first;     // [groups + 1], or null
    const int* shared;    // [groups] rows
    int groups;
    PagedPlan plan;
    // scratch
    const int2* starts;   // [B] first row of a sequence's own, its group or -1; [B]: whether groups
                          // ascend; null: few groups
    float* own_scores;
    float* pre_scores;
    float* own_part;
    float* pre_part;
    int g0, gs;           // this launch's kv heads
};
// Whether reading `rows` shared rows once for m sequences saves anything.  It saves the other members' reads,
// 2 es head_d bytes a row and kv head; but every query row's result then passes through the scratch in two
// parts, 16 head_d bytes (5 sequences of 281 tokens of 16 heads over 4 of 8192 dims, 19 rows shared: 1209 us
// read as their own, 2335 read once).
__host__ __device__ __forceinline__ bool saves_reads(int64_t rows, int m, int es, int rep, int T) {
    return m >= 2 && rows * (m - 1) * es > (int64_t)m * rep * T * 8;
}
// whole16: the rows of K, V and Q are whole 16-byte pieces that lie so.
PagedPlan paged_plan(int dtype, const PagedView& c, int H, int T, int groups, bool whole16,
                     size_t scratch_cap);
hipError_t launch_paged_attention(int dtype, PagedArgs a, void* scratch, hipStream_t st);
// its parts: head_d <= 256, bf16 with many query rows, head_d > 256
hipError_t launch_paged_narrow_f32(const PagedArgs& a, hipStream_t st);
hipError_t launch_paged_narrow_bf16(const PagedArgs& a, hipStream_t st);
hipError_t launch_paged_many(const PagedArgs& a, int pre, hipStream_t st);
hipError_t launch_paged_wide(int dtype, const PagedArgs& a, hipStream_t st);

}  // namespace atn

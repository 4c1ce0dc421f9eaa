// How a call of attention over a paged cache runs, its launches, and the merge of its parts
// (paged_attn_impl.hpp).
#include "paged_attn_impl.hpp"

namespace atn {

namespace {

constexpr int kInWave = 64;  // groups that a wave's lanes hold

// Many groups: where each sequence's own rows begin, and its group, once for the kernels that follow;
// behind them, whether first ascends: then the last group that begins at or before b is the one.
__global__ __launch_bounds__(256) void k_paged_starts(PagedArgs a, int2* starts) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    int down = 0;
    for (int i = threadIdx.x; i < a.groups; i += 256) down |= a.first[i + 1] < a.first[i];
    down = __syncthreads_or(down);
    if (b > a.c.B) return;
    if (b == a.c.B || down) {
        starts[b] = b == a.c.B ? make_int2(!down, 0) : make_int2(0, -1);
        return;
    }
    int lo = 0, hi = a.groups;  // groups [0, lo) begin at or before b, [hi, groups) behind it
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.first[mid] <= b) lo = mid + 1;
        else hi = mid;
    }
    int2 x = make_int2(0, -1);
    if (lo > 0) {
        const Groups g = group_at(a, lo - 1);
        if (g.rows > 0 && b >= g.first && b < g.end) x = make_int2(g.rows, lo - 1);
    }
    starts[b] = x;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Which kernel takes items of about R query rows, and its tile.  runs: rows are whole 16-byte pieces, and
// pages whole runs of 16 rows.  pairs: of segments and kv heads;
// keys: of an item, at most; may_be_whole: a workgroup may take a whole item.
enum Kind { kNarrow, kMany, kWide };
struct Tile {
    Kind kind;
    int rows;
    int whole;  // kMany: items whole
};
Tile tile_of(int dtype, int D, int64_t R, int64_t pairs, int64_t keys, bool runs, bool may_be_whole) {
    const bool bf = dtype == kDtypeBF16;
    // (64 rows where they leave no more than a fourth more rows empty than 32 do)
    if (D > kPagedNarrow)
        return {kWide, R <= 16 ? 16 : R > 32 && 4 * (ceil_div(R, 64) * 64) <= 5 * (ceil_div(R, 32) * 32)
                                       ? 64 : 32, 0};
    if (bf && runs && D <= 128 && R > 32 && keys >= 512) {
        // The least estimated time of three tiles, with whole items a workgroup (one a CU) or with
        // items in ranges, whose parts go through memory and a merge: 0.97 PFLOP/s in tiles of 256 rows,
        // tiles of 128 and 64 take 1.33 and 1.45 times as long (they read K and V from LDS for fewer
        // rows), a merge 12 us and its parts twice at 4.5 TB/s.  512 tokens over 8000 rows, 2 sequences of
        // 32 over 8 heads: 179 us in ranges of 256 rows, 210 in whole items of 128; 256 over 1000, 4
        // sequences: 76 and 49.
        Tile best{kMany, 0, 0};
        double least = 0;
        for (int rows : {256, 128, 64}) {
            const int64_t items = pairs * ceil_div(R, rows), rounds = ceil_div(items, 256) * 256;
            const double work = (double)items * rows * keys * D * 4 / 0.97e9 *
                                (rows == 256 ? 1. : rows == 128 ? 1.33 : 1.45);
            const double whole = work * rounds / items;
            const double split = work + 12 + (double)pairs * R * D * 16 / 4.5e6;
            const double time = may_be_whole ? std::min(whole, split) : split;
            if (least == 0 || time < least) {
                least = time;
                best = {kMany, rows, may_be_whole && whole <= split};
            }
        }
        return best;
    }
    return {kNarrow, R <= 16 ? 16 : R <= 32 || !bf || D > 64 ? 32 : 64, 0};
}

// A pass of `segments` segments of at most `most` query rows of a kv head (all: of all segments), over
// at most `keys` keys an item; kv: kv heads of a launch.
PagedPass plan_pass(int dtype, int D, Tile t, int64_t most, int64_t segments, int64_t all, int64_t keys,
                    int kv, bool may_be_whole, bool alone) {
    PagedPass p{};
    const bool bf = dtype == kDtypeBF16;
    p.many = t.kind == kMany;
    p.rows = t.rows;
    p.groups = 1;
    const int mt = p.rows / 16;
    int subs = 1;  // workgroups that share an item's rows (head_d > 256)
    int per_cu;    // workgroups that a CU holds at once (the kernels' registers and LDS)
    if (t.kind == kMany) {
        per_cu = 1;
        p.kb = p.rows == 64 ? 128 : 64;
        p.turn = 1;
    } else if (t.kind == kWide) {
        per_cu = mt == 1 && !bf ? 3 : 2;  // (of the values)
        p.kb = kPagedWideBlock;
        p.turn = kPagedWideTurn;
        subs = std::max(1, p.rows / kPagedWideRows);
        p.groups = (int)ceil_div(D, bf ? kPagedWideDims : kPagedWideDims / 2) * subs;
    } else {
        per_cu = std::max(1, (mt == 1 ? 4 : mt == 2 ? 3 : 2) - (D > 64) - (D > 128));
        p.kb = bf ? 32 : 16;
        p.turn = 4;
    }
    p.part_rows = (int)std::min<int64_t>(p.rows, most);
    p.tiles = (int)ceil_div(most, p.rows);
    p.items = kv * std::min(segments * p.tiles, ceil_div(all, p.rows) + segments);
    const int64_t slots = std::max<int64_t>(1, 256 * per_cu / p.groups);
    const int64_t blocks = ceil_div(keys, p.kb) + 1;
    p.ranges = (int)std::max<int64_t>(
        1, std::min(slots, ceil_div(p.items * (blocks + kPagedPad), 2 * p.turn)));
    p.line = p.items * (blocks + kPagedPad) + 2ll * p.turn * p.ranges;
    p.split = !may_be_whole || (p.items < 4 * slots && blocks > 7 * p.turn / 2);
    if (p.many && may_be_whole) p.split = !t.whole;
    // Few items of short contexts: each whole, by a workgroup of 8 waves, where that is estimated to take
    // less than ranges and their merge (8 us), at most 1024 of them, 256 where 4 waves each would take
    // them whole too.  A CU reads 50 (fp32 38) GB/s of rows of whole tiles of dims, all of them
    // 5.2 TB/s; 1 MiB an item at most, since the host knows no lengths but the bound and one long
    // sequence alone takes its time.  One token of 32 over 8 heads of 128 bf16 dims: 600 rows 15.1 in
    // ranges, 10.8 whole; 1500 rows 14.7 and 18.6; 32 sequences of 500 to 1000 rows 31.8 and 22.4, 100
    // of 16 heads over 8 75.6 and 72.8; 64 of 300 rows 17 by 4 waves and 21 by 8.
    // Tiles of 32 rows up to 128 dims (8 waves' results of more pass LDS): 32 sequences of 6 tokens over
    // 500 to 1000 rows 39.0 and 25.9.
    if (t.kind == kNarrow && alone && (p.rows == 16 || (p.rows == 32 && D <= 128))) {
        const double dim = 2. * keys * (bf ? 2 : 4), item = dim * ceil_div(D, 64) * 64;
        p.few = p.items <= (p.split ? 1024 : 256) && item <= 1 << 20 &&
                item / (bf ? 50e3 : 38e3) <= 8 + dim * D * p.items / 5.2e6;
    }
    if (p.few) p.split = 0;
    p.parts = p.ranges + p.items;
    // whole items in several runs of dims a workgroup, where there are workgroups enough
    if (t.kind == kWide && !p.split)
        p.groups = subs * (int)std::min<int64_t>(p.groups / subs, std::max<int64_t>(
                              1, 4 * 256 * per_cu / (p.items * subs)));
    p.scores = t.kind == kWide ? p.items * blocks * p.rows * kPagedWideBlock : 0;
    return p;
}

size_t to16(size_t n) { return (n + 15) / 16 * 16; }
size_t starts_bytes(int B, int groups) { return groups > kInWave ? to16(((size_t)B + 1) * sizeof(int2)) : 0; }
size_t part_bytes(const PagedPass& p, int D) {
    return to16((size_t)p.parts * p.part_rows * (D + 4) * sizeof(float));
}

// ... of the sequences of c in one pass
PagedPlan plan_sequences(int dtype, const PagedView& c, int H, int T, int groups, bool whole16,
                         size_t scratch_cap) {
    PagedPlan p{};
    const int D = c.D;
    p.seqs = c.B;
    const int64_t R = (int64_t)(H / c.G) * T, all = R * c.B;
    const bool runs = whole16 && c.page_rows % 16 == 0;
    Tile own = tile_of(dtype, D, R, (int64_t)c.B * c.G, c.rows, runs, true), pre = own;
    if (groups > 0) {
        // (groups are on the device: tiles for groups of equal size)
        pre = tile_of(dtype, D, ceil_div(c.B, groups) * R, (int64_t)groups * c.G, c.rows, runs,
                      false);
        // Prefixes of many query rows beside sequences of few: a launch of k_paged_many, which begins
        // with 24 us more than nothing and reads at 4.5 TB/s, or tiles of 32 (64) rows in the launch of
        // the sequences' own, each of which reads the prefix again, at 6 TB/s (from L2 for the most):
        // 8192 rows shared by 32 sequences of 64 to 1024 rows of their own, 32 over 8 heads of 128 dims,
        // 56 against 63 us; 4 times 16384 shared by 16 each 123 against 108.
        const int narrow = D > 64 ? 32 : 64;
        const double bytes = (double)c.rows * groups * c.G * D * 4;
        if (pre.kind == kMany && own.kind == kNarrow &&
            ceil_div(ceil_div(c.B, groups) * R, narrow) * bytes / 6e6 < 24 + bytes / 4.5e6)
            pre = {kNarrow, narrow, 0};
        // one launch takes both, in tiles of as many rows
        // (head_d > 256: or own 16, prefixes 32)
        if (pre.kind == kWide && own.rows == 16) pre.rows = std::min(pre.rows, 32);
        else if (pre.kind != kMany) own.rows = pre.rows = std::max(own.rows, pre.rows);
    }
    p.wide = own.kind == kWide;
    p.whole16 = whole16;
    // all kv heads at once, unless the scratch does not hold their parts and scores
    for (p.kv = c.G;; p.kv = (p.kv + 1) / 2) {
        p.own = plan_pass(dtype, D, own, R, c.B, all, c.rows, p.kv, true, groups == 0);
        if (groups > 0) {
            p.pre = plan_pass(dtype, D, pre, all, groups, all, c.rows, p.kv, false, false);
            p.pre.workgroups = (int64_t)p.pre.ranges * p.pre.groups;
            p.first = pre.kind == kMany ? 0 : (int)p.pre.workgroups;
        }
        if (!p.own.split) p.own.parts = (int64_t)c.B * p.kv * p.own.tiles;
        p.own.workgroups =
            (p.own.split ? p.own.ranges : (int64_t)c.B * p.kv * p.own.tiles) * p.own.groups;
        // scores: two workgroups a CU, where the dims give each wave two steps still
        int64_t blocks = p.own.scores / (p.own.rows * kPagedWideBlock);
        if (groups > 0) blocks += p.pre.scores / (p.pre.rows * kPagedWideBlock);
        p.shares = 1;
        while (p.wide && blocks * p.shares < 512 && p.shares < 8 &&
               D >= 2 * p.shares * 8 * (dtype == kDtypeBF16 ? 256 : 128))
            p.shares *= 2;
        size_t rest = starts_bytes(c.B, groups);
        if (groups > 0) rest += part_bytes(p.pre, D);
        if (groups > 0 || p.own.split) rest += part_bytes(p.own, D);
        for (;; p.shares /= 2) {
            p.scratch = rest + (size_t)(p.own.scores + p.pre.scores) * p.shares * sizeof(float);
            // (each share's scores are apart: fewer shares before the call is refused)
            if (p.scratch <= scratch_cap || p.kv > 1 || p.shares == 1) break;
        }
        p.score_grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(blocks * p.shares, 1024));
        if (p.scratch <= scratch_cap || p.kv == 1) break;
    }
    // A prefix needs parts, of a tile of rows each, and another bound of the lengths may have larger tiles:
    // a workspace that was asked for with it holds a half or a fourth of the ranges.
    for (int i = 0; i < 2 && groups > 0 && p.scratch > scratch_cap; ++i)
        for (PagedPass* x : {&p.pre, &p.own}) {
            if (x == &p.own && !x->split) continue;
            p.scratch -= part_bytes(*x, D);
            x->ranges = (x->ranges + 1) / 2;
            x->parts = x->ranges + x->items;
            x->workgroups = (int64_t)x->ranges * x->groups;
            p.scratch += part_bytes(*x, D);
            if (x == &p.pre && p.first > 0) p.first = (int)x->workgroups;
        }
    if (p.scratch > scratch_cap && groups == 0 && p.own.split) {  // items whole: no parts
        p.scratch -= part_bytes(p.own, D);
        p.own.split = 0;
        p.own.workgroups = (int64_t)c.B * p.kv * p.own.tiles * p.own.groups;
    }
    return p;
}

}  // namespace

PagedPlan paged_plan(int dtype, const PagedView& c, int H, int T, int groups, bool whole16,
                     size_t scratch_cap) {
    PagedView x = c;
    PagedPlan p = plan_sequences(dtype, x, H, T, groups, whole16, scratch_cap);
    // (head_d > 256: the scores of a part of the sequences at a time)
    while (p.scratch > scratch_cap && groups == 0 && x.B > 1) {
        x.B = (x.B + 1) / 2;
        p = plan_sequences(dtype, x, H, T, groups, whole16, scratch_cap);
    }
    return p;
}

hipError_t launch_paged_attention(int dtype, PagedArgs a, void* scratch, hipStream_t st) {
    char* at = static_cast<char*>(scratch);
    if (a.groups > kInWave) {
        int2* starts = reinterpret_cast<int2*>(at);
        hipLaunchKernelGGL(k_paged_starts, dim3((unsigned)(a.c.B / 256 + 1)), dim3(256), 0, st, a,
                           starts);
        a.starts = starts;
        at += starts_bytes(a.c.B, a.groups);
    }
    a.own_scores = reinterpret_cast<float*>(at);
    at += (size_t)a.plan.own.scores * a.plan.shares * sizeof(float);
    a.pre_scores = reinterpret_cast<float*>(at);
    at += (size_t)a.plan.pre.scores * a.plan.shares * sizeof(float);
    if (a.groups > 0) {
        a.pre_part = reinterpret_cast<float*>(at);
        at += part_bytes(a.plan.pre, a.c.D);
    }
    a.own_part = reinterpret_cast<float*>(at);
    const PagedArgs all = a;
    for (int b0 = 0; b0 < all.c.B; b0 += a.plan.seqs) {
        a.c.B = std::min(a.plan.seqs, all.c.B - b0);
        a.c.table = all.c.table + (int64_t)b0 * a.c.slots;
        a.c.len = all.c.len + b0;
        a.count = all.count ? all.count + b0 : nullptr;
        a.Q = (const char*)all.Q + b0 * a.qs[0] * a.es;
        a.out = (char*)all.out + b0 * a.os[0] * a.es;
        a.lse = all.lse ? all.lse + (int64_t)b0 * a.H * a.T : nullptr;
        for (a.g0 = 0; a.g0 < a.c.G; a.g0 += a.plan.kv) {
            a.gs = std::min(a.plan.kv, a.c.G - a.g0);
            PagedArgs x = a;
            if (!x.plan.own.split)
                x.plan.own.workgroups = (int64_t)x.c.B * x.gs * x.plan.own.tiles * x.plan.own.groups;
            hipError_t e = hipGetLastError();
            if (e == hipSuccess && x.plan.wide) e = launch_paged_wide(dtype, x, st);
            if (e == hipSuccess && x.plan.pre.many) e = launch_paged_many(x, 1, st);
            if (e == hipSuccess && x.plan.own.many) e = launch_paged_many(x, 0, st);
            if (e == hipSuccess && !x.plan.wide && !x.plan.own.many)
                e = dtype == kDtypeF32 ? launch_paged_narrow_f32(x, st) : launch_paged_narrow_bf16(x, st);
            if (e == hipSuccess && (x.groups > 0 || x.plan.own.split)) {
                if (dtype == kDtypeF32)
                    go_merge<float>(x, st);
                else
                    go_merge<uint16_t>(x, st);
                e = hipGetLastError();
            }
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace atn

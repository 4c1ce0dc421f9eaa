// How a call of attention over a paged cache runs, and its launches (paged_attn_impl.hpp).
#include "paged_attn_impl.hpp"

namespace atn {

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A pass of `segments` segments of about R query rows of a kv head, at most `most` (all: of all
// segments), over at most `keys` keys an item; kv: kv heads of a launch.
PagedPass plan_pass(int dtype, int D, int64_t R, int64_t most, int64_t segments, int64_t all,
                    int64_t keys, int kv, bool whole16) {
    PagedPass p{};
    const bool bf = dtype == kDtypeBF16, wide = D > kPagedNarrow;
    p.many = bf && whole16 && D <= 128 && R > 32;
    int per_cu;  // workgroups that a CU holds at once (the kernels' registers and LDS)
    if (p.many) {
        // the tile that leaves the fewest rows empty, the larger of equals
        p.rows = 64;
        for (int rows : {128, 256})
            if (ceil_div(R, rows) * rows <= ceil_div(R, p.rows) * p.rows) p.rows = rows;
        per_cu = 1;
        p.kb = p.rows == 256 ? 64 : 128;
        p.turn = 1;
    } else {
        p.rows = R <= 16 ? 16 : R <= 32 || !bf || D > 64 ? 32 : 64;
        const int mt = p.rows / 16;
        per_cu = wide ? (mt == 1 ? 2 : 1)
                      : std::max(1, (mt == 1 ? 4 : mt == 2 ? 3 : 2) - (D > 64) - (D > 128));
        p.kb = wide ? kPagedWideKeys : bf ? 32 : 16;
        p.turn = wide ? 1 : 4;
    }
    p.part_rows = (int)std::min<int64_t>(p.rows, most);
    p.tiles = (int)ceil_div(most, p.rows);
    const int dims = D > 1024 ? 2048 : D > 512 ? 1024 : 512;
    p.groups = wide ? (int)ceil_div(D, dims) : 1;
    const int64_t items = kv * std::min(segments * p.tiles, ceil_div(all, p.rows) + segments);
    const int64_t slots = std::max<int64_t>(1, 256 * per_cu / p.groups);
    const int64_t blocks = ceil_div(keys, p.kb) + 1;
    p.ranges =
        (int)std::max<int64_t>(1, std::min(slots, ceil_div(items * (blocks + kPagedPad), 2 * p.turn)));
    p.line = items * (blocks + kPagedPad) + 2ll * p.turn * p.ranges;
    p.split = items < 4 * slots && blocks > 7 * p.turn / 2;
    p.parts = p.ranges + items;
    return p;
}

size_t paged_starts_bytes(int B) { return ((size_t)B * sizeof(int2) + 15) / 16 * 16; }
size_t part_bytes(const PagedPass& p, int D) {
    return ((size_t)p.parts * p.part_rows * (D + 4) * sizeof(float) + 15) / 16 * 16;
}

}  // namespace

PagedPlan paged_plan(int dtype, const PagedView& c, int H, int T, int groups, bool whole16,
                     size_t scratch_cap) {
    PagedPlan p{};
    const int64_t R = (int64_t)(H / c.G) * T, all = R * c.B;
    whole16 = whole16 && c.page_rows % 16 == 0;
    // all kv heads at once, unless the scratch does not hold their parts
    for (p.kv = c.G;; p.kv = (p.kv + 1) / 2) {
        p.own = plan_pass(dtype, c.D, R, R, c.B, all, c.rows, p.kv, whole16);
        p.scratch = 0;
        if (groups > 0) {
            // (groups are on the device: tiles for groups of equal size)
            p.pre = plan_pass(dtype, c.D, ceil_div(c.B, groups) * R, all, groups, all, c.rows, p.kv,
                              whole16);
            p.pre.split = 1;
            p.scratch = paged_starts_bytes(c.B) + part_bytes(p.pre, c.D);
        }
        if (!p.own.split) p.own.parts = (int64_t)c.B * p.kv * p.own.tiles;
        if (groups > 0 || p.own.split) p.scratch += part_bytes(p.own, c.D);
        p.own.workgroups =
            (p.own.split ? p.own.ranges : (int64_t)c.B * p.kv * p.own.tiles) * p.own.groups;
        if (p.scratch <= scratch_cap || p.kv == 1) break;
    }
    if (p.scratch > scratch_cap && groups == 0) {  // items whole: no parts
        p.own.split = 0;
        p.own.workgroups = (int64_t)c.B * p.kv * p.own.tiles * p.own.groups;
        p.scratch = 0;
    }
    return p;
}

hipError_t launch_paged_attention(int dtype, PagedArgs a, void* scratch, hipStream_t st) {
    char* at = static_cast<char*>(scratch);
    if (a.groups > 0) {
        a.starts = reinterpret_cast<int2*>(at);
        a.pre_part = reinterpret_cast<float*>(at += paged_starts_bytes(a.c.B));
        at += part_bytes(a.plan.pre, a.c.D);
    }
    a.own_part = reinterpret_cast<float*>(at);
    for (a.g0 = 0; a.g0 < a.c.G; a.g0 += a.plan.kv) {
        a.gs = std::min(a.plan.kv, a.c.G - a.g0);
        const hipError_t e = dtype == kDtypeF32 ? launch_paged_f32(a, st) : launch_paged_bf16(a, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace atn

// C ABI of serving from a paged key/value cache: argument checks and dispatch onto rotary.hip and
// paged_attn.hip.  Every check runs before any HIP call.
#include <hip/hip_runtime.h>

#include "../kernels/paged.hpp"
#include "checks.hpp"

namespace {

constexpr int64_t kMaxTokens = (int64_t)1 << 23;  // workgroups of one token: threads below 2^32

size_t size_of(int dtype) { return dtype == ATN_DTYPE_F32 ? 4 : 2; }
bool is_dtype(int dtype) { return dtype == ATN_DTYPE_F32 || dtype == ATN_DTYPE_BF16; }

// A checked tensor [n0][n1][n2][D].
struct Tensor {
    const void* p = nullptr;
    int64_t s[3] = {0, 0, 0};
    int n[3] = {0, 0, 0};
    int D = 0;
    size_t es = 0;
    Range r{0, 0};
};
int tensor(const void* p, const int64_t* given, int n0, int n1, int n2, int D, size_t es, bool distinct,
           Tensor* t) {
    t->p = p;
    t->n[0] = n0, t->n[1] = n1, t->n[2] = n2;
    t->D = D;
    t->es = es;
    return check_tensor(p, given, n0, n1, n2, D, es, distinct, t->s, &t->r);
}
bool same(const Tensor& a, const Tensor& b) {
    return a.p == b.p && a.n[1] == b.n[1] && a.s[0] == b.s[0] && a.s[1] == b.s[1] && a.s[2] == b.s[2];
}
// No element in common.  Elements of a and b in one place are whole numbers n_i in [lo_i, hi_i] of steps
// u_i, and of single elements (between -(D - 1) and D - 1), that add up to b's distance from a: sought
// from the largest step down, among the n_i that leave a rest which the smaller steps reach.  Strides
// that nest leave two or three of them a step; where there are more the tensors count as meeting.
struct Steps {
    int n = 0;
    int64_t u[6], lo[6], hi[6];
    int64_t reach_lo[7], reach_hi[7];  // of the steps from i on
    bool hit(int64_t distance, int i, int* tries) const {
        if (distance < reach_lo[i] || distance > reach_hi[i]) return false;
        if (i == n || --*tries < 0) return true;
        // n_i u_i in [distance - reach_hi[i + 1], distance - reach_lo[i + 1]]
        const int64_t from = distance - reach_hi[i + 1], to = distance - reach_lo[i + 1], d = u[i];
        const int64_t first = std::max(lo[i], from / d + (from % d > 0));
        const int64_t last = std::min(hi[i], to / d - (to % d < 0));
        if (last - first > 8) return true;
        for (int64_t k = first; k <= last; ++k)
            if (hit(distance - k * d, i + 1, tries)) return true;
        return false;
    }
};
bool apart(const Tensor& a, const Tensor& b) {
    if (!meet(a.r, b.r)) return true;
    const int64_t bytes = (const char*)b.p - (const char*)a.p, es = (int64_t)a.es;
    if (bytes % es) return false;
    Steps x;
    auto add = [&](int64_t u, int64_t lo, int64_t hi) {
        if (u == 0 || lo == hi) return;
        int i = x.n++;
        for (; i > 0 && x.u[i - 1] < u; --i)
            x.u[i] = x.u[i - 1], x.lo[i] = x.lo[i - 1], x.hi[i] = x.hi[i - 1];
        x.u[i] = u, x.lo[i] = lo, x.hi[i] = hi;
    };
    for (int i = 0; i < 3; ++i) {
        if (a.s[i] == b.s[i]) {
            add(a.s[i], 1 - b.n[i], a.n[i] - 1);
        } else {  // (0 where a dimension has one index)
            add(a.s[i], 0, a.n[i] - 1);
            add(b.s[i], 1 - b.n[i], 0);
        }
    }
    x.reach_lo[x.n] = 1 - b.D;
    x.reach_hi[x.n] = a.D - 1;
    for (int i = x.n - 1; i >= 0; --i) {
        x.reach_lo[i] = x.reach_lo[i + 1] + x.lo[i] * x.u[i];
        x.reach_hi[i] = x.reach_hi[i + 1] + x.hi[i] * x.u[i];
    }
    int tries = 256;
    return !x.hit(bytes / es, 0, &tries);
}

struct Pool {
    Tensor k, v;
};
int check_paged(const atn_paged_cache* c, atn::PagedView* v, Pool* p) {
    if (!c) return ATN_ERR_NULL_POINTER;
    if (!is_dtype(c->dtype)) return ATN_ERR_BAD_ARGUMENT;
    if (!c->K || !c->V || !c->table || !c->len) return ATN_ERR_NULL_POINTER;
    if (c->batch < 1 || c->kv_heads < 1 || c->pages < 1 || c->page_rows < 1 || c->table_pages < 1 ||
        c->head_d < 1)
        return ATN_ERR_BAD_DIMENSION;
    if (c->head_d > ATN_CACHE_MAX_HEAD_D) return ATN_ERR_BAD_ARGUMENT;
    if ((int64_t)c->batch * c->kv_heads > 65535 ||
        (int64_t)c->table_pages * c->page_rows > (int64_t)1 << 30)
        return ATN_ERR_SIZE_OVERFLOW;
    const size_t es = size_of(c->dtype);
    int st = tensor(c->K, c->k_stride, c->pages, c->kv_heads, c->page_rows, c->head_d, es, true, &p->k);
    if (st == ATN_OK)
        st = tensor(c->V, c->v_stride, c->pages, c->kv_heads, c->page_rows, c->head_d, es, true, &p->v);
    if (st != ATN_OK) return st;
    // (the kernels address 16 rows of a page by 32-bit byte offsets)
    if (std::max(p->k.s[2], p->v.s[2]) * (int64_t)es > kMaxRow) return ATN_ERR_SIZE_OVERFLOW;
    if (!aligned(c->table, 4) || !aligned(c->len, 4)) return ATN_ERR_MISALIGNED;
    v->K = c->K;
    v->V = c->V;
    for (int i = 0; i < 3; ++i) v->ks[i] = p->k.s[i], v->vs[i] = p->v.s[i];
    v->table = c->table;
    v->len = c->len;
    v->B = c->batch;
    v->G = c->kv_heads;
    v->D = c->head_d;
    v->pages = c->pages;
    v->page_rows = c->page_rows;
    v->slots = c->table_pages;
    v->cap = v->rows = c->table_pages * c->page_rows;
    v->by_page = atn::divider(c->page_rows);
    return ATN_OK;
}
Range table_range(const atn_paged_cache* c) {
    return range(c->table, (int64_t)c->batch * c->table_pages * 4);
}
Range ints(const void* p, int64_t n) { return range(p, p ? n * 4 : 0); }

int check_sizes(const atn_paged_cache* c, const atn_drafts* d) {
    if (!d) return ATN_ERR_NULL_POINTER;
    if (d->heads < 1 || d->tokens < 1) return ATN_ERR_BAD_DIMENSION;
    if (d->heads % c->kv_heads != 0 || d->tokens > ATN_PAGED_MAX_TOKENS || d->mask)
        return ATN_ERR_BAD_ARGUMENT;
    if (d->heads > 65535 || (int64_t)c->batch * d->tokens >= kMaxTokens ||
        (int64_t)c->batch * d->tokens * (d->heads / c->kv_heads) >= (int64_t)1 << 30)
        return ATN_ERR_SIZE_OVERFLOW;
    return aligned(d->count, 4) ? ATN_OK : ATN_ERR_MISALIGNED;
}

int check_rotary(const atn_rotary* r, int D, int inverse, atn::RotaryView* v) {
    *v = atn::RotaryView{};
    if (!r) return ATN_OK;
    if (r->pairing != ATN_ROPE_INTERLEAVED && r->pairing != ATN_ROPE_HALF) return ATN_ERR_BAD_ARGUMENT;
    const int rot = r->rotary_dim == 0 ? D : r->rotary_dim;
    if (rot % 2 || rot < 2 || rot > D) return ATN_ERR_BAD_ROTARY;
    if (!r->freq) return ATN_ERR_NULL_POINTER;
    if (!aligned(r->freq, 4)) return ATN_ERR_MISALIGNED;
    if (!std::isfinite(r->amplitude)) return ATN_ERR_BAD_ARGUMENT;
    v->freq = r->freq;
    v->half = r->pairing == ATN_ROPE_HALF;
    v->rot = rot;
    v->amplitude = r->amplitude == 0.f ? 1.f : r->amplitude;
    v->sign = inverse ? -1.f : 1.f;
    return ATN_OK;
}

bool pieces16(const void* p, const int64_t s[3], size_t es) {
    return aligned(p, 16) && s[0] * (int64_t)es % 16 == 0 && s[1] * (int64_t)es % 16 == 0 &&
           s[2] * (int64_t)es % 16 == 0;
}
atn::RowJob job(const Tensor& in, const Tensor& out, int rotate, int paged) {
    atn::RowJob j{};
    j.in = in.p;
    j.out = const_cast<void*>(out.p);
    for (int i = 0; i < 3; ++i) j.is[i] = in.s[i], j.os[i] = out.s[i];
    j.heads = in.n[1];
    j.by_heads = atn::divider(j.heads);
    j.rotate = rotate;
    j.paged = paged;
    return j;
}
int go_rotary(int dtype, atn::RotaryArgs* a, void* stream) {
    a->by_t = atn::divider(a->T);
    a->by_pairs = atn::divider(std::max(1, a->r.rot / 2));
    int dev;
    const int st = atn_host::device(&dev);
    if (st != ATN_OK) return st;
    return launched(atn::launch_rotary(dtype, *a, (hipStream_t)stream));
}

// The parts of an attention call that its size query needs too.
int check_attention(const atn_paged_cache* cache, const atn_drafts* d, const atn_shared_prefix* prefix,
                    int max_len, atn::PagedArgs* a, Pool* p, Tensor* q, bool* whole16) {
    int st = check_paged(cache, &a->c, p);
    if (st == ATN_OK) st = check_sizes(cache, d);
    if (st != ATN_OK) return st;
    if (!d->Q) return ATN_ERR_NULL_POINTER;
    st = tensor(d->Q, d->q_stride, cache->batch, d->heads, d->tokens, cache->head_d,
                size_of(cache->dtype), false, q);
    if (st != ATN_OK) return st;
    if (max_len < 0) return ATN_ERR_BAD_DIMENSION;
    if (max_len > 0) a->c.rows = std::min(max_len, a->c.cap);
    if (prefix) {
        if (prefix->groups < 1) return ATN_ERR_BAD_DIMENSION;
        if (prefix->groups > cache->batch) return ATN_ERR_BAD_ARGUMENT;
        if (!prefix->first || !prefix->rows) return ATN_ERR_NULL_POINTER;
        if (!aligned(prefix->first, 4) || !aligned(prefix->rows, 4)) return ATN_ERR_MISALIGNED;
        // (prompts are shared by two at least)
        a->groups = cache->batch > 1 ? prefix->groups : 0;
        a->first = prefix->first;
        a->shared = prefix->rows;
    }
    *whole16 = cache->head_d * q->es % 16 == 0 && pieces16(q->p, q->s, q->es) &&
               pieces16(p->k.p, p->k.s, q->es) && pieces16(p->v.p, p->v.s, q->es);
    a->Q = d->Q;
    for (int i = 0; i < 3; ++i) a->qs[i] = q->s[i];
    a->count = d->count;
    a->H = d->heads;
    a->T = d->tokens;
    a->rep = d->heads / cache->kv_heads;
    a->es = (int)q->es;
    a->by_rep = atn::divider(a->rep);
    a->by_t = atn::divider(a->T);
    return ATN_OK;
}

// Whether the launches hold the plan.  (A dimension of a grid has less than 2^32 threads, workgroups of at
// most 512.)
bool lays_out(const atn::PagedPlan& p, int groups) {
    return p.own.workgroups + p.first < 1 << 23 && p.own.line <= INT32_MAX &&
           (groups == 0 || p.pre.line <= INT32_MAX);
}
// How a call runs in `room` bytes of scratch.  A prefix that does not fit is left out, its rows read as
// the sequences' own, where no workspace that the library asks for would hold its parts, or where no group
// can have anything to save, whatever its rows; else a larger workspace is worth asking for.
void plan_call(int dtype, bool whole16, size_t room, atn::PagedArgs* a) {
    auto plan = [&](size_t bytes) {
        return atn::paged_plan(dtype, a->c, a->H, a->T, a->groups, whole16, bytes);
    };
    a->plan = plan(room);
    if (a->groups == 0) return;
    const size_t cap = atn_host::workspace_cap();
    if (lays_out(a->plan, a->groups) &&
        (a->plan.scratch <= room ||
         (atn::saves_reads(a->c.rows, a->c.B, a->es, a->rep, a->T) && plan(cap).scratch <= cap)))
        return;
    a->groups = 0;
    a->first = a->shared = nullptr;
    a->plan = plan(room);
}

}  // namespace

extern "C" {

int atn_rope_frequencies(float* freq, int rotary_dim, double base, const atn_rope_scaling* scaling,
                         float* amplitude) {
    if (!freq) return ATN_ERR_NULL_POINTER;
    if (rotary_dim < 2 || rotary_dim % 2) return ATN_ERR_BAD_ROTARY;
    if (!std::isfinite(base) || base <= 0.0) return ATN_ERR_BAD_ARGUMENT;
    const atn_rope_scaling s = scaling ? *scaling : atn_rope_scaling{};
    const int kind = s.kind;
    if (kind < ATN_ROPE_SCALE_NONE || kind > ATN_ROPE_SCALE_PARTS) return ATN_ERR_BAD_ARGUMENT;
    if (kind != ATN_ROPE_SCALE_NONE && !(std::isfinite(s.factor) && s.factor >= 1.0))
        return ATN_ERR_BAD_ARGUMENT;
    double low = s.low, high = s.high;
    if (kind == ATN_ROPE_SCALE_PARTS) {
        if (s.original < 1) return ATN_ERR_BAD_DIMENSION;
        if (low == 0.0 && high == 0.0) low = 1.0, high = 32.0;
        if (!(std::isfinite(high) && low < high)) return ATN_ERR_BAD_ARGUMENT;
    }
    // (of two dims, whose one pair does not change with the base)
    if (kind == ATN_ROPE_SCALE_BASE && rotary_dim > 2)
        base *= std::pow(s.factor, (double)rotary_dim / (rotary_dim - 2));
    for (int i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rotary_dim);
        if (kind == ATN_ROPE_SCALE_LINEAR) f /= s.factor;
        if (kind == ATN_ROPE_SCALE_PARTS) {
            const double turns = s.original * f / 6.283185307179586;
            const double keep = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
            f = f * keep + f / s.factor * (1.0 - keep);
        }
        freq[i] = (float)f;
    }
    if (amplitude)
        *amplitude = kind == ATN_ROPE_SCALE_PARTS ? (float)(1.0 + 0.1 * std::log(s.factor)) : 1.f;
    return ATN_OK;
}

int atn_rotary_ex(int dtype, const atn_rotary* rotary, const atn_rotated* x, int n, int batch,
                  int tokens, int head_d, const int32_t* pos, int inverse, void* stream) {
    if (!is_dtype(dtype)) return ATN_ERR_BAD_ARGUMENT;
    if (!rotary || !x) return ATN_ERR_NULL_POINTER;
    if (n < 1 || batch < 1 || tokens < 1 || head_d < 1) return ATN_ERR_BAD_DIMENSION;
    if (n > 3 || head_d > ATN_CACHE_MAX_HEAD_D) return ATN_ERR_BAD_ARGUMENT;
    if ((int64_t)batch * tokens >= kMaxTokens) return ATN_ERR_SIZE_OVERFLOW;
    atn::RotaryArgs a{};
    int st = check_rotary(rotary, head_d, inverse, &a.r);
    if (st != ATN_OK) return st;
    if (!aligned(pos, 4)) return ATN_ERR_MISALIGNED;
    const size_t es = size_of(dtype);
    Tensor in[3], out[3];
    for (int i = 0; i < n; ++i) {
        if (!x[i].in || !x[i].out) return ATN_ERR_NULL_POINTER;
        if (x[i].heads < 1) return ATN_ERR_BAD_DIMENSION;
        if (x[i].heads > 65535) return ATN_ERR_SIZE_OVERFLOW;
        st = tensor(x[i].in, x[i].in_stride, batch, x[i].heads, tokens, head_d, es, false, &in[i]);
        if (st == ATN_OK)
            st = tensor(x[i].out, x[i].out_stride, batch, x[i].heads, tokens, head_d, es, true, &out[i]);
        if (st != ATN_OK) return st;
        a.job[i] = job(in[i], out[i], 1, 0);
    }
    for (int i = 0; i < n; ++i) {
        if (meet(out[i].r, ints(pos, (int64_t)batch * tokens)) ||
            meet(out[i].r, ints(rotary->freq, a.r.rot / 2)))
            return ATN_ERR_ALIASING;
        for (int j = 0; j < n; ++j) {
            if (!(i == j && same(out[i], in[i])) && !apart(out[i], in[j])) return ATN_ERR_ALIASING;
            if (j < i && !apart(out[i], out[j])) return ATN_ERR_ALIASING;
        }
    }
    a.jobs = n;
    a.pos = pos;
    a.B = batch;
    a.T = tokens;
    a.D = head_d;
    return go_rotary(dtype, &a, stream);
}

int atn_paged_append_ex(const atn_paged_cache* cache, const atn_drafts* d, const atn_rotary* rotary,
                        const int32_t* pos, void* q_out, const int64_t* q_out_stride, void* stream) {
    atn::RotaryArgs a{};
    Pool p;
    int st = check_paged(cache, &a.c, &p);
    if (st == ATN_OK) st = check_sizes(cache, d);
    if (st != ATN_OK) return st;
    if (!d->K || !d->V || (q_out && !d->Q)) return ATN_ERR_NULL_POINTER;
    const int B = cache->batch, G = cache->kv_heads, T = d->tokens, D = cache->head_d;
    st = check_rotary(rotary, D, 0, &a.r);
    if (st != ATN_OK) return st;
    if (!aligned(pos, 4)) return ATN_ERR_MISALIGNED;
    const size_t es = size_of(cache->dtype);
    Tensor q, qo, k, v;
    if (q_out) {
        st = tensor(d->Q, d->q_stride, B, d->heads, T, D, es, false, &q);
        if (st == ATN_OK) st = tensor(q_out, q_out_stride, B, d->heads, T, D, es, true, &qo);
        if (st != ATN_OK) return st;
    }
    st = tensor(d->K, d->k_stride, B, G, T, D, es, false, &k);
    if (st == ATN_OK) st = tensor(d->V, d->v_stride, B, G, T, D, es, false, &v);
    if (st != ATN_OK) return st;
    const Range lists[5] = {table_range(cache), ints(cache->len, B), ints(d->count, B),
                            ints(pos, (int64_t)B * T), ints(rotary ? rotary->freq : nullptr, a.r.rot / 2)};
    if (!apart(p.k, p.v)) return ATN_ERR_ALIASING;
    for (const Range& w : {p.k.r, p.v.r, qo.r})
        for (const Range& o : lists)
            if (meet(w, o)) return ATN_ERR_ALIASING;
    for (const Range& w : {p.k.r, p.v.r})
        for (const Range& o : {q.r, qo.r, k.r, v.r})
            if (meet(w, o)) return ATN_ERR_ALIASING;
    if (q_out) {
        if (!same(q, qo) && !apart(qo, q)) return ATN_ERR_ALIASING;
        if (!apart(qo, k) || !apart(qo, v)) return ATN_ERR_ALIASING;
        // (queries that nothing turns and that stay where they are: nothing to do)
        if (rotary || !same(q, qo)) a.job[a.jobs++] = job(q, qo, rotary != nullptr, 0);
    }
    a.job[a.jobs++] = job(k, p.k, rotary != nullptr, 1);
    a.job[a.jobs++] = job(v, p.v, 0, 1);
    a.pos = pos;
    a.count = d->count;
    a.B = B;
    a.T = T;
    a.D = D;
    a.with_cache = 1;
    return go_rotary(cache->dtype, &a, stream);
}

int atn_paged_advance_ex(const atn_paged_cache* cache, const atn_drafts* d, void* stream) {
    atn::PagedView c;
    Pool p;
    int st = check_paged(cache, &c, &p);
    if (st == ATN_OK) st = check_sizes(cache, d);
    if (st != ATN_OK) return st;
    if (meet(ints(cache->len, cache->batch), ints(d->count, cache->batch))) return ATN_ERR_ALIASING;
    int dev;
    st = atn_host::device(&dev);
    if (st != ATN_OK) return st;
    return launched(atn::launch_paged_advance(c, d->count, d->tokens, (hipStream_t)stream));
}

size_t atn_paged_attention_workspace_bytes(const atn_paged_cache* cache, const atn_drafts* tokens,
                                           const atn_shared_prefix* prefix, int max_len) {
    atn::PagedArgs a{};
    Pool p;
    Tensor q;
    bool whole16;
    if (check_attention(cache, tokens, prefix, max_len, &a, &p, &q, &whole16) != ATN_OK) return 0;
    const size_t cap = atn_host::workspace_cap();
    // Parts follow the tiles, which may be larger with a smaller bound of the lengths; and a prefix that this
    // bound leaves out may fit with a smaller one.  What is asked for serves them too.
    size_t most = 0;
    for (int rows = a.c.rows; rows >= 1; rows /= 2) {
        atn::PagedArgs x = a;
        x.c.rows = rows;
        plan_call(cache->dtype, whole16, cap, &x);
        most = std::max(most, x.plan.scratch);
        if (a.groups == 0) break;
        if (x.groups == 0 && atn::saves_reads(rows, x.c.B, x.es, x.rep, x.T)) most = std::max(most, cap);
    }
    return kSyncRegion + most;
}

int atn_paged_attention_ex(const atn_paged_cache* cache, const atn_drafts* tokens,
                           const atn_shared_prefix* prefix, void* out, const int64_t* out_stride,
                           float* lse, float scale, int max_len, void* workspace,
                           size_t workspace_bytes, void* stream) {
    atn::PagedArgs a{};
    Pool p;
    Tensor q, o;
    bool whole16;
    int st = check_attention(cache, tokens, prefix, max_len, &a, &p, &q, &whole16);
    if (st != ATN_OK) return st;
    if (!out) return ATN_ERR_NULL_POINTER;
    const int B = cache->batch;
    st = tensor(out, out_stride, B, a.H, a.T, a.c.D, q.es, true, &o);
    if (st != ATN_OK) return st;
    for (int i = 0; i < 3; ++i) a.os[i] = o.s[i];
    if (!aligned(lse, 4)) return ATN_ERR_MISALIGNED;
    const Range rl = range(lse, lse ? (int64_t)B * a.H * a.T * 4 : 0);
    if (any_meet({o.r, rl}, {p.k.r, p.v.r, q.r, table_range(cache), ints(cache->len, B),
                             ints(a.count, B), ints(a.first, a.groups + 1), ints(a.shared, a.groups)}))
        return ATN_ERR_ALIASING;
    st = check_scale(scale, a.c.D, &a.scale);
    if (st != ATN_OK) return st;
    a.out = out;
    a.lse = lse;
    size_t room = atn_host::workspace_cap();
    if (workspace != nullptr) {
        if (workspace_bytes < kSyncRegion) return ATN_ERR_WORKSPACE;
        room = workspace_bytes - kSyncRegion;
    }
    plan_call(cache->dtype, whole16, room, &a);
    if (!lays_out(a.plan, a.groups)) return ATN_ERR_SIZE_OVERFLOW;
    if (a.plan.scratch > room) return ATN_ERR_WORKSPACE;
    int dev;
    st = atn_host::device(&dev);
    if (st != ATN_OK) return st;
    void* ws;
    st = scratch(a.plan.scratch, workspace, workspace_bytes, (hipStream_t)stream, &ws);
    if (st != ATN_OK) return st;
    return launched(atn::launch_paged_attention(cache->dtype, a, ws, (hipStream_t)stream));
}

}  // extern "C"

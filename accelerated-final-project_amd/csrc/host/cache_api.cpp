// C ABI of decoding over a key/value cache: argument checks and dispatch onto
// tree_attn.hip and kv_cache.hip.  Every check runs before any HIP call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../kernels/kv_cache.hpp"
#include "attn_mi355x.h"
#include "host.hpp"

namespace {

using atn_host::kSyncRegion;

static_assert(ATN_TREE_MAX_TOKENS == atn::kTreeMaxTokens, "token limit");

constexpr int64_t kMaxRow = (int64_t)1 << 27;  // bytes from a row of K or V to the next

bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

// Bytes [lo, hi) that a call reads or writes.
struct Range {
    uintptr_t lo, hi;
};
Range range(const void* p, int64_t bytes) { return {(uintptr_t)p, (uintptr_t)p + (uint64_t)bytes}; }
bool meet(const Range& a, const Range& b) { return a.lo < b.hi && b.lo < a.hi; }

// A strided tensor [n0][n1][n2][D]: resolves all-zero strides to contiguous ones
// and gives its extent.  `distinct`: no two elements may share an address.
int check_tensor(const void* p, const int64_t* given, int n0, int n1, int n2, int D, size_t es,
                 bool distinct, int64_t out[3], Range* r) {
    if (!aligned(p, es)) return ATN_ERR_MISALIGNED;
    const int n[3] = {n0, n1, n2};
    int64_t s[3] = {0, 0, 0};
    if (given)
        for (int i = 0; i < 3; ++i) s[i] = given[i];
    constexpr int64_t kMax = INT64_MAX / 16;
    if (s[0] == 0 && s[1] == 0 && s[2] == 0) {
        s[2] = D;
        s[1] = s[2] * n2;
        if (s[1] > kMax / n1) return ATN_ERR_SIZE_OVERFLOW;
        s[0] = s[1] * n1;
    }
    int64_t last = D;
    for (int i = 0; i < 3; ++i) {
        if (s[i] < 0) return ATN_ERR_BAD_ARGUMENT;
        if (n[i] > 1 && s[i] > kMax / (n[i] - 1)) return ATN_ERR_SIZE_OVERFLOW;
        last += s[i] * (n[i] - 1);
        if (last > kMax) return ATN_ERR_SIZE_OVERFLOW;
    }
    if (distinct) {
        // from the smallest stride up, each dimension steps over all below it
        int o[3] = {0, 1, 2};
        std::sort(o, o + 3, [&](int a, int b) { return s[a] < s[b]; });
        int64_t extent = D;
        for (int i : o) {
            if (n[i] == 1) continue;
            if (s[i] < extent) return ATN_ERR_BAD_ARGUMENT;
            extent += s[i] * (n[i] - 1);
        }
    }
    for (int i = 0; i < 3; ++i) out[i] = n[i] == 1 ? 0 : s[i];
    *r = range(p, last * (int64_t)es);
    return ATN_OK;
}

struct Ranges {
    Range k, v, qd, kd, vd;
};

int check_cache(const atn_kv_cache* c, atn::CacheView* v, Ranges* r) {
    if (!c) return ATN_ERR_NULL_POINTER;
    if (c->dtype != ATN_DTYPE_F32 && c->dtype != ATN_DTYPE_BF16) return ATN_ERR_BAD_ARGUMENT;
    if (!c->K || !c->V || !c->len) return ATN_ERR_NULL_POINTER;
    if (c->batch < 1 || c->kv_heads < 1 || c->capacity < 1 || c->head_d < 1)
        return ATN_ERR_BAD_DIMENSION;
    if (c->head_d > ATN_CACHE_MAX_HEAD_D) return ATN_ERR_BAD_ARGUMENT;
    // (grids have a (sequence, kv head) per y; row numbers and steps past them are ints)
    if ((int64_t)c->batch * c->kv_heads > 65535 || c->capacity > 1 << 30) return ATN_ERR_SIZE_OVERFLOW;
    const size_t es = c->dtype == ATN_DTYPE_F32 ? 4 : 2;
    int st = check_tensor(c->K, c->k_stride, c->batch, c->kv_heads, c->capacity, c->head_d, es,
                          true, v->ks, &r->k);
    if (st == ATN_OK)
        st = check_tensor(c->V, c->v_stride, c->batch, c->kv_heads, c->capacity, c->head_d, es,
                          true, v->vs, &r->v);
    if (st != ATN_OK) return st;
    // (the kernels address the 32 rows of a block by 32-bit byte offsets)
    if (std::max(v->ks[2], v->vs[2]) * (int64_t)es > kMaxRow) return ATN_ERR_SIZE_OVERFLOW;
    for (const void* p : {(const void*)c->len, (const void*)c->seen, (const void*)c->weight,
                          (const void*)c->pos})
        if (!aligned(p, 4)) return ATN_ERR_MISALIGNED;
    v->K = c->K;
    v->V = c->V;
    v->len = c->len;
    v->weight = c->weight;
    v->pos = c->pos;
    v->seen = c->seen;
    v->B = c->batch;
    v->G = c->kv_heads;
    v->cap = c->capacity;
    v->D = c->head_d;
    v->rows = c->capacity;
    return ATN_OK;
}

// need_q, need_kv: the call reads the queries; keys and values must be given
int check_drafts(const atn_kv_cache* c, const atn_drafts* d, bool need_q, bool need_kv,
                 atn::DraftView* v, Ranges* r) {
    if (!d) return ATN_ERR_NULL_POINTER;
    if (d->heads < 1 || d->tokens < 1) return ATN_ERR_BAD_DIMENSION;
    if (d->heads % c->kv_heads != 0 || d->tokens > ATN_TREE_MAX_TOKENS) return ATN_ERR_BAD_ARGUMENT;
    if (need_q && !d->Q) return ATN_ERR_NULL_POINTER;
    if ((d->K == nullptr) != (d->V == nullptr) || (need_kv && !d->K)) return ATN_ERR_NULL_POINTER;
    const size_t es = c->dtype == ATN_DTYPE_F32 ? 4 : 2;
    *v = atn::DraftView{};
    r->qd = r->kd = r->vd = Range{0, 0};
    int st = ATN_OK;
    if (need_q)
        st = check_tensor(d->Q, d->q_stride, c->batch, d->heads, d->tokens, c->head_d, es, false,
                          v->qs, &r->qd);
    if (st == ATN_OK && d->K)
        st = check_tensor(d->K, d->k_stride, c->batch, c->kv_heads, d->tokens, c->head_d, es, false,
                          v->ks, &r->kd);
    if (st == ATN_OK && d->V)
        st = check_tensor(d->V, d->v_stride, c->batch, c->kv_heads, d->tokens, c->head_d, es, false,
                          v->vs, &r->vd);
    if (st != ATN_OK) return st;
    if (std::max(v->ks[2], v->vs[2]) * (int64_t)es > kMaxRow) return ATN_ERR_SIZE_OVERFLOW;
    if (!aligned(d->count, 4) || !aligned(d->mask, 4)) return ATN_ERR_MISALIGNED;
    v->Q = need_q ? d->Q : nullptr;
    v->K = d->K;
    v->V = d->V;
    v->count = d->count;
    v->mask = d->mask;
    v->H = d->heads;
    v->rep = d->heads / c->kv_heads;
    v->T = d->tokens;
    v->W = (d->tokens + 31) / 32;
    v->by_t = d->tokens > 1 ? (uint32_t)(((1ull << 32) + d->tokens - 1) / d->tokens) : 0;
    // (rows of a kv head times tokens below 2^32: the division by multiplication is exact)
    if ((int64_t)v->rep * d->tokens >= (1 << 24)) return ATN_ERR_SIZE_OVERFLOW;
    return ATN_OK;
}

int check_path(const int32_t* path, const int32_t* accepted, int path_len, atn::PathView* p) {
    if (path_len < 1) return ATN_ERR_BAD_DIMENSION;
    if (path_len > ATN_TREE_MAX_TOKENS) return ATN_ERR_BAD_ARGUMENT;
    if (!aligned(path, 4) || !aligned(accepted, 4)) return ATN_ERR_MISALIGNED;
    *p = atn::PathView{path, accepted, path_len};
    return ATN_OK;
}

// 1 / sqrtf(head_d) for 0, in units of log2
int check_scale(float scale, int D, float* out) {
    if (!std::isfinite(scale)) return ATN_ERR_BAD_ARGUMENT;
    if (scale == 0.f) scale = 1.f / std::sqrt((float)D);
    *out = scale * 1.4426950408889634f;
    return std::isnormal(*out) ? ATN_OK : ATN_ERR_BAD_ARGUMENT;
}

// lengths count up to max_len (0: the capacity)
int bound_rows(int max_len, atn::CacheView* c) {
    if (max_len < 0) return ATN_ERR_BAD_DIMENSION;
    if (max_len > 0) c->rows = std::min(max_len, c->cap);
    return ATN_OK;
}

// Scratch behind the sync region of the caller's workspace or the library's.
int scratch(size_t need, void* workspace, size_t workspace_bytes, hipStream_t stream, void** out) {
    *out = nullptr;
    if (need == 0) return ATN_OK;
    if (workspace != nullptr) {
        if (workspace_bytes < kSyncRegion + need) return ATN_ERR_WORKSPACE;
        if (!aligned(workspace, 16)) return ATN_ERR_MISALIGNED;
    } else {
        const int st = atn_host::workspace(kSyncRegion + need, stream, &workspace);
        if (st != ATN_OK) return st;
    }
    *out = static_cast<char*>(workspace) + kSyncRegion;
    return ATN_OK;
}

int launched(hipError_t e) { return e == hipSuccess ? ATN_OK : atn_host::fail(e); }

bool any_meet(std::initializer_list<Range> writes, std::initializer_list<Range> others) {
    for (auto w = writes.begin(); w != writes.end(); ++w) {
        for (const Range& o : others)
            if (meet(*w, o)) return true;
        for (auto x = w + 1; x != writes.end(); ++x)
            if (meet(*w, *x)) return true;
    }
    return false;
}

atn::TreePlan plan_tree(const atn::CacheView& c, const atn::DraftView& d, int dtype, size_t cap) {
    return atn::tree_plan(dtype, c.B, c.G, d.H, d.T, c.D, c.rows, d.K != nullptr, cap);
}

}  // namespace

extern "C" {

size_t atn_tree_attention_workspace_bytes(const atn_kv_cache* cache, const atn_drafts* drafts,
                                          int max_len) {
    atn::CacheView c;
    atn::DraftView d;
    Ranges r;
    if (check_cache(cache, &c, &r) != ATN_OK ||
        check_drafts(cache, drafts, true, false, &d, &r) != ATN_OK ||
        bound_rows(max_len, &c) != ATN_OK)
        return 0;
    return kSyncRegion + plan_tree(c, d, cache->dtype, atn_host::workspace_cap()).scratch;
}

int atn_tree_attention_ex(const atn_kv_cache* cache, const atn_drafts* drafts, void* out,
                          const int64_t* out_stride, float* lse, float scale, int max_len,
                          void* workspace, size_t workspace_bytes, void* stream) {
    atn::TreeArgs a{};
    Ranges r;
    int st = check_cache(cache, &a.c, &r);
    if (st != ATN_OK) return st;
    st = check_drafts(cache, drafts, true, false, &a.d, &r);
    if (st != ATN_OK) return st;
    if (!out) return ATN_ERR_NULL_POINTER;
    const size_t es = cache->dtype == ATN_DTYPE_F32 ? 4 : 2;
    Range ro, rl{0, 0};
    st = check_tensor(out, out_stride, a.c.B, a.d.H, a.d.T, a.c.D, es, true, a.os, &ro);
    if (st != ATN_OK) return st;
    if (!aligned(lse, 4)) return ATN_ERR_MISALIGNED;
    if (lse) rl = range(lse, (int64_t)a.c.B * a.d.H * a.d.T * 4);
    if (any_meet({ro, rl}, {r.k, r.v, r.qd, r.kd, r.vd})) return ATN_ERR_ALIASING;
    st = check_scale(scale, a.c.D, &a.scale);
    if (st == ATN_OK) st = bound_rows(max_len, &a.c);
    if (st != ATN_OK) return st;
    a.out = out;
    a.lse = lse;
    size_t room = atn_host::workspace_cap();
    if (workspace != nullptr) {
        if (workspace_bytes < kSyncRegion) return ATN_ERR_WORKSPACE;
        room = workspace_bytes - kSyncRegion;
    }
    a.plan = plan_tree(a.c, a.d, cache->dtype, room);
    // (a dimension of a grid has less than 2^32 threads; workgroups of at most 512)
    if (a.plan.workgroups >= 1 << 23 || a.plan.line > INT32_MAX) return ATN_ERR_SIZE_OVERFLOW;
    if (workspace != nullptr && a.plan.scratch > room) return ATN_ERR_WORKSPACE;
    int dev;
    st = atn_host::device(&dev);
    if (st != ATN_OK) return st;
    void* ws;
    st = scratch(a.plan.scratch, workspace, workspace_bytes, (hipStream_t)stream, &ws);
    if (st != ATN_OK) return st;
    a.scores = static_cast<float*>(ws);
    a.part = a.scores + a.plan.scores;
    return launched(atn::launch_tree_attention(cache->dtype, a, (hipStream_t)stream));
}

int atn_cache_commit_ex(const atn_kv_cache* cache, const atn_drafts* drafts, const int32_t* path,
                        const int32_t* accepted, int path_len, void* stream) {
    atn::CacheView c;
    atn::DraftView d;
    atn::PathView p;
    Ranges r;
    int st = check_cache(cache, &c, &r);
    if (st != ATN_OK) return st;
    st = check_drafts(cache, drafts, false, true, &d, &r);
    if (st != ATN_OK) return st;
    st = check_path(path, accepted, path_len, &p);
    if (st != ATN_OK) return st;
    if (c.pos && !c.seen) return ATN_ERR_NULL_POINTER;
    if (c.K == c.V || any_meet({r.k}, {r.kd, r.vd}) || any_meet({r.v}, {r.kd, r.vd}))
        return ATN_ERR_ALIASING;
    const int64_t mb = (int64_t)c.B * c.G * c.cap * 4;
    if (any_meet({range(c.weight, c.weight ? mb : 0), range(c.pos, c.pos ? mb : 0)},
                 {r.k, r.v, r.kd, r.vd}))
        return ATN_ERR_ALIASING;
    int dev;
    st = atn_host::device(&dev);
    if (st != ATN_OK) return st;
    return launched(atn::launch_cache_commit(cache->dtype, c, d, p, (hipStream_t)stream));
}

int atn_cache_weigh_ex(const atn_kv_cache* cache, const atn_drafts* drafts, const float* lse,
                       const int32_t* path, const int32_t* accepted, int path_len,
                       const float* weight_in, float scale, int max_len, void* stream) {
    atn::CacheView c;
    atn::DraftView d;
    atn::PathView p;
    Ranges r;
    int st = check_cache(cache, &c, &r);
    if (st != ATN_OK) return st;
    st = check_drafts(cache, drafts, true, false, &d, &r);
    if (st != ATN_OK) return st;
    st = check_path(path, accepted, path_len, &p);
    if (st != ATN_OK) return st;
    if (!lse || !c.weight) return ATN_ERR_NULL_POINTER;
    // (a query row per head and path entry)
    if ((int64_t)d.rep * path_len >= (1 << 24)) return ATN_ERR_SIZE_OVERFLOW;
    if (!aligned(lse, 4) || !aligned(weight_in, 4)) return ATN_ERR_MISALIGNED;
    const int64_t wb = (int64_t)c.B * c.G * c.cap * 4;
    const Range rw = range(c.weight, wb);
    if (any_meet({rw}, {r.k, r.v, r.qd, range(lse, (int64_t)c.B * d.H * d.T * 4)}))
        return ATN_ERR_ALIASING;
    // in place, or apart
    if (weight_in && weight_in != c.weight && meet(rw, range(weight_in, wb)))
        return ATN_ERR_ALIASING;
    float s = 0.f;
    st = check_scale(scale, c.D, &s);
    if (st == ATN_OK) st = bound_rows(max_len, &c);
    if (st != ATN_OK) return st;
    int dev;
    st = atn_host::device(&dev);
    if (st != ATN_OK) return st;
    return launched(atn::launch_cache_weigh(cache->dtype, c, d, p, lse, weight_in, s,
                                            (hipStream_t)stream));
}

size_t atn_cache_evict_workspace_bytes(const atn_kv_cache* cache, int budget) {
    atn::CacheView c;
    Ranges r;
    if (check_cache(cache, &c, &r) != ATN_OK || budget < 1) return 0;
    return kSyncRegion + atn::evict_scratch(c.B, c.G, c.cap, budget);
}

int atn_cache_evict_ex(const atn_kv_cache* cache, int budget, int recent, void* workspace,
                       size_t workspace_bytes, void* stream) {
    atn::CacheView c;
    Ranges r;
    int st = check_cache(cache, &c, &r);
    if (st != ATN_OK) return st;
    if (!c.weight || !c.pos || !c.seen) return ATN_ERR_NULL_POINTER;
    if (budget < 1) return ATN_ERR_BAD_DIMENSION;
    if (recent < 0 || recent > budget) return ATN_ERR_BAD_ARGUMENT;
    const int64_t mb = (int64_t)c.B * c.G * c.cap * 4;
    if (c.K == c.V || any_meet({range(c.weight, mb), range(c.pos, mb)}, {r.k, r.v}))
        return ATN_ERR_ALIASING;
    int dev;
    st = atn_host::device(&dev);
    if (st != ATN_OK) return st;
    void* ws;
    st = scratch(atn::evict_scratch(c.B, c.G, c.cap, budget), workspace, workspace_bytes,
                 (hipStream_t)stream, &ws);
    if (st != ATN_OK) return st;
    return launched(atn::launch_cache_evict(cache->dtype, c, budget, recent,
                                            static_cast<int*>(ws), (hipStream_t)stream));
}

int atn_cache_advance_ex(const atn_kv_cache* cache, const atn_drafts* drafts,
                         const int32_t* path, const int32_t* accepted, int path_len, int limit,
                         void* stream) {
    atn::CacheView c;
    atn::DraftView d{};
    atn::PathView p{};
    Ranges r;
    int st = check_cache(cache, &c, &r);
    if (st != ATN_OK) return st;
    if (limit < 0) return ATN_ERR_BAD_DIMENSION;
    if (drafts) {
        st = check_drafts(cache, drafts, false, false, &d, &r);
        if (st != ATN_OK) return st;
        st = check_path(path, accepted, path_len, &p);
        if (st != ATN_OK) return st;
    } else if (limit == 0) {
        return ATN_ERR_BAD_ARGUMENT;  // nothing to do
    }
    int dev;
    st = atn_host::device(&dev);
    if (st != ATN_OK) return st;
    return launched(atn::launch_cache_advance(c, cache->len, drafts ? &d : nullptr, p, limit,
                                              (hipStream_t)stream));
}

}  // extern "C"

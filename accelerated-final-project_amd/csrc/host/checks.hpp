// Argument checks that the calls on caches share.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "attn_mi355x.h"
#include "host.hpp"

namespace {

using atn_host::kSyncRegion;

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

// 1 / sqrtf(head_d) for 0, in units of log2
int check_scale(float scale, int D, float* out) {
    if (!std::isfinite(scale)) return ATN_ERR_BAD_ARGUMENT;
    if (scale == 0.f) scale = 1.f / std::sqrt((float)D);
    *out = scale * 1.4426950408889634f;
    return std::isnormal(*out) ? ATN_OK : ATN_ERR_BAD_ARGUMENT;
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

}  // namespace

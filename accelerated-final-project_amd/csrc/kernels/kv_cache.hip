// The key/value cache of a decoding program: accepted drafts written into it,
// eviction of the lightest rows, and its lengths.
#include <algorithm>

#include "kv_cache.hpp"

namespace atn {

namespace {

// One row of D elements by one wave, `vec` elements (16 bytes) at a time
// where both rows allow it.
template <typename T>
__device__ __forceinline__ void copy_row(T* __restrict__ dst, const T* __restrict__ src, int D,
                                         bool vec, int lane) {
    constexpr int N = 16 / sizeof(T);
    if (vec) {
        for (int d = lane * N; d < D; d += 64 * N)
            *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(src + d);
    } else {
        for (int d = lane; d < D; d += 64) dst[d] = src[d];
    }
}

// One wave per accepted row and kv head.  Nothing to compute: a chain of
// latencies (lengths, path, row).
template <typename T>
__global__ __launch_bounds__(256) void k_commit(CacheView c, DraftView d, PathView p, int vec) {
    const int lane = threadIdx.x & 63;
    const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (long)c.B * c.G * p.n) return;
    const int i = (int)(id % p.n), g = (int)((id / p.n) % c.G), b = (int)(id / p.n / c.G);
    const int A = rows_accepted(c, d, p, b);
    if (i >= A) return;
    const int row = rows_in_use(c, b) + i, t = path_at(p, b, i);
    copy_row((T*)c.K + b * c.ks[0] + g * c.ks[1] + row * c.ks[2],
             (const T*)d.K + b * d.ks[0] + g * d.ks[1] + t * d.ks[2], c.D, vec, lane);
    copy_row((T*)c.V + b * c.vs[0] + g * c.vs[1] + row * c.vs[2],
             (const T*)d.V + b * d.vs[0] + g * d.vs[1] + t * d.vs[2], c.D, vec, lane);
    const size_t m = ((size_t)b * c.G + g) * c.cap + row;
    if (lane == 0 && c.weight) c.weight[m] = 0.f;
    if (lane == 0 && c.pos) c.pos[m] = c.seen[b] + i;
}

__global__ __launch_bounds__(64) void k_advance(CacheView c, int* len, DraftView d, PathView p,
                                                int add, int limit) {
    const int b = blockIdx.x;
    int L = rows_in_use(c, b);
    const int A = add ? rows_accepted(c, d, p, b) : 0;
    if (threadIdx.x == 0) {
        L += A;
        len[b] = limit > 0 ? min(L, limit) : L;
        if (c.seen && add) c.seen[b] += A;
    }
}

// ---------------------------------------------------------------- eviction
// Rank of a row as an unsigned key: recent rows above all, then weights in
// their order (-0 as 0), NaN below all.
__device__ __forceinline__ uint32_t rank_key(float w, int pos, int since) {
    if (pos >= since) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One workgroup per (sequence, kv head): the key of rank `budget` by three
// histograms of its digits (11, 11 and 10 bits), then the rows below it that
// leave slots under `budget` free and the kept rows from `budget` on, in
// order, as the lists of moves.
// scratch: [B G] counts, then [B G][slots][2] (to, from).
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

__global__ __launch_bounds__(kSelThreads) void k_evict_select(CacheView c, int budget, int recent,
                                                              int slots, int* scratch) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t wsum[kSelWaves];
    __shared__ uint32_t pick[2];
    __shared__ int cnt[3][kSelWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bg = blockIdx.x, b = bg / c.G;
    const int L = rows_in_use(c, b);
    if (L <= budget) {
        if (tid == 0) scratch[bg] = 0;
        return;
    }
    const float* w = c.weight + (size_t)bg * c.cap;
    const int* pos = c.pos + (size_t)bg * c.cap;
    // (a position is at least seen - recent; in 64 bits, so that no difference wraps)
    const long lo = (long)c.seen[b] - recent;
    const int since = lo < INT32_MIN ? INT32_MIN : (int)lo;
    uint32_t prefix = 0, mask = 0, need = (uint32_t)budget;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t bins = pass == 2 ? 1024 : 2048;
        for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int r = tid; r < L; r += kSelThreads) {
            const uint32_t k = rank_key(w[r], pos[r], since);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        // thread t holds bins 2047 - 2t and 2046 - 2t: sums from the top down
        const uint32_t h0 = hist[2047 - 2 * tid], h1 = hist[2046 - 2 * tid];
        uint32_t s = h0 + h1;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = __shfl_up(s, o);
            if (lane >= o) s += v;
        }
        if (lane == 63) wsum[wave] = s;
        __syncthreads();
        uint32_t above = s - h0 - h1;
        for (int i = 0; i < wave; ++i) above += wsum[i];
        if (above < need && need <= above + h0 + h1) {
            const bool first = need <= above + h0;
            pick[0] = 2047 - 2 * tid - (first ? 0 : 1);
            pick[1] = need - above - (first ? 0 : h0);
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        mask |= (bins - 1) << shift;
        need = pick[1];  // rows of this prefix that stay
        __syncthreads();
    }
    // rows with the key `prefix` stay up to the need-th; each wave takes a
    // consecutive part of the rows
    const int per = ((L + kSelWaves - 1) / kSelWaves + 63) / 64 * 64;
    const int r0 = wave * per, r1 = min(L, r0 + per);
    int eq = 0;
    for (int r = r0 + lane; r < r0 + per; r += 64)
        eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(
            r < r1 && rank_key(w[r], pos[r], since) == prefix));
    if (lane == 0) cnt[0][wave] = eq;
    __syncthreads();
    int eq0 = 0;
    for (int i = 0; i < wave; ++i) eq0 += cnt[0][i];
    const uint64_t below = (1ull << lane) - 1;
    int to = 0, from = 0;
    for (int round = 0; round < 2; ++round) {
        int e = eq0;
        for (int r = r0 + lane; r < r0 + per; r += 64) {
            const bool on = r < r1;
            const uint32_t k = on ? rank_key(w[r], pos[r], since) : 0u;
            const uint64_t same = __builtin_amdgcn_ballot_w64(on && k == prefix);
            const bool keep =
                on && (k > prefix ||
                       (k == prefix &&
                        e + __builtin_popcountll(same & below) < (int)need));
            e += __builtin_popcountll(same);
            const uint64_t free_ = __builtin_amdgcn_ballot_w64(on && !keep && r < budget);
            const uint64_t move = __builtin_amdgcn_ballot_w64(keep && r >= budget);
            if (round) {
                int* list = scratch + c.B * c.G + (size_t)bg * slots * 2;
                if (on && !keep && r < budget)
                    list[2 * (to + __builtin_popcountll(free_ & below))] = r;
                if (keep && r >= budget)
                    list[2 * (from + __builtin_popcountll(move & below)) + 1] = r;
            }
            to += __builtin_popcountll(free_);
            from += __builtin_popcountll(move);
        }
        if (round == 0) {
            if (lane == 0) cnt[1][wave] = to, cnt[2][wave] = from;
            __syncthreads();
            if (tid == 0) {
                int n = 0;
                for (int i = 0; i < kSelWaves; ++i) n += cnt[1][i];
                scratch[bg] = n;
            }
            to = from = 0;
            for (int i = 0; i < wave; ++i) to += cnt[1][i], from += cnt[2][i];
        }
    }
}

// One wave per move, the moves of a head dealt to gridDim.x workgroups.
// Sources lie at or past `budget`, targets below it: no order among them.
template <typename T>
__global__ __launch_bounds__(256) void k_evict_move(CacheView c, int slots, const int* scratch,
                                                    int vec) {
    const int lane = threadIdx.x & 63, bg = blockIdx.y, g = bg % c.G, b = bg / c.G;
    const int n = min(scratch[bg], slots);
    const int* list = scratch + c.B * c.G + (size_t)bg * slots * 2;
    T* K = (T*)c.K + b * c.ks[0] + g * c.ks[1];
    T* V = (T*)c.V + b * c.vs[0] + g * c.vs[1];
    for (int i = blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += gridDim.x * 4) {
        const int to = list[2 * i], from = list[2 * i + 1];
        copy_row(K + to * c.ks[2], K + from * c.ks[2], c.D, vec, lane);
        copy_row(V + to * c.vs[2], V + from * c.vs[2], c.D, vec, lane);
        const size_t m = (size_t)bg * c.cap;
        if (lane == 0) c.weight[m + to] = c.weight[m + from];
        if (lane == 0) c.pos[m + to] = c.pos[m + from];
    }
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool rows16(const void* p, const int64_t s[3], int D, size_t es) {
    if (!al16(p) || (D * es) % 16) return false;
    for (int i = 0; i < 3; ++i)
        if ((s[i] * (int64_t)es) % 16) return false;
    return true;
}

}  // namespace

hipError_t launch_cache_commit(int dtype, const CacheView& c, const DraftView& d,
                               const PathView& p, hipStream_t st) {
    const size_t es = dtype == kDtypeF32 ? 4 : 2;
    const int vec = rows16(c.K, c.ks, c.D, es) && rows16(c.V, c.vs, c.D, es) &&
                    rows16(d.K, d.ks, c.D, es) && rows16(d.V, d.vs, c.D, es);
    const dim3 grid((unsigned)(((long)c.B * c.G * p.n + 3) / 4));
    if (dtype == kDtypeF32)
        hipLaunchKernelGGL(k_commit<float>, grid, dim3(256), 0, st, c, d, p, vec);
    else
        hipLaunchKernelGGL(k_commit<uint16_t>, grid, dim3(256), 0, st, c, d, p, vec);
    return hipGetLastError();
}

hipError_t launch_cache_advance(const CacheView& c, int* len, const DraftView* d,
                                const PathView& p, int limit, hipStream_t st) {
    hipLaunchKernelGGL(k_advance, dim3(c.B), dim3(64), 0, st, c, len, d ? *d : DraftView{}, p,
                       d != nullptr, limit);
    return hipGetLastError();
}

size_t evict_scratch(int B, int G, int cap, int budget) {
    const size_t slots = (size_t)std::max(0, std::min(budget, cap - budget));
    return ((size_t)B * G * (1 + 2 * slots)) * sizeof(int);
}

hipError_t launch_cache_evict(int dtype, const CacheView& c, int budget, int recent, int* scratch,
                              hipStream_t st) {
    const int slots = std::min(budget, c.cap - budget);
    if (slots <= 0) return hipSuccess;  // no row can lie past the budget
    const size_t es = dtype == kDtypeF32 ? 4 : 2;
    const int vec = rows16(c.K, c.ks, c.D, es) && rows16(c.V, c.vs, c.D, es);
    const int BG = c.B * c.G;
    hipLaunchKernelGGL(k_evict_select, dim3(BG), dim3(kSelThreads), 0, st, c, budget, recent,
                       slots, scratch);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)std::max(1, std::min((slots + 3) / 4, 8192 / std::min(BG, 8192))),
                    (unsigned)BG);
    if (dtype == kDtypeF32)
        hipLaunchKernelGGL(k_evict_move<float>, grid, dim3(256), 0, st, c, slots, scratch, vec);
    else
        hipLaunchKernelGGL(k_evict_move<uint16_t>, grid, dim3(256), 0, st, c, slots, scratch, vec);
    return hipGetLastError();
}

}  // namespace atn

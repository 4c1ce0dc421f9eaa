// The key/value cache of a decoding program: accepted drafts written into it,
// eviction of the lightest rows, and its lengths.
#include <algorithm>
#include <type_traits>

#include "kv_cache.hpp"

namespace atn {

namespace {

// A K row and a V row of D elements copied by `width` lanes, 16 bytes at a time where all of
// them lie so (vec); four loads go out before the first store.
template <typename T>
__device__ __forceinline__ void copy_rows(T* __restrict__ k, const T* __restrict__ k0,
                                          T* __restrict__ v, const T* __restrict__ v0, int D,
                                          bool vec, int lane, int width) {
    constexpr int N = 16 / sizeof(T);
    if (vec) {
        for (int d = lane * N; d < D; d += 2 * width * N) {
            const int e = d + width * N;
            const bool two = e < D;
            const uint4 a = *reinterpret_cast<const uint4*>(k0 + d);
            const uint4 b = *reinterpret_cast<const uint4*>(v0 + d);
            uint4 x{}, y{};
            if (two) {
                x = *reinterpret_cast<const uint4*>(k0 + e);
                y = *reinterpret_cast<const uint4*>(v0 + e);
            }
            *reinterpret_cast<uint4*>(k + d) = a;
            *reinterpret_cast<uint4*>(v + d) = b;
            if (two) {
                *reinterpret_cast<uint4*>(k + e) = x;
                *reinterpret_cast<uint4*>(v + e) = y;
            }
        }
    } else {
        for (int d = lane; d < D; d += width) {
            const T a = k0[d], b = v0[d];
            k[d] = a;
            v[d] = b;
        }
    }
}

// `width` lanes per accepted row and kv head: a row of D elements in 16-byte pieces, a power of
// two up to a wave.  Nothing to compute: a chain of latencies (lengths, path, row) for few rows
// (2.7 us), the copy for many (272 rows of 8 kv heads of 1024 fp32 dims: 36 MB in 9.6 us).
template <typename T>
__global__ __launch_bounds__(256) void k_commit(CacheView c, DraftView d, PathView p, int vec,
                                                int width) {
    const int lane = threadIdx.x & (width - 1);
    const long id = ((long)blockIdx.x * 256 + threadIdx.x) / width;
    const bool on = id < (long)c.B * c.G * p.n;
    const int row_id = (int)(on ? id : 0), i = row_id % p.n, g = row_id / p.n % c.G;
    const int b = row_id / p.n / c.G;
    // (the rows of a wave may be of several sequences)
    const int A = rows_accepted_by(c, d, p, b, i, lane, width);
    if (!on || i >= A) return;
    const int row = rows_in_use(c, b) + i, t = path_at(p, b, i);
    copy_rows((T*)c.K + b * c.ks[0] + g * c.ks[1] + row * c.ks[2],
              (const T*)d.K + b * d.ks[0] + g * d.ks[1] + t * d.ks[2],
              (T*)c.V + b * c.vs[0] + g * c.vs[1] + row * c.vs[2],
              (const T*)d.V + b * d.vs[0] + g * d.vs[1] + t * d.vs[2], c.D, vec, lane, width);
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
// scratch: [B G] counts, then (at an even place) [B G][slots][2] (to, from).
__host__ __device__ inline int list_at(int pairs) { return (pairs + 1) & ~1; }
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

// The sum over the waves below this one, and over all, of a value per wave (two barriers).
__device__ __forceinline__ int below_waves(int* slot, int x, int wave, int lane, int* all) {
    if (lane == 0) slot[wave] = x;
    __syncthreads();
    const int upto = wave_scan(lane < kSelWaves ? slot[lane] : 0);
    __syncthreads();
    *all = __builtin_amdgcn_readlane(upto, 63);
    return __builtin_amdgcn_readlane(upto, wave) - x;
}

// Moves first, first + step, ... of n of a head, `width` lanes each.  Sources lie at or past
// `budget`, targets below it: no order among them.
template <typename T>
__device__ __forceinline__ void move_rows(const CacheView& c, int bg, const int* list, int n,
                                          int first, int step, int vec, int lane, int width) {
    const int g = bg % c.G, b = bg / c.G;
    T* K = (T*)c.K + b * c.ks[0] + g * c.ks[1];
    T* V = (T*)c.V + b * c.vs[0] + g * c.vs[1];
    const size_t m = (size_t)bg * c.cap;
    for (int i = first; i < n; i += step) {
        const int to = list[2 * i], from = list[2 * i + 1];
        float w = 0.f;
        int p = 0;
        if (lane == 0) w = c.weight[m + from], p = c.pos[m + from];
        copy_rows(K + to * c.ks[2], K + from * c.ks[2], V + to * c.vs[2], V + from * c.vs[2], c.D, vec,
                  lane, width);
        if (lane == 0) c.weight[m + to] = w, c.pos[m + to] = p;
    }
}

// KPT keys a thread come from memory at once and stay in LDS, each read by its own thread alone: a
// wave's are 64 KPT consecutive rows.  Heads of more than 1024 KPT rows go through it in chunks,
// read again for each digit (KPT = 16, 16384 rows a chunk).  One read of little
// data: what bounds it is the code, fetched as the launch runs through it, so the loops stay loops
// (KPT = 16: 7.7 KB, 18 us for 32 heads of 12000 to 16384 rows; 19 KB with keys in registers,
// 21.5 us; one load after another 44 us.  KPT = 1: 2.5 KB and 6 us against 7.6 KB and 8 us.
// Several copies of a histogram, for weights that share their first digit: 4 us more).
// T: the workgroup moves the rows itself, where a head has few of them (a cache that is cut
// whenever it is a little over its bound): a second launch takes longer than they do (58 of 570
// rows at most: 10.7 against 14.2 us, both with a copy that restores the cache).  void: it leaves
// them to k_evict_move.
template <int KPT, typename T>
__global__ __launch_bounds__(kSelThreads) void k_evict_select(CacheView c, int budget, int recent,
                                                              int slots, int* scratch, int vec,
                                                              int width) {
    constexpr int CHUNK = kSelThreads * KPT;
    __shared__ uint32_t keys[CHUNK];
    __shared__ uint32_t hist[2048];
    __shared__ int slot[kSelWaves];
    __shared__ uint32_t pick[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = of_wave(tid >> 6);
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
    const int chunks = (L + CHUNK - 1) / CHUNK, mine = wave * 64 * KPT + lane;
    auto load = [&](int chunk) {
        float x[KPT];
        int y[KPT];
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
            const int r = min(chunk * CHUNK + mine + 64 * k, L - 1);
            x[k] = w[r];
            y[k] = pos[r];
        }
#pragma unroll
        for (int k = 0; k < KPT; ++k) keys[mine + 64 * k] = rank_key(x[k], y[k], since);
    };
    for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    uint32_t prefix = 0, mask = 0, need = (uint32_t)budget;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t bins = pass == 2 ? 1024 : 2048;
#pragma unroll 1
        for (int chunk = 0; chunk < chunks; ++chunk) {
            if (pass == 0 || chunks > 1) load(chunk);
#pragma unroll 4
            for (int k = 0; k < KPT; ++k) {
                const uint32_t key = keys[mine + 64 * k];
                if (chunk * CHUNK + mine + 64 * k < L && (key & mask) == prefix)
                    atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
            }
        }
        __syncthreads();
        // thread t holds bins 2047 - 2t and 2046 - 2t (and clears them): sums from the top down
        const uint32_t h0 = hist[2047 - 2 * tid], h1 = hist[2046 - 2 * tid];
        hist[2047 - 2 * tid] = hist[2046 - 2 * tid] = 0;
        const int s = wave_scan((int)(h0 + h1));
        int total;
        const uint32_t above = (uint32_t)(below_waves(slot, __builtin_amdgcn_readlane(s, 63), wave,
                                                      lane, &total) +
                                          s) -
                               h0 - h1;
        if (above < need && need <= above + h0 + h1) {
            const bool first = need <= above + h0;
            pick[0] = 2047 - 2 * tid - (first ? 0 : 1);
            pick[1] = need - above - (first ? 0 : h0);
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        mask |= (bins - 1) << shift;
        need = pick[1];  // rows of this prefix that stay
    }
    // rows with the key `prefix` stay up to the need-th, in their order
    const uint64_t below = (1ull << lane) - 1;
    int* list = scratch + list_at(c.B * c.G) + (size_t)bg * slots * 2;
    int eq0 = 0, to0 = 0, from0 = 0;  // of the chunks before
#pragma unroll 1
    for (int chunk = 0; chunk < chunks; ++chunk) {
        if (chunks > 1) load(chunk);
        const int r0 = chunk * CHUNK + mine;
        int eq = 0;
#pragma unroll 2
        for (int k = 0; k < KPT; ++k)
            eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(
                r0 + 64 * k < L && keys[mine + 64 * k] == prefix));
        int all;
        int e = eq0 + below_waves(slot, eq, wave, lane, &all);
        eq0 += all;
        uint32_t keep = 0;   // bit k: row k of this thread stays
        uint32_t moves = 0;  // slots left free below budget; rows kept past it, times 2^16
#pragma unroll 2
        for (int k = 0; k < KPT; ++k) {
            const int r = r0 + 64 * k;
            const uint32_t key = keys[mine + 64 * k];
            const bool on = r < L, tie = on && key == prefix;
            const uint64_t same = __builtin_amdgcn_ballot_w64(tie);
            const bool stay = (on && key > prefix) ||
                              (tie && e + __builtin_popcountll(same & below) < (int)need);
            e += __builtin_popcountll(same);
            keep |= (uint32_t)stay << k;
            moves += __builtin_popcountll(__builtin_amdgcn_ballot_w64(on && !stay && r < budget));
            moves += __builtin_popcountll(__builtin_amdgcn_ballot_w64(stay && r >= budget)) << 16;
        }
        static_assert(CHUNK < 1 << 16, "a chunk's moves in 16 bits");
        int moves_all;
        const uint32_t at = (uint32_t)below_waves(slot, (int)moves, wave, lane, &moves_all);
        int to = to0 + (int)(at & 0xffffu), from = from0 + (int)(at >> 16);
        to0 += moves_all & 0xffff;
        from0 += (int)((uint32_t)moves_all >> 16);
#pragma unroll 2
        for (int k = 0; k < KPT; ++k) {
            const int r = r0 + 64 * k;
            const bool stay = (keep >> k) & 1u, free_ = r < L && !stay && r < budget;
            const bool move = stay && r >= budget;
            const uint64_t f = __builtin_amdgcn_ballot_w64(free_);
            const uint64_t v = __builtin_amdgcn_ballot_w64(move);
            if (free_) list[2 * (to + __builtin_popcountll(f & below))] = r;
            if (move) list[2 * (from + __builtin_popcountll(v & below)) + 1] = r;
            to += __builtin_popcountll(f);
            from += __builtin_popcountll(v);
        }
    }
    if constexpr (std::is_void_v<T>) {
        if (tid == 0) scratch[bg] = to0;
    } else {
        __syncthreads();  // (the lists are written)
        move_rows<T>(c, bg, list, to0, tid / width, kSelThreads / width, vec, tid & (width - 1), width);
    }
}

// `width` lanes per move, the moves of a head dealt to gridDim.x workgroups.  The copy bounds it:
// 64 MB in 11 us (rows of 256 bytes).
template <typename T>
__global__ __launch_bounds__(256) void k_evict_move(CacheView c, int slots, const int* scratch,
                                                    int vec, int width) {
    const int bg = blockIdx.y, per = 256 / width;
    const int* list = scratch + list_at(c.B * c.G) + (size_t)bg * slots * 2;
    move_rows<T>(c, bg, list, min(scratch[bg], slots), blockIdx.x * per + threadIdx.x / width,
                 gridDim.x * per, vec, threadIdx.x & (width - 1), width);
}

// lanes of a row: its 16-byte pieces, a power of two up to a wave
int lanes_of(int D, size_t es) {
    int w = 1;
    while (w < 64 && w * 16 < (int)(D * es)) w *= 2;
    return w;
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
    const int width = lanes_of(c.D, es);
    const dim3 grid((unsigned)(((long)c.B * c.G * p.n * width + 255) / 256));
    if (dtype == kDtypeF32)
        hipLaunchKernelGGL(k_commit<float>, grid, dim3(256), 0, st, c, d, p, vec, width);
    else
        hipLaunchKernelGGL(k_commit<uint16_t>, grid, dim3(256), 0, st, c, d, p, vec, width);
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
    return (list_at(B * G) + (size_t)B * G * 2 * slots) * sizeof(int);
}

template <typename T>
static void select(const CacheView& c, int budget, int recent, int slots, int* scratch, int vec,
                   int width, hipStream_t st) {
    const dim3 grid((unsigned)(c.B * c.G)), block(kSelThreads);
    if (c.cap <= kSelThreads)
        hipLaunchKernelGGL((k_evict_select<1, T>), grid, block, 0, st, c, budget, recent, slots,
                           scratch, vec, width);
    else if (c.cap <= 4 * kSelThreads)
        hipLaunchKernelGGL((k_evict_select<4, T>), grid, block, 0, st, c, budget, recent, slots,
                           scratch, vec, width);
    else
        hipLaunchKernelGGL((k_evict_select<16, T>), grid, block, 0, st, c, budget, recent, slots,
                           scratch, vec, width);
}

hipError_t launch_cache_evict(int dtype, const CacheView& c, int budget, int recent, int* scratch,
                              hipStream_t st) {
    const int slots = std::min(budget, c.cap - budget);
    if (slots <= 0) return hipSuccess;  // no row can lie past the budget
    const size_t es = dtype == kDtypeF32 ? 4 : 2;
    const int vec = rows16(c.K, c.ks, c.D, es) && rows16(c.V, c.vs, c.D, es);
    const int BG = c.B * c.G, width = lanes_of(c.D, es), per = 256 / width;
    // the bytes of a head's moves that one workgroup still copies in less time than a launch takes
    const bool few = (int64_t)slots * c.D * es * 2 <= 64 * 1024;
    if (few && dtype == kDtypeF32)
        select<float>(c, budget, recent, slots, scratch, vec, width, st);
    else if (few)
        select<uint16_t>(c, budget, recent, slots, scratch, vec, width, st);
    else
        select<void>(c, budget, recent, slots, scratch, vec, width, st);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || few) return e;
    const dim3 grid((unsigned)std::max(1, std::min((slots + per - 1) / per, 4096 / std::min(BG, 4096))),
                    (unsigned)BG);
    if (dtype == kDtypeF32)
        hipLaunchKernelGGL(k_evict_move<float>, grid, dim3(256), 0, st, c, slots, scratch, vec, width);
    else
        hipLaunchKernelGGL(k_evict_move<uint16_t>, grid, dim3(256), 0, st, c, slots, scratch, vec,
                           width);
    return hipGetLastError();
}

}  // namespace atn

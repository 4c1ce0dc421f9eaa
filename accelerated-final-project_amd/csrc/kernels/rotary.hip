// Rotation of tokens by their positions, and the append of new keys and values to the pages of a
// cache with that rotation on the way.  Pair (x1, x2) of a token at position p becomes
//   a (x1 cos - x2 sin), a (x1 sin + x2 cos),  angle = p freq_i,
// the inverse (its transpose, so the gradient) with the angle's sign turned.  dims >= rot and
// values are copied.
//
// Nothing but the bytes bounds it, once each angle is computed once for all heads: a workgroup
// takes a few tokens, puts their cosines and sines into LDS and goes through the tokens' rows of
// all tensors 16 bytes a lane.  4 sequences of 4096 tokens, 40 heads of 128 bf16 dims: 67 us, 5.0
// TB/s; prompts of 14338 tokens (8 of 2048 or 1366) into the cache, 48 heads, 75 us, 4.7 TB/s; a few
// tokens 7 us, of which the call is 4.
// Angles: p freq in fp64 (24 + 31 bits: exact to 2^-53), reduced to half turns there, so that
// positions far into a context lose nothing; the rest is fp32, rounded to the type once.
#include <algorithm>
#include <type_traits>

#include "cache_tiles.hpp"
#include "paged.hpp"

namespace atn {

namespace {

constexpr int kThreads = 256;

// Element i of a piece as fp32, and two elements put back.
template <typename T, typename P>
__device__ __forceinline__ float get(const P& p, int i) {
    if constexpr (sizeof(T) == 4)
        return __uint_as_float(p.w[i]);
    else
        return __uint_as_float(i & 1 ? p.w[i / 2] & 0xffff0000u : p.w[i / 2] << 16);
}
template <typename T, typename P>
__device__ __forceinline__ void put2(P& p, int i, float a, float b) {
    if constexpr (sizeof(T) == 4)
        p.w[i] = __float_as_uint(a), p.w[i + 1] = __float_as_uint(b);
    else
        p.w[i / 2] = pack2(a, b);
}

// A row's work: `turned` pieces of 16 bytes (two of them where pairs are halves apart) and `copied`
// ones, then the pairs and the elements that are left over, one at a time.  Rows need only element
// alignment.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryArgs a, int tokens_wg,
                                                     Divider by_tokens) {
    constexpr int W = 16 / (int)sizeof(T);
    using P = Words<T, 16>;
    extern __shared__ float2 turn[];               // [tokens][pairs]
    __shared__ int seq[kThreads], place[kThreads];  // of each token: sequence, row in the cache or -1
    const int tid = threadIdx.x, pairs = a.r.rot / 2;
    const int tok0 = blockIdx.x * tokens_wg, toks = min(tokens_wg, a.B * a.T - tok0);
    if (tid < toks) {
        const int b = over(tok0 + tid, a.by_t), t = tok0 + tid - b * a.T;
        const int n = a.count ? min(max(a.count[b], 0), a.T) : a.T;
        seq[tid] = b;
        place[tid] = t < n ? t + (a.with_cache ? rows_in_use(a.c, b) : 0) : -1;
    }
    __syncthreads();
    for (int e = tid; e < toks * pairs; e += kThreads) {
        const int k = over(e, a.by_pairs), i = e - k * pairs, row = place[k];
        if (row < 0) continue;
        const int p = a.pos ? a.pos[tok0 + k] : row;
        const double turns = (double)p * (double)a.r.freq[i] * 0.15915494309189535;
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        turn[e] = make_float2(c * a.r.amplitude, s * a.r.amplitude * a.r.sign);
    }
    __syncthreads();
#pragma unroll 1
    for (int j = 0; j < a.jobs; ++j) {
        const RowJob& job = a.job[j];
        const int rot = job.rotate ? a.r.rot : 0, apart = a.r.half ? rot / 2 : 1;
        const int turned = (a.r.half ? rot / 2 : rot) / W, copied = (a.D - rot) / W;
        const int pairs_left = a.r.half ? rot / 2 - turned * W : (rot - turned * W) / 2;
        const int left = a.D - rot - copied * W;
        const int tasks = turned + copied + pairs_left + left, rows = tokens_wg * job.heads;
        // (rows that follow one another in memory go to lanes that follow one another)
        const bool by_head = job.is[1] < job.is[2];
        int width = 1;
        while (width < kThreads && width < tasks) width *= 2;
        const int lane = tid & (width - 1), per = kThreads / width * (int)gridDim.y;
        const T* in = (const T*)job.in;
        T* out = (T*)job.out;
        // (rows are dealt to the y workgroups too; one at a time: with two or four rows' loads in flight a
        // lane, fewer waves fit, 71 and 87 us where one takes 67)
        for (int r = blockIdx.y * (kThreads / width) + tid / width; r < rows; r += per) {
            const int x = over(r, by_head ? job.by_heads : by_tokens);
            const int k = by_head ? x : r - x * tokens_wg, h = by_head ? r - x * job.heads : x;
            if (k >= toks) continue;
            const int row = place[k], b = seq[k], t = tok0 + k - b * a.T;
            if (row < 0) continue;
            const T* from = in + b * job.is[0] + h * job.is[1] + t * job.is[2];
            T* to = out + b * job.os[0] + h * job.os[1] + t * job.os[2];
            if (job.paged) {
                if (row >= a.c.cap) continue;
                const int slot = over(row, a.c.by_page);
                const int page = a.c.table[(size_t)b * a.c.slots + slot];
                if (!is_page(a.c, page)) continue;
                to = out + page * job.os[0] + h * job.os[1] + (row - slot * a.c.page_rows) * job.os[2];
            }
            const float2* cs = turn + k * pairs;
            for (int d = lane; d < tasks; d += width) {
                if (d < turned + copied) {
                    const bool two = d < turned && a.r.half;
                    const int e0 = d < turned ? d * W : rot + (d - turned) * W, e1 = e0 + apart;
                    P x = ld_words<16>(from + e0), y;
                    if (two) {
                        y = ld_words<16>(from + e1);
#pragma unroll
                        for (int i = 0; i < W; i += 2) {
                            const float2 z = cs[e0 + i], w = cs[e0 + i + 1];
                            const float p = get<T>(x, i), q = get<T>(y, i);
                            const float r = get<T>(x, i + 1), s = get<T>(y, i + 1);
                            put2<T>(x, i, p * z.x - q * z.y, r * w.x - s * w.y);
                            put2<T>(y, i, p * z.y + q * z.x, r * w.y + s * w.x);
                        }
                    } else if (d < turned) {
#pragma unroll
                        for (int i = 0; i < W; i += 2) {
                            const float2 z = cs[(e0 + i) / 2];
                            const float p = get<T>(x, i), q = get<T>(x, i + 1);
                            put2<T>(x, i, p * z.x - q * z.y, p * z.y + q * z.x);
                        }
                    }
                    __builtin_memcpy(to + e0, &x, 16);
                    if (two) __builtin_memcpy(to + e1, &y, 16);
                } else {
                    const int s = d - turned - copied;
                    if (s < pairs_left) {
                        const int e0 = turned * W + (a.r.half ? s : 2 * s);
                        const float2 z = cs[a.r.half ? e0 : e0 / 2];
                        const float p = Elem<T>::ld(from, e0), q = Elem<T>::ld(from, e0 + apart);
                        Elem<T>::st(to, e0, p * z.x - q * z.y);
                        Elem<T>::st(to, e0 + apart, p * z.y + q * z.x);
                    } else {
                        const int e0 = rot + copied * W + s - pairs_left;
                        to[e0] = from[e0];
                    }
                }
            }
        }
    }
}

__global__ __launch_bounds__(256) void k_paged_advance(PagedView c, const int* count, int T) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= c.B) return;
    const int n = count ? min(max(count[b], 0), T) : T, L = rows_in_use(c, b);
    c.len[b] = min(c.cap - L, n) + L;
}

}  // namespace

hipError_t launch_rotary(int dtype, const RotaryArgs& a, hipStream_t st) {
    const int64_t tokens = (int64_t)a.B * a.T;
    const int64_t pairs = std::max(1, a.r.rot / 2), es = dtype == kDtypeF32 ? 4 : 2;
    int64_t heads = 0;
    for (int j = 0; j < a.jobs; ++j) heads += a.job[j].heads;
    // a workgroup's tokens: 48 KiB of rows, with four angles a thread at most, where that leaves
    // four workgroups a CU
    const int64_t row = heads * a.D * es;
    int64_t per = std::min<int64_t>({49152 / std::max<int64_t>(1, row), 4 * kThreads / pairs,
                                     tokens / 1024, kThreads});
    per = std::max<int64_t>(1, per);
    const int64_t wgs = (tokens + per - 1) / per;
    // few tokens: their rows over several workgroups, of 8 KiB at least
    const int64_t share = std::max<int64_t>(
        1, std::min<int64_t>({1024 / std::max<int64_t>(1, wgs), per * row / 8192, 64}));
    const dim3 grid((unsigned)wgs, (unsigned)share);
    const Divider by = divider((int)per);
    const size_t lds = (size_t)(a.r.rot > 0 ? per * pairs : 1) * sizeof(float2);
    if (dtype == kDtypeF32)
        hipLaunchKernelGGL(k_rotary<float>, grid, dim3(kThreads), lds, st, a, (int)per, by);
    else
        hipLaunchKernelGGL(k_rotary<uint16_t>, grid, dim3(kThreads), lds, st, a, (int)per, by);
    return hipGetLastError();
}

hipError_t launch_paged_advance(const PagedView& c, const int* count, int T, hipStream_t st) {
    hipLaunchKernelGGL(k_paged_advance, dim3((unsigned)((c.B + 255) / 256)), dim3(256), 0, st, c,
                       count, T);
    return hipGetLastError();
}

}  // namespace atn

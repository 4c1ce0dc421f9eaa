// Rotation of tokens by their positions, and the append of new keys and values to the pages of a
// cache with that rotation on the way.  Pair (x1, x2) of a token at position p becomes
//   a (x1 cos - x2 sin), a (x1 sin + x2 cos),  angle = p freq_i,
// the inverse (its transpose, so the gradient) with the angle's sign turned.  dims >= rot and
// values are copied.
//
// Nothing but the bytes bounds it, once each angle is computed once for all heads: a workgroup
// takes a few tokens, puts their cosines and sines into LDS and goes through the tokens' rows of
// all tensors 16 bytes a lane.
// Angles: p freq in fp64 (24 + 31 bits: exact to 2^-53), reduced to half turns there, so that
// positions far into a context lose nothing; the rest is fp32, rounded to the type once.
#include <algorithm>
#include <type_traits>

#include "cache_tiles.hpp"
#include "paged.hpp"

namespace atn {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 4096;  // of a workgroup's tokens: 32 KiB

// One piece of a row: N pairs (and the two pieces of memory that hold them), or, `plain`, 2 N
// elements copied.
template <typename T, int N>
struct Piece {
    T a[N], b[N];
};

// (rows that a lane holds at once: their loads are in flight together)
constexpr int kAtOnce = 4;

// VEC: pieces of 16 bytes; else pairs and elements one at a time.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryArgs a, int tokens_wg) {
    constexpr int W = VEC ? 16 / (int)sizeof(T) : 1;
    using P = Words<T, VEC ? 16 : 4>;
    __shared__ float2 turn[kMaxPairs];
    const int tid = threadIdx.x, pairs = a.r.rot / 2;
    const int tok0 = blockIdx.x * tokens_wg, toks = min(tokens_wg, a.B * a.T - tok0);
    __shared__ int seq[kThreads], place[kThreads];  // of each token: sequence, row in the cache or -1
    if (tid < toks) {
        const int b = over(tok0 + tid, a.by_t), t = tok0 + tid - b * a.T;
        const int n = a.count ? min(max(a.count[b], 0), a.T) : a.T;
        seq[tid] = b;
        place[tid] = t < n ? t + (a.with_cache ? rows_in_use(a.c, b) : 0) : -1;
    }
    __syncthreads();
    for (int e = tid; e < toks * pairs; e += kThreads) {
        const int k = e / pairs, i = e - k * pairs, row = place[k];
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
        const int rot = job.rotate ? a.r.rot : 0;
        // pieces of a row: rotated ones (of two places where pairs are halves apart), then copies
        const int step = VEC ? (a.r.half ? 2 * W : W) : 2;
        const int turned = rot / step, pieces = turned + (a.D - rot) / W;
        const int rows = toks * job.heads;
        int width = 1;
        while (width < kThreads && width < pieces) width *= 2;
        const int lane = tid & (width - 1), per = kThreads / width;
        const T* in = (const T*)job.in;
        T* out = (T*)job.out;
        // rows of a head are dealt to the y workgroups too
        for (int r0 = blockIdx.y * per + tid / width; r0 < rows; r0 += per * gridDim.y * kAtOnce) {
            for (int d = lane; d < pieces; d += width) {
                P x[kAtOnce], y[kAtOnce];
                int tk[kAtOnce];
                T* to[kAtOnce];
                const bool two = d < turned && (!VEC || a.r.half);
                // elements of the piece's two places
                int e0, e1 = 0;
                if (d >= turned) {
                    e0 = rot + (d - turned) * W;
                } else if (VEC) {
                    e0 = d * W;
                    e1 = e0 + rot / 2;
                } else {
                    e0 = a.r.half ? d : 2 * d;
                    e1 = a.r.half ? d + rot / 2 : 2 * d + 1;
                }
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const int r = r0 + u * per * gridDim.y;
                    tk[u] = -1;
                    if (r >= rows) continue;
                    const int k = r / job.heads, h = r - k * job.heads, row = place[k], b = seq[k];
                    if (row < 0) continue;
                    const int t = tok0 + k - b * a.T;
                    if (job.paged) {
                        if (row >= a.c.cap) continue;
                        const int slot = over(row, a.c.by_page);
                        const int page = a.c.table[(size_t)b * a.c.slots + slot];
                        if (!is_page(a.c, page)) continue;
                        to[u] = out + page * job.os[0] + h * job.os[1] +
                                (row - slot * a.c.page_rows) * job.os[2];
                    } else {
                        to[u] = out + b * job.os[0] + h * job.os[1] + t * job.os[2];
                    }
                    tk[u] = k;
                    const T* from = in + b * job.is[0] + h * job.is[1] + t * job.is[2];
                    if constexpr (VEC) {
                        x[u] = ld_words<16>(from + e0);
                        if (two) y[u] = ld_words<16>(from + e1);
                    } else {
                        x[u] = ld_some<4>(from + e0, 1);
                        if (two) y[u] = ld_some<4>(from + e1, 1);
                    }
                }
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    if (tk[u] < 0) continue;
                    if (d < turned) {
                        const float2* cs = turn + tk[u] * pairs;
                        auto get = [](const P& p, int i) {
                            if constexpr (sizeof(T) == 4)
                                return __uint_as_float(p.w[i]);
                            else
                                return __uint_as_float(i & 1 ? p.w[i / 2] & 0xffff0000u
                                                             : p.w[i / 2] << 16);
                        };
                        float f[W], g[W];
                        if (two) {
                            const int i0 = VEC ? e0 : d;
#pragma unroll
                            for (int i = 0; i < W; ++i) {
                                const float2 z = cs[i0 + i];
                                const float p = get(x[u], i), q = get(y[u], i);
                                f[i] = p * z.x - q * z.y;
                                g[i] = p * z.y + q * z.x;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i + 1 < W; i += 2) {
                                const float2 z = cs[(e0 + i) / 2];
                                const float p = get(x[u], i), q = get(x[u], i + 1);
                                f[i] = p * z.x - q * z.y;
                                f[i + 1] = p * z.y + q * z.x;
                            }
                        }
                        auto put = [](P& p, const float(&v)[W]) {
                            if constexpr (sizeof(T) == 4) {
#pragma unroll
                                for (int i = 0; i < W; ++i) p.w[i] = __float_as_uint(v[i]);
                            } else if constexpr (W == 1) {
                                p.w[0] = pack2(v[0], 0.f) & 0xffffu;
                            } else {
#pragma unroll
                                for (int i = 0; i < W; i += 2) p.w[i / 2] = pack2(v[i], v[i + 1]);
                            }
                        };
                        put(x[u], f);
                        if (two) put(y[u], g);
                    }
                    if constexpr (VEC) {
                        __builtin_memcpy(to[u] + e0, &x[u], 16);
                        if (two) __builtin_memcpy(to[u] + e1, &y[u], 16);
                    } else {
                        __builtin_memcpy(to[u] + e0, &x[u], sizeof(T));
                        if (two) __builtin_memcpy(to[u] + e1, &y[u], sizeof(T));
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
    const int64_t pairs = std::max(1, a.r.rot / 2);
    int64_t rows = 0;
    for (int j = 0; j < a.jobs; ++j) rows += a.job[j].heads;
    // as many tokens as give every thread an angle, where that leaves two workgroups a CU
    int64_t per = std::max<int64_t>(1, std::min<int64_t>(kThreads / pairs, tokens / 512));
    per = std::min<int64_t>(per, std::min<int64_t>(kThreads, kMaxPairs / pairs));
    const int64_t wgs = (tokens + per - 1) / per;
    // few tokens: their rows over several workgroups, of 16 KiB at least
    const int64_t bytes = per * rows * a.D * (dtype == kDtypeF32 ? 4 : 2);
    const int64_t share = std::max<int64_t>(
        1, std::min<int64_t>({512 / std::max<int64_t>(1, wgs), bytes / 16384, 64}));
    const dim3 grid((unsigned)wgs, (unsigned)share);
    if (dtype == kDtypeF32) {
        if (a.vec)
            hipLaunchKernelGGL((k_rotary<float, true>), grid, dim3(kThreads), 0, st, a, (int)per);
        else
            hipLaunchKernelGGL((k_rotary<float, false>), grid, dim3(kThreads), 0, st, a, (int)per);
    } else {
        if (a.vec)
            hipLaunchKernelGGL((k_rotary<uint16_t, true>), grid, dim3(kThreads), 0, st, a, (int)per);
        else
            hipLaunchKernelGGL((k_rotary<uint16_t, false>), grid, dim3(kThreads), 0, st, a, (int)per);
    }
    return hipGetLastError();
}

hipError_t launch_paged_advance(const PagedView& c, const int* count, int T, hipStream_t st) {
    hipLaunchKernelGGL(k_paged_advance, dim3((unsigned)((c.B + 255) / 256)), dim3(256), 0, st, c,
                       count, T);
    return hipGetLastError();
}

}  // namespace atn

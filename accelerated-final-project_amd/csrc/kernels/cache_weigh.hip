// The attention weight of a cache's rows: for the accepted drafts i of a
// sequence (the path's, in order) and the heads of the row's kv head,
//   weight[r] = weight_in[r] + sum over (head, i) with r <= len + i
//               of exp2(scale q . k_r - log2(e) lse),
// scores as in tree_attn.hip; V is not read.  One pass over K: the query rows
// are few (heads times path), the sum over them ends in a row of 16 lanes, and a
// row's weight has one writer and one order of sums.  The read of K bounds it: 8 sequences of 1000
// to 8191 rows, 8 kv heads of 128 bf16 dims 17.2 to 18.5 us, 4.2 to 4.5 TB/s; fp32, 512 dims, 2 of
// 2000 to 4091 rows, 4 kv heads 14.2 us, 3.5 TB/s.
#include <algorithm>

#include "cache_tiles.hpp"

namespace atn {

namespace {

constexpr int kWaves = 4;
constexpr int kRows = 64;  // query rows of a pass (rep times path rows: more take further passes)
constexpr float kLog2e = 1.4426950408889634f;

struct WeighArgs {
    CacheView c;
    DraftView d;
    PathView p;
    const float* lse;
    const float* weight_in;
    float scale;
};

// Query row `row` (head times A + path entry) of a pair.
struct QueryRow {
    int head, tok, entry;
};
__device__ __forceinline__ QueryRow query_row(const WeighArgs& a, int b, int g, int A, int row) {
    QueryRow x;
    x.head = g * a.d.rep + row / A;
    x.entry = row % A;
    x.tok = path_at(a.p, b, x.entry);
    return x;
}

// the last cache row that a query row attends (-1: none), and its lse in units of log2
__device__ __forceinline__ float2 reach_of(const WeighArgs& a, int b, int g, int L, int A, int row,
                                           int R) {
    if (row >= R) return make_float2(__int_as_float(-1), 0.f);
    const QueryRow x = query_row(a, b, g, A, row);
    const float z = a.lse[((size_t)b * a.d.H + x.head) * a.d.T + x.tok];
    return make_float2(__int_as_float(z == -INFINITY ? -1 : L + x.entry), z * kLog2e);
}

// Lane (col, q) of a 16-lane row holds its row's sums for keys k0 + 4 q + e: lanes col 0..3 write
// one each.
__device__ __forceinline__ void put_weights(const WeighArgs& a, size_t at, bool first, float4 sum,
                                            int r0, int end, int col) {
    const float x = col & 2 ? (col & 1 ? sum.w : sum.z) : (col & 1 ? sum.y : sum.x);
    const int r = r0 + col;
    if (col < 4 && r < end) {
        const float old = !first ? a.c.weight[at + r] : a.weight_in ? a.weight_in[at + r] : 0.f;
        a.c.weight[at + r] = old + x;
    }
}

// head_d <= 256: a wave holds a block of keys in registers and runs the pass's query rows over
// it from LDS, the next block's keys on their way.
template <typename T, int DP, int MODE>
__global__ __launch_bounds__(64 * kWaves, 2) void k_weigh_narrow(WeighArgs a) {
    using N = CacheTiles<T, DP, 1, MODE>;
    constexpr int KB = N::KB, SUB = N::SUB, KS = N::KS;
    __shared__ typename N::KPiece qs[kRows / 16 * KS * 64];
    __shared__ float2 reach[kRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    const int bg = blockIdx.y, g = bg % a.c.G, b = bg / a.c.G, D = a.c.D;
    const int L = of_wave(rows_in_use(a.c, b)), A = of_wave(rows_accepted(a.c, a.d, a.p, b));
    const int end = L + A, blocks = (end + KB - 1) / KB, R = a.d.rep * A;
    const T* kc = (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1];
    const int i0 = blockIdx.x * kWaves + wave, step = gridDim.x * kWaves;
    if ((int)blockIdx.x * kWaves >= blocks) return;
    for (int row0 = 0; row0 == 0 || row0 < R; row0 += kRows) {
        typename N::Keys k;
        auto load_k = [&](int i) {
            N::load_k(k, kc + (int64_t)i * KB * a.c.ks[2], a.c.ks[2], end - i * KB, D, lane);
        };
        if (i0 < blocks) load_k(i0);
        const int tiles = (min(kRows, R - row0) + 15) / 16;
        __syncthreads();
        for (int e = threadIdx.x; e < tiles * KS * 64; e += 64 * kWaves) {
            const int el = e & 63, i = (e >> 6) % KS, t = (e >> 6) / KS;
            const int row = row0 + 16 * t + (el & 15);
            typename N::KPiece z{};
            if (row < R) {
                const QueryRow x = query_row(a, b, g, A, row);
                z = N::piece((const T*)a.d.Q + b * a.d.qs[0] + x.head * a.d.qs[1] +
                                 x.tok * a.d.qs[2],
                             16 * (el >> 4), i, el >> 4, D);
            }
            qs[e] = z;
        }
        if (threadIdx.x < kRows) reach[threadIdx.x] = reach_of(a, b, g, L, A, row0 + threadIdx.x, R);
        __syncthreads();
        for (int i = i0; i < blocks; i += step) {
            float sum[SUB][4];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[u][e] = 0.f;
            for (int t = 0; t < tiles; ++t) {
                v4f s[SUB];
#pragma unroll
                for (int u = 0; u < SUB; ++u) s[u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < KS; ++e) {
                    const typename N::KPiece f = qs[(t * KS + e) * 64 + lane];
#pragma unroll
                    for (int u = 0; u < SUB; ++u) s[u] = N::dot(k.p[u][e], f, s[u]);
                }
                const float2 z = reach[16 * t + col];
                const int last = __float_as_int(z.x);
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = exp2_(fmaf(s[u][e], a.scale, -z.y));
                        sum[u][e] += i * KB + 16 * u + 4 * q + e <= last ? p : 0.f;
                    }
            }
            const int nx = i + step;
            if (nx < blocks) load_k(nx);
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const float4 w = make_float4(row16_sum(sum[u][0]), row16_sum(sum[u][1]),
                                             row16_sum(sum[u][2]), row16_sum(sum[u][3]));
                put_weights(a, (size_t)bg * a.c.cap, row0 == 0, w, i * KB + 16 * u + 4 * q, end, col);
            }
        }
    }
}

// head_d > 256: 8 waves share the dims of a block of 16 SUB keys and add up through LDS.
constexpr int kScoreWaves = 8;

template <typename T, int MT, bool AHEAD, int SUB>
__global__ __launch_bounds__(64 * kScoreWaves) void k_weigh_wide(WeighArgs a) {
    constexpr int kBlock = 16 * SUB;
    __shared__ v4f red[kScoreWaves][MT * SUB * 64];
    __shared__ float part[MT][kBlock];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    const int bg = blockIdx.y, g = bg % a.c.G, b = bg / a.c.G, D = a.c.D;
    const int L = of_wave(rows_in_use(a.c, b)), A = of_wave(rows_accepted(a.c, a.d, a.p, b));
    const int end = L + A, j0 = blockIdx.x * kBlock, rows = min(kBlock, end - j0);
    const int R = a.d.rep * A;
    if (rows <= 0) return;
    const T* kp[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u)
        kp[u] = (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1] +
                (int64_t)(j0 + min(16 * u + col, rows - 1)) * a.c.ks[2];
    for (int row0 = 0; row0 == 0 || row0 < R; row0 += 16 * MT) {
        v4f s[MT][SUB] = {};
        if (R > 0) {
            const T* qp[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const QueryRow x = query_row(a, b, g, A, min(row0 + 16 * t + col, R - 1));
                qp[t] = (const T*)a.d.Q + b * a.d.qs[0] + x.head * a.d.qs[1] + x.tok * a.d.qs[2];
            }
            wide_scores<T, MT, AHEAD>(s, kp, qp, D, wave, kScoreWaves, q);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int u = 0; u < SUB; ++u) red[wave][(t * SUB + u) * 64 + lane] = s[t][u];
        __syncthreads();
        if (threadIdx.x < MT * SUB * 64) {  // one thread per query row and 4 keys
            const int u = (threadIdx.x >> 6) % SUB, t = (threadIdx.x >> 6) / SUB;
            v4f x = red[0][threadIdx.x];
#pragma unroll
            for (int w = 1; w < kScoreWaves; ++w) x += red[w][threadIdx.x];
            const float2 z = reach_of(a, b, g, L, A, row0 + 16 * t + col, R);
            const int last = __float_as_int(z.x), k0 = 16 * u + 4 * q;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = exp2_(fmaf(x[e], a.scale, -z.y));
                y[e] = row16_sum(j0 + k0 + e <= last ? p : 0.f);
            }
            if (col == 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) part[t][k0 + e] = y[e];
            }
        }
        __syncthreads();
        if (threadIdx.x < rows) {
            const size_t at = (size_t)bg * a.c.cap + j0 + threadIdx.x;
            float w = row0 > 0 ? a.c.weight[at] : a.weight_in ? a.weight_in[at] : 0.f;
#pragma unroll
            for (int t = 0; t < MT; ++t) w += part[t][threadIdx.x];
            a.c.weight[at] = w;
        }
    }
}

template <typename T, int DP>
void go_narrow(const WeighArgs& a, dim3 grid, hipStream_t st) {
    if (a.c.D == DP)
        hipLaunchKernelGGL((k_weigh_narrow<T, DP, kExact>), grid, dim3(64 * kWaves), 0, st, a);
    else if (DP > 64 || a.c.D >= 16 / (int)sizeof(T))
        hipLaunchKernelGGL((k_weigh_narrow<T, DP, kClamp>), grid, dim3(64 * kWaves), 0, st, a);
    else if constexpr (DP == 64)
        hipLaunchKernelGGL((k_weigh_narrow<T, DP, kElem>), grid, dim3(64 * kWaves), 0, st, a);
}

template <typename T, int MT, int SUB>
void go_wide(const WeighArgs& a, dim3 grid, hipStream_t st) {
    // (a wave of more than a step of 128 bf16 or 64 fp32 dims)
    if (a.c.D > kScoreWaves * 256 / (int)sizeof(T))
        hipLaunchKernelGGL((k_weigh_wide<T, MT, true, SUB>), grid, dim3(64 * kScoreWaves), 0, st, a);
    else
        hipLaunchKernelGGL((k_weigh_wide<T, MT, false, SUB>), grid, dim3(64 * kScoreWaves), 0, st, a);
}

template <typename T, int MT>
void go_wide(const WeighArgs& a, int keys, int BG, hipStream_t st) {
    const int blocks = (keys + 31) / 32;
    // (blocks of 32 keys read Q half as often, blocks of 16 reach more of the card where there are
    // fewer than two of 32 a CU: fp32, 8192 dims, 1163 rows of 3 kv heads 47 -> 33.5 us)
    if ((int64_t)blocks * BG < 512)
        go_wide<T, MT, 1>(a, dim3((unsigned)((keys + 15) / 16), (unsigned)BG), st);
    else
        go_wide<T, MT, 2>(a, dim3((unsigned)blocks, (unsigned)BG), st);
}

template <typename T>
void go(const WeighArgs& a, hipStream_t st) {
    const int D = a.c.D, BG = a.c.B * a.c.G;
    const int keys = std::min(a.c.cap, a.c.rows + a.p.n);
    if (D > 256) {
        const int R = a.d.rep * a.p.n;  // at most
        if (R <= 16) return go_wide<T, 1>(a, keys, BG, st);
        if (R <= 32) return go_wide<T, 2>(a, keys, BG, st);
        return go_wide<T, 4>(a, keys, BG, st);
    }
    const int kb = sizeof(T) == 2 ? 32 : 16;
    const int most = (keys + kb * kWaves - 1) / (kb * kWaves);
    // about four workgroups a CU, each wave walking its blocks
    const dim3 grid((unsigned)std::max(1, std::min(most, (1024 + BG - 1) / BG)), (unsigned)BG);
    if (D <= 64) go_narrow<T, 64>(a, grid, st);
    else if (D <= 128) go_narrow<T, 128>(a, grid, st);
    else if (D <= 192) go_narrow<T, 192>(a, grid, st);
    else go_narrow<T, 256>(a, grid, st);
}

}  // namespace

hipError_t launch_cache_weigh(int dtype, const CacheView& c, const DraftView& d,
                              const PathView& p, const float* lse, const float* weight_in,
                              float scale, hipStream_t st) {
    const WeighArgs a{c, d, p, lse, weight_in, scale};
    if (dtype == kDtypeF32)
        go<float>(a, st);
    else
        go<uint16_t>(a, st);
    return hipGetLastError();
}

}  // namespace atn

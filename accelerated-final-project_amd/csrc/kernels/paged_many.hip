// Attention over a paged cache, many query rows (paged_attn_impl.hpp has what its kernels share).
#include "paged_attn_impl.hpp"

namespace atn {

namespace {

// ---------------------------------------------------------------- many query rows
// bf16, at most 128 dims in whole 16-byte pieces, more than 32 query rows of an item: products and
// softmax weigh as much as the reads.  Each wave has 32 query rows, the workgroup's WAVES of them
// share K and V through LDS, KEYS keys a stage.  MFMA 32 x 32: S^T = K Q^T leaves a lane the scores
// of query L % 32 for 4 consecutive keys of every 8, which are the operand of O^T = V^T P^T as they
// lie; V's comes by the transposing LDS read.  The scores of the next stage are computed beside
// the softmax of this one, so that matrix and vector units both have work in every wave.
typedef float v16f __attribute__((ext_vector_type(16)));

template <int DP_, int WAVES_, int KEYS_>
struct PagedMany {
    static constexpr int DP = DP_, WAVES = WAVES_, KEYS = KEYS_;
    static constexpr int ROWS = 32 * WAVES;
    static constexpr int CH = DP / 8;                    // 16-byte pieces of a row
    static constexpr int NT = KEYS / 32;                 // tiles of keys
    static constexpr int QS = DP / 16, DT = DP / 32;     // steps of the scores, tiles of dims
    static constexpr int kStage = KEYS * DP * 2;
    static constexpr int X = KEYS * CH / (64 * WAVES);   // pieces of K (and of V) a lane a stage
    static constexpr int SUB = KEYS / 16, AHEAD = 64 / SUB;
    static_assert(X * 64 * WAVES == KEYS * CH, "whole pieces a lane");
    // Pieces lie at a place of their row that changes with it, so that the rows which one LDS
    // cycle reads lie in different banks: 16 keys at one piece (K), 4 keys at four (V).
    static __device__ __forceinline__ int k_place(int key, int c) {
        return DP == 128 ? c ^ (key & 15) : c ^ ((key >> 1) & 7);
    }
    static __device__ __forceinline__ int v_place(int key, int c) {
        return DP == 128 ? c ^ (4 * (key & 3)) : c ^ (4 * ((key >> 1) & 1));
    }
};

template <int DP, int WAVES, int KEYS, int PRE>
__global__ __launch_bounds__(64 * WAVES, 2) void k_paged_many(PagedArgs a) {
    using N = PagedMany<DP, WAVES, KEYS>;
    using T = uint16_t;
    using W16 = Words<T, 16>;
    // (registers: with four waves a lane loads twice the pieces, so K's go to LDS before V's come)
    constexpr bool kLate = N::X * DP >= 512;
    constexpr int CH = N::CH, NT = N::NT, QS = N::QS, DT = N::DT, X = N::X, SUB = N::SUB;
    __shared__ __align__(16) char kbuf[2][N::kStage];
    __shared__ __align__(16) char vbuf[2][N::kStage];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int D = a.c.D, pieces = D / 8;
    const float scale = fabsf(a.scale);
    if (PRE && blockIdx.x == 0) write_starts(a);

    each_span<PRE>(a, blockIdx.x, KEYS, lane, [&](const Span& sp) {
        const T* kp = (const T*)a.c.K + sp.g * a.c.ks[1];
        const T* vp = (const T*)a.c.V + sp.g * a.c.vs[1];
        const int row0 = sp.tile * N::ROWS, lo = sp.s.lo;
        const int last = min(sp.last, tile_end<PRE>(a, sp.s, sp.tile, KEYS));
        const int mine = row0 + 32 * wave + col;  // this lane's query row
        const int upto = attended<PRE>(a, sp, mine);
        const int w0 = (lo + KEYS - 1) / KEYS, w1 = of_wave(attended<PRE>(a, sp, row0)) / KEYS;

        // pages of 16 keys: lane l those of stage `at` + l / SUB, run l % SUB
        int at = sp.first;
        auto fetch = [&](int i) {
            return page_of(a.c, sp.s.first, (i + lane / SUB) * KEYS + 16 * (lane % SUB));
        };
        int now = fetch(at), next = fetch(at + N::AHEAD);
        auto go = [&](int i) {
            if (i < at + N::AHEAD) return;
            at += N::AHEAD;
            now = next;
            next = fetch(at + N::AHEAD);
        };
        auto run = [&](int i, int s) {
            const int x = (i - at) * SUB + s;
            return __builtin_amdgcn_readlane(x < 64 ? now : next, x & 63);
        };
        auto there_of = [&](int i) {
            uint64_t x = 0;
#pragma unroll
            for (int s = 0; s < SUB; ++s)
                x |= is_page(a.c, run(i, s)) ? (uint64_t)0xffff << (16 * s) : 0;
            return x;
        };
        // piece x of this lane: row (x WAVES + wave) 64 / CH + lane / CH of the stage, piece lane % CH
        const int lrow = lane / CH, lc = lane % CH;
        const bool has = lc < pieces;
        auto load = [&](W16 (&to)[X], const T* pool, const int64_t (&st)[3], int i) {
#pragma unroll
            for (int x = 0; x < X; ++x) {
                const int r0 = (x * WAVES + wave) * (64 / CH);  // (of one run of 16)
                const int r = i * KEYS + r0, in = r - over(r, a.c.by_page) * a.c.page_rows;
                const int page = run(i, r0 / 16);
                const T* base = pool + (is_page(a.c, page) ? page : 0) * st[0] + in * st[2];
                to[x] = ld_words<16>(base + lrow * (uint32_t)st[2] + 8 * min(lc, pieces - 1));
            }
        };
        auto put_k = [&](const W16 (&from)[X], char* buf) {
#pragma unroll
            for (int x = 0; x < X; ++x) {
                const int r = (x * WAVES + wave) * (64 / CH) + lrow;
                W16 z = from[x];
                if (!has) z = W16{};
                reinterpret_cast<W16*>(buf)[r * CH + N::k_place(r, lc)] = z;
            }
        };
        // whether some row does not attend some key of stage i
        auto is_part = [&](int i) { return i < w0 || i >= w1 || there_of(i) != ~0ull >> (64 - KEYS); };
        bool odd = false;  // an infinity or NaN was left out
        auto put_v = [&](W16 (&from)[X], char* buf, int i) {
            if (is_part(i)) {
                // (an infinity or NaN times a weight of 0 would reach rows that do not attend its key:
                // V enters without them, and they are written over the results of the rows that do)
                uint32_t bad = 0;
#pragma unroll
                for (int x = 0; x < X; ++x)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t& z = from[x].w[w];
                        const uint32_t hi = (z & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
                        const uint32_t lo = (z & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
                        z &= ~(hi | lo);
                        bad |= hi | lo;
                    }
                odd |= bad != 0;
            }
#pragma unroll
            for (int x = 0; x < X; ++x) {
                const int r = (x * WAVES + wave) * (64 / CH) + lrow;
                W16 z = from[x];
                if (!has) z = W16{};
                reinterpret_cast<W16*>(buf)[r * CH + N::v_place(r, lc)] = z;
            }
        };

        W16 kr[X], vr[X];
        const bool any = sp.first < last;
        if (any) {
            load(kr, kp, a.c.ks, sp.first);
            load(vr, vp, a.c.vs, sp.first);
        }
        // Q: this lane's row (those of no token: some token's; nobody reads their results)
        W16 qf[QS];
        {
            const T* q = (const T*)a.Q + q_at<PRE>(a, sp, mine);
#pragma unroll
            for (int s = 0; s < QS; ++s) {
                const int c = 2 * s + half;
                qf[s] = ld_words<16>(q + 8 * min(c, pieces - 1));
                if (c >= pieces) qf[s] = W16{};
                if (a.scale < 0.f)
#pragma unroll
                    for (int w = 0; w < 4; ++w) qf[s].w[w] ^= 0x80008000u;
            }
        }
        v16f o[DT];
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[c][e] = 0.f;
        float m = -INFINITY, l = 0.f, used = 0.f;
        __syncthreads();  // (the last span's stages have been read)
        if (any) {
            put_k(kr, kbuf[0]);
            put_v(vr, vbuf[0], sp.first);
            if (sp.first + 1 < last) {
                load(kr, kp, a.c.ks, sp.first + 1);
                put_k(kr, kbuf[1]);
            }
        }
        __syncthreads();

        auto k_at = [&](const char* buf, int t, int e) {
            const int key = 32 * t + col;
            return reinterpret_cast<const W16*>(buf)[key * CH + N::k_place(key, 2 * e + half)];
        };
        // V^T's operand: dims 32 c + lane % 32 of the keys that words [8 u, 8 u + 8) of tile t's
        // weights are
        const int sub = lane & 15, dhalf = lane >> 4 & 1;
        auto v_at = [&](const char* buf, int t, int u, int c) {
            W16 v;
            const int key = 32 * t + 16 * u + 4 * half + (sub >> 2);
            const int piece = 4 * c + 2 * dhalf + ((sub & 3) >> 1);
            const uint16_t* p = reinterpret_cast<const uint16_t*>(buf);
            const uint2 x = lds_tr16(p + (key * CH + N::v_place(key, piece)) * 8 + 4 * (sub & 1));
            const uint2 y =
                lds_tr16(p + ((key + 8) * CH + N::v_place(key + 8, piece)) * 8 + 4 * (sub & 1));
            v.w[0] = x.x, v.w[1] = x.y, v.w[2] = y.x, v.w[3] = y.y;
            return v;
        };
        auto mfma = [](const W16& x, const W16& y, const v16f& z) {
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x),
                                                           __builtin_bit_cast(bf16x8, y), z, 0, 0, 0);
        };
        v16f s0[NT], s1[NT];
        if (any) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                s0[t] = v16f{};
#pragma unroll
                for (int e = 0; e < QS; ++e) s0[t] = mfma(k_at(kbuf[0], t, e), qf[e], s0[t]);
            }
        }
        // One stage: its scores s into weights, beside them the next stage's scores n (of what the
        // buffer holds where there is none), then the product with V.
        auto stage = [&](int i, v16f (&s)[NT], v16f (&n)[NT], const char* kb, char* kfree,
                         const char* vb, char* vfree) {
            const bool more = i + 1 < last, more2 = i + 2 < last;
            const uint64_t there = there_of(i);
            if (more) {
                go(i + 1);
                if (more2) load(kr, kp, a.c.ks, i + 2);
                if (!kLate) load(vr, vp, a.c.vs, i + 1);
            }
            if (i < w0 || i >= w1 || there != ~0ull >> (64 - KEYS)) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int j0 = i * KEYS + 32 * t;
                    const uint32_t on = ((uint32_t)(there >> (32 * t)) & below(upto - j0) &
                                         ~below(lo - j0)) >>
                                        (4 * half);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!(on >> (8 * (e >> 2) + (e & 3)) & 1u)) s[t][e] = -INFINITY;
                }
            }
            // softmax, as weights() does it
            float top = s[0][0];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, s[t][e]);
            if (__builtin_amdgcn_ballot_w64(top * scale > m + 8.f)) {
                const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top),
                                                                __float_as_uint(top), false, false);
                top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
                const float m_new = fmaxf(m, top * scale), f = exp2_(m - base_of(m_new));
                m = m_new;
                l *= f;
                used *= f;
#pragma unroll
                for (int c = 0; c < DT; ++c) o[c] *= f;
            }
            const float base = base_of(m);
            W16 p[NT][2];
            constexpr int STEPS = NT * QS, PER = 16 * NT / STEPS;  // scores beside a product
            W16 k = k_at(kb, 0, 0);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < QS; ++e) {
                    const int step = t * QS + e;
                    const W16 now_k = k;
                    if (step + 1 < STEPS) k = k_at(kb, (step + 1) / QS, (step + 1) % QS);
                    n[t] = mfma(now_k, qf[e], e == 0 ? v16f{} : n[t]);
#pragma unroll
                    for (int y = step * PER; y < (step + 1) * PER; y += 2) {
                        const int ty = y / 16, ey = y % 16;
                        const float x0 = exp2_(fmaf(s[ty][ey], scale, -base));
                        const float x1 = exp2_(fmaf(s[ty][ey + 1], scale, -base));
                        l += x0 + x1;
                        // (rounded: see CacheTiles::accumulate)
                        const uint32_t w = pack2(x0, x1);
                        used = add2(w, used);
                        p[ty][ey / 8].w[ey % 8 / 2] = w;
                        // (what the compiler knows to be needed later alone it computes later, with
                        // the scores kept in registers until then)
                        asm volatile("" : "+v"(p[ty][ey / 8].w[ey % 8 / 2]), "+v"(l), "+v"(used));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            if (kLate && more) {
                if (more2) put_k(kr, kfree);
                load(vr, vp, a.c.vs, i + 1);
            }
            W16 v = v_at(vb, 0, 0, 0);
#pragma unroll
            for (int y = 0; y < 2 * NT * DT; ++y) {
                const int t = y / (2 * DT), u = y / DT % 2, c = y % DT;
                const W16 now_v = v;
                if (y + 1 < 2 * NT * DT)
                    v = v_at(vb, (y + 1) / (2 * DT), (y + 1) / DT % 2, (y + 1) % DT);
                o[c] = mfma(now_v, p[t][u], o[c]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!kLate && more2) put_k(kr, kfree);
            if (more) put_v(vr, vfree, i + 1);
            __syncthreads();
        };
#pragma unroll 1
        for (int i = sp.first; i < last; i += 2) {
            stage(i, s0, s1, kbuf[1], kbuf[0], vbuf[0], vbuf[1]);
            if (i + 1 >= last) break;
            stage(i + 1, s1, s0, kbuf[0], kbuf[1], vbuf[1], vbuf[0]);
        }
        // (a row's keys lie in two lanes)
        auto both = [](float v) {
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                            false);
            return __uint_as_float(x[0]) + __uint_as_float(x[1]);
        };
        l = both(l);
        used = both(used);
        const int late = opaque(lane), lcol = late & 31, lh = late >> 5;
        const int r = 32 * wave + lcol;
        const Row to = row_of<PRE>(a, sp, row0 + r);
        const float4 z = make_float4(m, l, used, 0.f);
        const bool parted = PRE || sp.part >= 0, on = to.b >= 0;
        const size_t pr = part_row<PRE>(a, max(sp.part, 0), r);
        if (lh == 0 && on) {
            if (parted)
                part_stats<PRE>(a)[pr] = z;
            else if (a.lse)
                a.lse[((size_t)to.b * a.H + to.h) * a.T + to.tok] = lse_of(z);
        }
        const float inv = parted ? 1.f : used == 0.f ? 0.f : 1.f / used;
        float* dims = part_dims<PRE>(a) + pr * D;
        T* out = (T*)a.out + to.b * a.os[0] + to.h * a.os[1] + to.tok * a.os[2];
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = 32 * c + 2 * e + 4 * lh;
                if (d >= D || !on) continue;
                float y[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) y[x] = !parted && used == 0.f ? 0.f : o[c][e + x] * inv;
                if (parted)
                    store4(dims + d, y, 4);
                else
                    store4(out + d, y, 4);
            }
        if (__syncthreads_or(odd)) {
            __threadfence_block();  // (this wave's own stores, from other lanes)
#pragma unroll 1
            for (int x = 0; x < 32; ++x) {
                const int row = row0 + 32 * wave + x;
                const Row w = row_of<PRE>(a, sp, row);
                const float lx = __shfl(l, x);
                if (w.b < 0 || lx != lx) continue;  // (NaN scores: NaN in every dim)
                const int end = min(attended<PRE>(a, sp, row), last * KEYS);
#pragma unroll 1
                for (int d = late; d < D; d += 64) {
                    float sum = 0.f;
#pragma unroll 1
                    for (int j = max(lo, sp.first * KEYS); j < end; ++j) {
                        const int page = page_of(a.c, sp.s.first, j);
                        if (!is_page(a.c, page)) continue;
                        const int in = j - over(j, a.c.by_page) * a.c.page_rows;
                        const float y = Elem<T>::ld(vp + page * a.c.vs[0] + in * a.c.vs[2], d);
                        sum += fabsf(y) < INFINITY ? 0.f : y;
                    }
                    if (fabsf(sum) < INFINITY) continue;
                    if (parted)
                        part_dims<PRE>(a)[part_row<PRE>(a, max(sp.part, 0), 32 * wave + x) * D + d] = sum;
                    else
                        Elem<T>::st((T*)a.out + w.b * a.os[0] + w.h * a.os[1] + w.tok * a.os[2], d, sum);
                }
            }
        }
    });
}

template <int DP, int PRE>
void go_many(const PagedArgs& a, dim3 grid, hipStream_t st) {
    const int rows = pass_of<PRE>(a).rows;
    if (rows == 64)
        hipLaunchKernelGGL((k_paged_many<DP, 2, 32, PRE>), grid, dim3(128), 0, st, a);
    else if (rows == 128)
        hipLaunchKernelGGL((k_paged_many<DP, 4, 64, PRE>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_paged_many<DP, 8, 64, PRE>), grid, dim3(512), 0, st, a);
}

}  // namespace

hipError_t launch_paged_many(const PagedArgs& a, int pre, dim3 grid, hipStream_t st) {
    if (a.c.D <= 64) {
        if (pre) go_many<64, 1>(a, grid, st);
        else go_many<64, 0>(a, grid, st);
    } else {
        if (pre) go_many<128, 1>(a, grid, st);
        else go_many<128, 0>(a, grid, st);
    }
    return hipGetLastError();
}

}  // namespace atn

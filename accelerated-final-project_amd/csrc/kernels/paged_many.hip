// Attention over a paged cache, many query rows (paged_attn_impl.hpp has what its kernels share).
#include "paged_attn_impl.hpp"

namespace atn {

namespace {

// ---------------------------------------------------------------- many query rows
// bf16, at most 128 dims in whole 16-byte pieces, more than 32 query rows of an item: products and
// softmax weigh as much as the reads.  A workgroup's 8 waves are RG groups of 32 query rows times
// KG = 8 / RG groups of KEYS keys of every stage, which comes straight into LDS while the stage
// before is worked on.  MFMA 32 x 32: S^T = K Q^T leaves a lane the scores of query L % 32 for 4
// consecutive keys of every 8, which are the operand of O^T = V^T P^T as they lie; V's comes by the
// transposing LDS read.  The scores of the next stage are computed beside the softmax of this one,
// so that matrix and vector units both have work in every wave.
// 2 sequences of 512 and 342 tokens over 8000 rows, 32 over 8 heads of 128 dims: 163 us in tiles of 256
// rows, 0.71 PFLOP/s of the attended products, bound by the issue of both units and the barrier of
// every stage; the kernel begins with 20 us more than nothing.  Prefixes of 64 query rows: 4 of 16384
// rows, 68 us, 3.9 TB/s.  Fewer than 512 keys go to k_paged_narrow, which begins in 9 us (8 sequences of
// 100 tokens over 100 to 200 rows, 16 over 8 heads: 14 against 22 us).
typedef float v16f __attribute__((ext_vector_type(16)));

template <int DP_, int RG_, int KEYS_>
struct PagedMany {
    static constexpr int DP = DP_, RG = RG_, KG = 8 / RG_, KEYS = KEYS_;
    static constexpr int ALL = KG * KEYS;                // keys of a stage
    static constexpr int ROWS = 32 * RG;
    static constexpr int CH = DP / 8;                    // 16-byte pieces of a row
    static constexpr int NT = KEYS / 32;                 // tiles of a wave's keys
    static constexpr int QS = DP / 16, DT = DP / 32;     // steps of the scores, tiles of dims
    static constexpr int kStage = ALL * DP * 2;
    static constexpr int X = ALL * CH / 512;             // pieces of K (and of V) a lane a stage
    static constexpr int SUB = ALL / 16, AHEAD = 64 / SUB;
    static_assert(X * 512 == ALL * CH, "whole pieces a lane");
    // the results of a key group but the first: slabs of 64 rows, one a buffer where they fit it
    static constexpr bool kInBuffers = KG > 1 && kStage >= 64 * DP * 4;
    static_assert(!kInBuffers || (KG - 1) * ROWS / 64 <= 3, "slabs");
    static constexpr int kSlabs = KG > 1 && !kInBuffers ? (KG - 1) * ROWS * DP / 4 : 1;
    // Pieces lie at a place of their row that changes with it, so that the rows which one LDS
    // cycle reads lie in different banks: 16 keys at one piece (K), 4 keys at four (V).
    static __device__ __forceinline__ int k_place(int key, int c) {
        return DP == 128 ? c ^ (key & 15) : c ^ ((key >> 1) & 7);
    }
    // a lane's 16 bytes from `of` bytes behind a uniform base to LDS: lane L's at to + 16 L
    static __device__ __forceinline__ void load16(const uint16_t* base, uint32_t of, char* to) {
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)((const char*)base + of),
            (__attribute__((address_space(3))) void*)to, 16, 0, 0);
    }
    static __device__ __forceinline__ int v_place(int key, int c) {
        return DP == 128 ? c ^ (4 * (key & 3)) : c ^ (4 * ((key >> 1) & 1));
    }
};

constexpr int kDepth = 3;

template <int DP, int RG, int KEYS, int PRE>
__global__ __launch_bounds__(512, 2) void k_paged_many(PagedArgs a) {
    using N = PagedMany<DP, RG, KEYS>;
    using T = uint16_t;
    using W16 = Words<T, 16>;
    constexpr int CH = N::CH, NT = N::NT, QS = N::QS, DT = N::DT, X = N::X, SUB = N::SUB;
    constexpr int ALL = N::ALL, KG = N::KG, AHEAD = N::AHEAD, ROWS_X = 64 / CH;  // rows of a wave's load
    // (each an object of its own: the compiler lets reads of one pass loads into another)
    __shared__ __align__(16) char k0[N::kStage], k1[N::kStage], v0[N::kStage], v1[N::kStage];
    __shared__ float4 slabs[N::kSlabs];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5, rg = wave % RG, kg = wave / RG;
    const int D = a.c.D, pieces = D / 8;
    const float scale = fabsf(a.scale);
    // Places of pieces past the row's end are 0 (and stay so, but where a span leaves its results there).
    auto clear = [&]() {
        for (int e = 16 * tid; e < N::kStage; e += 16 * 512)
            for (char* z : {k0, k1, v0, v1}) *reinterpret_cast<uint4*>(z + e) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    };
    if (KG == 1 && pieces < CH) clear();
    // This wave's rows of a stage, of one run of 16: lane L loads place L % CH of row L / CH, load x
    // those ROWS_X rows on.  Which piece lies there: PagedMany's places.
    const int wrow = wave * X * ROWS_X, wrun = wrow / 16;
    auto load_k = [&](const T* base, char* buf) {
        const int late = opaque(lane);  // (or each load's offsets are kept in registers)
#pragma unroll
        for (int x = 0; x < X; ++x) {
            const int r = (wrow & 15) + x * ROWS_X + late / CH, c = N::k_place(r, late % CH);
            const uint32_t of = (r * (uint32_t)a.c.ks[2] + 8 * c) * 2;
            if (c < pieces) N::load16(base, of, buf + (wrow + x * ROWS_X) * CH * 16);
        }
    };
    auto load_v = [&](const T* base, char* buf) {
        const int late = opaque(lane);
#pragma unroll
        for (int x = 0; x < X; ++x) {
            const int r = (wrow & 15) + x * ROWS_X + late / CH, c = N::v_place(r, late % CH);
            const uint32_t of = (r * (uint32_t)a.c.vs[2] + 8 * c) * 2;
            if (c < pieces) N::load16(base, of, buf + (wrow + x * ROWS_X) * CH * 16);
        }
    };
    auto landed = [&]() {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __syncthreads();
    };
    // operands: K's piece 2 e + half of key 32 t + col
    // (the place of piece p is that of piece 0 with p's bits turned: one lane value a stage, not one a
    // piece kept in registers)
    auto k_at = [&](const char* buf, int lane_at, int t, int e) {
        return __builtin_bit_cast(
            W16, *reinterpret_cast<const uint4*>(buf + 32 * t * CH * 16 + (lane_at ^ (32 * e))));
    };
    const int k_lane = ((kg * KEYS + col) * CH + N::k_place(col, half)) * 16;
    // ... V's dims 32 c + lane % 32 of the keys that words [8 u, 8 u + 8) of tile t's weights are
    const int sub = lane & 15, dhalf = lane >> 4 & 1;
    const int v_key = 4 * half + (sub >> 2);
    const int v_lane = ((kg * KEYS + v_key) * CH + N::v_place(v_key, 2 * dhalf + ((sub & 3) >> 1))) * 16 +
                       8 * (sub & 1);
    auto v_at = [&](const char* buf, int lane_at, int t, int u, int c) {
        W16 v;
        const char* p = buf + (32 * t + 16 * u) * CH * 16 + (lane_at ^ (64 * c));
        const uint2 x = lds_tr16(reinterpret_cast<const uint16_t*>(p));
        const uint2 y = lds_tr16(reinterpret_cast<const uint16_t*>(p + 8 * CH * 16));
        v.w[0] = x.x, v.w[1] = x.y, v.w[2] = y.x, v.w[3] = y.y;
        return v;
    };
    auto mfma = [](const W16& x, const W16& y, const v16f& z) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x),
                                                       __builtin_bit_cast(bf16x8, y), z, 0, 0, 0);
    };

    each_span<PRE>(a, blockIdx.x, ALL, lane, [&](const Span& sp) {
        const T* kp = (const T*)a.c.K + sp.g * a.c.ks[1];
        const T* vp = (const T*)a.c.V + sp.g * a.c.vs[1];
        const int row0 = sp.tile * N::ROWS, lo = sp.s.lo;
        const int last = min(sp.last, tile_end<PRE>(a, sp.s, sp.tile, ALL));
        const int mine = row0 + 32 * rg + col;  // this lane's query row
        const int upto = attended<PRE>(a, sp, mine);
        // stages [w0, w1) are attended whole by every row
        const int w0 = (lo + ALL - 1) / ALL, w1 = of_wave(attended<PRE>(a, sp, row0)) / ALL;

        // pages of 16 keys: lane l those of stage `at` + l / SUB, run l % SUB; `there`: which are pages
        int at = sp.first;
        auto fetch = [&](int i) {
            return page_of(a.c, sp.s.first, (i + lane / SUB) * ALL + 16 * (lane % SUB));
        };
        int now = fetch(at), next = fetch(at + AHEAD);
        uint64_t there = __builtin_amdgcn_ballot_w64(is_page(a.c, now));
        // of a stage (asked for in their order): where this wave's run begins, and its runs' pages
        struct Run {
            const T *k, *v;
            uint32_t ok;
        };
        auto run_of = [&](int i) {
            if (i >= at + AHEAD) {
                at += AHEAD;
                now = next;
                next = fetch(at + AHEAD);
                there = __builtin_amdgcn_ballot_w64(is_page(a.c, now));
            }
            const int x = (i - at) * SUB, r = i * ALL + 16 * wrun;
            const int p = __builtin_amdgcn_readlane(now, x + wrun), page = is_page(a.c, p) ? p : 0;
            const int in = r - over(r, a.c.by_page) * a.c.page_rows;
            Run y;
            y.k = kp + page * a.c.ks[0] + in * a.c.ks[2];
            y.v = vp + page * a.c.vs[0] + in * a.c.vs[2];
            y.ok = (uint32_t)(there >> x) & ((1u << SUB) - 1);
            return y;
        };
        bool odd = false;  // an infinity or NaN was left out

        const bool any = sp.first < last;
        __syncthreads();  // (the last span's stages have been read)
        if (KG > 1 && pieces < CH) clear();
        Run r0{}, r1{};   // of the stage at work, and the next one
        if (any) {
            r0 = run_of(sp.first);
            load_k(r0.k, k0);
            load_v(r0.v, v0);
            if (sp.first + 1 < last) {
                r1 = run_of(sp.first + 1);
                load_k(r1.k, k1);
            }
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
        for (int c = 0; c < DT; ++c) o[c] = v16f{};
        float m = -INFINITY, l = 0.f, used = 0.f;
        landed();

        v16f s0[NT], s1[NT];
        if (any) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                s0[t] = v16f{};
#pragma unroll
                for (int e = 0; e < QS; ++e) s0[t] = mfma(k_at(k0, k_lane, t, e), qf[e], s0[t]);
            }
        }
        __syncthreads();  // (the first stage loads into the buffer just read)
        auto highest = [&](const v16f (&z)[NT]) {
            float top = z[0][0];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, z[t][e]);
            return top;
        };
        float top = any ? highest(s0) : 0.f;  // of the stage's scores in this lane
        // One stage: its scores s into weights, beside them the next stage's scores n (of what the
        // buffer holds where there is none), then the product with V.
        auto stage = [&](int i, v16f (&s)[NT], v16f (&n)[NT], const char* kb, char* kfree, char* vb,
                         char* vfree) {
            Run r2{};
            if (i + 1 < last) {
                load_v(r1.v, vfree);
                if (i + 2 < last) {
                    r2 = run_of(i + 2);
                    load_k(r2.k, kfree);
                }
            }
            if (i < w0 || i >= w1 || r0.ok != (1u << SUB) - 1) {
                // (some row does not attend some key)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int j0 = i * ALL + kg * KEYS + 32 * t, run = (kg * KEYS + 32 * t) / 16;
                    const uint32_t has = (r0.ok >> run & 1u ? 0xffffu : 0u) |
                                         (r0.ok >> (run + 1) & 1u ? 0xffff0000u : 0u);
                    const uint32_t on = (has & below(upto - j0) & ~below(lo - j0)) >> (4 * half);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!(on >> (8 * (e >> 2) + (e & 3)) & 1u)) s[t][e] = -INFINITY;
                }
                // An infinity or NaN times a weight of 0 would reach rows that do not attend its key: V
                // enters without them, and they are written over the results of the rows that do (of
                // keys that nobody attends, or of no page, there are none).
                const int end = of_wave(attended<PRE>(a, sp, row0 + N::ROWS - 1));
                uint32_t bad = 0;
#pragma unroll 1
                for (int e = opaque(tid); e < ALL * CH; e += 512) {
                    W16 z = reinterpret_cast<W16*>(vb)[e];
                    const int key = e / CH, j = i * ALL + key;
                    uint32_t any = 0;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t hi = (z.w[w] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
                        const uint32_t lw = (z.w[w] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
                        z.w[w] &= ~(hi | lw);
                        any |= hi | lw;
                    }
                    reinterpret_cast<W16*>(vb)[e] = z;
                    if (j >= lo && j < end && (r0.ok >> (key / 16) & 1u)) bad |= any;
                }
                odd |= bad != 0;
                __syncthreads();
                top = highest(s);
            }
            // softmax, as weights() does it
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
            // Products: the next scores', then V's.  Their operands come from LDS DEPTH products ahead.
            // Beside the first half of the weights stand the scores' products, beside the second half
            // V's of the first, beside the rest the next scores' maximum: the vector units have about
            // as much to do in each as the matrix units.
            constexpr int NK = NT * QS, NV = 2 * NT * DT, HALF = 8 * NT, DEPTH = kDepth;
            W16 p[NT][2], x[DEPTH];
            const int kl = opaque(k_lane), vl = opaque(v_lane);
            auto operand = [&](int y) {
                if (y < NK) return k_at(kb, kl, y % NT, y / NT);
                y -= NK;
                return v_at(vb, vl, y / (2 * DT), y / DT % 2, y % DT);
            };
            auto weigh = [&](int z) {  // scores z, z + 1
                const int tz = z / 16, ez = z % 16;
                const float f0 = exp2_(fmaf(s[tz][ez], scale, -base));
                const float f1 = exp2_(fmaf(s[tz][ez + 1], scale, -base));
                l += f0 + f1;
                // (rounded: see CacheTiles::accumulate)
                uint32_t& w = p[tz][ez / 8].w[ez % 8 / 2];
                w = pack2(f0, f1);
                used = add2(w, used);
                // (what the compiler knows to be needed later alone it computes later, with the
                // scores kept in registers until then)
                asm volatile("" : "+v"(w), "+v"(l), "+v"(used));
            };
#pragma unroll
            for (int y = 0; y < DEPTH; ++y) x[y] = operand(y);
#pragma unroll
            for (int y = 0; y < NK; ++y) {
                const int t = y % NT, e = y / NT;
                n[t] = mfma(x[y % DEPTH], qf[e], e == 0 ? v16f{} : n[t]);
                x[y % DEPTH] = operand(y + DEPTH);
#pragma unroll
                for (int z = y * HALF / NK / 2 * 2; z < (y + 1) * HALF / NK / 2 * 2; z += 2) weigh(z);
                __builtin_amdgcn_sched_barrier(0);
            }
            top = n[0][0];
#pragma unroll
            for (int y = 0; y < NV; ++y) {
                const int t = y / (2 * DT), u = y / DT % 2, c = y % DT;
                o[c] = mfma(x[(NK + y) % DEPTH], p[t][u], o[c]);
                if (y + DEPTH < NV) x[(NK + y) % DEPTH] = operand(NK + y + DEPTH);
                if (y < NV / 2) {
#pragma unroll
                    for (int z = y * HALF / (NV / 2); z < (y + 1) * HALF / (NV / 2); z += 2)
                        weigh(HALF + z);
                } else {
                    constexpr int PER = 16 * NT / (NV / 2);
#pragma unroll
                    for (int z = (y - NV / 2) * PER; z < (y - NV / 2 + 1) * PER; ++z)
                        top = fmaxf(top, n[z / 16][z % 16]);
                    asm volatile("" : "+v"(top));
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            r0 = r1;
            r1 = r2;
            landed();
        };
#pragma unroll 1
        for (int i = sp.first; i < last; i += 2) {
            stage(i, s0, s1, k1, k0, v0, v1);
            if (i + 1 >= last) break;
            stage(i + 1, s1, s0, k0, k1, v1, v0);
        }
        // (a row's keys lie in two lanes)
        auto both = [](float v) {
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                            false);
            return __uint_as_float(x[0]) + __uint_as_float(x[1]);
        };
        l = both(l);
        used = both(used);
        if constexpr (KG > 1) {
            // The key groups' results added up: all but the first leave theirs in LDS (a row's pieces
            // of 4 dims at places that change with it, against bank conflicts).
            constexpr int P = DP / 4;
            // (computed here: hoisted out of the loop over spans, these take the loop's registers)
            const int here = opaque(lane), hcol = here & 31, hhalf = here >> 5, turn = hcol & (P - 1);
            float4* stats = reinterpret_cast<float4*>(k0);
            auto slab = [&](int g) {
                const int x = (g - 1) * (N::ROWS / 64) + rg / 2, row = 32 * (rg & 1) + hcol;
                if (!N::kInBuffers) return slabs + (64 * x + row) * P;
                return reinterpret_cast<float4*>(x == 0 ? v0 : x == 1 ? v1 : k1) + row * P;
            };
            if (kg > 0) {
                if (hhalf == 0) stats[(kg - 1) * N::ROWS + 32 * rg + hcol] = make_float4(m, l, used, 0.f);
                float4* to = slab(kg);
#pragma unroll
                for (int c = 0; c < DT; ++c)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        to[(8 * c + e / 2 + hhalf) ^ turn] =
                            make_float4(o[c][e], o[c][e + 1], o[c][e + 2], o[c][e + 3]);
            }
            __syncthreads();
            if (kg == 0) {
                float4 z[KG];
                float top = m;
#pragma unroll
                for (int g = 1; g < KG; ++g) {
                    z[g] = stats[(g - 1) * N::ROWS + 32 * rg + hcol];
                    top = fmaxf(top, z[g].x);
                }
                const float base = base_of(top), f0 = exp2_(m - base);
                m = top;
                l *= f0;
                used *= f0;
#pragma unroll
                for (int c = 0; c < DT; ++c) o[c] *= f0;
#pragma unroll
                for (int g = 1; g < KG; ++g) {
                    const float f = exp2_(z[g].x - base);
                    l += z[g].y * f;
                    used += z[g].z * f;
                    const float4* from = slab(g);
#pragma unroll
                    for (int c = 0; c < DT; ++c)
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const float4 y = from[(8 * c + e / 2 + hhalf) ^ turn];
                            o[c][e] += y.x * f, o[c][e + 1] += y.y * f;
                            o[c][e + 2] += y.z * f, o[c][e + 3] += y.w * f;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                }
            }
        }
        const int late = opaque(lane), lcol = late & 31, lh = late >> 5;
        const int r = 32 * rg + lcol;
        const Row to = row_of<PRE>(a, sp, row0 + r);
        const float4 z = make_float4(m, l, used, 0.f);
        const bool parted = PRE || sp.part >= 0, on = to.b >= 0 && kg == 0;
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
        if (__syncthreads_or(odd) && kg == 0) {
            // V's rows once more, dims 2 L and 2 L + 1 in lane L: for each of the two the rows (a bit each) that
            // attend an infinity or NaN there (two parts of 512 tokens over 3000 rows, one infinity: 90 us,
            // 57 without).
            const bool live = to.b >= 0 && l == l;  // (NaN scores: NaN in every dim)
            const int mine_upto = attended<PRE>(a, sp, row0 + r);
            const int d = 2 * late, end = min(of_wave(attended<PRE>(a, sp, row0 + 32 * rg + 31)), last * ALL);
            uint32_t pos[2] = {0, 0}, neg[2] = {0, 0}, nan[2] = {0, 0};
#pragma unroll 1
            for (int j0 = max(lo, sp.first * ALL) & -16; j0 < end; j0 += 16) {
                const int page = of_wave(page_of(a.c, sp.s.first, j0));
                if (!is_page(a.c, page)) continue;
                const int in = j0 - over(j0, a.c.by_page) * a.c.page_rows;
                const T* v = vp + page * a.c.vs[0] + in * a.c.vs[2] + min(d, D - 2);
                uint32_t y[16];
#pragma unroll
                for (int u = 0; u < 16; ++u) __builtin_memcpy(&y[u], v + u * a.c.vs[2], 4);
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    const bool lw = (y[u] & 0x7f80u) == 0x7f80u, hi = (y[u] & 0x7f800000u) == 0x7f800000u;
                    if (!__builtin_amdgcn_ballot_w64(lw || hi) || j0 + u < lo) continue;
                    const uint32_t rows = (uint32_t)__builtin_amdgcn_ballot_w64(live && mine_upto > j0 + u);
                    if (lw) (y[u] & 0x7fu ? nan : y[u] & 0x8000u ? neg : pos)[0] |= rows;
                    if (hi) (y[u] & 0x7f0000u ? nan : y[u] >> 31 ? neg : pos)[1] |= rows;
                }
            }
            __threadfence_block();  // (this wave's own stores, from other lanes)
#pragma unroll 1
            for (int x = 0; x < 32; ++x) {
                const Row w = row_of<PRE>(a, sp, row0 + 32 * rg + x);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (d >= D || !((pos[h] | neg[h] | nan[h]) >> x & 1u)) continue;
                    const float y = (nan[h] | (pos[h] & neg[h])) >> x & 1u ? __builtin_nanf("")
                                    : pos[h] >> x & 1u ? INFINITY : -INFINITY;
                    if (parted)
                        part_dims<PRE>(a)[part_row<PRE>(a, max(sp.part, 0), 32 * rg + x) * D + d + h] = y;
                    else
                        Elem<T>::st((T*)a.out + w.b * a.os[0] + w.h * a.os[1] + w.tok * a.os[2], d + h, y);
                }
            }
        }
    });
}

template <int DP, int PRE>
void go_many(const PagedArgs& a, dim3 grid, hipStream_t st) {
    const int rows = pass_of<PRE>(a).rows;
    const dim3 block(512);
    if (rows == 64)
        hipLaunchKernelGGL((k_paged_many<DP, 2, 32, PRE>), grid, block, 0, st, a);
    else if (rows == 128)
        hipLaunchKernelGGL((k_paged_many<DP, 4, 32, PRE>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((k_paged_many<DP, 8, 64, PRE>), grid, block, 0, st, a);
}

}  // namespace

hipError_t launch_paged_many(const PagedArgs& a, int pre, hipStream_t st) {
    const dim3 grid((unsigned)(pre ? a.plan.pre.workgroups : a.plan.own.workgroups));
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

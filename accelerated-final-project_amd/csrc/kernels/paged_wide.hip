// Attention over a paged cache, head_d > 256 (paged_attn_impl.hpp has what its kernels share).  No
// output tile fits a wave's registers, so two kernels with the scores between them: k_paged_scores
// writes x (a row's are few floats beside K and V's rows of head_d), each workgroup's 8 waves
// sharing a tile's dims, or its share of them, and adding up through LDS; k_paged_values is the
// softmax over them and the product with V, each wave 16 VL dims of the output.  Keys lie in blocks
// of 32.  Both take the prefixes' items and the sequences' own in one launch.  The reads of K, then of V
// bound them: fp32, one token of 4 heads of 2048 dims, 8 sequences of 100 to 500 rows under 1000
// shared ones, 30 and 39 us, 3.7 and 2.8 TB/s.
#include "paged_attn_impl.hpp"

namespace atn {

namespace {

constexpr int kBlock = 32;
constexpr int kScoreWaves = 8;
constexpr int kWaves = 4;        // of a value workgroup
constexpr int kValueKeys = 128;  // keys between barriers of k_paged_values

// Scores of a block: [share][place in the line without padding][rows][32], to be added over the shares.
template <int PRE>
__device__ __forceinline__ float* scores_of(const PagedArgs& a, int share, int place) {
    const int64_t block = pass_of<PRE>(a).rows * kBlock;
    return (PRE ? a.pre_scores : a.own_scores) + share * pass_of<PRE>(a).scores + place * block;
}

// K's 32 rows and a tile's query rows, 128 bytes of each at a time, in a wave's own part of LDS: rows
// are loaded 8 lanes each (a load straight into the products' operands takes 16 bytes of every row
// from a cache that delivers 64 a cycle), pieces at places that change with the row, so that the 16
// rows of an operand lie in different banks.
constexpr int kRowBytes = 128;
template <int MT>
struct Stage {
    static constexpr int ROWS = kBlock + 16 * MT, LOADS = ROWS / 8;
    static constexpr int kBytes = ROWS * kRowBytes;  // (also what the partial scores need)
    static_assert(kBytes >= MT * (kBlock / 16) * 64 * 16, "partial scores");
    static __device__ __forceinline__ int place(int row, int piece) { return piece ^ (row >> 1 & 7); }
};

// The scores of a wave's share of the dims (every `waves`-th 128 bytes from `wave` on), from LDS.
template <typename T, int MT, int PRE>
__device__ __forceinline__ void staged_scores(v4f (&s)[MT][2], const PagedArgs& a, const Span& sp, int j0,
                                              int row0, int wave, int waves, char* lds, int lane) {
    using S = Stage<MT>;
    using N = CacheTiles<T, 64, MT, kExact>;
    const int q = lane >> 4, col = lane & 15, bytes = a.c.D * (int)sizeof(T);
    // load x: rows 8 x + lane / 8 (keys, then queries), the piece that lies at place lane % 8 there
    const char* from[S::LOADS];
#pragma unroll
    for (int x = 0; x < S::LOADS; ++x) {
        const int row = 8 * x + lane / 8;
        if (x < kBlock / 8) {  // (past the last row: that one again)
            const int r = min(j0 + row, max(j0, sp.s.hi - 1)), page = page_of(a.c, sp.s.first, r);
            from[x] = (const char*)((const T*)a.c.K + (is_page(a.c, page) ? page : 0) * a.c.ks[0] +
                                    sp.g * a.c.ks[1] +
                                    (r - over(r, a.c.by_page) * a.c.page_rows) * a.c.ks[2]);
        } else {
            from[x] = (const char*)((const T*)a.Q + q_at<PRE>(a, sp, row0 + row - kBlock));
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[t][u] = v4f{0.f, 0.f, 0.f, 0.f};
    auto at = [&](int row, int piece) {
        return __builtin_bit_cast(typename N::KPiece, *reinterpret_cast<const uint4*>(
                                                          lds + row * kRowBytes + 16 * S::place(row, piece)));
    };
#pragma unroll 1
    for (int step = wave; step * kRowBytes < bytes; step += waves) {
        const int left = bytes - step * kRowBytes;
        if (left < kRowBytes) {  // (pieces past the row's end are 0)
            for (int e = 16 * lane; e < S::kBytes; e += 16 * 64)
                *reinterpret_cast<uint4*>(lds + e) = make_uint4(0, 0, 0, 0);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): LDS has been read and written
        const int mine = opaque(lane);
#pragma unroll
        for (int x = 0; x < S::LOADS; ++x) {
            const int of = 16 * S::place(8 * x + mine / 8, mine % 8);
            if (of < left)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void*)(from[x] + step * kRowBytes + of),
                    (__attribute__((address_space(3))) void*)(lds + 8 * x * kRowBytes), 16, 0, 0);
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        asm volatile("" ::: "memory");
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            typename N::KPiece k[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) k[u] = at(16 * u + col, 4 * e + q);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const typename N::KPiece f = at(kBlock + 16 * t + col, 4 * e + q);
#pragma unroll
                for (int u = 0; u < 2; ++u) s[t][u] = N::dot(k[u], f, s[t][u]);
            }
        }
    }
}

template <typename T, int MT, int PRE, bool STAGED>
__device__ __forceinline__ void block_scores(const PagedArgs& a, const Groups& gr, const Line& line,
                                             int unit, char* lds) {
    constexpr int SUB = kBlock / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15;
    const int shares = a.plan.shares, place = (unsigned)unit / (unsigned)shares;
    const int share = unit - place * shares;
    const Place p = place_at<PRE>(a, gr, line, place, kBlock, lane, 0);
    Span sp;
    sp.s = segment<PRE>(a, gr, p.seg);
    sp.s.lo = of_wave(sp.s.lo), sp.s.hi = of_wave(sp.s.hi), sp.s.len = of_wave(sp.s.len);
    sp.s.first = of_wave(sp.s.first), sp.s.members = of_wave(sp.s.members);
    const int off = place - p.start, item = (unsigned)off / (unsigned)p.n;
    const int tiles = of_wave(sp.s.tiles), g = (unsigned)item / (unsigned)max(1, tiles);
    sp.g = a.g0 + min(g, a.gs - 1);
    sp.tile = item - g * tiles;
    const int i = sp.s.lo / kBlock + off - item * p.n;
    if (i >= tile_end<PRE>(a, sp.s, sp.tile, kBlock)) return;
    const int row0 = sp.tile * 16 * MT;
    uint32_t there = 0;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
        const bool is = is_page(a.c, page_of(a.c, sp.s.first, i * kBlock + 16 * u + col));
        there |= ((uint32_t)__builtin_amdgcn_ballot_w64(is) & 0xffffu) << (16 * u);
    }
    v4f s[MT][SUB];
    const int w = share * kScoreWaves + wave, waves = shares * kScoreWaves;
    __syncthreads();  // (the block before has been read)
    char* mine = lds + wave * Stage<MT>::kBytes;
    if constexpr (STAGED) {
        staged_scores<T, MT, PRE>(s, a, sp, i * kBlock, row0, w, waves, mine, lane);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // (this wave's part of LDS has been read)
    } else {
        const T* kp[SUB];
        const T* qp[MT];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const int r = min(i * kBlock + 16 * u + col, max(i * kBlock, sp.s.hi - 1));
            const int page = page_of(a.c, sp.s.first, r);
            kp[u] = (const T*)a.c.K + (is_page(a.c, page) ? page : 0) * a.c.ks[0] + sp.g * a.c.ks[1] +
                    (r - over(r, a.c.by_page) * a.c.page_rows) * a.c.ks[2];
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) qp[t] = (const T*)a.Q + q_at<PRE>(a, sp, row0 + 16 * t + col);
        wide_scores<T, MT, true>(s, kp, qp, a.c.D, w, waves, q);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < SUB; ++u)
            reinterpret_cast<v4f*>(mine)[(t * SUB + u) * 64 + lane] = s[t][u];
    __syncthreads();
    // one thread per row and 4 keys
    if (threadIdx.x >= MT * SUB * 64) return;
    const int u = wave % SUB, t = wave / SUB;
    v4f x = reinterpret_cast<const v4f*>(lds)[threadIdx.x];
#pragma unroll
    for (int w = 1; w < kScoreWaves; ++w)
        x += reinterpret_cast<const v4f*>(lds + w * Stage<MT>::kBytes)[threadIdx.x];
    const uint32_t see = seen<SUB>(i * kBlock, sp.s.lo, attended<PRE>(a, sp, row0 + 16 * t + col), there,
                                   q) >> (4 * u);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = see >> e & 1u ? x[e] * a.scale : -INFINITY;
    float* to = scores_of<PRE>(a, share, place) + (16 * t + col) * kBlock + 16 * u + 4 * q;
    *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
}

// STAGED: rows are whole 16-byte pieces that lie so.
template <typename T, int OWN, int PRE, bool STAGED>
__global__ __launch_bounds__(64 * kScoreWaves) void k_paged_scores(PagedArgs a) {
    __shared__ __align__(16) char lds[kScoreWaves * Stage<(OWN > PRE ? OWN : PRE)>::kBytes];
    const int lane = threadIdx.x & 63;
    const Groups gr = groups_of(a, lane);
    Line pre{};
    if (a.groups > 0) pre = line_of<1>(a, gr, kBlock, lane, 0);
    const Line own = line_of<0>(a, gr, kBlock, lane, 0);
    const int first = pre.total * a.plan.shares, all = first + own.total * a.plan.shares;
#pragma unroll 1
    for (int u = blockIdx.x; u < all; u += gridDim.x) {
        if (u < first)
            block_scores<T, PRE, 1, STAGED>(a, gr, pre, u, lds);
        else
            block_scores<T, OWN, 0, STAGED>(a, gr, own, u - first, lds);
    }
}

template <typename T>
constexpr int wide_dims() {  // of a value workgroup
    return (sizeof(T) == 2 ? 128 : 64) * kWaves;
}

template <typename T, int MT>
struct Values : CacheTiles<T, (sizeof(T) == 2 ? 128 : 64), MT, kClamp> {
    static constexpr int LDP = kValueKeys + 16 / (int)sizeof(T);
    T pl[2][16 * MT * LDP];
    float alpha[2][16 * MT];
    float4 fin[16 * MT];
};

template <typename T, int MT, int PRE>
__device__ __forceinline__ void paged_values(const PagedArgs& a, int id, Values<T, MT>& x_) {
    constexpr bool kBf = sizeof(T) == 2;
    // (a wave's dims: one V step of 128 in bf16, 64 in fp32; where the row ends before, its last
    // ones; those before d0 are the wave's before)
    using N = Values<T, MT>;
    constexpr int VL = N::VL, WD = N::VD, ROWS = N::ROWS, PK = N::KB, NB = kValueKeys / PK;
    constexpr int LDP = N::LDP, STEP = kValueKeys / kBlock;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, col = lane & 15, D = a.c.D;
    // (workgroups of an item: runs of dims, times tiles of ROWS of the item's rows)
    const int all = pass_of<PRE>(a).groups, subs = pass_of<PRE>(a).rows / ROWS, groups = all / subs;
    const int unit = (unsigned)id / (unsigned)all, mine = id - unit * all;
    const int sub = subs > 1 ? mine % subs : 0, chunk0 = mine / subs;
    // softmax: 16 threads a row, 8 keys each, one pass per 16 rows
    const int sr = threadIdx.x >> 4, sk = (threadIdx.x & 15) * 8;

    each_span<PRE, true>(a, unit, kBlock, lane, [&](const Span& sp) {
      // (short items: a workgroup takes several runs of dims, one after another)
#pragma unroll 1
      for (int chunk = chunk0; chunk * kWaves * WD < D; chunk += groups) {
        const int d0 = (chunk * kWaves + wave) * WD;
        const bool busy = d0 < D;
        const T* vp = (const T*)a.c.V + sp.g * a.c.vs[1] + d0;
        const int row0 = sp.tile * pass_of<PRE>(a).rows + sub * ROWS, lo = sp.s.lo, b0 = lo / kBlock;
        const int last = min(sp.last, tile_end<PRE>(a, sp.s, sp.tile, kBlock));
        // rows of keys that any row attends
        const int end = max(lo + 1, min(last * kBlock, PRE ? sp.s.hi : of_wave(attended<PRE>(
                                                           a, sp, row0 + ROWS - 1))));
        const int whole0 = (lo + PK - 1) / PK, whole1 = of_wave(attended<PRE>(a, sp, row0)) / PK;
        const float* sc = scores_of<PRE>(a, 0, sp.blocks_before);
        float m[MT], l[MT], used[MT], x[MT][8];
        v4f o[MT][1][VL];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            m[t] = -INFINITY;
            l[t] = used[t] = 0.f;
#pragma unroll
            for (int c = 0; c < VL; ++c) o[t][0][c] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        // scores of the step at block i
        auto load_x = [&](int i) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float* from = sc + (int64_t)(i - b0 + sk / kBlock) * (pass_of<PRE>(a).rows * kBlock) +
                                    (sub * ROWS + 16 * t + sr) * kBlock + sk % kBlock;
                v4f u = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, w = u;
                if (sk < (last - i) * kBlock) {
                    u = *reinterpret_cast<const v4f*>(from);
                    w = *reinterpret_cast<const v4f*>(from + 4);
                    for (int y = 1; y < a.plan.shares; ++y) {
                        from += pass_of<PRE>(a).scores;
                        u += *reinterpret_cast<const v4f*>(from);
                        w += *reinterpret_cast<const v4f*>(from + 4);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[t][e] = u[e], x[t][4 + e] = w[e];
            }
        };
        // pages of a step's keys lane and 64 + lane
        struct Pair {
            int lo, hi;
        };
        auto pages_of = [&](int i) {
            Pair p;
            p.lo = page_of(a.c, sp.s.first, i * kBlock + lane);
            p.hi = page_of(a.c, sp.s.first, i * kBlock + 64 + lane);
            return p;
        };
        // V of keys [k, k + PK) of the step at block i
        auto load_v = [&](typename N::Vals& to, const Pair& pg, int i, int k) {
#pragma unroll
            for (int j = 0; j < N::KEYS; ++j) {
                // (past the last row: that one again)
                const int key = min(k + N::key_of(lane, j), end - 1 - i * kBlock), r = i * kBlock + key;
                const int p = __shfl(key < 64 ? pg.lo : pg.hi, key & 63);
                const T* row = vp + (is_page(a.c, p) ? p : 0) * a.c.vs[0] +
                               (r - over(r, a.c.by_page) * a.c.page_rows) * a.c.vs[2];
                to.p[j][0] = N::v_piece(row, 0, 0, D - d0, lane);
                // (all rows' addresses at once would take the registers of the output)
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // Two buffers of weights: a wave past a barrier writes the other one, and comes to write
        // this one only after the next barrier, when every wave has read it.
        typename N::Vals v0, v1;
        __syncthreads();  // (the last span's)
        Pair now{}, next{};
        const bool any = sp.first < last;
        if (any) {
            load_x(sp.first);
            now = pages_of(sp.first);
            next = pages_of(sp.first + STEP);
            if (busy) load_v(v0, now, sp.first, 0);
        }
        int buf = 0;
#pragma unroll 1
        for (int i = sp.first; i < last; i += STEP, buf ^= 1) {
            // scores into weights
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                float top = x[t][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) top = fmaxf(top, x[t][e]);
                top = fmaxf(top, dpp<kDppQuadXor1>(top));
                top = fmaxf(top, dpp<kDppQuadXor2>(top));
                top = fmaxf(top, dpp<kDppRowHalfMirror>(top));
                top = fmaxf(top, dpp<kDppRowMirror>(top));
                const float m_new = fmaxf(m[t], top), base = base_of(m_new);
                const float f = exp2_(m[t] - base);
                m[t] = m_new;
                l[t] *= f;
                used[t] *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[t][e] = exp2_(x[t][e] - base);
                    l[t] += x[t][e];
                }
                if ((threadIdx.x & 15) == 0) x_.alpha[buf][16 * t + sr] = f;
                T* to = x_.pl[buf] + (16 * t + sr) * LDP + sk;
                if constexpr (kBf) {  // (rounded: see CacheTiles::accumulate)
                    uint32_t w[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        w[h] = pack2(x[t][2 * h], x[t][2 * h + 1]);
                        used[t] = add2(w[h], used[t]);
                    }
                    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    *reinterpret_cast<float4*>(to) =
                        make_float4(x[t][0], x[t][1], x[t][2], x[t][3]);
                    *reinterpret_cast<float4*>(to + 4) =
                        make_float4(x[t][4], x[t][5], x[t][6], x[t][7]);
                }
            }
            if (i + STEP < last) load_x(i + STEP);
            __syncthreads();
            if (busy) {
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const float f = x_.alpha[buf][16 * t + col];
                    if (__builtin_amdgcn_ballot_w64(f != 1.f)) {
#pragma unroll
                        for (int c = 0; c < VL; ++c) o[t][0][c] *= f;
                    }
                }
                // each PK keys' V on their way while the ones before are used
                auto use = [&](typename N::Vals& v, int k) {
                    const int j0 = i * kBlock + k, b = j0 / PK;
                    const uint32_t there =
                        (uint32_t)(__builtin_amdgcn_ballot_w64(is_page(a.c, k < 64 ? now.lo : now.hi)) >>
                                   (k & 63)) & below(PK);
                    if ((b < whole0 || b >= whole1 || there != below(PK)) && not_finite<T>(v)) {
                        uint32_t see[MT];
#pragma unroll
                        for (int t = 0; t < MT; ++t)
                            see[t] = seen<N::SUB>(j0, lo, attended<PRE>(a, sp, row0 + 16 * t + col),
                                                  there, q);
                        spread_not_finite<T, N, MT>(o, v, see);
                    }
                    N::accumulate_lds(o, v, x_.pl[buf] + k, LDP, lane);
                };
                const int nb = min(NB, (end - i * kBlock + PK - 1) / PK);
#pragma unroll 1
                for (int k = 0; k < nb; k += 2) {
                    if (k + 1 < nb) load_v(v1, now, i, (k + 1) * PK);
                    __builtin_amdgcn_sched_barrier(0);
                    use(v0, k * PK);
                    if (k + 2 < nb)
                        load_v(v0, now, i, (k + 2) * PK);
                    else if (i + STEP < last)  // the next step's first
                        load_v(v0, next, i + STEP, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    if (k + 1 < nb) use(v1, (k + 1) * PK);
                }
            }
            now = next;
            next = pages_of(i + 2 * STEP);
        }
        // sums of the rows, for the waves that hold their outputs
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float y = row16_sum(l[t]), z = kBf ? row16_sum(used[t]) : y;
            if ((threadIdx.x & 15) == 0) x_.fin[16 * t + sr] = make_float4(m[t], y, z, 0.f);
        }
        __syncthreads();
        if (!busy) continue;
        // (computed here: hoisted out of the loop over spans, these take the loop's registers)
        const int late = opaque(lane), lq = late >> 4, lc = late & 15;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = 16 * t + lc;
            const Row to = row_of<PRE>(a, sp, row0 + r);
            if (to.b < 0) continue;
            const float4 z = x_.fin[r];
            const bool parted = PRE || sp.part >= 0, zero = !parted && z.z == 0.f;
            const size_t pr = part_row<PRE>(a, max(sp.part, 0), sub * ROWS + r);
            const float inv = parted ? 1.f : 1.f / z.z;
            if (lq == 0 && d0 == 0) {
                if (parted)
                    part_stats<PRE>(a)[pr] = z;
                else if (a.lse)
                    a.lse[((size_t)to.b * a.H + to.h) * a.T + to.tok] = lse_of(z);
            }
            float* dims = part_dims<PRE>(a) + pr * D + d0;
            T* out = (T*)a.out + to.b * a.os[0] + to.h * a.os[1] + to.tok * a.os[2] + d0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = N::dim_of(0, 4 * lq + e, D - d0);
#pragma unroll
                for (int c = 0; c < VL; c += 4) {
                    float y[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] = zero ? 0.f : o[t][0][c + r][e] * inv;
                    if (d + c >= 0) {
                        if (parted)
                            store4(dims + d + c, y, 4);
                        else
                            store4(out + d + c, y, 4);
                    } else {  // (a row's last dims, fewer than a piece)
#pragma unroll
                        for (int r = 1; r < 4; ++r)
                            if (d + c + r >= 0) {
                                if (parted)
                                    dims[d + c + r] = y[r];
                                else
                                    Elem<T>::st(out, d + c + r, y[r]);
                            }
                    }
                }
            }
        }
      }
    });
}

template <typename T, int OWN, int PRE>
__global__ __launch_bounds__(64 * kWaves, OWN + PRE == 2 && sizeof(T) == 4 ? 3 : 2) void k_paged_values(
    PagedArgs a) {
    constexpr size_t kOwn = sizeof(Values<T, OWN>), kPre = sizeof(Values<T, PRE>);
    __shared__ __align__(16) char lds[kOwn > kPre ? kOwn : kPre];
    const int id = (int)blockIdx.x - a.plan.first;
    if (id < 0)
        paged_values<T, PRE, 1>(a, blockIdx.x, *reinterpret_cast<Values<T, PRE>*>(lds));
    else
        paged_values<T, OWN, 0>(a, id, *reinterpret_cast<Values<T, OWN>*>(lds));
}

// OWN, PRE: 16 rows of tiles of the scores; the values' are of 32 rows at most
template <typename T, int OWN, int PRE>
void go(const PagedArgs& a, hipStream_t st) {
    const dim3 grid(a.plan.score_grid), block(64 * kScoreWaves);
    if (a.plan.whole16)
        hipLaunchKernelGGL((k_paged_scores<T, OWN, PRE, true>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((k_paged_scores<T, OWN, PRE, false>), grid, block, 0, st, a);
    hipLaunchKernelGGL((k_paged_values<T, (OWN > 2 ? 2 : OWN), (PRE > 2 ? 2 : PRE)>),
                       dim3((unsigned)(a.plan.first + a.plan.own.workgroups)), dim3(64 * kWaves), 0, st,
                       a);
}
template <typename T>
void go_rows_wide(const PagedArgs& a, hipStream_t st) {
    const int pre = a.groups > 0 ? a.plan.pre.rows : 16;
    if (a.plan.own.rows == 64) go<T, 4, 4>(a, st);
    else if (a.plan.own.rows == 32) go<T, 2, 2>(a, st);
    else if (pre == 32) go<T, 1, 2>(a, st);
    else go<T, 1, 1>(a, st);
}

}  // namespace

static_assert(wide_dims<float>() == kPagedWideDims / 2 && wide_dims<uint16_t>() == kPagedWideDims,
              "dims of a value workgroup");
static_assert(kBlock == kPagedWideBlock && kValueKeys == kBlock * kPagedWideTurn, "blocks");

hipError_t launch_paged_wide(int dtype, const PagedArgs& a, hipStream_t st) {
    if (dtype == kDtypeF32) go_rows_wide<float>(a, st);
    else go_rows_wide<uint16_t>(a, st);
    return hipGetLastError();
}

}  // namespace atn

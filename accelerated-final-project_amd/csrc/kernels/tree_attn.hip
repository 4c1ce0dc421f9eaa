// Attention of drafted tokens over a key/value cache: row (h, t) attends
// every cache row in use and the drafts that its mask names,
//   x_j = scale q . k_j,  m = max x,  l = sum exp(x - m),
//   out = sum exp(x - m) v / l,  lse = m + log l.
#include "kv_cache.hpp"

namespace atn {

namespace {

// One workgroup per row: keys in blocks of 256 (a wave per key, lanes over
// the dims), the running maximum and sum in fp32, the output's dims in
// registers (32 per thread at head_d 8192).
constexpr int kDimsPerThread = 32;

template <typename T>
__global__ __launch_bounds__(256) void k_tree_rows(TreeArgs a) {
    __shared__ float p[256];
    __shared__ float red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x % a.d.T, h = (blockIdx.x / a.d.T) % a.d.H;
    const int b = blockIdx.x / (a.d.T * a.d.H), g = h / (a.d.H / a.c.G);
    const int L = rows_in_use(a.c, b), n = drafts_of(a.d, b), D = a.c.D;
    if (t >= n) return;
    const T* q = (const T*)a.d.Q + b * a.d.qs[0] + h * a.d.qs[1] + t * a.d.qs[2];
    const T* kc = (const T*)a.c.K + b * a.c.ks[0] + g * a.c.ks[1];
    const T* vc = (const T*)a.c.V + b * a.c.vs[0] + g * a.c.vs[1];
    const T* kd = (const T*)a.d.K + b * a.d.ks[0] + g * a.d.ks[1];
    const T* vd = (const T*)a.d.V + b * a.d.vs[0] + g * a.d.vs[1];
    const int keys = L + (a.d.K ? n : 0);
    float m = -INFINITY, l = 0.f, acc[kDimsPerThread];
#pragma unroll
    for (int i = 0; i < kDimsPerThread; ++i) acc[i] = 0.f;
    for (int k0 = 0; k0 < keys; k0 += 256) {
        const int nk = min(256, keys - k0);
        for (int i = wave; i < nk; i += 4) {
            const int j = k0 + i;
            float s = -INFINITY;
            if (j < L || sees(a.d, b, t, j - L)) {
                const T* k = j < L ? kc + j * a.c.ks[2] : kd + (j - L) * a.d.ks[2];
                float x = 0.f;
                for (int d = lane; d < D; d += 64) x = fmaf(Elem<T>::ld(q, d), Elem<T>::ld(k, d), x);
                s = wave_sum(x) * a.scale;
            }
            if (lane == 0) p[i] = s;
        }
        __syncthreads();
        const float s = threadIdx.x < nk ? p[threadIdx.x] : -INFINITY;
        const float wm = wave_max(s);
        if (lane == 0) red[wave] = wm;
        __syncthreads();
        const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        // no key seen so far: nothing to scale, and no key of this block counts
        const float base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = m == -INFINITY ? 0.f : exp2f(m - base);
        const float e = exp2f(s - base);
        const float ws = wave_sum(e);
        __syncthreads();
        if (lane == 0) red[wave] = ws;
        if (threadIdx.x < nk) p[threadIdx.x] = e;
        __syncthreads();
        l = l * alpha + (red[0] + red[1]) + (red[2] + red[3]);
        m = m_new;
#pragma unroll
        for (int i = 0; i < kDimsPerThread; ++i) acc[i] *= alpha;
        for (int i = 0; i < nk; ++i) {
            const int j = k0 + i;
            if (j >= L && !sees(a.d, b, t, j - L)) continue;  // its V may be anything
            const T* v = j < L ? vc + j * a.c.vs[2] : vd + (j - L) * a.d.vs[2];
#pragma unroll
            for (int c = 0; c < kDimsPerThread; ++c) {
                const int d = threadIdx.x + 256 * c;
                if (d < D) acc[c] = fmaf(p[i], Elem<T>::ld(v, d), acc[c]);
            }
        }
        __syncthreads();
    }
    T* o = (T*)a.out + b * a.os[0] + h * a.os[1] + t * a.os[2];
    // (l == 0: nothing visible, or no score above -infinity)
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < kDimsPerThread; ++c) {
        const int d = threadIdx.x + 256 * c;
        if (d < D) Elem<T>::st(o, d, l == 0.f ? 0.f : acc[c] * inv);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[((size_t)b * a.d.H + h) * a.d.T + t] =
            l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

}  // namespace

TreePlan tree_plan(int, int B, int, int H, int T, int, int, size_t) {
    return TreePlan{1, 1, 1, 0, (int64_t)B * H * T};
}

hipError_t launch_tree_attention(int dtype, const TreeArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)a.c.B * a.d.H * a.d.T);
    if (dtype == kDtypeF32)
        hipLaunchKernelGGL(k_tree_rows<float>, grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(k_tree_rows<uint16_t>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace atn

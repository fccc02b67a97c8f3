// Group normalisation with an activation on channels-last activations [B][P][C] (P pixels):
//   mean, var over the P * (C/G) values of one sample's group;  xh = (x - mean) * rstd
//   p = xh * gamma + beta;  y = act(p)                      act: none, ReLU, SiLU
// and its backward: dp = dy * act'(p);  dbeta = sum dp;  dgamma = sum dp * xh
//   dx = rstd * (gamma*dp - s1 - xh*s2),  s1, s2 = group means of gamma*dp, gamma*dp*xh
// Memory-bound (a few operations per value).  Two forms:
//   one pass ("resident"): a block owns a slab of whole groups of one sample and holds it in
//     registers between the statistics and the result, so every value is read once;
//   two passes: a slab too large for a block is cut into chunks of pixels; the second pass merges
//     the per-chunk partials first (a launch of its own does where they are many), then
//     applies them.  Measured (training, forward and backward, 16 x 256^2 x 64 fp32, 268 MB):
//     58 + 86 and 115 + 138 us, 4.6 to 6.2 TB/s each against 4.8 of a plain copy; the second
//     readings come from the memory-side cache in part.  Two passes in one launch, one part
//     of the batch behind the other, were slower (428 us against 398 in all).
// Statistics are centred: (mean, M2) of short runs merged by Chan's rule, or the mean first
// and squares of differences after, never sum(x^2) - n*mean^2.  No atomics: every sum has a
// fixed order.
#include "common.h"
#include "vecio.h"

namespace ugpg {

// SiLU's exponential is exp2 of the rounded p * log2(e): off by (2|p| + 4) half steps of itself,
// which reaches the result times |p| s (1 - s), at most 2 half steps of 1 in all.
__device__ __forceinline__ float gn_act(float p, int act) {
    if (act == UGPG_ACT_RELU) return p < 0.f ? 0.f : p;  // (a NaN stays one)
    if (act == UGPG_ACT_SILU) return p / (1.f + __expf(-p));
    return p;
}
// dy * act'(p)
__device__ __forceinline__ float gn_act_bwd(float dy, float p, int act) {
    if (act == UGPG_ACT_RELU) return p > 0.f ? dy : (p != p ? p : 0.f);
    if (act == UGPG_ACT_SILU) {
        const float s = 1.f / (1.f + __expf(-p));
        return dy * (s * fmaf(p, 1.f - s, 1.f));
    }
    return dy;
}

// ---------------------------------------------------------------- two passes
// Block (b, chunk, column block): cb vector columns x `rows` pixel rows of threads, each
// thread keeps its V channels and steps over the chunk's pixels.
constexpr int GN_NT = 512;  // threads of a block
// pixels a thread has in flight: 4 of x, 2 of x and dy (8 and 4 time the same; 512 threads
// beat 256 by 7 % and 1024 by 3 % over forward and backward of 16 x 256^2 x 64 fp32)
constexpr int GN_U = 4, GN_UB = 2;
constexpr int GN_FG = 256;       // groups a block folds itself at most
constexpr int GN_FOLD = 1 << 14;  // partials of a sample that a block folds itself at most

struct GnGeom {
    int64_t P, ppc;  // pixels of a sample, pixels per chunk
    int C, G, cpg;
    int cb, rows, ncol, nchunk;
    int fold;  // the second pass merges the partials itself (no merge launch)
};
struct GnPos {
    int b, chunk, c, row;  // c: first channel of the thread's vector
    bool on;
    int64_t p0, p1;
};
template <int V> __device__ __forceinline__ GnPos gn_pos(const GnGeom& g, unsigned id) {
    GnPos r;
    const int col = id % g.ncol;
    const unsigned rest = id / g.ncol;
    r.chunk = rest % g.nchunk;
    r.b = rest / g.nchunk;
    r.row = threadIdx.x / g.cb;
    r.c = (col * g.cb + threadIdx.x % g.cb) * V;
    r.on = r.row < g.rows && r.c < g.C;
    r.p0 = (int64_t)r.chunk * g.ppc;
    r.p1 = r.p0 + g.ppc < g.P ? r.p0 + g.ppc : g.P;
    return r;
}
__device__ __forceinline__ double gn_count(const GnGeom& g, int chunk) {
    const int64_t left = g.P - (int64_t)chunk * g.ppc;
    return (double)(left < g.ppc ? left : g.ppc);
}

// per-channel (mean, M2) of a chunk -> part[b][chunk][2][C]
template <typename T, int V>
__global__ void __launch_bounds__(GN_NT) gn_stats_kernel(const T* x, GnGeom g, float* part) {
    constexpr int U = GN_U;
    __shared__ float s_mean[GN_NT * V], s_m2[GN_NT * V], s_n[GN_NT];
    const GnPos q = gn_pos<V>(g, blockIdx.x);
    float n = 0.f, mean[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
    if (q.on) {
        const T* xb = x + ((size_t)q.b * g.P) * g.C + q.c;
        int64_t p = q.p0 + q.row;
        const int64_t step = g.rows;
        for (; p + (U - 1) * step < q.p1; p += U * step) {
            Pack<T, V> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u].load(xb + (size_t)(p + u * step) * g.C);
            const float rn = 1.f / (n + U);
            const float wb = U * rn, wq = n * U * rn;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float s = 0.f, d2 = 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u) s += v[u].get(e);
                const float mb = s * (1.f / U);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float d = v[u].get(e) - mb;
                    d2 = fmaf(d, d, d2);
                }
                const float dm = mb - mean[e];
                mean[e] = fmaf(dm, wb, mean[e]);
                m2[e] += fmaf(dm * dm, wq, d2);
            }
            n += U;
        }
        for (; p < q.p1; p += step) {
            Pack<T, V> v;
            v.load(xb + (size_t)p * g.C);
            n += 1.f;
            const float rn = 1.f / n;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = v.get(e) - mean[e];
                mean[e] = fmaf(d, rn, mean[e]);
                m2[e] = fmaf(d, v.get(e) - mean[e], m2[e]);
            }
        }
    }
    const int t = threadIdx.x;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        s_mean[e * GN_NT + t] = mean[e];
        s_m2[e * GN_NT + t] = m2[e];
    }
    s_n[t] = n;
    int top = 1;
    while (top < g.rows) top <<= 1;
    for (int s = top >> 1; s > 0; s >>= 1) {
        __syncthreads();
        if (q.on && q.row < s && q.row + s < g.rows) {
            const int o = t + s * g.cb;
            const float nb = s_n[o];
            if (nb > 0.f) {
                const float rn = 1.f / (n + nb);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float dm = s_mean[e * GN_NT + o] - mean[e];
                    mean[e] = fmaf(dm, nb * rn, mean[e]);
                    m2[e] += fmaf(dm * dm, n * nb * rn, s_m2[e * GN_NT + o]);
                    s_mean[e * GN_NT + t] = mean[e];
                    s_m2[e * GN_NT + t] = m2[e];
                }
                n += nb;
                s_n[t] = n;
            }
        }
    }
    if (q.on && q.row == 0) {
        float* o = part + ((size_t)(q.b * (int64_t)g.nchunk + q.chunk) * 2) * g.C + q.c;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            o[e] = mean[e];
            o[g.C + e] = m2[e];
        }
    }
}

// block per (sample, group): the chunks' partials -> mean, rstd (4 x 37 x 41 x 1000 fp32 in 8
// groups, 127 chunks of 125 channels: the whole forward 28 us, with a wave per group 59)
__global__ void __launch_bounds__(256) gn_merge_kernel(const float* part, GnGeom g, float eps, float* mean,
                                                       float* rstd) {
    __shared__ double red[2][4];
    const int b = blockIdx.x / g.G, gr = blockIdx.x % g.G, t = threadIdx.x;
    const float* pb = part + (size_t)b * g.nchunk * 2 * g.C + gr * g.cpg;
    const int ct = g.cpg < 256 ? g.cpg : 256, parts = 256 / ct, cl = t % ct, pi = t / ct;
    const double cnt = (double)g.P * g.cpg;
    // about the first partial's mean: the squares cancel nothing
    const double ref = pb[0];
    double s = 0, q = 0;
    if (pi < parts)
        for (int c = cl; c < g.cpg; c += ct) {
#pragma unroll 4
            for (int ch = pi; ch < g.nchunk; ch += parts) {
                const double np = gn_count(g, ch), d = (double)pb[(size_t)ch * 2 * g.C + c] - ref;
                s += np * d;
                q += (double)pb[((size_t)ch * 2 + 1) * g.C + c] + np * d * d;
            }
        }
    s = wave_sum_d(s);
    q = wave_sum_d(q);
    if ((t & 63) == 0) {
        red[0][t / 64] = s;
        red[1][t / 64] = q;
    }
    __syncthreads();
    if (t == 0) {
        s = (red[0][0] + red[0][1] + red[0][2] + red[0][3]) / cnt;
        q = (red[1][0] + red[1][1] + red[1][2] + red[1][3]) / cnt - s * s;
        mean[blockIdx.x] = (float)(ref + s);
        rstd[blockIdx.x] = (float)(1.0 / sqrt((q > 0 ? q : q != q ? q : 0.0) + (double)eps));
    }
}

// Group sums of two per-channel quantities: `each(c, first, step)` gives the caller's share of
// channel c over the partials first, first + step, ... (a few dozen at most, summed in fp32); L lanes a
// group add the shares in fp64, in a fixed order.  Every thread of the block calls it; the
// sums are in f->gs.  (Sums of a share in fp64 cost every block of the second pass 10 us where
// 1024 blocks merge 64 chunks of 128 channels.)
struct GnFold {
    double red[2][GN_NT];
    double gs[2][GN_FG];
};
template <typename F>
__device__ __forceinline__ void gn_fold(const GnGeom& g, GnFold* f, F each) {
    const int t = threadIdx.x;
    const int ct = g.C < GN_NT ? g.C : GN_NT, parts = GN_NT / ct;
    for (int k = t; k < g.G; k += GN_NT) f->gs[0][k] = f->gs[1][k] = 0;
    for (int c0 = 0; c0 < g.C; c0 += ct) {
        const int cl = t % ct, pi = t / ct, c = c0 + cl;
        double a = 0, b = 0;
        if (pi < parts && pi < g.nchunk && c < g.C) each(c, pi, parts, a, b);
        f->red[0][t] = a;
        f->red[1][t] = b;
        __syncthreads();
        const int c1 = c0 + ct < g.C ? c0 + ct : g.C;
        const int k0 = c0 / g.cpg, k1 = (c1 - 1) / g.cpg;
        int L = 64;
        while (L > 1 && (k1 - k0 + 1) * L > GN_NT) L >>= 1;
        const int l = t & (L - 1);
        for (int kb = k0; kb <= k1; kb += GN_NT / L) {
            const int k = kb + t / L;
            double x = 0, y = 0;
            if (k <= k1) {
                const int lo = (k * g.cpg > c0 ? k * g.cpg : c0) - c0;
                const int wd = ((k + 1) * g.cpg < c1 ? (k + 1) * g.cpg : c1) - c0 - lo;
                for (int j = l; j < wd * parts; j += L) {
                    const int at = j / wd * ct + lo + j % wd;
                    x += f->red[0][at];
                    y += f->red[1][at];
                }
            }
            for (int o = L >> 1; o > 0; o >>= 1) {
                x += __shfl_xor(x, o, 64);
                y += __shfl_xor(y, o, 64);
            }
            // (a group that spans tiles: one tile after the other, a barrier between)
            if (l == 0 && k <= k1) {
                f->gs[0][k] += x;
                f->gs[1][k] += y;
            }
        }
        __syncthreads();
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(GN_NT) gn_apply_kernel(const T* x, GnGeom g, const float* part,
                                                         float eps, float* mean, float* rstd,
                                                         const float* gamma, const float* beta,
                                                         int act, T* y) {
    constexpr int U = GN_U;
    __shared__ GnFold fold;
    GnFold* const f = &fold;
    // the last block of the first pass first: its values are the likeliest still cached
    const GnPos q = gn_pos<V>(g, gridDim.x - 1 - blockIdx.x);
    const size_t base = ((size_t)q.b * g.P) * g.C + q.c;
    const int64_t step = g.rows;
    int64_t p = q.p0 + q.row;
    Pack<T, V> v[U];
    bool full = q.on && p + (U - 1) * step < q.p1;
    if (full) {  // on their way while the statistics are merged
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].load(x + base + (size_t)(p + u * step) * g.C);
    }
    if (g.fold) {
        const float* pb = part + (size_t)q.b * g.nchunk * 2 * g.C;
        gn_fold(g, f, [&](int c, int first, int step, double& s, double& v) {
            // a share about its own first mean, then about the group's: a chunk far from the
            // others must not cost the others their digits
            const float own = pb[(size_t)first * 2 * g.C + c];
            const int64_t rest = g.P - (int64_t)(g.nchunk - 1) * g.ppc;
            const float whole = (float)g.ppc, last = (float)rest;
            float fs = 0.f, fv = 0.f;
#pragma unroll 8
            for (int ch = first; ch < g.nchunk; ch += step) {
                const float np = ch == g.nchunk - 1 ? last : whole;
                const float d = pb[(size_t)ch * 2 * g.C + c] - own;
                fs = fmaf(np, d, fs);
                fv += fmaf(np * d, d, pb[((size_t)ch * 2 + 1) * g.C + c]);
            }
            const int m = (g.nchunk - 1 - first) / step;  // chunks before the share's last
            const double n = (double)m * g.ppc + (first + m * step == g.nchunk - 1 ? rest : g.ppc);
            const double e = (double)own - pb[c / g.cpg * g.cpg];
            s = fs + n * e;
            v = fv + e * (2.0 * fs + n * e);
        });
        const double cnt = (double)g.P * g.cpg;
        for (int k = threadIdx.x; k < g.G; k += GN_NT) {
            const double s = f->gs[0][k] / cnt, v = f->gs[1][k] / cnt - s * s;
            const double m = (double)pb[k * g.cpg] + s;
            const double r = 1.0 / sqrt((v > 0 ? v : v != v ? v : 0.0) + (double)eps);
            f->gs[0][k] = m;
            f->gs[1][k] = r;
            if (q.chunk == 0) {
                mean[(size_t)q.b * g.G + k] = (float)m;
                rstd[(size_t)q.b * g.G + k] = (float)r;
            }
        }
        __syncthreads();
    }
    if (!q.on) return;
    float mu[V], a[V], h[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int k = (q.c + e) / g.cpg;
        mu[e] = g.fold ? (float)f->gs[0][k] : mean[(size_t)q.b * g.G + k];
        a[e] = (g.fold ? (float)f->gs[1][k] : rstd[(size_t)q.b * g.G + k]) * (gamma ? gamma[q.c + e] : 1.f);
        h[e] = beta ? beta[q.c + e] : 0.f;
    }
    auto one = [&](const Pack<T, V>& in, int64_t at) {
        Pack<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.set(e, gn_act(fmaf(in.get(e) - mu[e], a[e], h[e]), act));
        o.store(y + base + (size_t)at * g.C);
    };
    while (full) {
        Pack<T, V> w[U];
        const int64_t pn = p + U * step;
        const bool next = pn + (U - 1) * step < q.p1;
        if (next) {
#pragma unroll
            for (int u = 0; u < U; ++u) w[u].load(x + base + (size_t)(pn + u * step) * g.C);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) one(v[u], p + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = w[u];
        p = pn;
        full = next;
    }
    for (; p < q.p1; p += step) {
        v[0].load(x + base + (size_t)p * g.C);
        one(v[0], p);
    }
}

// per-channel (sum dp, sum dp*xh[, sum xh]) of a chunk -> part[b][chunk][2 or 3][C]
template <typename T, typename TD, int V, bool X>
__global__ void __launch_bounds__(GN_NT) gn_bwd_reduce_kernel(const TD* dy, const T* x, GnGeom g,
                                                              const float* mean, const float* rstd,
                                                              const float* gamma, const float* beta,
                                                              int act, float* part) {
    constexpr int U = GN_UB, K = X ? 3 : 2;
    __shared__ float sh[GN_NT * V];
    const GnPos q = gn_pos<V>(g, blockIdx.x);
    float sum[K][V], mu[V], rs[V], w[V], h[V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[k][e] = 0.f;
    if (q.on) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int gi = q.b * g.G + (q.c + e) / g.cpg;
            mu[e] = mean[gi];
            rs[e] = rstd[gi];
            w[e] = gamma ? gamma[q.c + e] : 1.f;
            h[e] = beta ? beta[q.c + e] : 0.f;
        }
        const size_t base = ((size_t)q.b * g.P) * g.C + q.c;
        const int64_t step = g.rows;
        int64_t p = q.p0 + q.row;
        auto add = [&](const Pack<T, V>& v, const Pack<TD, V>& d) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (v.get(e) - mu[e]) * rs[e];
                const float dp = gn_act_bwd(d.get(e), fmaf(xh, w[e], h[e]), act);
                sum[0][e] += dp;
                sum[1][e] = fmaf(dp, xh, sum[1][e]);
                if constexpr (X) sum[2][e] += xh;
            }
        };
        for (; p + (U - 1) * step < q.p1; p += U * step) {
            Pack<T, V> v[U];
            Pack<TD, V> d[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                v[u].load(x + base + (size_t)(p + u * step) * g.C);
                d[u].load(dy + base + (size_t)(p + u * step) * g.C);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) add(v[u], d[u]);
        }
        for (; p < q.p1; p += step) {
            Pack<T, V> v;
            Pack<TD, V> d;
            v.load(x + base + (size_t)p * g.C);
            d.load(dy + base + (size_t)p * g.C);
            add(v, d);
        }
    }
    const int t = threadIdx.x;
    int top = 1;
    while (top < g.rows) top <<= 1;
    float* o = part + ((size_t)(q.b * (int64_t)g.nchunk + q.chunk) * K) * g.C + q.c;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) sh[e * GN_NT + t] = sum[k][e];
        for (int s = top >> 1; s > 0; s >>= 1) {
            __syncthreads();
            if (q.on && q.row < s && q.row + s < g.rows) {
#pragma unroll
                for (int e = 0; e < V; ++e) sh[e * GN_NT + t] += sh[e * GN_NT + t + s * g.cb];
            }
        }
        if (q.on && q.row == 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) o[k * g.C + e] = sh[e * GN_NT + t];
        }
    }
}

// block per (sample, group): the chunks' sums per channel (part with K = 3) -> tot[b][3][C],
// and the group's s1, s2 -> sums[b][G][2]
__global__ void __launch_bounds__(256) gn_bwd_merge_kernel(const float* part, GnGeom g,
                                                           const float* gamma, float* tot,
                                                           float* sums) {
    __shared__ double sh[3][256];
    const int b = blockIdx.x / g.G, gr = blockIdx.x % g.G, t = threadIdx.x;
    const int ct = g.cpg < 256 ? g.cpg : 256, parts = 256 / ct;
    const int cl = t % ct, pi = t / ct;
    const double cnt = (double)g.P * g.cpg;
    double s1 = 0, s2 = 0;
    for (int c0 = 0; c0 < g.cpg; c0 += ct) {
        const int c = gr * g.cpg + c0 + cl;
        const bool on = pi < parts && c0 + cl < g.cpg;
        double a = 0, bb = 0, xx = 0;
        if (on) {
#pragma unroll 4
            for (int ch = pi; ch < g.nchunk; ch += parts) {
                const float* pb = part + ((size_t)(b * (int64_t)g.nchunk + ch) * 3) * g.C + c;
                a += pb[0];
                bb += pb[g.C];
                xx += pb[2 * g.C];
            }
        }
        sh[0][t] = a;
        sh[1][t] = bb;
        sh[2][t] = xx;
        __syncthreads();
        if (on && pi == 0) {
            for (int k = 1; k < parts; ++k) {
                a += sh[0][k * ct + cl];
                bb += sh[1][k * ct + cl];
                xx += sh[2][k * ct + cl];
            }
            float* o = tot + (size_t)b * 3 * g.C + c;
            o[0] = (float)a;
            o[g.C] = (float)bb;
            o[2 * g.C] = (float)xx;
            const double w = gamma ? (double)gamma[c] : 1.0;
            s1 += w * a;
            s2 += w * bb;
        }
        __syncthreads();
    }
    sh[0][t] = s1;
    sh[1][t] = s2;
    __syncthreads();
    for (int s = 128; s > 0; s >>= 1) {
        if (t < s) {
            sh[0][t] += sh[0][t + s];
            sh[1][t] += sh[1][t + s];
        }
        __syncthreads();
    }
    if (t == 0) {
        sums[2 * blockIdx.x] = (float)(sh[0][0] / cnt);
        sums[2 * blockIdx.x + 1] = (float)(sh[1][0] / cnt);
    }
}

// dgamma, dbeta and the sum of dx per channel (the gradient of a bias added to x), from the
// samples' totals: sum_p dx = rstd * (gamma*A - P*s1 - s2*X) per sample, A = sum dp, X = sum xh
__device__ __forceinline__ void gn_param_grads(int c, int B, int64_t P, int C, int G, int cpg,
                                               const float* tot, const float* sums,
                                               const float* rstd, const float* gamma,
                                               float* dgamma, float* dbeta, float* dxsum) {
    double a = 0, bb = 0, d = 0;
    const int gr = c / cpg;
    const double w = gamma ? (double)gamma[c] : 1.0;
    for (int b = 0; b < B; ++b) {
        const float* o = tot + (size_t)b * 3 * C + c;
        a += o[0];
        bb += o[C];
        const float* s = sums + 2 * ((size_t)b * G + gr);
        d += (double)rstd[(size_t)b * G + gr] *
             (w * o[0] - (double)P * s[0] - (double)s[1] * o[2 * C]);
    }
    if (dbeta) dbeta[c] = (float)a;
    if (dgamma) dgamma[c] = (float)bb;
    if (dxsum) dxsum[c] = (float)d;
}

// the parameters' gradients of 64 channels a block: over all the chunks' partials (fold), or
// over the samples' totals
__device__ __forceinline__ void gn_params(const GnGeom& g, int B, unsigned id, const float* part,
                                          const float* tot, const float* sums, const float* rstd,
                                          const float* gamma, float* dgamma, float* dbeta, float* dxsum) {
    const int c = id * 64 + (threadIdx.x & 63), pi = threadIdx.x / 64;
    if (!g.fold) {
        if (c < g.C && pi == 0)
            gn_param_grads(c, B, g.P, g.C, g.G, g.cpg, tot, sums, rstd, gamma, dgamma, dbeta, dxsum);
        return;
    }
    __shared__ double red[2][GN_NT];
    double a = 0, b = 0;
    if (c < g.C) {
#pragma unroll 8
        for (int64_t k = pi; k < (int64_t)B * g.nchunk; k += GN_NT / 64) {
            a += part[(size_t)k * 2 * g.C + c];
            b += part[((size_t)k * 2 + 1) * g.C + c];
        }
    }
    red[0][threadIdx.x] = a;
    red[1][threadIdx.x] = b;
    __syncthreads();
    if (c < g.C && pi == 0) {
        for (int k = 1; k < GN_NT / 64; ++k) {
            a += red[0][threadIdx.x + 64 * k];
            b += red[1][threadIdx.x + 64 * k];
        }
        if (dbeta) dbeta[c] = (float)a;
        if (dgamma) dgamma[c] = (float)b;
    }
}

// dx; the first `nparam` blocks sum the parameters' gradients, 64 channels each
template <typename T, typename TD, typename TO, int V>
__global__ void __launch_bounds__(GN_NT) gn_bwd_apply_kernel(
    const TD* dy, const T* x, GnGeom g, int B, unsigned nparam, const float* mean, const float* rstd,
    const float* gamma, const float* beta, int act, const float* part, const float* tot,
    const float* sums, TO* dx, float* dgamma, float* dbeta, float* dxsum) {
    constexpr int U = GN_UB;
    __shared__ GnFold fold;
    GnFold* const f = &fold;
    if (blockIdx.x < nparam) {
        gn_params(g, B, blockIdx.x, part, tot, sums, rstd, gamma, dgamma, dbeta, dxsum);
        return;
    }
    const GnPos q = gn_pos<V>(g, gridDim.x - 1 - blockIdx.x);
    const size_t base = ((size_t)q.b * g.P) * g.C + q.c;
    const int64_t step = g.rows;
    int64_t p = q.p0 + q.row;
    Pack<T, V> v[U];
    Pack<TD, V> d[U];
    bool full = q.on && p + (U - 1) * step < q.p1;
    if (full) {  // on their way while the sums are merged
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u].load(x + base + (size_t)(p + u * step) * g.C);
            d[u].load(dy + base + (size_t)(p + u * step) * g.C);
        }
    }
    if (g.fold) {
        const float* pb = part + (size_t)q.b * g.nchunk * 2 * g.C;
        gn_fold(g, f, [&](int c, int first, int step, double& s, double& t) {
            float a = 0.f, b = 0.f;
#pragma unroll 8
            for (int ch = first; ch < g.nchunk; ch += step) {
                a += pb[(size_t)ch * 2 * g.C + c];
                b += pb[((size_t)ch * 2 + 1) * g.C + c];
            }
            const double w = gamma ? gamma[c] : 1.f;
            s = w * a;
            t = w * b;
        });
    }
    if (!q.on) return;
    const double rcnt = 1.0 / ((double)g.P * g.cpg);
    float mu[V], rs[V], w[V], h[V], s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int k = (q.c + e) / g.cpg, gi = q.b * g.G + k;
        mu[e] = mean[gi];
        rs[e] = rstd[gi];
        w[e] = gamma ? gamma[q.c + e] : 1.f;
        h[e] = beta ? beta[q.c + e] : 0.f;
        s1[e] = g.fold ? (float)(f->gs[0][k] * rcnt) : sums[2 * gi];
        s2[e] = g.fold ? (float)(f->gs[1][k] * rcnt) : sums[2 * gi + 1];
    }
    auto one = [&](const Pack<T, V>& v, const Pack<TD, V>& d, int64_t at) {
        Pack<TO, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float xh = (v.get(e) - mu[e]) * rs[e];
            const float dp = gn_act_bwd(d.get(e), fmaf(xh, w[e], h[e]), act);
            o.set(e, rs[e] * fmaf(-xh, s2[e], fmaf(w[e], dp, -s1[e])));
        }
        o.store(dx + base + (size_t)at * g.C);
    };
    while (full) {
        Pack<T, V> vn[U];
        Pack<TD, V> dn[U];
        const int64_t pn = p + U * step;
        const bool next = pn + (U - 1) * step < q.p1;
        if (next) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                vn[u].load(x + base + (size_t)(pn + u * step) * g.C);
                dn[u].load(dy + base + (size_t)(pn + u * step) * g.C);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) one(v[u], d[u], p + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = vn[u];
            d[u] = dn[u];
        }
        p = pn;
        full = next;
    }
    for (; p < q.p1; p += step) {
        v[0].load(x + base + (size_t)p * g.C);
        d[0].load(dy + base + (size_t)p * g.C);
        one(v[0], d[0], p);
    }
}

// ---------------------------------------------------------------- one pass
// Block = (sample, slab of gb whole groups): thread (row, col) holds the V channels `col` of
// the pixels row, row + rows, ...  (NV of them at most) in registers as loaded.  V divides a
// group, so a thread's vector lies in one group.
struct GnSlab {
    int64_t P;
    int C, G, cpg, gb, nslab, scv, rows;
};
struct GnSlabPos {
    int b, g0, ng, col, row, c, gl;
    bool on;
};
template <int V> __device__ __forceinline__ GnSlabPos gn_slab_pos(const GnSlab& g) {
    GnSlabPos r;
    r.b = blockIdx.x / g.nslab;
    r.g0 = (blockIdx.x % g.nslab) * g.gb;
    r.ng = g.G - r.g0 < g.gb ? g.G - r.g0 : g.gb;
    r.col = threadIdx.x % g.scv;
    r.row = threadIdx.x / g.scv;
    r.gl = r.col * V / g.cpg;
    r.c = r.g0 * g.cpg + r.col * V;
    r.on = r.row < g.rows && r.gl < r.ng;
    return r;
}

// sum of v over the block's threads of the caller's group (one wave per group, fixed order)
template <int V>
__device__ __forceinline__ float gn_group_sum(float v, const GnSlab& g, const GnSlabPos& q,
                                              float* red, float* out) {
    __syncthreads();
    red[threadIdx.x] = q.on ? v : 0.f;
    __syncthreads();
    const int nw = blockDim.x / 64, w = threadIdx.x / 64, lane = threadIdx.x & 63;
    const int vpg = g.cpg / V, n = vpg * g.rows;
    for (int k = w; k < q.ng; k += nw) {
        float s = 0.f;
        for (int j = lane; j < n; j += 64) s += red[j / vpg * g.scv + k * vpg + j % vpg];
        s = wave_sum(s);
        if (lane == 0) out[k] = s;
    }
    __syncthreads();
    return q.on ? out[q.gl] : 0.f;
}

constexpr int GN_GB = 64;  // groups of a slab at most

template <typename T, int V, int NV>
__global__ void __launch_bounds__(1024) gn_fwd_res_kernel(const T* x, GnSlab g, const float* gamma,
                                                          const float* beta, float eps, int act,
                                                          T* y, float* mean, float* rstd) {
    __shared__ float red[1024], out[GN_GB];
    const GnSlabPos q = gn_slab_pos<V>(g);
    const size_t base = ((size_t)q.b * g.P) * g.C + q.c;
    Pack<T, V> v[NV];
    float w[V], h[V];
    if (q.on) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t p = q.row + (int64_t)i * g.rows;
            if (p < g.P) v[i].load(x + base + (size_t)p * g.C);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[e] = gamma ? gamma[q.c + e] : 1.f;
            h[e] = beta ? beta[q.c + e] : 0.f;
        }
    }
    float s = 0.f;
    if (q.on) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (q.row + (int64_t)i * g.rows < g.P) {
#pragma unroll
                for (int e = 0; e < V; ++e) s += v[i].get(e);
            }
    }
    const float rn = 1.f / ((float)g.P * (float)g.cpg);
    const float mu = gn_group_sum<V>(s, g, q, red, out) * rn;
    s = 0.f;
    if (q.on) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (q.row + (int64_t)i * g.rows < g.P) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float d = v[i].get(e) - mu;
                    s = fmaf(d, d, s);
                }
            }
    }
    const float var = gn_group_sum<V>(s, g, q, red, out) * rn;
    const float rs = 1.f / sqrtf(var + eps);
    if (!q.on) return;
    if (q.row == 0 && q.col * V % g.cpg == 0) {
        mean[(size_t)q.b * g.G + q.g0 + q.gl] = mu;
        rstd[(size_t)q.b * g.G + q.g0 + q.gl] = rs;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] *= rs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t p = q.row + (int64_t)i * g.rows;
        if (p < g.P) {
            Pack<T, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e)
                o.set(e, gn_act(fmaf(v[i].get(e) - mu, w[e], h[e]), act));
            o.store(y + base + (size_t)p * g.C);
        }
    }
}

// per-channel sums over the block's rows: each thread's v[V] -> tot[scv * V]
template <int V>
__device__ __forceinline__ void gn_channel_sums(const float (&v)[V], const GnSlab& g, bool on,
                                                float* red, float* tot) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) red[e * 1024 + threadIdx.x] = on ? v[e] : 0.f;
    __syncthreads();
    const int nw = blockDim.x / 64, w = threadIdx.x / 64, lane = threadIdx.x & 63;
    for (int k = w; k < g.scv * V; k += nw) {
        const float* r = red + (k % V) * 1024 + k / V;
        float s = 0.f;
        for (int j = lane; j < g.rows; j += 64) s += r[j * g.scv];
        s = wave_sum(s);
        if (lane == 0) tot[k] = s;
    }
}

// Eight vectors of 8 bf16 values need more than the 128 registers of 1024 threads: with a float32 dy
// 186 of them spill (16 x 64^2 x 256 in 32 groups: 143 us where the floor is 28 and float32
// vectors of 4 take 61; 1 x 64^2 x 256: 103 and 19), with a bf16 dy 24.
template <typename T, typename TD, typename TO, int V, int NV>
__global__ void __launch_bounds__(1024) gn_bwd_res_kernel(
    const TD* dy, const T* x, GnSlab g, const float* mean, const float* rstd, const float* gamma,
    const float* beta, int act, TO* dx, float* tot, float* sums) {
    __shared__ float red[1024 * V], ta[1024], tb[1024], tx[1024], s12[2 * GN_GB];
    const GnSlabPos q = gn_slab_pos<V>(g);
    const size_t base = ((size_t)q.b * g.P) * g.C + q.c;
    Pack<T, V> v[NV];
    Pack<TD, V> d[NV];
    float w[V], h[V], sa[V], sb[V], sx[V], mu = 0.f, rs = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) sa[e] = sb[e] = sx[e] = w[e] = h[e] = 0.f;
    if (q.on) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t p = q.row + (int64_t)i * g.rows;
            if (p < g.P) {
                v[i].load(x + base + (size_t)p * g.C);
                d[i].load(dy + base + (size_t)p * g.C);
            }
        }
        mu = mean[(size_t)q.b * g.G + q.g0 + q.gl];
        rs = rstd[(size_t)q.b * g.G + q.g0 + q.gl];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[e] = gamma ? gamma[q.c + e] : 1.f;
            h[e] = beta ? beta[q.c + e] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (q.row + (int64_t)i * g.rows < g.P) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = (v[i].get(e) - mu) * rs;
                    const float dp = gn_act_bwd(d[i].get(e), fmaf(xh, w[e], h[e]), act);
                    sa[e] += dp;
                    sb[e] = fmaf(dp, xh, sb[e]);
                    sx[e] += xh;
                }
            }
    }
    gn_channel_sums<V>(sa, g, q.on, red, ta);
    gn_channel_sums<V>(sb, g, q.on, red, tb);
    gn_channel_sums<V>(sx, g, q.on, red, tx);
    __syncthreads();
    const int nw = blockDim.x / 64, wv = threadIdx.x / 64, lane = threadIdx.x & 63;
    const float rn = 1.f / ((float)g.P * (float)g.cpg);
    for (int k = wv; k < q.ng; k += nw) {
        float s1 = 0.f, s2 = 0.f;
        for (int j = lane; j < g.cpg; j += 64) {
            const int c = k * g.cpg + j;
            const float gm = gamma ? gamma[q.g0 * g.cpg + c] : 1.f;
            s1 = fmaf(gm, ta[c], s1);
            s2 = fmaf(gm, tb[c], s2);
        }
        s1 = wave_sum(s1) * rn;
        s2 = wave_sum(s2) * rn;
        if (lane == 0) {
            s12[2 * k] = s1;
            s12[2 * k + 1] = s2;
            float* o = sums + 2 * ((size_t)q.b * g.G + q.g0 + k);
            o[0] = s1;
            o[1] = s2;
        }
    }
    for (int k = threadIdx.x; k < q.ng * g.cpg; k += blockDim.x) {
        float* o = tot + (size_t)q.b * 3 * g.C + q.g0 * g.cpg + k;
        o[0] = ta[k];
        o[g.C] = tb[k];
        o[2 * g.C] = tx[k];
    }
    __syncthreads();
    if (!q.on) return;
    const float s1 = s12[2 * q.gl], s2 = s12[2 * q.gl + 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t p = q.row + (int64_t)i * g.rows;
        if (p < g.P) {
            Pack<TO, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (v[i].get(e) - mu) * rs;
                const float dp = gn_act_bwd(d[i].get(e), fmaf(xh, w[e], h[e]), act);
                o.set(e, rs * fmaf(-xh, s2, fmaf(w[e], dp, -s1)));
            }
            o.store(dx + base + (size_t)p * g.C);
        }
    }
}

__global__ void __launch_bounds__(256) gn_params_kernel(int B, int64_t P, int C, int G,
                                                        const float* tot, const float* sums,
                                                        const float* rstd, const float* gamma,
                                                        float* dgamma, float* dbeta, float* dxsum) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < C) gn_param_grads(c, B, P, C, G, C / G, tot, sums, rstd, gamma, dgamma, dbeta, dxsum);
}

// ---------------------------------------------------------------- host side
// The one-pass form, where a slab of whole groups fits the registers of a block: at most
// `nvmax` vectors a thread, 1024 threads.  A pixel's slab is 128 bytes (whole lines) where
// that leaves 256 blocks, else 64; never less unless the pixel is.  Returns the vectors a
// thread holds (0: does not fit) and the block size.
static int gn_slab(int B, int64_t P, int C, int G, int V, int es, int nvmax, GnSlab* o, int* nt) {
    const int cpg = C / G;
    if (cpg % V) return 0;
    for (int target = 128; target >= 64; target -= 64) {
        int gb = (int)cdiv(target, (int64_t)cpg * es);
        if (gb > G) gb = G;
        if (gb > GN_GB) gb = GN_GB;
        const int64_t scv = (int64_t)gb * cpg / V;
        if ((int64_t)gb * cpg > 1024) continue;  // (the block's per-channel sums)
        const int nslab = (int)cdiv(G, gb);
        if (target == 128 && (int64_t)B * nslab < 256 && cpg * es < 128) continue;
        for (int n = 256; n <= 1024; n *= 2) {
            const int rows = n / (int)scv;
            if (rows == 0) continue;
            const int64_t nv = cdiv(P, rows);
            if (nv > (n < 1024 ? 4 : nvmax)) continue;
            *o = GnSlab{P, C, G, cpg, gb, nslab, (int)scv, rows};
            *nt = n;
            return (int)nv;
        }
    }
    return 0;
}

// widest vector (values) that divides C and that every tensor's address allows
static int gn_vec(int C, int es_max, const void* a, int ea, const void* b, int eb, const void* c,
                  int ec) {
    for (int v = es_max; v > 1; v >>= 1) {
        if (C % v) continue;
        auto ok = [v](const void* p, int es) {
            const int n = v * es < 16 ? v * es : 16;
            return ((uintptr_t)p % n) == 0;
        };
        if (ok(a, ea) && ok(b, eb) && ok(c, ec)) return v;
    }
    return 1;
}

// The vector width of a call: the widest at which the one-pass form fits (its vectors lie in
// one group), else the widest that C and the addresses allow.
static int gn_pick(int B, int64_t P, int C, int G, int vmax, int es, int nvmax) {
    GnSlab o;
    int nt;
    for (int v = vmax; v >= 1; v >>= 1)
        if (gn_slab(B, P, C, G, v, es, nvmax, &o, &nt)) return v;
    return vmax;
}

static GnGeom gn_geom(int B, int64_t P, int C, int G, int V) {
    GnGeom g;
    g.P = P;
    g.C = C;
    g.G = G;
    g.cpg = C / G;
    const int cv = C / V;
    g.ncol = (int)cdiv(cv, GN_NT);
    g.cb = (int)cdiv(cv, g.ncol);
    g.rows = GN_NT / g.cb;
    // about 1024 blocks (4 per CU), no chunk below 4 pixels a thread, at most 1024 chunks
    int64_t want = cdiv(1024, (int64_t)B * g.ncol);
    const int64_t most = cdiv(P, (int64_t)g.rows * 4);
    if (want > most) want = most;
    if (want > 1024) want = 1024;
    if (want < 1) want = 1;
    // every block of the second pass merges a sample's partials again: at most 4096 of them,
    // or down to 512 blocks (16 x 128^2 x 128 bf16 forward: 44 us at 32 chunks, 52 at 64;
    // 16 x 256^2 x 64 fp32 forward and backward: 398 us at 1024 blocks, 426 at 512)
    const int64_t light = 4096 / C > 1 ? 4096 / C : 1;
    const int64_t fill = cdiv(512, (int64_t)B * g.ncol);
    if (want > light) want = light > fill ? light : (want < fill ? want : fill);
    g.ppc = cdiv(P, want);
    g.nchunk = (int)cdiv(P, g.ppc);
    g.fold = g.ncol == 1 && G <= GN_FG && (int64_t)g.nchunk * C <= GN_FOLD;
    return g;
}

static int gn_check(const char* what, const ugpg_group_norm_t* p, bool tensors) {
    if (!p) {
        set_error("%s: no descriptor", what);
        return UGPG_ERR_INVALID;
    }
    if (p->B <= 0 || p->HW <= 0 || p->C <= 0 || p->G <= 0 || p->C % p->G ||
        (p->dtype != UGPG_DT_F32 && p->dtype != UGPG_DT_BF16) || p->act < UGPG_ACT_NONE ||
        p->act > UGPG_ACT_SILU || !(p->eps >= 0.f)) {
        set_error("%s: bad arguments (dtype=%d B=%d HW=%lld C=%d groups=%d eps=%g act=%d)", what,
                  p->dtype, p->B, (long long)p->HW, p->C, p->G, (double)p->eps, p->act);
        return UGPG_ERR_INVALID;
    }
    if (tensors && (!p->x || !p->mean || !p->rstd || (uintptr_t)p->x % (p->dtype == UGPG_DT_F32 ? 4 : 2))) {
        set_error("%s: x, mean and rstd must be given, x aligned to its type", what);
        return UGPG_ERR_INVALID;
    }
    // (grids: B*G blocks of up to 1024 threads, below 2^32 in all; B * column blocks; offsets
    // are 64-bit)
    if (p->C > (1 << 20) || (int64_t)p->B * p->G >= (1 << 22) ||
        (int64_t)p->B * cdiv(p->C, 256) > (1 << 22) || p->HW > ((int64_t)1 << 40) ||
        (double)p->B * (double)p->HW * (double)p->C > 1e15) {
        set_error("%s: B=%d HW=%lld C=%d is too large", what, p->B, (long long)p->HW, p->C);
        return UGPG_ERR_INVALID;
    }
    return UGPG_OK;
}

// chunk count at the narrowest vector bounds it at every vector width (rows only shrinks)
static size_t gn_part_floats(int B, int64_t P, int C, int G, int per) {
    size_t most = 0;
    for (int v = 8; v >= 1; v >>= 1) {
        if (C % v) continue;
        const GnGeom g = gn_geom(B, P, C, G, v);
        const size_t n = (size_t)B * g.nchunk * per * C;
        if (n > most) most = n;
    }
    return most;
}

}  // namespace ugpg

using namespace ugpg;

extern "C" size_t ugpg_group_norm_workspace(const ugpg_group_norm_t* p, int backward) {
    if (gn_check("group_norm_workspace", p, false)) return 0;
    if (!backward) return gn_part_floats(p->B, p->HW, p->C, p->G, 2) * 4;
    return (gn_part_floats(p->B, p->HW, p->C, p->G, 3) + (size_t)p->B * 3 * p->C +
            (size_t)p->B * p->G * 2) * 4;
}

template <typename T, int V>
static int gn_fwd_run(const ugpg_group_norm_t* d, void* y, void* ws, hipStream_t s) {
    const void* x = d->x;
    const int B = d->B, C = d->C, G = d->G, act = d->act;
    const int64_t P = d->HW;
    const float *gamma = d->gamma, *beta = d->beta;
    const float eps = d->eps;
    float *mean = d->mean, *rstd = d->rstd;
    const T* xt = static_cast<const T*>(x);
    GnSlab sl;
    int nt;
    if (const int nv = gn_slab(B, P, C, G, V, sizeof(T), 16, &sl, &nt)) {
        const dim3 grid((unsigned)((int64_t)B * sl.nslab));
#define GN_RES(NV) \
    hipLaunchKernelGGL((gn_fwd_res_kernel<T, V, NV>), grid, dim3(nt), 0, s, xt, sl, gamma, beta, eps, act, \
                       static_cast<T*>(y), mean, rstd)
        if (nv <= 4) GN_RES(4);
        else if (nv <= 8) GN_RES(8);
        else GN_RES(16);
#undef GN_RES
        return check_launch("group_norm_fwd");
    }
    const GnGeom g = gn_geom(B, P, C, G, V);
    const unsigned nb = (unsigned)((int64_t)B * g.nchunk * g.ncol);
    float* part = static_cast<float*>(ws);
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), dim3(nb), dim3(GN_NT), 0, s, xt, g, part);
    if (!g.fold)
        hipLaunchKernelGGL(gn_merge_kernel, dim3((unsigned)((int64_t)B * G)), dim3(256), 0, s, part, g,
                           eps, mean, rstd);
    hipLaunchKernelGGL((gn_apply_kernel<T, V>), dim3(nb), dim3(GN_NT), 0, s, xt, g, part, eps, mean,
                       rstd, gamma, beta, act, static_cast<T*>(y));
    return check_launch("group_norm_fwd");
}

static int gn_ws_check(const char* what, const ugpg_group_norm_t* p, int backward, const void* ws,
                       size_t n) {
    const size_t need = ugpg_group_norm_workspace(p, backward);
    if (!ws || n < need) {
        set_error("%s: workspace %zu < %zu", what, n, need);
        return UGPG_ERR_WORKSPACE;
    }
    return UGPG_OK;
}

extern "C" int ugpg_group_norm_fwd(const ugpg_group_norm_t* p, void* y, void* ws, size_t ws_bytes,
                                   void* stream) {
    if (int rc = gn_check("group_norm_fwd", p, true)) return rc;
    if (!y || (uintptr_t)y % (p->dtype == UGPG_DT_F32 ? 4 : 2)) {
        set_error("group_norm_fwd: no output, or not aligned to its type");
        return UGPG_ERR_INVALID;
    }
    if (int rc = gn_ws_check("group_norm_fwd", p, 0, ws, ws_bytes)) return rc;
    const int es = p->dtype == UGPG_DT_F32 ? 4 : 2;
    const int v = gn_pick(p->B, p->HW, p->C, p->G, gn_vec(p->C, 16 / es, p->x, es, y, es, nullptr, es),
                          es, 16);
    hipStream_t s = as_stream(stream);
#define GN_FWD(T, V) gn_fwd_run<T, V>(p, y, ws, s)
    if (es == 4) return v == 4 ? GN_FWD(float, 4) : v == 2 ? GN_FWD(float, 2) : GN_FWD(float, 1);
    return v == 8 ? GN_FWD(__bf16, 8) : v == 4 ? GN_FWD(__bf16, 4) : v == 2 ? GN_FWD(__bf16, 2)
                                                                         : GN_FWD(__bf16, 1);
#undef GN_FWD
}

template <typename T, typename TD, typename TO, int V>
static int gn_bwd_run(const ugpg_group_norm_t* p, const void* dy, void* dx, float* dgamma,
                      float* dbeta, float* dxsum, void* ws, hipStream_t s) {
    const void* x = p->x;
    const int B = p->B, C = p->C, G = p->G, act = p->act;
    const int64_t P = p->HW;
    const float *gamma = p->gamma, *beta = p->beta, *mean = p->mean, *rstd = p->rstd;
    const T* xt = static_cast<const T*>(x);
    const TD* dt = static_cast<const TD*>(dy);
    float* tot = static_cast<float*>(ws);
    float* sums = tot + (size_t)B * 3 * C;
    float* part = sums + (size_t)B * G * 2;
    const unsigned pblocks = dgamma || dbeta || dxsum ? (unsigned)cdiv(C, 256) : 0;
    GnSlab sl;
    int nt;
    if (const int nv = gn_slab(B, P, C, G, V, sizeof(TD), 8, &sl, &nt)) {
        const dim3 grid((unsigned)((int64_t)B * sl.nslab));
#define GN_RES(NV) \
    hipLaunchKernelGGL((gn_bwd_res_kernel<T, TD, TO, V, NV>), grid, dim3(nt), 0, s, dt, xt, sl, mean, rstd, \
                       gamma, beta, act, static_cast<TO*>(dx), tot, sums)
        if (nv <= 4) GN_RES(4);
        else GN_RES(8);
#undef GN_RES
        if (pblocks)
            hipLaunchKernelGGL(gn_params_kernel, dim3(pblocks), dim3(256), 0, s, B, P, C, G, tot, sums,
                               rstd, gamma, dgamma, dbeta, dxsum);
        return check_launch("group_norm_bwd");
    }
    GnGeom g = gn_geom(B, P, C, G, V);
    g.fold = g.fold && !dxsum;  // (the sum of dx needs the totals)
    const unsigned nb = (unsigned)((int64_t)B * g.nchunk * g.ncol);
    if (g.fold) {
        hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, TD, V, false>), dim3(nb), dim3(GN_NT), 0, s, dt, xt, g,
                           mean, rstd, gamma, beta, act, part);
    } else {
        hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, TD, V, true>), dim3(nb), dim3(GN_NT), 0, s, dt, xt, g,
                           mean, rstd, gamma, beta, act, part);
        hipLaunchKernelGGL(gn_bwd_merge_kernel, dim3((unsigned)((int64_t)B * G)), dim3(256), 0, s, part,
                           g, gamma, tot, sums);
    }
    const unsigned np = dgamma || dbeta || dxsum ? (unsigned)cdiv(C, 64) : 0;
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, TD, TO, V>), dim3(nb + np), dim3(GN_NT), 0, s, dt, xt, g, B,
                       np, mean, rstd, gamma, beta, act, part, tot, sums, static_cast<TO*>(dx), dgamma,
                       dbeta, dxsum);
    return check_launch("group_norm_bwd");
}

extern "C" int ugpg_group_norm_bwd(const ugpg_group_norm_t* p, const void* dy, int dy_dtype, void* dx,
                                   int dx_dtype, float* dgamma, float* dbeta, float* dxsum, void* ws,
                                   size_t ws_bytes, void* stream) {
    if (int rc = gn_check("group_norm_bwd", p, true)) return rc;
    const int F = UGPG_DT_F32, H = UGPG_DT_BF16, dtype = p->dtype;
    const bool fff = dtype == F && dy_dtype == F && dx_dtype == F;
    const bool hhh = dtype == H && dy_dtype == H && dx_dtype == H;
    const bool hfh = dtype == H && dy_dtype == F && dx_dtype == H;
    const bool hff = dtype == H && dy_dtype == F && dx_dtype == F;
    if (!dy || !dx || !(fff || hhh || hfh || hff) || (uintptr_t)dy % (dy_dtype == F ? 4 : 2) ||
        (uintptr_t)dx % (dx_dtype == F ? 4 : 2)) {
        set_error("group_norm_bwd: bad arguments or alignment (x, dy, dx types %d %d %d)", dtype, dy_dtype,
                  dx_dtype);
        return UGPG_ERR_INVALID;
    }
    if (int rc = gn_ws_check("group_norm_bwd", p, 1, ws, ws_bytes)) return rc;
    const int ex = dtype == F ? 4 : 2, ed = dy_dtype == F ? 4 : 2, eo = dx_dtype == F ? 4 : 2;
    const int v = gn_pick(p->B, p->HW, p->C, p->G, gn_vec(p->C, 16 / ex, p->x, ex, dy, ed, dx, eo), ed, 8);
    hipStream_t s = as_stream(stream);
#define GN_BWD(T, TD, TO, V) gn_bwd_run<T, TD, TO, V>(p, dy, dx, dgamma, dbeta, dxsum, ws, s)
#define GN_BWD_H(TD, TO)                              \
    (v == 8 ? GN_BWD(__bf16, TD, TO, 8) : v == 4 ? GN_BWD(__bf16, TD, TO, 4) \
     : v == 2 ? GN_BWD(__bf16, TD, TO, 2) : GN_BWD(__bf16, TD, TO, 1))
    if (fff)
        return v == 4 ? GN_BWD(float, float, float, 4)
               : v == 2 ? GN_BWD(float, float, float, 2) : GN_BWD(float, float, float, 1);
    if (hhh) return GN_BWD_H(__bf16, __bf16);
    if (hfh) return GN_BWD_H(float, __bf16);
    return GN_BWD_H(float, float);
#undef GN_BWD
#undef GN_BWD_H
}

// A teacher's top logits, and the distillation loss that reads them.
//
// Record of a teacher's row t over V classes at temperature T: its k largest logits, sorted
// by value then by the lower index, and `rest` = T * logsumexp(t_v / T over the others): the
// logit of one class that carries all the others' mass.
//
// Loss of a student's row z against a record: both distributions live on k + 1 classes,
//   q = softmax([t_1 .. t_k, rest] / T),   p = softmax(z / T) with the classes beyond the
//   kept ones added up,   KL = sum_j q_j (log q_j - log p_j)
//   loss = scale * T^2 * sum_r w_r KL_r
//   dz_v = scale * T * w_r * (p_v - q_v)                          v kept
//        = scale * T * w_r * (p_rest - q_rest) * r_v              else, r_v = p_v / p_rest
// The kept classes are left out of the rest's sums (by a bitmap), never subtracted from a
// total: both distributions may have almost all their mass in the kept classes.
//
// Bandwidth-bound: a row's logits are read for the sums and again for the gradient, which
// finds them in the caches; sums over a row are fp32 (runs of 4 or 8 per thread, then trees),
// the few terms of the k + 1 classes fp64.  No float atomics; orders are fixed.
#include "common.h"
#include "vecio.h"

namespace ugpg {

constexpr int DK_MAX = 256;              // entries of a record
constexpr float NEG_INF = -__builtin_inff();
constexpr double LOG2E = 1.4426950408889634074;
constexpr double LN2 = 0.69314718055994530942;

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T> struct RowVec { static constexpr int N = 16 / (int)sizeof(T); };

// The elements [lo, hi) of a row in vectors of N: slot 0 is the part before the first
// 16-byte boundary, then whole vectors, then the tail.  f(slot, first index, pack, count);
// a partial pack is filled up with -inf.
template <typename T> struct RowSpan {
    static constexpr int N = RowVec<T>::N;
    const T* z;
    int lo, hi, head, nv;
    __device__ __forceinline__ RowSpan(const T* row, int l, int h) : z(row), lo(l), hi(h) {
        const int mis = (int)(((uintptr_t)(row + l) & 15) / sizeof(T));
        head = mis ? N - mis : 0;
        if (head > hi - lo) head = hi - lo;
        nv = (hi - lo - head) / N;
    }
    __device__ __forceinline__ int bits() const { return (nv + 2) * N; }
    // position of element idx in the bitmap (N bits a slot)
    __device__ __forceinline__ int bit(int idx) const {
        const int o = idx - lo;
        return o < head ? o : o - head + N;
    }
    __device__ __forceinline__ Pack<T, N> partial(int i0, int cnt) const {
        Pack<T, N> v;
#pragma unroll
        for (int e = 0; e < N; ++e) v.set(e, e < cnt ? (float)z[i0 + e] : NEG_INF);
        return v;
    }
    template <int U, typename F> __device__ __forceinline__ void scan(int tid, int nt, F f) const {
        const T* b = z + lo + head;
        int i = tid;
        for (; i + (U - 1) * nt < nv; i += U * nt) {
            Pack<T, N> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u].load(b + (size_t)(i + u * nt) * N);
#pragma unroll
            for (int u = 0; u < U; ++u) f(i + u * nt + 1, lo + head + (i + u * nt) * N, v[u], N);
        }
        for (; i < nv; i += nt) {
            Pack<T, N> v;
            v.load(b + (size_t)i * N);
            f(i + 1, lo + head + i * N, v, N);
        }
        ends(tid, nt, f);
    }
    // the same from the row's end: what an earlier scan read last is the likeliest in the caches
    template <int U, typename F> __device__ __forceinline__ void scan_back(int tid, int nt, F f) const {
        const T* b = z + lo + head;
        int i = (nv - tid - 1) / nt * nt + tid;  // the thread's last vector
        if (tid < nv) {
            for (; i - (U - 1) * nt >= 0; i -= U * nt) {
                Pack<T, N> v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v[u].load(b + (size_t)(i - u * nt) * N);
#pragma unroll
                for (int u = 0; u < U; ++u) f(i - u * nt + 1, lo + head + (i - u * nt) * N, v[u], N);
            }
            for (; i >= 0; i -= nt) {
                Pack<T, N> v;
                v.load(b + (size_t)i * N);
                f(i + 1, lo + head + i * N, v, N);
            }
        }
        ends(tid, nt, f);
    }
    // the parts that are no whole vector
    template <typename F> __device__ __forceinline__ void ends(int tid, int nt, F f) const {
        if (tid == 0 && head > 0) f(0, lo, partial(lo, head), head);
        const int t0 = lo + head + nv * N;
        if (tid == 64 % nt && t0 < hi) f(nv + 1, t0, partial(t0, hi - t0), hi - t0);
    }
};

// (max, sum of exp2((v - max) * c)); max -inf: nothing yet
struct MaxSum {
    float m, s;
    __device__ __forceinline__ void merge(float m2, float s2, float c) {
        const float mm = fmaxf(m, m2);
        if (mm == NEG_INF) {
            s += s2;  // (0, or a NaN that must stay)
            return;
        }
        s = s * exp2_raw((m - mm) * c) + s2 * exp2_raw((m2 - mm) * c);
        m = mm;
    }
    // the maximum first: one exponential a lane, not one a step
    __device__ __forceinline__ void wave(float c) {
        float mm = m;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
        s = wave_sum(m == mm ? s : s * exp2_raw((m - mm) * c));  // (all -inf: s is 0, or a NaN)
        m = mm;
    }
};
// Where |m * c| is below this, exp2(v * c - mc) is one fma and one exp2: the rounding of mc =
// fl(m * c), at most 2^-5, is a factor common to all terms, which done() takes out again.  Beyond
// (logits masked with -1e10, say, or a temperature near 0) that factor would leave float32
// itself: the difference is taken first, exp2((v - m) * c).
constexpr float EXP_SAFE = 0x1p20f;
// what mc leaves of m * c
__device__ __forceinline__ float exp_off(float m, float mc, float c) {
    return fabsf(mc) < EXP_SAFE ? fmaf(m, c, -mc) : 0.f;
}
// A thread's running form: s = the sum of exp2(v * c - mc), or of exp2((v - m) * c).
struct RunSum {
    float m = NEG_INF, mc = NEG_INF, s = 0.f;
    __device__ __forceinline__ void raise(float v, float c) {
        if (v > m) {
// (s is relative to mc as stored: mc - vc with the rounded vc, never one fma of v * c)
#pragma clang fp contract(off)
            const float vc = v * c;
            float d = mc - vc;
            if (!(fmaxf(fabsf(mc), fabsf(vc)) < EXP_SAFE)) d = (m - v) * c + (exp_off(v, vc, c) - exp_off(m, mc, c));
            s *= exp2_raw(d);
            m = v;
            mc = vc;
        }
    }
    // n values (compile-time n, a power of two), mx their maximum
    __device__ __forceinline__ void add(const float* v, int n, float mx, float c) {
        raise(mx, c);
        float t[8];
        if (fabsf(mc) < EXP_SAFE) {
            for (int e = 0; e < n; ++e) t[e] = exp2_raw(fmaf(v[e], c, -mc));
        } else if (m == NEG_INF) {  // nothing, or values that are no numbers: nor is the sum then
            for (int e = 0; e < n; ++e) t[e] = v[e] == NEG_INF ? 0.f : v[e];
        } else {
            for (int e = 0; e < n; ++e) t[e] = exp2_raw((v[e] - m) * c);
        }
        for (int h = n / 2; h > 0; h >>= 1)
            for (int e = 0; e < h; ++e) t[e] += t[e + h];
        s += t[0];
    }
    __device__ __forceinline__ void add1(float v, float c) { add(&v, 1, v, c); }
    __device__ __forceinline__ MaxSum done(float c) const {
        return MaxSum{m, s * exp2_raw(-exp_off(m, mc, c))};
    }
};

// block-wide merge; every thread returns the result (sm: 2 floats per wave)
__device__ __forceinline__ MaxSum block_maxsum(MaxSum a, float c, float* sm) {
    a.wave(c);
    const int w = threadIdx.x / 64, nw = blockDim.x / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        sm[2 * w] = a.m;
        sm[2 * w + 1] = a.s;
    }
    __syncthreads();
    MaxSum r{sm[0], 0.f};
    for (int i = 1; i < nw; ++i) r.m = fmaxf(r.m, sm[2 * i]);
    for (int i = 0; i < nw; ++i)
        r.s += sm[2 * i] == r.m ? sm[2 * i + 1] : sm[2 * i + 1] * exp2_raw((sm[2 * i] - r.m) * c);
    return r;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// ---------------------------------------------------------------- the loss: arguments
struct DistillArgs {
    const void* logits;
    const void* values;
    const void* indices;
    const float* rest;
    const float* weight;
    int64_t rows, inner, stride;  // row r = (r / inner, r % inner)
    int V, k, v16, i64;           // v16: values in bf16; i64: indices in 64 bits
    double T, coef;               // coef = scale; loss coef*T*T*w*KL, gradient coef*T*w*(p - q)
    float c;                      // log2(e) / T
    const float* gout;            // upstream gradient: NULL (1), a scalar, or one per row
    int gout_rows, skip_one;      // skip_one: nothing to do where the scalar is 1
    double* row_loss;             // weighted loss per row (or per block, class maps), or NULL
    float* row_out;               // reduction "none": the loss of each row, or NULL
    void* dz;                     // gradient, packed rows [rows][V] / maps [N][V][inner], or NULL
};

__device__ __forceinline__ bool distill_skip(const DistillArgs& a) {
    return a.skip_one && a.gout[0] == 1.f;
}
// entry j of record row (n, p): position in [N][k][inner]
__device__ __forceinline__ int distill_index(const DistillArgs& a, size_t at) {
    if (a.i64) {
        const int64_t i = static_cast<const int64_t*>(a.indices)[at];
        return i >= 0 && i < a.V ? (int)i : -1;
    }
    const int i = static_cast<const int*>(a.indices)[at];
    return i >= 0 && i < a.V ? i : -1;
}
__device__ __forceinline__ float distill_value(const DistillArgs& a, size_t at) {
    return a.v16 ? (float)static_cast<const __bf16*>(a.values)[at]
                 : static_cast<const float*>(a.values)[at];
}

// Entries 0 .. K - 1 of a pixel's record at `at` (absent beyond the k it has).  All loads go out
// before the first value is looked at: a choice of type per entry made the loads wait for one
// another (16 maps of 8 x 256^2 with 3 entries and the gradient: 37 us against 32).
template <int K>
__device__ __forceinline__ void map_entries(const DistillArgs& a, size_t at, int k, int* idx, float* t) {
    int lo[K], hi[K];
    uint32_t v[K];
    if (a.i64) {
#pragma unroll
        for (int e = 0; e < K; ++e) {
            const int2 q = static_cast<const int2*>(a.indices)[at + (size_t)(e < k ? e : k - 1) * a.inner];
            lo[e] = q.x;
            hi[e] = q.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < K; ++e) {
            lo[e] = static_cast<const int*>(a.indices)[at + (size_t)(e < k ? e : k - 1) * a.inner];
            hi[e] = 0;
        }
    }
    if (a.v16) {
#pragma unroll
        for (int e = 0; e < K; ++e)
            v[e] = static_cast<const uint16_t*>(a.values)[at + (size_t)(e < k ? e : k - 1) * a.inner];
    } else {
#pragma unroll
        for (int e = 0; e < K; ++e)
            v[e] = static_cast<const uint32_t*>(a.values)[at + (size_t)(e < k ? e : k - 1) * a.inner];
    }
#pragma unroll
    for (int e = 0; e < K; ++e) {
        idx[e] = e < k && hi[e] == 0 && (uint32_t)lo[e] < (uint32_t)a.V ? lo[e] : -1;
        t[e] = __uint_as_float(a.v16 ? v[e] << 16 : v[e]);
    }
}

// What a row's k + 1 classes give (computed by one wave over entries in LDS), in fp64: a loss is
// the difference of logarithms of nearly equal probabilities, and fp32 exponentials alone
// put a single row's KL 2e-7 off.  1 / T is c * ln 2 with the rounded c that the rest's fp32
// exponentials use: all parts share one temperature, 2^-24 beside the given one at most,
// which moves the KL by as little of itself, not of 1.
struct RowTerms {
    double kl;         // NaN / inf as they come out
    double M, m, iT;   // the teacher's and the student's maximum, 1 / T
    double rsq, rs;    // 1 / sums
    double restdiff;   // (p_rest - q_rest) / s_rest (0 where the student's rest is empty)
    bool empty;        // the record says nothing: no loss, no gradient
    __device__ __forceinline__ double q(float t) const { return exp(((double)t - M) * iT); }
    __device__ __forceinline__ double p(float z) const { return exp(((double)z - m) * iT); }
    __device__ __forceinline__ float grad(double g, float t, float z) const {
        return (float)(g * (p(z) * rs - q(t) * rsq));
    }
};

// one wave; idx < 0: absent.  r: the student's rest
__device__ __forceinline__ RowTerms row_terms(const int* idx, const float* t, const float* z, int k,
                                              float rest, MaxSum r, float c) {
    const int lane = threadIdx.x & 63;
    RowTerms o;
    o.iT = (double)c * LN2;
    float M = rest, m = r.m;
    for (int j = lane; j < k; j += 64)
        if (idx[j] >= 0) {
            M = fmaxf(M, t[j]);
            m = fmaxf(m, z[j]);
        }
    o.M = M = wave_max(M);
    o.m = m = wave_max(m);
    double sq = 0, ss = 0, kl = 0;
    for (int j = lane; j < k; j += 64)
        if (idx[j] >= 0) {
            const double e = o.q(t[j]);
            sq += e;
            ss += o.p(z[j]);
            if (!(e == 0.0)) kl += e * (((double)t[j] - o.M) - ((double)z[j] - o.m));
        }
    sq = wave_sum_d(sq);
    ss = wave_sum_d(ss);
    kl = wave_sum_d(kl) * o.iT;
    const double er = rest == NEG_INF ? 0.0 : o.q(rest);
    const double sr = r.m == NEG_INF ? (double)r.s : (double)r.s * o.p(r.m);  // (empty: 0, or a NaN)
    // the rest's log q - log p, but for the logarithms of the sums
    if (!(er == 0.0))
        kl += er * (r.m == NEG_INF ? (double)__builtin_inff()
                                   : (((double)rest - o.M) - ((double)r.m - o.m)) * o.iT - log((double)r.s));
    sq += er;
    ss += sr;
    o.rsq = 1.0 / sq;
    o.rs = 1.0 / ss;
    o.kl = kl * o.rsq + log(ss * o.rsq);  // (the q_j add up to 1)
    o.restdiff = r.m == NEG_INF ? 0.0 : (sr * o.rs - er * o.rsq) / (double)r.s;
    o.empty = M == NEG_INF;
    return o;
}

// ---------------------------------------------------------------- rows, a block each
struct RowShared {
    alignas(16) int idx[DK_MAX];
    float t[DK_MAX], z[DK_MAX], ms[2 * 16];
    int dup;
    float a, mr;
    double g;
    RowTerms o;
};

// the bitmap of the kept classes within the span
template <typename T>
__device__ __forceinline__ void row_marks(const DistillArgs& a, int64_t r, const RowSpan<T>& sp, uint32_t* bits) {
    const int tid = threadIdx.x, nt = blockDim.x;
    for (int i = tid; i < (sp.bits() + 31) / 32; i += nt) bits[i] = 0;
    __syncthreads();
    for (int j = tid; j < a.k; j += nt) {
        const int i = distill_index(a, (size_t)r * a.k + j);
        if (i >= sp.lo && i < sp.hi) atomicOr(&bits[sp.bit(i) >> 5], 1u << (sp.bit(i) & 31));
    }
    __syncthreads();
}

// the record's entries into LDS, the student's logits at them, and that bitmap; an index given
// twice counts the first time only
template <typename T>
__device__ __forceinline__ void row_entries(const DistillArgs& a, int64_t r, const RowSpan<T>& sp,
                                            RowShared& s, uint32_t* bits) {
    const int tid = threadIdx.x, nt = blockDim.x;
    for (int i = tid; i < (sp.bits() + 31) / 32; i += nt) bits[i] = 0;
    if (tid == 0) s.dup = 0;
    const int kp = (a.k + 3) & ~3;
    for (int j = tid; j < kp; j += nt) {
        int i = -1;
        if (j < a.k) {
            const size_t at = (size_t)r * a.k + j;
            i = distill_index(a, at);
            s.t[j] = distill_value(a, at);
            s.z[j] = i >= 0 ? (float)sp.z[i] : NEG_INF;
        }
        s.idx[j] = i;
    }
    __syncthreads();
    // entries up to j that equal j's index (four a read): one, unless it occurred before
    auto upto = [&](int j) {
        const int i = s.idx[j];
        int n = 0;
        for (int l = 0; l <= j; l += 4) {
            const int4 q = *reinterpret_cast<const int4*>(&s.idx[l]);
            n += (q.x == i) + (l + 1 <= j && q.y == i) + (l + 2 <= j && q.z == i) + (l + 3 <= j && q.w == i);
        }
        return n;
    };
    for (int j = tid; j < a.k; j += nt) {
        const int i = s.idx[j];
        if (i >= sp.lo && i < sp.hi) {
            const int b = sp.bit(i);
            const uint32_t old = atomicOr(&bits[b >> 5], 1u << (b & 31));
            if (old >> (b & 31) & 1) s.dup = 1;
        } else if (i >= 0 && upto(j) > 1) {  // outside the span: no bitmap to ask
            s.dup = 1;
        }
    }
    __syncthreads();
    if (s.dup) {  // (no correct record has one)
        unsigned drop = 0;
        for (int q = 0, j = tid; j < a.k; j += nt, ++q) drop |= (unsigned)(upto(j) > 1) << q;
        __syncthreads();
        for (int q = 0, j = tid; j < a.k; j += nt, ++q)
            if (drop >> q & 1) s.idx[j] = -1;
        __syncthreads();
    }
}

// sums over the span's classes outside the record
template <typename T>
__device__ __forceinline__ MaxSum row_rest(const DistillArgs& a, const RowSpan<T>& sp,
                                           const uint32_t* bits) {
    constexpr int N = RowVec<T>::N;
    RunSum acc;
    const float c = a.c;
    sp.template scan<4>(threadIdx.x, blockDim.x, [&](int slot, int i0, const Pack<T, N>& v, int cnt) {
        const uint32_t w = (bits[slot * N >> 5] >> (slot * N & 31)) & ((1u << N) - 1);
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = v.get(e);
        if (__builtin_expect(w != 0, 0)) {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = w >> e & 1 ? NEG_INF : x[e];
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < N; ++e) mx = fmaxf(mx, x[e]);
        acc.add(x, N, mx, c);
    });
    return acc.done(c);
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void row_grad(const DistillArgs& a, int64_t r, const RowSpan<T>& sp,
                                         RowShared& s) {
    constexpr int N = RowVec<T>::N;
    T* d = static_cast<T*>(a.dz) + (size_t)r * a.V;
    const float f = s.a, mr = s.mr, c = a.c;
    auto put = [&](int i0, const Pack<T, N>& o, int cnt) {
        if (ALIGNED && cnt == N) {
            o.store(d + i0);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (e < cnt) d[i0 + e] = (T)o.get(e);
        }
    };
    if (f == 0.f || mr == NEG_INF) {  // (f NaN: written as such below)
        Pack<T, N> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.set(e, 0.f);
        sp.template scan<1>(threadIdx.x, blockDim.x, [&](int, int i0, const Pack<T, N>&, int cnt) { put(i0, o, cnt); });
    } else if (const float mc = mr * c; fabsf(mc) < EXP_SAFE) {
        const float fc = f * exp2_raw(-fmaf(mr, c, -mc));  // (as RunSum::done)
        sp.template scan_back<4>(threadIdx.x, blockDim.x, [&](int, int i0, const Pack<T, N>& v, int cnt) {
            Pack<T, N> o;
#pragma unroll
            for (int e = 0; e < N; ++e) o.set(e, fc * exp2_raw(fmaf(v.get(e), c, -mc)));
            put(i0, o, cnt);
        });
    } else {
        sp.template scan<1>(threadIdx.x, blockDim.x, [&](int, int i0, const Pack<T, N>& v, int cnt) {
            Pack<T, N> o;
#pragma unroll
            for (int e = 0; e < N; ++e) o.set(e, f * exp2_raw((v.get(e) - mr) * c));
            put(i0, o, cnt);
        });
    }
    __syncthreads();  // the kept classes over what the scan wrote there
    if (s.o.empty || s.g == 0.0) return;
    for (int j = threadIdx.x; j < a.k; j += blockDim.x) {
        const int i = s.idx[j];
        if (i >= sp.lo && i < sp.hi) d[i] = (T)s.o.grad(s.g, s.t[j], s.z[j]);
    }
}

// wave 0: the row's terms; every thread of the block calls it
__device__ __forceinline__ void row_finish(const DistillArgs& a, int64_t r, MaxSum rest, bool first,
                                           RowShared& s) {
    const float w = a.weight ? a.weight[r] : 1.f;
    if (threadIdx.x < 64) {
        const float tr = a.rest ? a.rest[r] : NEG_INF;
        const RowTerms o = row_terms(s.idx, s.t, s.z, a.k, tr, rest, a.c);
        if (threadIdx.x == 0) {
            const bool none = o.empty || w == 0.f;
            const double l = none ? 0.0 : a.coef * a.T * a.T * (double)w * o.kl;
            if (first && a.row_loss) a.row_loss[r] = l;
            if (first && a.row_out) a.row_out[r] = (float)l;
            const double go = a.gout ? (double)a.gout[a.gout_rows ? r : 0] : 1.0;
            s.g = none ? 0.0 : a.coef * a.T * (double)w * go;
            s.a = none ? 0.f : (float)(s.g * o.restdiff);
            s.mr = rest.m;
            s.o = o;
            s.o.empty = none;
        }
    }
    __syncthreads();
}

template <typename T, bool ALIGNED, int NT>
__global__ void __launch_bounds__(NT) distill_row_kernel(DistillArgs a) {
    extern __shared__ uint32_t bits[];
    __shared__ RowShared s;
    if (distill_skip(a)) return;
    const int64_t r = blockIdx.x;
    const RowSpan<T> sp(static_cast<const T*>(a.logits) + r * a.stride, 0, a.V);
    row_entries<T>(a, r, sp, s, bits);
    const MaxSum rest = block_maxsum(row_rest(a, sp, bits), a.c, s.ms);
    row_finish(a, r, rest, true, s);
    if (a.dz) row_grad<T, ALIGNED>(a, r, sp, s);
}

// few or very long rows: `split` blocks a row, sums first ...
template <typename T>
__global__ void __launch_bounds__(256) distill_part_kernel(DistillArgs a, int split, int chunk,
                                                           float* part) {
    extern __shared__ uint32_t bits[];
    __shared__ float ms[8];
    if (distill_skip(a)) return;
    const int64_t r = blockIdx.x / split;
    const int c = blockIdx.x % split, lo = c * chunk;
    const RowSpan<T> sp(static_cast<const T*>(a.logits) + r * a.stride, lo < a.V ? lo : a.V,
                        lo + chunk < a.V ? lo + chunk : a.V);
    row_marks<T>(a, r, sp, bits);
    const MaxSum rest = block_maxsum(row_rest(a, sp, bits), a.c, ms);
    if (threadIdx.x == 0) {
        part[2 * blockIdx.x] = rest.m;
        part[2 * blockIdx.x + 1] = rest.s;
    }
}
// ... then the row's terms (every block of a row, the same way) and its share of the gradient
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) distill_join_kernel(DistillArgs a, int split, int chunk,
                                                           int gsplit, int gchunk,
                                                           const float* part) {
    extern __shared__ uint32_t bits[];
    __shared__ RowShared s;
    if (distill_skip(a)) return;
    const int64_t r = blockIdx.x / gsplit;
    const int c = blockIdx.x % gsplit, lo = c * gchunk;
    const RowSpan<T> sp(static_cast<const T*>(a.logits) + r * a.stride, lo < a.V ? lo : a.V,
                        lo + gchunk < a.V ? lo + gchunk : a.V);
    row_entries<T>(a, r, sp, s, bits);
    MaxSum rest{NEG_INF, 0.f};
    for (int i = threadIdx.x; i < split; i += blockDim.x)
        rest.merge(part[2 * (r * split + i)], part[2 * (r * split + i) + 1], a.c);
    rest = block_maxsum(rest, a.c, s.ms);
    row_finish(a, r, rest, c == 0, s);
    if (a.dz) row_grad<T, ALIGNED>(a, r, sp, s);
}

// the sum of the waves' losses -> row_loss[block] (256 threads)
__device__ __forceinline__ void block_loss(const DistillArgs& a, double l) {
    __shared__ double red[4];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = l;
    __syncthreads();
    if (threadIdx.x == 0 && a.row_loss) a.row_loss[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// ---------------------------------------------------------------- short rows, a wave each
constexpr int DW_MAX = 512;  // classes
struct WaveShared {
    int idx[DK_MAX];
    float t[DK_MAX], z[DK_MAX];
    uint32_t bits[DW_MAX / 32];
};

// LDS written and read by one wave: its operations stay in order, the compiler must too
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// NV values a lane; returns the row's weighted loss (every lane)
template <typename T, int NV>
__device__ __forceinline__ double distill_wave_row(const DistillArgs& a, int64_t r, WaveShared& s) {
    const int lane = threadIdx.x & 63;
    const T* z = static_cast<const T*>(a.logits) + r * a.stride;
    float v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = lane + 64 * i < a.V ? (float)z[lane + 64 * i] : NEG_INF;
    if (lane < DW_MAX / 32) s.bits[lane] = 0;
    wave_sync();
    bool dup = false;
    for (int j = lane; j < a.k; j += 64) {
        const size_t at = (size_t)r * a.k + j;
        const int i = distill_index(a, at);
        s.idx[j] = i;
        s.t[j] = distill_value(a, at);
        s.z[j] = i >= 0 ? (float)z[i] : NEG_INF;
        if (i >= 0) dup |= atomicOr(&s.bits[i >> 5], 1u << (i & 31)) >> (i & 31) & 1;
    }
    wave_sync();
    if (__any(dup)) {
        unsigned drop = 0;
        for (int q = 0, j = lane; j < a.k; j += 64, ++q)
            for (int l = 0; l < j; ++l) drop |= (unsigned)(s.idx[l] == s.idx[j]) << q;
        wave_sync();
        for (int q = 0, j = lane; j < a.k; j += 64, ++q)
            if (drop >> q & 1) s.idx[j] = -1;
        wave_sync();
    }
    const float w = a.weight ? a.weight[r] : 1.f;
    RunSum acc;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int x = lane + 64 * i;
        if (x < a.V && !(s.bits[x >> 5] >> (x & 31) & 1)) acc.add1(v[i], a.c);
    }
    MaxSum rest = acc.done(a.c);
    rest.wave(a.c);
    const float tr = a.rest ? a.rest[r] : NEG_INF;
    const RowTerms o = row_terms(s.idx, s.t, s.z, a.k, tr, rest, a.c);
    const bool none = o.empty || w == 0.f;
    const double l = none ? 0.0 : a.coef * a.T * a.T * (double)w * o.kl;
    if (a.dz) {
        T* d = static_cast<T*>(a.dz) + (size_t)r * a.V;
        const double go = a.gout ? (double)a.gout[a.gout_rows ? r : 0] : 1.0;
        const double g = none ? 0.0 : a.coef * a.T * (double)w * go;
        const float f = none || rest.m == NEG_INF ? 0.f : (float)(g * o.restdiff);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int x = lane + 64 * i;
            if (x < a.V && !(s.bits[x >> 5] >> (x & 31) & 1))
                d[x] = (T)(f == 0.f ? 0.f : f * exp2_raw((v[i] - rest.m) * a.c));
        }
        for (int j = lane; j < a.k; j += 64)
            if (s.idx[j] >= 0)
                d[s.idx[j]] = (T)(none ? 0.f : o.grad(g, s.t[j], s.z[j]));
    }
    wave_sync();  // the next row reuses the LDS
    return l;
}

// one block for everything: also sums the rows (loss out)
template <typename T, int NV>
__global__ void __launch_bounds__(1024) distill_wave_one_kernel(DistillArgs a, float* loss) {
    __shared__ WaveShared s[16];
    __shared__ double sum[16];
    if (distill_skip(a)) return;
    const int w = threadIdx.x / 64, nw = blockDim.x / 64;
    double acc = 0;
    for (int64_t r = w; r < a.rows; r += nw) {
        const double l = distill_wave_row<T, NV>(a, r, s[w]);
        if (a.row_out && (threadIdx.x & 63) == 0) a.row_out[r] = (float)l;
        acc += l;
    }
    if ((threadIdx.x & 63) == 0) sum[w] = acc;
    __syncthreads();
    if (threadIdx.x == 0 && loss) {
        for (int i = 1; i < nw; ++i) acc += sum[i];
        loss[0] = (float)acc;
    }
}
// the blocks step over the rows; row_loss: a block's sum
template <typename T, int NV>
__global__ void __launch_bounds__(256) distill_wave_kernel(DistillArgs a) {
    __shared__ WaveShared s[4];
    if (distill_skip(a)) return;
    double acc = 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; r < a.rows; r += (int64_t)gridDim.x * 4) {
        const double l = distill_wave_row<T, NV>(a, r, s[threadIdx.x / 64]);
        if (a.row_out && (threadIdx.x & 63) == 0) a.row_out[r] = (float)l;
        acc += l;
    }
    block_loss(a, acc);
}

// ---------------------------------------------------------------- class maps, a thread each
// The teacher's exp2(x).  Below float32's range it still counts: against a student's logit of the
// type's lowest value, 3e38, a probability of 2^-130 is a loss of 0.2.
__device__ __forceinline__ double teacher_exp2(float x) {
    double e = exp2_raw(x);
    if (__builtin_expect(x < -100.f, 0)) {
        const float n = fmaxf(rintf(x), -2000.f);
        e = x < -2000.f ? 0.0 : ldexp((double)exp2_raw(x - n), (int)n);
    }
    return e;
}

// At most VR classes and KR entries: a pixel's logits and record stay in registers, read once.
// Exponentials are fp32 here, sums and differences fp64: a pixel's KL is off by 2^-19 of a unit
// at most (1e-7 in the mean over a map; fp64 exponentials, as a row's terms have, would be k + 1
// for every pixel).  16 maps of 8 x 256^2 fp32 at 3 entries, with the gradient: 30 us (55 with marks in LDS
// and the classes read twice); its floor, 113 MB at a copy's 4.8 TB/s, is 24.
template <typename T, int VR, int KR> __global__ void __launch_bounds__(256) distill_map_small_kernel(DistillArgs a) {
    if (distill_skip(a)) return;
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    double l = 0;
    if (r < a.rows) {
        const int64_t n = r / a.inner, p = r % a.inner;
        const T* z = static_cast<const T*>(a.logits) + (size_t)n * a.V * a.inner + p;
        const size_t rec = (size_t)n * a.k * a.inner + p;
        const float c = a.c;
        const double iT = (double)c * LN2;  // (see RowTerms)
        float x[VR], t[KR], zj[KR];
        int idx[KR];
#pragma unroll
        for (int i = 0; i < VR; ++i) x[i] = i < a.V ? (float)z[(size_t)i * a.inner] : NEG_INF;
        map_entries<KR>(a, rec, a.k, idx, t);
        const float w = a.weight ? a.weight[r] : 1.f;
        const float rest = a.rest ? a.rest[r] : NEG_INF;
        uint32_t mask = 0;
        float M = rest, m = NEG_INF;
#pragma unroll
        for (int j = 0; j < KR; ++j) {
            const uint32_t b = idx[j] >= 0 ? 1u << idx[j] : 0u;
            if (mask & b) idx[j] = -1;  // an index seen before is absent
            mask |= b;
            zj[j] = NEG_INF;
#pragma unroll
            for (int i = 0; i < VR; ++i) zj[j] = idx[j] == i ? x[i] : zj[j];
            if (idx[j] >= 0) {
                M = fmaxf(M, t[j]);
                m = fmaxf(m, zj[j]);
            }
        }
        RunSum acc;
#pragma unroll
        for (int i0 = 0; i0 < VR; i0 += 8) {
            float y[8], mx = NEG_INF;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] = mask >> (i0 + e) & 1 ? NEG_INF : x[i0 + e];
                mx = fmaxf(mx, y[e]);
            }
            acc.add(y, 8, mx, c);
        }
        const MaxSum rs = acc.done(c);
        const bool has = rs.m != NEG_INF;
        m = fmaxf(m, rs.m);
        // as row_terms
        double sq = 0, ss = 0, kl = 0;
        float eq[KR], ep[KR];
#pragma unroll
        for (int j = 0; j < KR; ++j) {
            eq[j] = ep[j] = 0.f;
            if (idx[j] >= 0) {
                const double e = teacher_exp2((t[j] - M) * c);
                eq[j] = (float)e;
                ep[j] = exp2_raw((zj[j] - m) * c);
                sq += e;
                ss += ep[j];
                if (!(e == 0.0)) kl += e * (((double)t[j] - M) - ((double)zj[j] - m));
            }
        }
        kl *= iT;
        const double er = rest == NEG_INF ? 0.0 : teacher_exp2((rest - M) * c);
        const float sr = has ? rs.s * exp2_raw((rs.m - m) * c) : rs.s;
        if (!(er == 0.0))
            kl += has ? er * ((((double)rest - M) - ((double)rs.m - m)) * iT - log((double)rs.s))
                      : (double)__builtin_inff();
        sq += er;
        ss += sr;
        const double rsq = 1.0 / sq, rss = 1.0 / ss;
        const bool none = M == NEG_INF || w == 0.f;
        l = none ? 0.0 : a.coef * a.T * a.T * (double)w * (kl * rsq + log(ss * rsq));
        if (a.row_out) a.row_out[r] = (float)l;
        if (a.dz) {
            T* d = static_cast<T*>(a.dz) + (size_t)n * a.V * a.inner + p;
            const double go = a.gout ? (double)a.gout[a.gout_rows ? r : 0] : 1.0;
            const double g = none ? 0.0 : a.coef * a.T * (double)w * go;
            const float f = none || !has ? 0.f : (float)(g * ((double)sr * rss - er * rsq) / (double)rs.s);
            float dk[KR];
#pragma unroll
            for (int j = 0; j < KR; ++j) dk[j] = none ? 0.f : (float)(g * ((double)ep[j] * rss - (double)eq[j] * rsq));
#pragma unroll
            for (int i = 0; i < VR; ++i) {
                if (i >= a.V) break;
                float v = f == 0.f ? 0.f : f * exp2_raw((x[i] - rs.m) * c);
#pragma unroll
                for (int j = 0; j < KR; ++j) v = idx[j] == i ? dk[j] : v;
                d[(size_t)i * a.inner] = (T)v;
            }
        }
    }
    block_loss(a, wave_sum_d(l));
}

// More classes or entries: a thread a pixel, or (S = 4, more than 32 classes: the pixels alone may
// not fill the card) four threads of different waves, each a part of the classes; the first
// reads the record and joins the parts.  Marks of the kept classes lie in LDS.  2 maps of 64 x
// 256^2 fp32, 8 entries, with the gradient: 35 us (a thread a pixel, entries read three times:
// 87); one of 1000 x 128^2: 67 (690); 8 maps of 16 x 256^2 with 12 entries, the loss: 37, with
// S = 4 153.  Bound by the record's steps and the classes' second reading.
constexpr int DM_MAX = 1024;  // classes
template <typename T, int KR, int S> __global__ void __launch_bounds__(256) distill_map_kernel(DistillArgs a) {
    constexpr int PX = 256 / S;
    extern __shared__ uint32_t bits[];  // [ceil(V / 32)][PX]
    __shared__ float sm[256], ss[256];
    if (distill_skip(a)) return;
    const int tid = threadIdx.x, px = tid % PX, sl = tid / PX;
    const int64_t at = (int64_t)blockIdx.x * PX + px;
    const bool on = at < a.rows;
    const int64_t r = on ? at : a.rows - 1;  // (a thread beyond the last pixel reads that one)
    const int64_t n = r / a.inner, p = r % a.inner;
    const T* z = static_cast<const T*>(a.logits) + (size_t)n * a.V * a.inner + p;
    const size_t rec = (size_t)n * a.k * a.inner + p;
    uint32_t* mine = bits + px;
    const float c = a.c;
    for (int i = sl; i < (a.V + 31) / 32; i += S) mine[PX * i] = 0;
    __syncthreads();
    // The record's entries, each index once: read on pass 0, which marks them, and kept in
    // registers, up to KR; or read on every pass, with the marks set, cleared and set again.
    int ri[KR > 0 ? KR : 1];
    float rt[KR > 0 ? KR : 1], rz[KR > 0 ? KR : 1];
    auto entries = [&](int pass, auto f) {
        if constexpr (KR > 0) {
            if (pass == 0) {
#pragma unroll
                for (int e = 0; e < KR; e += 8) {
                    for (int i = e; i < e + 8; ++i) ri[i] = -1;
                    if (e < a.k) map_entries<8>(a, rec + (size_t)e * a.inner, a.k - e, ri + e, rt + e);
                }
#pragma unroll
                for (int e = 0; e < KR; ++e) rz[e] = ri[e] >= 0 ? (float)z[(size_t)ri[e] * a.inner] : NEG_INF;
#pragma unroll
                for (int e = 0; e < KR; ++e)
                    if (ri[e] >= 0) {
                        uint32_t& word = mine[PX * (ri[e] >> 5)];
                        const uint32_t b = 1u << (ri[e] & 31);
                        if (word & b) ri[e] = -1;
                        else word |= b;
                    }
            }
#pragma unroll
            for (int e = 0; e < KR; ++e)
                if (ri[e] >= 0) f(ri[e], rt[e], rz[e]);
            return;
        }
        for (int j0 = 0; j0 < a.k; j0 += 4) {
            int i[4];
            float t[4], zi[4];
            map_entries<4>(a, rec + (size_t)j0 * a.inner, a.k - j0, i, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) zi[e] = i[e] >= 0 ? (float)z[(size_t)i[e] * a.inner] : NEG_INF;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i[e] < 0) continue;
                uint32_t& word = mine[PX * (i[e] >> 5)];
                const uint32_t b = 1u << (i[e] & 31);
                if (((word & b) != 0) == (pass != 1)) continue;
                word ^= b;
                f(i[e], t[e], zi[e]);
            }
        }
    };
    const float w = a.weight ? a.weight[r] : 1.f;
    const float rest = a.rest ? a.rest[r] : NEG_INF;
    float M = rest, m = NEG_INF;
    if (sl == 0)
        entries(0, [&](int, float t, float zi) {
            M = fmaxf(M, t);
            m = fmaxf(m, zi);
        });
    __syncthreads();
    // classes in eights, so that a group's marks lie in one word
    const int per = (a.V + 8 * S - 1) / (8 * S) * 8, v0 = sl * per < a.V ? sl * per : a.V, v1 = v0 + per < a.V ? v0 + per : a.V;
    auto each = [&](auto f) {
        for (int i0 = v0; i0 < v1; i0 += 8) {
            const uint32_t b = mine[PX * (i0 >> 5)] >> (i0 & 31);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)z[(size_t)(i0 + e < v1 ? i0 + e : v1 - 1) * a.inner];
            f(i0, b, x);
        }
    };
    RunSum acc;
    each([&](int i0, uint32_t b, float (&x)[8]) {
        float mx = NEG_INF;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (b >> e & 1 || i0 + e >= v1) x[e] = NEG_INF;
            mx = fmaxf(mx, x[e]);
        }
        acc.add(x, 8, mx, c);
    });
    MaxSum rs = acc.done(c);
    sm[tid] = rs.m;
    ss[tid] = rs.s;
    __syncthreads();
    double l = 0;
    if (sl == 0) {
        for (int q = px + PX; q < 256; q += PX) rs.merge(sm[q], ss[q], c);
        const bool has = rs.m != NEG_INF;
        m = fmaxf(m, rs.m);
        double sq = 0, sp = 0;
        entries(1, [&](int, float t, float zi) {
            sq += teacher_exp2((t - M) * c);
            sp += exp2_raw((zi - m) * c);
        });
        const double er = rest == NEG_INF ? 0.0 : teacher_exp2((rest - M) * c);
        const double iT = (double)c * LN2;  // (see RowTerms)
        const double logr = has ? ((double)rs.m - (double)m) * iT + log((double)rs.s) : (double)NEG_INF;
        const float sr = has ? rs.s * exp2_raw((rs.m - m) * c) : rs.s;
        sq += er;
        sp += sr;
        const double lq = log(sq), ls = log(sp), rsq = 1.0 / sq, rsp = 1.0 / sp;
        const bool none = M == NEG_INF || w == 0.f;
        const double go = a.gout ? (double)a.gout[a.gout_rows ? r : 0] : 1.0;
        const double g = none ? 0.0 : a.coef * a.T * (double)w * go;
        T* d = static_cast<T*>(a.dz) + (a.dz ? (size_t)n * a.V * a.inner + p : 0);
        double kl = 0;
        entries(2, [&](int i, float t, float zi) {
            const double q = teacher_exp2((t - M) * c) * rsq;
            if (!(q == 0.0))
                kl += q * ((((double)t - (double)M) * iT - lq) - (((double)zi - (double)m) * iT - ls));
            if (a.dz && on)
                d[(size_t)i * a.inner] = (T)(none ? 0.f : (float)(g * ((double)exp2_raw((zi - m) * c) * rsp - q)));
        });
        const double qr = er * rsq;
        if (!(qr == 0.0)) kl += qr * ((((double)rest - (double)M) * iT - lq) - (logr - ls));
        l = none || !on ? 0.0 : a.coef * a.T * a.T * (double)w * kl;
        if (a.row_out && on) a.row_out[r] = (float)l;
        sm[px] = rs.m;
        ss[px] = none || !has ? 0.f : (float)(g * (((double)sr * rsp - qr) / (double)rs.s));
    }
    if (a.dz) {
        __syncthreads();
        const float mr = sm[px], f = ss[px];
        T* d = static_cast<T*>(a.dz) + (size_t)n * a.V * a.inner + p;
        each([&](int i0, uint32_t b, float (&x)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (on && !(b >> e & 1) && i0 + e < v1)
                    d[(size_t)(i0 + e) * a.inner] = (T)(f == 0.f ? 0.f : f * exp2_raw((x[e] - mr) * c));
        });
    }
    block_loss(a, wave_sum_d(l));
}

__global__ void __launch_bounds__(1024) distill_sum_kernel(const double* part, int64_t n, float* loss) {
    __shared__ double s[16];
    double acc = 0;
#pragma unroll 16
    for (int64_t i = threadIdx.x; i < n; i += 1024) acc += part[i];
    acc = wave_sum_d(acc);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x / 64] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) acc += s[i];
        loss[0] = (float)acc;
    }
}

// ---------------------------------------------------------------- a teacher's top logits
// Order of a row: the larger value first, then the lower index; a NaN counts as the largest.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);  // (-0 is 0)
    return v != v ? 0xffffffffu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// larger is earlier
__device__ __forceinline__ uint64_t order_pair(uint32_t key, int idx) {
    return (uint64_t)key << 32 | (uint32_t)~idx;
}

struct TopArgs {
    const void* logits;
    int64_t rows, inner, stride;
    int V, k;
    float T, c;  // temperature, log2(e) / T
    int first;   // the first segment is this part of the tiles
    void* values;
    int64_t* indices;
    float* rest;
};

__device__ __forceinline__ float rest_logit(MaxSum r, float T) {
    // (+inf among the others: their sum of exp is not a number, their logit is +inf)
    if (r.m == __builtin_inff()) return r.m;
    return r.m == NEG_INF ? NEG_INF + r.s : (float)((double)r.m + (double)T * log((double)r.s));
}

constexpr int TK_NEAR = 512;  // values at or above the last bound that are ranked at most
// CAP: vectors set aside at most
template <int CAP> struct TopShared {
    uint4 raw[CAP];
    uint32_t key[CAP], idx[CAP];  // the maximum's key; first index
    uint8_t cnt[CAP];             // values of the vector
    uint64_t near[TK_NEAR], sum[8];
    float mx[512], ms[32];
    uint32_t hist[256];
    int n, nn, eq[9];
    uint32_t tau;
};

// Exact selection by key digits, for rows the threshold does not thin out (many equal values,
// masked rows, NaN): the k-th key by four histograms, then the larger ones and the first of
// the equal ones in index order.  Leaves the k entries in s.near; returns the rest's sums.
template <typename T, typename S>
__device__ MaxSum top_exact(const TopArgs& a, const RowSpan<T>& sp, S& s) {
    constexpr int N = RowVec<T>::N;
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, w = tid / 64, nw = nt / 64;
    uint32_t prefix = 0;
    int need = a.k;  // entries still to take among the keys that match the prefix
    for (int d = 24; d >= 0; d -= 8) {
        for (int i = tid; i < 256; i += nt) s.hist[i] = 0;
        __syncthreads();
        const uint32_t high = d == 24 ? 0u : 0xffffffffu << (d + 8);
        sp.template scan<1>(tid, nt, [&](int, int, const Pack<T, N>& v, int cnt) {
            for (int e = 0; e < cnt; ++e) {
                const uint32_t key = order_key(v.get(e));
                const bool in = ((key ^ prefix) & high) == 0;
                const uint32_t dig = key >> d & 255;
                // equal digits across the wave (a row of one value): one addition
                const uint32_t first = __builtin_amdgcn_readfirstlane(dig);
                const uint64_t act = __ballot(1), same = __ballot(in && dig == first);
                if (same == act) {
                    if ((int)(__ffsll((unsigned long long)act) - 1) == lane) atomicAdd(&s.hist[first], (uint32_t)__popcll(act));
                } else if (in) {
                    atomicAdd(&s.hist[dig], 1u);
                }
            }
        });
        __syncthreads();
        // digit of the k-th key: the largest b with (count of digits >= b) >= need
        if (tid == 0) {
            int left = need, b = 255;
            for (; b > 0 && left > (int)s.hist[b]; --b) left -= s.hist[b];
            s.eq[0] = left;
            s.tau = prefix | (uint32_t)b << d;
        }
        __syncthreads();
        need = s.eq[0];
        prefix = s.tau;
        __syncthreads();
    }
    // prefix: the k-th key; `need` of the values equal to it belong to the record
    if (tid == 0) s.nn = 0;
    __syncthreads();
    RunSum acc;
    int taken = 0;
    const int lo = sp.lo, hi = sp.hi;
    for (int base = lo; base < hi; base += nt) {
        const int i = base + tid;
        const uint32_t key = i < hi ? order_key((float)sp.z[i]) : 0u;
        const bool eq = i < hi && key == prefix;
        bool take = i < hi && key > prefix;
        if (taken < need) {  // (uniform)
            const uint64_t m = __ballot(eq);
            if (lane == 0) s.eq[1 + w] = __popcll(m);
            __syncthreads();
            int before = taken, all = taken;
            for (int q = 0; q < nw; ++q) {
                if (q < w) before += s.eq[1 + q];
                all += s.eq[1 + q];
            }
            const int pos = before + __popcll(m & ((1ull << lane) - 1));
            take |= eq && pos < need;
            taken = all;
            __syncthreads();
        }
        if (take) {
            const int at = atomicAdd(&s.nn, 1);  // (their order does not matter)
            s.near[at] = order_pair(key, i);
        } else if (i < hi) {
            acc.add1((float)sp.z[i], a.c);
        }
    }
    __syncthreads();
    return acc.done(a.c);
}

// one wave: the upper 16 bits of the k-th largest of n <= 64 * R keys (key(i): the i-th),
// counting with ballots (shuffles would cost several times the comparisons)
template <int R, typename F> __device__ __forceinline__ uint32_t kth_prefix_of(int n, int k, F key) {
    const int lane = threadIdx.x & 63;
    uint32_t v[R];
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = lane + 64 * i < n ? key(lane + 64 * i) >> 16 : 0u;
    uint32_t t = 0;
    for (int b = 14; b >= 0; b -= 2) {  // two bits a step: three independent counts
        const uint32_t u1 = t | 1u << b, u2 = t | 2u << b, u3 = t | 3u << b;
        int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            c1 += __popcll(__ballot(v[i] >= u1));
            c2 += __popcll(__ballot(v[i] >= u2));
            c3 += __popcll(__ballot(v[i] >= u3));
        }
        t = c3 >= k ? u3 : c2 >= k ? u2 : c1 >= k ? u1 : t;
    }
    return t;
}
template <typename F> __device__ __forceinline__ uint32_t kth_prefix(int n, int k, F key) {
    if (n <= 256) return kth_prefix_of<4>(n, k, key);
    if (n <= 512) return kth_prefix_of<8>(n, k, key);
    if (n <= 1024) return kth_prefix_of<16>(n, k, key);
    return kth_prefix_of<32>(n, k, key);
}
// that prefix as a value that bounds the k-th from below
__device__ __forceinline__ float prefix_value(uint32_t t) {
    t <<= 16;
    // (keys below that of -inf belong to no value; a NaN's cannot be a bound)
    return t <= 0x007fffffu ? NEG_INF : t >= 0xff800000u ? __builtin_inff() : key_value(t);
}

// A row is read once, in segments: the first quarter, up to the half, the rest.  A vector
// whose maximum reaches a lower bound tau of the k-th largest value is set aside as loaded; the
// others go into the rest's sums at once.  tau comes from the threads' maxima over the first
// quarter (which is read a second time, from the caches) and rises to the k-th maximum of
// what is set aside before each further segment, which so adds about k vectors.  At the end
// the values of the vectors set aside are told apart: those near the k-th are ranked by
// counting, the others join the rest.  A thread's sum is V / (NT * N) additions deep, V / NT in
// the exact selection: V / 512 for wide rows.  A row has one block whatever its length: 65537 fp32
// values take 19 us, 2^20 131, 2^22 628.  What bounds many rows is the instructions: setting single
// values aside took 196 us for 2048 x 131072 bf16 (22 vector instructions a value), and so did
// two readings of whole rows; rows held in registers 299 (a block a CU).
template <typename T, int NT, int CAP> __global__ void __launch_bounds__(NT, 8) top_row_kernel(TopArgs a) {
    constexpr int N = RowVec<T>::N, U = 4;
    __shared__ TopShared<CAP> s;
    constexpr int nt = NT;
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t r = blockIdx.x;
    const RowSpan<T> sp(static_cast<const T*>(a.logits) + r * a.stride, 0, a.V);
    const T* const body = sp.z + sp.head;
    const float c = a.c;
    float tau = NEG_INF;
    RunSum acc;
    auto top_of = [](const Pack<T, N>& v) {
        float m = v.get(0);
#pragma unroll
        for (int e = 1; e < N; ++e) m = fmaxf(m, v.get(e));
        return m;
    };
    auto eat = [&](int i0, const Pack<T, N>& v, int cnt) {
        float x[N], mx = top_of(v);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = v.get(e);
        if (__builtin_expect(!(mx < tau), 0)) {
            const int at = atomicAdd(&s.n, 1);
            if (at < CAP) {
                s.raw[at] = v.raw;
                s.key[at] = order_key(mx);
                s.idx[at] = i0;
                s.cnt[at] = (uint8_t)cnt;
            }
            mx = NEG_INF;
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = NEG_INF;
        }
        acc.add(x, N, mx, c);
    };
    // tiles of nt vectors; the row's ends belong to the first segment
    const int tiles = (sp.nv + nt - 1) / nt;
    int end = (tiles + a.first - 1) / a.first;
    float mx = NEG_INF;
    const int last = end * nt < sp.nv ? end * nt : sp.nv;
    int i = tid;
    for (; i + (U - 1) * nt < last; i += U * nt) {
        Pack<T, N> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].load(body + (size_t)(i + u * nt) * N);
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, top_of(v[u]));
    }
    for (; i < last; i += nt) {
        Pack<T, N> v;
        v.load(body + (size_t)i * N);
        mx = fmaxf(mx, top_of(v));
    }
    sp.ends(tid, nt, [&](int, int, const Pack<T, N>& v, int) { mx = fmaxf(mx, top_of(v)); });
    s.mx[tid] = mx;
    __syncthreads();
    if (tid < 64) {
        const uint32_t t = kth_prefix(nt, a.k, [&](int i) { return order_key(s.mx[i]); });
        if (lane == 0) s.tau = t;
    }
    if (tid == 0) s.n = s.nn = 0;
    __syncthreads();
    tau = prefix_value(s.tau);
    sp.ends(tid, nt, [&](int, int i0, const Pack<T, N>& v, int cnt) { eat(i0, v, cnt); });
    int n = 0;
    for (int t = 0;;) {
        for (; t + U <= end; t += U) {
            Pack<T, N> v[U];
            const int i = t * nt + tid;
            if (i + (U - 1) * nt < sp.nv) {
#pragma unroll
                for (int u = 0; u < U; ++u) v[u].load(body + (size_t)(i + u * nt) * N);
#pragma unroll
                for (int u = 0; u < U; ++u) eat(sp.head + (i + u * nt) * N, v[u], N);
            } else {
                for (int u = 0; u < U; ++u)
                    if (i + u * nt < sp.nv) {
                        v[0].load(body + (size_t)(i + u * nt) * N);
                        eat(sp.head + (i + u * nt) * N, v[0], N);
                    }
            }
        }
        for (; t < end; ++t) {
            const int i = t * nt + tid;
            if (i < sp.nv) {
                Pack<T, N> v;
                v.load(body + (size_t)i * N);
                eat(sp.head + i * N, v, N);
            }
        }
        __syncthreads();
        n = s.n;
        if (end >= tiles || n > CAP) break;
        if (n >= a.k) {
            if (tid < 64) {
                const uint32_t p = kth_prefix(n, a.k, [&](int i) { return s.key[i]; });
                if (lane == 0) s.tau = p;
            }
            __syncthreads();
            tau = fmaxf(tau, prefix_value(s.tau));
        }
        end = 2 * end < tiles ? 2 * end : tiles;
    }
    MaxSum rest = block_maxsum(acc.done(c), c, s.ms);
    // the values of the vectors set aside: the key of value e of vector i, f(pair) for each
    auto key_of = [&](int i, int e) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(&s.raw[i])[e * (int)sizeof(T) / 4];
        return order_key(sizeof(T) == 4 ? __uint_as_float(w) : __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16));
    };
    auto each = [&](auto f) {
        for (int j = tid; j < n * N; j += nt)
            if (j % N < (int)s.cnt[j / N]) f(order_pair(key_of(j / N, j % N), (int)s.idx[j / N] + j % N));
    };
    bool exact = n > CAP || rest.s != rest.s;  // too much near the top, or a NaN below it
    if (!exact) {
        // bounds of the k-th: the last tau and the vectors' k-th maximum, or, where that leaves most
        // of a short row, the k-th value's own prefix (8192 x 2000 bf16, k = 250: 260 us, 512
        // without, mostly in exact selections; of 3000 it would take 275 instead of 205)
        uint32_t low = order_key(tau);
        const bool few = n * 4 > 3 * sp.nv && n * N <= 2048;  // (so wherever n < k <= 256: all are set aside)
        if (n > 64 || few) {
            if (tid < 64) {
                const uint32_t p =
                    few ? kth_prefix(n * N, a.k, [&](int j) { return j % N < (int)s.cnt[j / N] ? key_of(j / N, j % N) : 0u; })
                        : kth_prefix(n, a.k, [&](int i) { return s.key[i]; });
                if (lane == 0) s.tau = p;
            }
            __syncthreads();
            low = s.tau << 16 > low ? s.tau << 16 : low;
        }
        each([&](uint64_t p) {
            if ((uint32_t)(p >> 32) >= low) {
                const int at = atomicAdd(&s.nn, 1);
                if (at < TK_NEAR) s.near[at] = p;
            }
        });
        __syncthreads();
        exact = s.nn > TK_NEAR;
    }
    if (exact) {
        __syncthreads();
        rest = block_maxsum(top_exact<T>(a, sp, s), c, s.ms);
    }
    const int nn = s.nn;
    T* val = static_cast<T*>(a.values) + (size_t)r * a.k;
    int64_t* idx = a.indices + (size_t)r * a.k;
    for (int i = tid; i < nn; i += nt) {
        const uint64_t p = s.near[i];
        int b = 0;
        for (int j = 0; j < nn; ++j) b += s.near[j] > p;
        if (b < a.k) {
            val[b] = (T)key_value((uint32_t)(p >> 32));
            idx[b] = (int64_t)(uint32_t)~(uint32_t)p;
        }
        if (b == a.k - 1) s.sum[0] = p;
    }
    __syncthreads();
    if (!exact) {
        // what is below the k-th joins the rest.  The vectors' order is the atomics', so their
        // exponentials are added as integers, 2^-40 of the largest
        const uint64_t edge = s.sum[0];
        float em = NEG_INF;
        int bad = 0;
        each([&](uint64_t p) {
            if (p < edge) {
                const float v = key_value((uint32_t)(p >> 32));
                em = fmaxf(em, v);
                bad |= v != v;
            }
        });
        bad = __syncthreads_or(bad);
        const MaxSum e = block_maxsum(MaxSum{em, 0.f}, c, s.ms);
        uint64_t add = 0;
        if (e.m != NEG_INF && e.m != __builtin_inff())
            each([&](uint64_t p) {
                if (p < edge)
                    add += (uint64_t)((double)exp2_raw((key_value((uint32_t)(p >> 32)) - e.m) * c) * 0x1p40 + 0.5);
            });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) add += __shfl_xor((unsigned long long)add, o, 64);
        if (lane == 0) s.sum[tid / 64] = add;
        __syncthreads();
        add = 0;
        for (int i = 0; i < nt / 64; ++i) add += s.sum[i];
        rest.merge(e.m, e.m == __builtin_inff() ? 1.f : (float)((double)add * 0x1p-40), c);
        if (bad) rest.s = __builtin_nanf("");
    }
    if (tid == 0) a.rest[r] = rest_logit(rest, a.T);
}

// at most 64 classes: a wave a row, a class a lane, ranked by counting
template <typename T> __global__ void __launch_bounds__(256) top_wave_kernel(TopArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (r >= a.rows) return;
    const float v = lane < a.V ? (float)static_cast<const T*>(a.logits)[r * a.stride + lane] : NEG_INF;
    const uint32_t key = lane < a.V ? order_key(v) : 0u;
    int rank = 0;
    for (int j = 0; j < a.V; ++j) {
        const uint32_t kj = __builtin_amdgcn_readlane(key, j);
        rank += kj > key || (kj == key && j < lane);
    }
    const bool kept = lane < a.V && rank < a.k;
    RunSum acc;
    if (!kept && lane < a.V) acc.add1(v, a.c);
    MaxSum rest = acc.done(a.c);
    rest.wave(a.c);
    if (kept) {
        static_cast<T*>(a.values)[(size_t)r * a.k + rank] = (T)key_value(key);
        a.indices[(size_t)r * a.k + rank] = lane;
    }
    if (lane == 0) a.rest[r] = rest_logit(rest, a.T);
}

// At most 64 * R classes: a wave a row, R classes a lane in registers.  The k-th key is found two
// bits a step by counting with ballots, until exactly k keys reach the prefix; the entries go
// to LDS by their index and are ranked there.  No barrier and no second reading: a block a row
// took 233 us for 7804 x 539 bf16, k = 104, this 50; 8192 x 512, k = 50: 26.
template <typename T, int R> __global__ void __launch_bounds__(256) top_wide_wave_kernel(TopArgs a) {
    __shared__ uint32_t skey[4][DK_MAX + 4];
    __shared__ int sidx[4][DK_MAX];
    const int lane = threadIdx.x & 63, w = threadIdx.x / 64;
    const int64_t r = (int64_t)blockIdx.x * 4 + w;
    if (r >= a.rows) return;
    const T* z = static_cast<const T*>(a.logits) + r * a.stride;
    uint32_t key[R];
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = lane + 64 * i < a.V ? order_key((float)z[lane + 64 * i]) : 0u;
    uint32_t t = 0;
    int reach = 64 * R;  // keys that reach t
    for (int b = 30; b >= 0 && reach != a.k; b -= 2) {
        const uint32_t u1 = t | 1u << b, u2 = t | 2u << b, u3 = t | 3u << b;
        int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            c1 += __popcll(__ballot(key[i] >= u1));
            c2 += __popcll(__ballot(key[i] >= u2));
            c3 += __popcll(__ballot(key[i] >= u3));
        }
        t = c3 >= a.k ? u3 : c2 >= a.k ? u2 : c1 >= a.k ? u1 : t;
        reach = c3 >= a.k ? c3 : c2 >= a.k ? c2 : c1 >= a.k ? c1 : reach;
    }
    // more than k: t is the k-th key itself, and of those equal to it the first belong to the record
    const bool all = reach == a.k;
    int spare = a.k, base = 0;
    if (!all) {
#pragma unroll
        for (int i = 0; i < R; ++i) spare -= __popcll(__ballot(key[i] > t));
    }
    const uint64_t below = (1ull << lane) - 1;
    RunSum acc;
    float y[R < 8 ? R : 8], mx = NEG_INF;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int x = lane + 64 * i;
        bool take = x < a.V && key[i] >= t;
        if (!all) {
            const uint64_t eq = __ballot(take && key[i] == t);
            take = take && (key[i] > t || __popcll(eq & below) < spare);
            spare -= __popcll(eq) < spare ? __popcll(eq) : spare;
        }
        const uint64_t m = __ballot(take);
        if (take) {
            const int at = base + __popcll(m & below);
            skey[w][at] = key[i];
            sidx[w][at] = x;
        }
        base += __popcll(m);
        y[i % 8] = take || x >= a.V ? NEG_INF : key_value(key[i]);
        mx = fmaxf(mx, y[i % 8]);
        if (i % 8 == 7 || i == R - 1) {
            acc.add(y, R < 8 ? R : 8, mx, a.c);
            mx = NEG_INF;
        }
    }
    if (lane < 4) skey[w][a.k + lane] = 0;  // (the ranking reads four at a time)
    MaxSum rest = acc.done(a.c);
    rest.wave(a.c);
    wave_sync();
    T* val = static_cast<T*>(a.values) + (size_t)r * a.k;
    int64_t* idx = a.indices + (size_t)r * a.k;
    for (int j = lane; j < a.k; j += 64) {
        const uint32_t kj = skey[w][j];
        int rank = 0;
        for (int l = 0; l < a.k; l += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t kl = skey[w][l + e];
                rank += kl > kj || (kl == kj && l + e < j);
            }
        val[rank] = (T)key_value(kj);
        idx[rank] = sidx[w][j];
    }
    if (lane == 0) a.rest[r] = rest_logit(rest, a.T);
}

// Signed keys in order_key's order, and back; a place not taken is -inf.
constexpr int MAP_NINF = (int)0x807fffffu, MAP_EMPTY = MAP_NINF - 1, MAP_TOP = 0x7fffffff;
__device__ __forceinline__ int map_key(float v) {
    const int b = __float_as_int(v + 0.f);  // (-0 is 0)
    return v != v ? MAP_TOP : b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float map_value(int k) {
    k = k > MAP_NINF ? k : MAP_NINF;
    return __int_as_float(k ^ (k >> 31 & 0x7fffffff));
}
// KR places in order; a class that enters pushes the last one out.  Classes come by their
// index, so one that equals a place stays behind it.
template <int KR> struct MapTop {
    int key[KR], id[KR];
    // `used` places, the last ones
    __device__ __forceinline__ void clear(int used) {
#pragma unroll
        for (int e = 0; e < KR; ++e) {
            key[e] = e < KR - used ? MAP_TOP : MAP_EMPTY;
            id[e] = -1;
        }
    }
    // x: the key that is left over
    __device__ __forceinline__ void put(int& x, int i) {
        const int over = x < key[KR - 1] ? x : key[KR - 1];
#pragma unroll
        for (int e = KR - 1; e > 0; --e) {
            const bool here = x > key[e], before = x > key[e - 1];
            id[e] = before ? id[e - 1] : here ? i : id[e];
            const int up = x > key[e] ? x : key[e];
            key[e] = up < key[e - 1] ? up : key[e - 1];
        }
        id[0] = x > key[0] ? i : id[0];
        key[0] = x > key[0] ? x : key[0];
        x = over;
    }
};

// Class maps: a thread a pixel, or S threads of different waves a pixel, each a part of the
// classes, whose lists are joined.  One reading gives KR entries and the sums of what is
// pushed out; more than KR take a reading for each KR.  A round of "the next in order"
// for every entry took 62 us where 4 maps of 32 x 256^2 keep 8 classes, this
// 21; 2 maps of 64 classes 166 against 30, one of 1000 at 128^2 with 5 entries 2012 against 70.
template <typename T, int KR, int S> __global__ void __launch_bounds__(256) top_map_kernel(TopArgs a) {
    constexpr int PX = 256 / S;
    __shared__ int sk[S > 1 ? 256 * KR : 1], si[S > 1 ? 256 * KR : 1];
    __shared__ float sm[S > 1 ? 256 : 1], ss[S > 1 ? 256 : 1];
    const int tid = threadIdx.x, px = tid % PX, sl = tid / PX;
    const int64_t at = (int64_t)blockIdx.x * PX + px;
    const bool on = at < a.rows;
    const int64_t r = on ? at : a.rows - 1;  // (a thread beyond the last pixel reads that one)
    const int64_t n = r / a.inner, p = r % a.inner;
    const T* z = static_cast<const T*>(a.logits) + (size_t)n * a.V * a.inner + p;
    const int per = (a.V + S - 1) / S, v0 = sl * per < a.V ? sl * per : a.V, v1 = v0 + per < a.V ? v0 + per : a.V;
    int lastk = MAP_TOP, lasti = -1;
    for (int j0 = 0;; j0 += KR) {
        const int used = a.k - j0 < KR ? a.k - j0 : KR;
        const bool fin = j0 + KR >= a.k;
        MapTop<KR> top;
        top.clear(used);
        RunSum acc;
        for (int i0 = v0; i0 < v1; i0 += 8) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (float)z[(size_t)(i0 + e < v1 ? i0 + e : v1 - 1) * a.inner];
            int x[8], mx = MAP_EMPTY;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = i0 + e < v1 ? map_key(y[e]) : MAP_EMPTY;
                if (j0 > 0 && !(x[e] < lastk || (x[e] == lastk && i0 + e > lasti))) x[e] = MAP_EMPTY;
                mx = mx > x[e] ? mx : x[e];
            }
            if (mx > top.key[KR - 1]) {
#pragma unroll
                for (int e = 0; e < 8; ++e) top.put(x[e], i0 + e);
            }
            if (fin) {
                float m = NEG_INF;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[e] = map_value(x[e]);
                    m = fmaxf(m, y[e]);
                }
                acc.add(y, 8, m, a.c);
            }
        }
        if constexpr (S > 1) {
            __syncthreads();  // (the last round's entries have been read)
            if (sl > 0) {
                const MaxSum o = acc.done(a.c);
                sm[tid] = o.m;
                ss[tid] = o.s;
#pragma unroll
                for (int e = 0; e < KR; ++e) {
                    sk[e * 256 + tid] = top.key[e];
                    si[e * 256 + tid] = top.id[e];
                }
            }
            __syncthreads();
            if (sl == 0)
                for (int q = px + PX; q < 256; q += PX)
#pragma unroll
                    for (int e = 0; e < KR; ++e)
                        if (e >= KR - used) {
                            int x = sk[e * 256 + q];
                            top.put(x, si[e * 256 + q]);
                            if (fin) acc.add1(map_value(x), a.c);
                        }
        }
        if (sl == 0 && on) {
            T* val = static_cast<T*>(a.values) + (size_t)n * a.k * a.inner + p;
            int64_t* idx = a.indices + (size_t)n * a.k * a.inner + p;
#pragma unroll
            for (int e = 0; e < KR; ++e)
                if (e >= KR - used) {
                    const size_t j = (size_t)(j0 + e - (KR - used)) * a.inner;
                    val[j] = (T)map_value(top.key[e]);
                    idx[j] = top.id[e];
                }
        }
        if (fin) {
            if (sl == 0) {
                MaxSum rest = acc.done(a.c);
                if constexpr (S > 1)
                    for (int q = px + PX; q < 256; q += PX) rest.merge(sm[q], ss[q], a.c);
                if (on) a.rest[r] = rest_logit(rest, a.T);
            }
            break;
        }
        lastk = top.key[KR - 1];
        lasti = top.id[KR - 1];
        if constexpr (S > 1) {
            if (sl == 0) {
                sk[px] = lastk;  // (places 0 .. PX - 1 hold no list)
                si[px] = lasti;
            }
            __syncthreads();
            lastk = sk[px];
            lasti = si[px];
        }
    }
}

// ---------------------------------------------------------------- host side
// shared by both operators: N rows of V (inner == 1, row stride >= V) or N maps of V x inner
static int rows_check(const char* what, const void* logits, int dtype, int64_t N, int V, int64_t inner,
                      int64_t stride, int k, double T) {
    if (!logits || (dtype != UGPG_DT_F32 && dtype != UGPG_DT_BF16) || N <= 0 || V <= 0 || inner <= 0 ||
        k < 1 || k > V || !(T >= 9e-31) || !(T <= 1.1e30)) {
        set_error("%s: bad arguments (dtype=%d N=%lld V=%d inner=%lld k=%d T=%g)", what, dtype,
                  (long long)N, V, (long long)inner, k, T);
        return UGPG_ERR_INVALID;
    }
    if (k > DK_MAX) {
        set_error("%s: k=%d entries, at most %d", what, k, DK_MAX);
        return UGPG_ERR_INVALID;
    }
    if (inner == 1 ? stride < V && N > 1 : stride != (int64_t)V * inner) {
        set_error("%s: row stride %lld does not fit V=%d inner=%lld", what, (long long)stride, V,
                  (long long)inner);
        return UGPG_ERR_INVALID;
    }
    // (grids below 2^32 threads, up to four a pixel in blocks of 64 pixels; V leaves room for a
    // span's padding in 32 bits)
    if (V > (1 << 30) || (inner == 1 ? N > (1 << 22) : N > (int64_t)((1 << 30) - 64) / inner)) {
        set_error("%s: N=%lld V=%d inner=%lld is too large", what, (long long)N, V, (long long)inner);
        return UGPG_ERR_INVALID;
    }
    if ((uintptr_t)logits % (dtype == UGPG_DT_F32 ? 4 : 2)) {
        set_error("%s: logits are not aligned to their type", what);
        return UGPG_ERR_INVALID;
    }
    return UGPG_OK;
}

// A row's blocks: one where the rows alone fill the card (256 CUs) and its bitmap fits
// (2^18 classes, 32 KB), else enough that about 512 run, of at least 4096 classes each.
struct Split {
    int n, chunk;
};
static Split row_split(int64_t rows, int V) {
    int64_t n = rows >= 256 ? 1 : cdiv(512, rows);
    const int64_t most = V / 4096 > 1 ? V / 4096 : 1, least = cdiv(V, 1 << 18);
    if (n > most) n = most;
    if (n < least) n = least;
    Split s;
    s.chunk = (int)(cdiv(cdiv(V, n), 64) * 64);
    s.n = (int)cdiv(V, s.chunk);
    return s;
}

}  // namespace ugpg

using namespace ugpg;

constexpr int TOPW_MAX = 1024;  // classes of a row that one wave holds

extern "C" int ugpg_top_logits(const void* logits, int dtype, int64_t N, int V, int64_t inner,
                               int64_t stride, int k, float temperature, void* values,
                               int64_t* indices, float* rest, void* stream) {
    if (int rc = rows_check("top_logits", logits, dtype, N, V, inner, stride, k, temperature)) return rc;
    if (!values || !indices || !rest) {
        set_error("top_logits: values, indices and rest must be given");
        return UGPG_ERR_INVALID;
    }
    TopArgs a{logits, N * inner, inner, stride, V, k, temperature, (float)(LOG2E / temperature), 4, values, indices, rest};
    // few rows wait for their own steps, not for memory: a bound from the whole row, read twice,
    // saves two of them (64 x 131072 bf16, k = 128: 28 us against 36; 512 rows: 55 against 49)
    if (N <= 128) a.first = 1;
    hipStream_t s = as_stream(stream);
    const bool f32 = dtype == UGPG_DT_F32;
#define TOP_GO(KF, KH, grid, nt)                                              \
    do {                                                                      \
        if (f32) hipLaunchKernelGGL(KF, dim3((unsigned)(grid)), dim3(nt), 0, s, a); \
        else hipLaunchKernelGGL(KH, dim3((unsigned)(grid)), dim3(nt), 0, s, a);     \
    } while (0)
    if (inner > 1) {
        // the classes of a pixel in four parts where there are many, or few pixels
        const bool four = V > 32 || (V > 16 && a.rows < (1 << 17));
        const int64_t g = cdiv(a.rows, four ? 64 : 256);
#define TOP_MAP(KR)                                                                                       \
    do {                                                                                                  \
        if (four) TOP_GO((top_map_kernel<float, KR, 4>), (top_map_kernel<__bf16, KR, 4>), g, 256);        \
        else TOP_GO((top_map_kernel<float, KR, 1>), (top_map_kernel<__bf16, KR, 1>), g, 256);             \
    } while (0)
        if (k <= 2) TOP_MAP(2);
        else if (k <= 4) TOP_MAP(4);
        else TOP_MAP(8);
#undef TOP_MAP
    } else if (V <= 64) {
        TOP_GO((top_wave_kernel<float>), (top_wave_kernel<__bf16>), cdiv(N, 4), 256);
    } else if (V <= 256) {
        TOP_GO((top_wide_wave_kernel<float, 4>), (top_wide_wave_kernel<__bf16, 4>), cdiv(N, 4), 256);
    } else if (V <= 512) {
        TOP_GO((top_wide_wave_kernel<float, 8>), (top_wide_wave_kernel<__bf16, 8>), cdiv(N, 4), 256);
    } else if (V <= TOPW_MAX) {
        TOP_GO((top_wide_wave_kernel<float, 16>), (top_wide_wave_kernel<__bf16, 16>), cdiv(N, 4), 256);
    } else {
        // twice as many maxima as entries keep the first bound near the k-th; about 3.2 k vectors
        // are set aside
        if (k <= 64 && V <= 4096) TOP_GO((top_row_kernel<float, 128, 256>), (top_row_kernel<__bf16, 128, 256>), N, 128);
        else if (k <= 128 && V <= 16384) TOP_GO((top_row_kernel<float, 256, 512>), (top_row_kernel<__bf16, 256, 512>), N, 256);
        else TOP_GO((top_row_kernel<float, 512, 1024>), (top_row_kernel<__bf16, 512, 1024>), N, 512);
    }
#undef TOP_GO
    return check_launch("top_logits");
}

// pixels of a block: a thread a pixel, or four
static int map_pixels(int V) { return V <= 32 ? 256 : 64; }

// blocks of four waves for short rows: up to 16 rounds of the card's 2048
static int64_t wave_blocks(int64_t rows) {
    const int64_t n = cdiv(rows, 4);
    return n < 32768 ? n : 32768;
}

static int distill_check(const char* what, const ugpg_distill_t* p) {
    if (!p) {
        set_error("%s: no descriptor", what);
        return UGPG_ERR_INVALID;
    }
    if (int rc = rows_check(what, p->logits, p->dtype, p->N, p->V, p->inner, p->stride, p->k, p->temperature))
        return rc;
    if (!p->values || !p->indices || (p->values_dtype != UGPG_DT_F32 && p->values_dtype != UGPG_DT_BF16) ||
        (p->index_bits != 32 && p->index_bits != 64) || !(p->scale == p->scale)) {
        set_error("%s: bad record (values type %d, %d-bit indices) or scale %g", what, p->values_dtype,
                  p->index_bits, p->scale);
        return UGPG_ERR_INVALID;
    }
    if (p->inner == 1 && p->V > DW_MAX && (double)p->N * row_split(p->N, p->V).n * 512 > 4e9) {
        set_error("%s: N=%lld V=%d is too large", what, (long long)p->N, p->V);
        return UGPG_ERR_INVALID;
    }
    if (p->inner > 1 && p->V > DM_MAX) {
        set_error("%s: class maps of %d classes, at most %d", what, p->V, DM_MAX);
        return UGPG_ERR_INVALID;
    }
    return UGPG_OK;
}

extern "C" size_t ugpg_distill_workspace(const ugpg_distill_t* p, int backward) {
    if (distill_check("distill_workspace", p)) return 0;
    if (p->inner > 1) return backward ? 0 : (size_t)cdiv(p->N * p->inner, map_pixels(p->V)) * 8;
    size_t n = backward ? 0 : (size_t)p->N * 8;  // the rows' losses, then the parts of split rows
    if (p->V > DW_MAX) {
        const Split sp = row_split(p->N, p->V);
        if (sp.n > 1) n += (size_t)p->N * sp.n * 8;
    }
    return n;
}

template <typename T>
static int distill_run(const ugpg_distill_t* p, DistillArgs a, float* loss, bool backward, void* ws,
                       hipStream_t s) {
    const int es = sizeof(T);
    const int64_t rows = a.rows;
    int64_t nsum = rows;
    a.row_loss = loss ? static_cast<double*>(ws) : nullptr;
    if (p->inner > 1) {
        nsum = cdiv(rows, map_pixels(a.V));
        const dim3 grid((unsigned)nsum);
        const unsigned marks = (unsigned)(cdiv(a.V, 32) * 4 * map_pixels(a.V));
        if (a.V > 32) {
            if (a.k <= 8) hipLaunchKernelGGL((distill_map_kernel<T, 8, 4>), grid, dim3(256), marks, s, a);
            else if (a.k <= 16) hipLaunchKernelGGL((distill_map_kernel<T, 16, 4>), grid, dim3(256), marks, s, a);
            else hipLaunchKernelGGL((distill_map_kernel<T, 0, 4>), grid, dim3(256), marks, s, a);
        } else if (a.k > 8) {
            if (a.k <= 16) hipLaunchKernelGGL((distill_map_kernel<T, 16, 1>), grid, dim3(256), marks, s, a);
            else hipLaunchKernelGGL((distill_map_kernel<T, 0, 1>), grid, dim3(256), marks, s, a);
        } else if (a.V <= 8 && a.k <= 4)
            hipLaunchKernelGGL((distill_map_small_kernel<T, 8, 4>), grid, dim3(256), 0, s, a);
        else if (a.V <= 16 && a.k <= 8)
            hipLaunchKernelGGL((distill_map_small_kernel<T, 16, 8>), grid, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL((distill_map_small_kernel<T, 32, 8>), grid, dim3(256), 0, s, a);
    } else if (a.V <= DW_MAX) {
        // up to 64 rows: one block of 16 waves, which also sums them
        const bool one = rows <= 64;
        const int nv = (int)cdiv(a.V, 64);
        if (!one) nsum = wave_blocks(rows);
#define DISTILL_WAVE(NV)                                                                          \
    do {                                                                                          \
        if (one)                                                                                  \
            hipLaunchKernelGGL((distill_wave_one_kernel<T, NV>), dim3(1), dim3(1024), 0, s, a, loss); \
        else                                                                                      \
            hipLaunchKernelGGL((distill_wave_kernel<T, NV>), dim3((unsigned)nsum), dim3(256), 0, s, a);   \
    } while (0)
        if (nv <= 1) DISTILL_WAVE(1);
        else if (nv <= 4) DISTILL_WAVE(4);
        else DISTILL_WAVE(8);
#undef DISTILL_WAVE
        if (one) return check_launch("distill");
    } else {
        // 16-byte stores where the gradient's rows lie as the logits' do
        const bool al = !a.dz || (((uintptr_t)a.dz ^ (uintptr_t)a.logits) % 16 == 0 &&
                                  (a.stride - a.V) * es % 16 == 0);
        const Split sp = row_split(rows, a.V);
        auto lds = [&](int span) { return (unsigned)(((span + 3 * RowVec<T>::N + 31) / 32) * 4); };
        if (sp.n == 1) {
#define DISTILL_ROW(AL, NT) \
    hipLaunchKernelGGL((distill_row_kernel<T, AL, NT>), dim3((unsigned)rows), dim3(NT), lds(a.V), s, a)
            // (4096 x 32768 bf16 with its gradient: 135 us at 512 threads, 143 at 256, 154 at 1024;
            // rows held in registers instead of read again: 173)
            if (a.V <= 8192) {
                if (al) DISTILL_ROW(true, 256);
                else DISTILL_ROW(false, 256);
            } else {
                if (al) DISTILL_ROW(true, 512);
                else DISTILL_ROW(false, 512);
            }
#undef DISTILL_ROW
        } else {
            float* part = reinterpret_cast<float*>(static_cast<double*>(ws) + (backward ? 0 : rows));
            const unsigned g = (unsigned)(rows * sp.n);
            hipLaunchKernelGGL((distill_part_kernel<T>), dim3(g), dim3(256), lds(sp.chunk), s, a, sp.n, sp.chunk, part);
            // without a gradient one block a row joins them, over no classes of its own
            const int gn = a.dz ? sp.n : 1, gc = a.dz ? sp.chunk : 0;
            const unsigned gg = (unsigned)(rows * gn);
            if (al)
                hipLaunchKernelGGL((distill_join_kernel<T, true>), dim3(gg), dim3(256), lds(gc), s, a, sp.n, sp.chunk, gn, gc, part);
            else
                hipLaunchKernelGGL((distill_join_kernel<T, false>), dim3(gg), dim3(256), lds(gc), s, a, sp.n, sp.chunk, gn, gc, part);
        }
    }
    if (loss)
        hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, s, a.row_loss, nsum, loss);
    return check_launch("distill");
}

static DistillArgs distill_args(const ugpg_distill_t* p) {
    DistillArgs a{};
    a.logits = p->logits;
    a.values = p->values;
    a.indices = p->indices;
    a.rest = p->rest;
    a.weight = p->weight;
    a.rows = p->N * p->inner;
    a.inner = p->inner;
    a.stride = p->stride;
    a.V = p->V;
    a.k = p->k;
    a.v16 = p->values_dtype == UGPG_DT_BF16;
    a.i64 = p->index_bits == 64;
    a.T = p->temperature;
    a.coef = p->scale;
    a.c = (float)(LOG2E / p->temperature);
    return a;
}

static int distill_ws_check(const char* what, const ugpg_distill_t* p, int backward, const void* ws,
                            size_t n) {
    const size_t need = ugpg_distill_workspace(p, backward);
    if (need && (!ws || n < need)) {
        set_error("%s: workspace %zu < %zu", what, n, need);
        return UGPG_ERR_WORKSPACE;
    }
    return UGPG_OK;
}

extern "C" int ugpg_distill_fwd(const ugpg_distill_t* p, float* loss, float* row_loss, void* dlogits,
                                void* ws, size_t ws_bytes, void* stream) {
    if (int rc = distill_check("distill_fwd", p)) return rc;
    if ((!loss && !row_loss) || (uintptr_t)dlogits % (p->dtype == UGPG_DT_F32 ? 4 : 2)) {
        set_error("distill_fwd: neither loss nor row_loss given, or dlogits not aligned to its type");
        return UGPG_ERR_INVALID;
    }
    if (int rc = distill_ws_check("distill_fwd", p, 0, ws, ws_bytes)) return rc;
    DistillArgs a = distill_args(p);
    a.row_out = row_loss;
    a.dz = dlogits;
    return p->dtype == UGPG_DT_F32 ? distill_run<float>(p, a, loss, false, ws, as_stream(stream))
                                   : distill_run<__bf16>(p, a, loss, false, ws, as_stream(stream));
}

extern "C" int ugpg_distill_bwd(const ugpg_distill_t* p, const float* gout, int per_row, int skip_one,
                                void* dlogits, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = distill_check("distill_bwd", p)) return rc;
    if (!gout || !dlogits || (per_row && skip_one) || (uintptr_t)dlogits % (p->dtype == UGPG_DT_F32 ? 4 : 2)) {
        set_error("distill_bwd: bad arguments (per_row=%d skip_one=%d)", per_row, skip_one);
        return UGPG_ERR_INVALID;
    }
    if (int rc = distill_ws_check("distill_bwd", p, 1, ws, ws_bytes)) return rc;
    DistillArgs a = distill_args(p);
    a.gout = gout;
    a.gout_rows = per_row != 0;
    a.skip_one = skip_one != 0;
    a.dz = dlogits;
    return p->dtype == UGPG_DT_F32 ? distill_run<float>(p, a, nullptr, true, ws, as_stream(stream))
                                   : distill_run<__bf16>(p, a, nullptr, true, ws, as_stream(stream));
}

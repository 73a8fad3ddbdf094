// Losses that train a policy on preferences or rewards, over logits [rows, vocab] (bf16 or fp32): log-probabilities of the labels, the paired
// log-ratio loss, the clipped policy loss with a KL term, and the gradients in the logits.
//
// With z = x / tau, row t and label l_t:
//   lse_t = log sum_j exp z_tj,   logp_t = z_t,l - lse_t,   d logp_t / d x_tj = (1[j = l_t] - exp(z_tj - lse_t)) / tau
// so every loss of the log-probabilities has the gradient  c_t (1[j = l_t] - p_tj) / tau  with one coefficient c_t per row.  A row whose label is
// ignore_index, or no index into the vocabulary at all, is masked: its logits are never read, its log-probability, log-sum-exp and coefficient are 0
// and its gradient is written as zeros.
//
// All kernels stream the logits and are bound by HBM; one workgroup owns one row, so no sum crosses workgroups and every result is the same from run to run.
#include "ie_common.h"

#include <math.h>

#include <algorithm>

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));   // 16 bytes at any element's address: rows of an odd vocabulary start anywhere

template <bool BF> struct Elem;
template <> struct Elem<true> {
    typedef bf16_t T;
    static constexpr int N = 8;
    static __device__ __forceinline__ u32x4 ninf() { return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}; }
    static __device__ __forceinline__ float get(const T* p) { return bf2f(*p); }
    static __device__ __forceinline__ void put(T* p, float f) { *p = f2bf(f); }
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = bflo(v[i]); f[2 * i + 1] = bfhi(v[i]); }
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pack2bf(f[2 * i], f[2 * i + 1]);
        return v;
    }
};
template <> struct Elem<false> {
    typedef float T;
    static constexpr int N = 4;
    static __device__ __forceinline__ u32x4 ninf() { return u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}; }
    static __device__ __forceinline__ float get(const T* p) { return *p; }
    static __device__ __forceinline__ void put(T* p, float f) { *p = f; }
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[i]);
        return v;
    }
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr double kLog2e = 1.44269504088896340736;
constexpr double kLn2 = 0.693147180559945309417;

// S (of loads alone: L): past the caches (non-temporal)
template <bool S> __device__ __forceinline__ u32x4 ldv(const void* p) { return S ? __builtin_nontemporal_load((const u32x4_any*)p) : *(const u32x4_any*)p; }
template <bool S> __device__ __forceinline__ void stv(void* p, const u32x4& v) {
    if (S) __builtin_nontemporal_store(v, (u32x4_any*)p);
    else *(u32x4_any*)p = v;
}

// Sums of exponentials.  With k = log2(e) / tau:  exp((x - m) / tau) = 2^(x k - r), r = fl(m k): one fma and one exponential an element, m the largest logit so far; what
// rounding m k loses, up to half its last place, is the same factor in every term and goes out again when a thread's sum joins the others'.  That holds while the factor is
// near 1: up to |m k| = 2^20 it lies within 2^(1/16) either way, at 2^33 it would be 2^512 and the sum lost.  Rows whose maximum lies beyond (logits of 7e5 at a
// temperature of 1, a vocabulary forbidden as a whole by a finite value, temperatures of 1e-5 and less, a maximum of +inf or -inf) are done over as
// 2^((x - m) k) (F = false).  NaN and +inf make the sum NaN.
// A thread whose own maximum lies below -2^21 gets the reference 0, and its terms are 0 as they should be beside a row maximum above -2^20; between the two
// bounds it is joined like any other.
constexpr float kRange = 1048576.f, kLow = -2097152.f;
__device__ __forceinline__ bool usable(float m, float k) { return m * k >= kLow; }   // (false for NaN)
__device__ __forceinline__ float ref(float m, float k) { return usable(m, k) ? m * k : 0.f; }
__device__ __forceinline__ bool in_range(float m, float k) { return fabsf(m * k) <= kRange; }
template <bool F> __device__ __forceinline__ float term(float x, float k, float r) { return exp2_(F ? __builtin_fmaf(x, k, -r) : (x - r) * k); }

// Sums of hundreds of log-probabilities show any error that all rows share.  The hardware's exponential is 3.3e-9 low on average (measured: every argument range from
// [-1, 0) to [-30, -29) the same to 1 %), which log_sum below puts right for the terms; what multiplies a whole sum uses this instead:
// 2^d for d <= 0 by the Taylor series of 2^f, off by 2e-10 for |f| <= 1/2 (by 2e-9 at 5/8, the most that what a thread's reference lost adds), and one rounding to the nearest.
constexpr double kExpLow = 3.3e-9;
__device__ __forceinline__ float exp2_near(float f, float n) {   // 2^(f + n), n whole
    float p = 1.3215486790e-6f;
#pragma unroll
    for (const float c : {1.5252733804e-5f, 1.5403530394e-4f, 1.3333558146e-3f, 9.6181291076e-3f, 5.5504108665e-2f, 2.4022650696e-1f, 6.9314718056e-1f, 1.f}) p = __builtin_fmaf(p, f, c);
    return ldexpf(p, (int)fmaxf(n, -200.f));
}

// log2(e) / tau lies between two fp32 numbers, log2(e) itself 1.3e-8 off the nearer: the same way in every term of every row, which the 500 log-probabilities of a sequence
// add up to 6e-5.  So the share of threads that its place between them says takes the upper one (a second fma an element would take the error out too: + 4 to 7 %).
struct Scale {
    double inv_tau;
    float lo, hi, rest;   // rest: log2(e) / tau - lo
    unsigned cut;         // of 2^32
    explicit Scale(double it) : inv_tau(it) {
        const double e = it * kLog2e;
        const float f = (float)e;
        lo = (double)f <= e ? f : nextafterf(f, 0.f);
        hi = nextafterf(lo, INFINITY);
        rest = (float)(e - (double)lo);
        cut = (unsigned)(4294967295.0 * ((e - (double)lo) / ((double)hi - (double)lo)));
    }
    __device__ __forceinline__ float mine() const { return threadIdx.x * 0x9e3779b1u < cut ? hi : lo; }   // (multiples of the golden ratio: evenly spread over any threads)
};

struct RowStat {
    float m, s;   // s = sum exp((x - m) / tau)
    bool fast;
    __device__ __forceinline__ double log_sum() const { return log((double)s) + kExpLow * (1.0 - 1.0 / (double)s); }   // (the largest term is 1, and exact)
    __device__ __forceinline__ double lse(double inv_tau) const { return (double)m * inv_tau + log_sum(); }
    __device__ __forceinline__ double logp(float x, double inv_tau) const { return ((double)x - (double)m) * inv_tau - log_sum(); }
};

// exp(d / tau) 2^lost: whole sums are multiplied by it, so the exponent is taken apart into a whole number and a remainder and nothing of it is rounded away
__device__ __forceinline__ float shift(float d, float lost, const Scale& sc) {
    const float n = rintf(d * sc.lo);
    if (!(n >= -160.f)) return exp2_(n);   // (0, or NaN)
    return exp2_near(__builtin_fmaf(d, sc.lo, -n) + __builtin_fmaf(d, sc.rest, lost), n);
}
// factor that brings a thread's terms 2^(x k - ref(m, k)) to exp((x - to) / tau)
__device__ __forceinline__ float to_max(float m, float k, float to, const Scale& sc) { return shift(m - to, __builtin_fmaf(-m, k, ref(m, k)), sc); }

// (m, s) of every thread, s at reference ref(m, k) -> of the workgroup; every thread returns the same.  sh: 2 NT / 64 floats.
template <int NT>
__device__ __forceinline__ RowStat join_stats(float m, float s, float k, const Scale& sc, float* sh) {
    constexpr int NW = NT / 64;
    const float wm = wave_max(m);
    s = wave_sum(s == 0.f ? 0.f : s * to_max(m, k, wm, sc));
    if (NW == 1) return {wm, s, in_range(wm, sc.lo)};
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6] = wm; sh[NW + (threadIdx.x >> 6)] = s; }
    __syncthreads();
    m = sh[threadIdx.x & (NW - 1)];
    s = sh[NW + (threadIdx.x & (NW - 1))];
    float b = m;
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) b = fmaxf(b, __shfl_xor(b, o, 64));
    s = s == 0.f ? 0.f : s * shift(m - b, 0.f, sc);
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    return {b, s, in_range(b, sc.lo)};
}

// Sum of N values (a power of two) as a tree: a term next to 1 -- the label's, in a trained model -- meets log2 N roundings, where one sum from left to right would
// round the others away one by one
template <int N>
__device__ __forceinline__ float tree_sum(const float* v) {
    float t[N];
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = v[e];
#pragma unroll
    for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
        for (int e = 0; e < w; ++e) t[e] += t[e + w];
    return t[0];
}

template <int N>
__device__ __forceinline__ void add_values(const float* v, float k, float& m, float& s) {
    float c = v[0];
#pragma unroll
    for (int e = 1; e < N; ++e) c = fmaxf(c, v[e]);
    if (c > m) {
        const float d = ref(m, k) - ref(c, k), n = rintf(d);
        s = s == 0.f ? 0.f : s * exp2_near(d - n, n);
        m = c;
    }
    const float r = ref(m, k);
    float t[N];
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = term<true>(v[e], k, r);
    s += tree_sum<N>(t);
}

__device__ __forceinline__ float max_ref(float m) { return m == -INFINITY ? 0.f : m; }

// The row whose maximum m is out of the fast form's range, again.  sh as in join_stats, free to be written after the barrier at its start.
template <bool BF, int NT>
__device__ __noinline__ RowStat row_stat_again(const typename Elem<BF>::T* x, int vocab, float m, float k, float* sh) {
    constexpr int NW = NT / 64;
    const float r = max_ref(m);
    float s = 0.f;
    for (int i = threadIdx.x; i < vocab; i += NT) s += term<false>(Elem<BF>::get(x + i), k, r);
    s = wave_sum(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.f;
    for (int w = 0; w < NW; ++w) s += sh[w];
    return {m, s, false};
}

// One pass over the row, U 16-byte loads a thread in flight.
template <bool BF, int NT, int U, bool S>
__device__ __forceinline__ RowStat row_stat(const typename Elem<BF>::T* x, int vocab, const Scale& sc, float* sh) {
    constexpr int N = Elem<BF>::N;
    const float k = sc.mine();
    float m = -INFINITY, s = 0.f;
    const int nv = vocab / N;
    int i = threadIdx.x;
    for (; i + (U - 1) * NT < nv; i += U * NT) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = ldv<S>(x + (int64_t)(i + u * NT) * N);
        float v[U * N];
#pragma unroll
        for (int u = 0; u < U; ++u) Elem<BF>::unpack(w[u], v + u * N);
        add_values<U * N>(v, k, m, s);
    }
    if (i < nv) {   // fewer than U vectors left: loaded together too, what is not there stays -inf
        u32x4 w[U - 1];
#pragma unroll
        for (int u = 0; u < U - 1; ++u) {
            w[u] = Elem<BF>::ninf();
            if (i + u * NT < nv) w[u] = ldv<S>(x + (int64_t)(i + u * NT) * N);
        }
#pragma unroll
        for (int u = 0; u < U - 1; ++u) {
            float v[N];
            Elem<BF>::unpack(w[u], v);
            add_values<N>(v, k, m, s);
        }
    }
    if ((int)threadIdx.x < vocab - nv * N) {
        const float v = Elem<BF>::get(x + nv * N + threadIdx.x);
        add_values<1>(&v, k, m, s);
    }
    const RowStat st = join_stats<NT>(m, s, k, sc, sh);
    return st.fast ? st : row_stat_again<BF, NT>(x, vocab, st.m, sc.lo, sh);
}

__device__ __forceinline__ bool row_label(const int64_t* labels, int64_t row, int64_t ignore_index, int vocab, int& lab) {
    const int64_t l = labels[row];
    lab = (int)l;
    return l != ignore_index && l >= 0 && l < vocab;
}

// The thread that writes element `lab` of a row in the loops below: its own later store puts the label's element right.
template <bool BF, int NT>
__device__ __forceinline__ bool owns(int lab, int vocab) {
    constexpr int N = Elem<BF>::N;
    const int nv = vocab / N;
    return (int)threadIdx.x == (lab < nv * N ? (lab / N) % NT : lab - nv * N);
}

template <bool BF, bool F>
__device__ __forceinline__ u32x4 grad_vector(const u32x4& w, float k, float r, float g_p) {
    float v[Elem<BF>::N];
    Elem<BF>::unpack(w, v);
#pragma unroll
    for (int e = 0; e < Elem<BF>::N; ++e) v[e] = -g_p * term<F>(v[e], k, r);
    return Elem<BF>::pack(v);
}

// d = g 1[j = label] - g_p 2^(x k - r) for the whole row: with the row's reference and sum g_p = g / s, with its log-sum-exp as reference g_p = g.  xl: the label's
// logit, read before any store (dlogits may be the logits themselves).
template <bool BF, int NT, int U, bool L, bool S, bool F>
__device__ __forceinline__ void row_grad(const typename Elem<BF>::T* x, typename Elem<BF>::T* d, int vocab, float k, float r, float g, float g_p, int lab, float xl) {
    constexpr int N = Elem<BF>::N;
    const int nv = vocab / N;
    int i = threadIdx.x;
    for (; i + (U - 1) * NT < nv; i += U * NT) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = ldv<L>(x + (int64_t)(i + u * NT) * N);
#pragma unroll
        for (int u = 0; u < U; ++u) stv<S>(d + (int64_t)(i + u * NT) * N, grad_vector<BF, F>(w[u], k, r, g_p));
    }
    if (U > 1) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U - 1; ++u)
            if (i + u * NT < nv) w[u] = ldv<L>(x + (int64_t)(i + u * NT) * N);
#pragma unroll
        for (int u = 0; u < U - 1; ++u)
            if (i + u * NT < nv) stv<S>(d + (int64_t)(i + u * NT) * N, grad_vector<BF, F>(w[u], k, r, g_p));
    }
    i = nv * N + threadIdx.x;
    if (i < vocab) Elem<BF>::put(d + i, -g_p * term<F>(Elem<BF>::get(x + i), k, r));
    if (owns<BF, NT>(lab, vocab)) Elem<BF>::put(d + lab, g - g_p * term<F>(xl, k, r));
}

// the same for a row out of the fast form's range
template <bool BF, int NT>
__device__ __noinline__ void row_grad_again(const typename Elem<BF>::T* x, typename Elem<BF>::T* d, int vocab, float k, float r, float g, float g_p, int lab, float xl) {
    row_grad<BF, NT, 1, false, false, false>(x, d, vocab, k, r, g, g_p, lab, xl);
}

// A log-sum-exp in 32 bits is off by up to half its last place, and so is every probability formed with it: 2^-18 of it below 128, 2^-14 below 2048.  Beyond
// what the gradient's type shows of that (small temperatures, logits far from zero) a row's sums are formed again.
template <bool BF> constexpr float kFar = BF ? 2048.f * 1.4426950f : 128.f * 1.4426950f;   // (in units of log 2)

template <bool BF, int NT, bool L, bool S>
__device__ __forceinline__ void row_grad_far(const typename Elem<BF>::T* x, typename Elem<BF>::T* d, int vocab, float g, int lab, const Scale& sc, float* sh) {
    const float xl = Elem<BF>::get(x + lab);
    const RowStat st = row_stat<BF, NT, 2, L>(x, vocab, sc, sh);
    __syncthreads();   // the row is read before any store may replace it
    const float k = sc.lo, g_p = g / st.s;
    if (!st.fast) { row_grad_again<BF, NT>(x, d, vocab, k, max_ref(st.m), g, g_p, lab, xl); return; }
    const float r = st.m * k;
    row_grad<BF, NT, 2, L, S, true>(x, d, vocab, k, r, g, g_p * exp2_(__builtin_fmaf(-st.m, k, r)), lab, xl);
}

template <bool BF, int NT, bool S>
__device__ __forceinline__ void row_zero(typename Elem<BF>::T* d, int vocab) {
    constexpr int N = Elem<BF>::N;
    const int nv = vocab / N;
    const u32x4 z = {0, 0, 0, 0};
    for (int i = threadIdx.x; i < nv; i += NT) stv<S>(d + (int64_t)i * N, z);
    if (nv * N + (int)threadIdx.x < vocab) Elem<BF>::put(d + nv * N + threadIdx.x, 0.f);
}

// ------------------------------------------------------------------------------------------ log-probabilities
// coef (may be null) is cleared: the loss kernels behind this one set it for the rows of their sequences only; low comes with it, what logp loses in 32 bits, for sums of
// many.
template <bool BF, int NT, bool S>
__global__ __launch_bounds__(NT) void logprob_fwd_k(const void* __restrict__ logits, int64_t ld, const int64_t* __restrict__ labels, float* __restrict__ logp,
                                                    float* __restrict__ lse, float* __restrict__ coef, float* __restrict__ low, int vocab, int64_t ignore_index, Scale sc,
                                                    int64_t row0) {
    __shared__ float sh[NT / 32];
    const int64_t row = row0 + blockIdx.x;
    int lab;
    if (!row_label(labels, row, ignore_index, vocab, lab)) {
        if (threadIdx.x == 0) {
            logp[row] = 0.f;
            lse[row] = 0.f;
            if (coef) { coef[row] = 0.f; low[row] = 0.f; }
        }
        return;
    }
    const typename Elem<BF>::T* x = (const typename Elem<BF>::T*)logits + row * ld;
    const float xl = Elem<BF>::get(x + lab);
    const RowStat st = row_stat<BF, NT, 4, S>(x, vocab, sc, sh);
    if (threadIdx.x == 0) {
        const double lp = st.logp(xl, sc.inv_tau);
        lse[row] = (float)st.lse(sc.inv_tau);
        const float l = (float)lp;
        logp[row] = l;
        if (coef) { coef[row] = 0.f; low[row] = fabsf(l) < INFINITY ? (float)(lp - (double)l) : 0.f; }   // (a label of logit -inf: nothing is lost, and inf - inf is NaN)
    }
}

// `parts` workgroups a row, one vector a thread and no loop: the chip's reads and writes then move through memory as one dense front, which HBM serves at 6.2 TB/s of
// mixed traffic where workgroups that walk a row each get 5.5.  16 384 x 92 544 bf16, 40 % masked: 775 us (a workgroup a row: 871).
// What a workgroup needs before its first vector is asked for in two rounds, the launch's arguments and then the row's numbers, each as a whole (the compiler would
// put every scalar load next to its use, six rounds one after the other): with one vector a thread the kernel waits for them longer than it works.
struct Divisor {   // n / d for any 32-bit n by one product (Granlund and Montgomery, 1994)
    unsigned d, mul, s1, s2;
    explicit Divisor(unsigned d_) : d(d_) {
        unsigned l = 0;
        while (l < 32 && (uint64_t(1) << l) < d) ++l;
        mul = (unsigned)(((uint64_t(1) << 32) * ((uint64_t(1) << l) - d)) / d + 1);
        s1 = l < 1 ? l : 1;
        s2 = l > 1 ? l - 1 : 0;
    }
    __device__ __forceinline__ unsigned of(unsigned n) const {
        const unsigned t = __umulhi(mul, n);
        return (t + ((n - t) >> s1)) >> s2;
    }
};
template <typename T> __device__ __forceinline__ T sload(const T* p, int64_t i) {   // a scalar load: p[i] is not written while the kernel runs
    return ((const __attribute__((address_space(4))) T*)p)[i];
}
struct BwdArgs {
    const void* logits;
    void* dlogits;
    int64_t ld, ldd;
    const int64_t* labels;
    const float *lse, *coef, *dloss;   // dloss: any readable number if there is none
    int64_t ignore_index;
    double log2e;                      // lse in units of the kernel's x k
    float mul, dloss_or;               // 1 / tau and the caller's factor; dloss counts if dloss_or is 0
    int vocab;
};

template <bool BF, int NT, bool L, bool S>
__global__ __launch_bounds__(NT) void logprob_bwd_k(BwdArgs a, Scale sc, Divisor parts, int64_t row0) {
    typedef typename Elem<BF>::T T;
    constexpr int N = Elem<BF>::N;
    __shared__ float sh[NT / 32];
    asm volatile("" :: "s"(a.logits), "s"(a.dlogits), "s"(a.ld), "s"(a.ldd), "s"(a.labels), "s"(a.lse), "s"(a.coef), "s"(a.dloss), "s"(a.ignore_index), "s"(a.log2e),
                 "s"(a.mul), "s"(a.dloss_or), "s"(a.vocab), "s"(row0), "s"(sc.lo));
    const int vocab = a.vocab;
    const unsigned slice = parts.of(blockIdx.x);
    const int64_t row = row0 + slice;
    const int64_t label = sload(a.labels, row);
    const float coef = sload(a.coef, row), lse = sload(a.lse, row), dloss = sload(a.dloss, 0);
    asm volatile("" :: "s"(label), "s"(coef), "s"(lse), "s"(dloss));
    const int part = (int)(blockIdx.x - slice * parts.d), nv = vocab / N, i = part * NT + threadIdx.x, lab = (int)label;
    T* d = (T*)a.dlogits + row * a.ldd;
    const T* x = (const T*)a.logits + row * a.ld;
    const bool valid = label != a.ignore_index && label >= 0 && label < vocab;
    const float g = valid ? coef * a.mul * (a.dloss_or == 0.f ? dloss : a.dloss_or) : 0.f;
    const int e = part == (int)parts.d - 1 ? nv * N + (int)threadIdx.x : vocab;   // the row's last elements, fewer than a vector
    if (!valid || g == 0.f) {
        if (i < nv) stv<S>(d + (int64_t)i * N, u32x4{0, 0, 0, 0});
        if (e < vocab) Elem<BF>::put(d + e, 0.f);
        return;
    }
    // p = 2^(x k - l), l = lse log2(e): what rounding l to 32 bits loses goes into the factor
    const float k = sc.lo;
    const double l = (double)lse * a.log2e;
    const float r = (float)l;
    if (!(fabsf(r) <= kFar<BF>)) {   // the row's sums again, by one workgroup
        if (part == 0) row_grad_far<BF, NT, L, S>(x, d, vocab, g, lab, sc, sh);
        return;
    }
    const float g_p = g * exp2_((float)((double)r - l));
    if (i < nv) {
        const u32x4 w = ldv<L>(x + (int64_t)i * N);
        float v[N];
        Elem<BF>::unpack(w, v);
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = -g_p * term<true>(v[q], k, r);
        if ((unsigned)(lab - i * N) < (unsigned)N) {
#pragma unroll
            for (int q = 0; q < N; ++q) v[q] += i * N + q == lab ? g : 0.f;
        }
        stv<S>(d + (int64_t)i * N, Elem<BF>::pack(v));
    }
    if (e < vocab) Elem<BF>::put(d + e, (e == lab ? g : 0.f) - g_p * term<true>(Elem<BF>::get(x + e), k, r));
}

// ------------------------------------------------------------------------------------------ sums over a workgroup in 64 bits, fixed order
template <int NW>
__device__ __forceinline__ double block_sum_d(double v, double* scratch) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < NW; ++i) t += scratch[i];
    return t;
}

// rows [begin, end) of sequence s, inside [0, rows) whatever the offsets say
__device__ __forceinline__ void seq_range(const int32_t* cu, int64_t s, int64_t rows, int64_t& begin, int64_t& end) {
    begin = min(max((int64_t)cu[s], (int64_t)0), rows);
    end = min(max((int64_t)cu[s + 1], begin), rows);
}

// ------------------------------------------------------------------------------------------ preference loss
struct PrefArgs {
    int kind, average;
    double beta, smoothing, margin;
};

// log(sigmoid(z)) without overflow
__device__ __forceinline__ double log_sigmoid(double z) { return (z < 0.0 ? z : 0.0) - log1p(exp(-fabs(z))); }

// loss of one pair at the log-ratio h, and its slope
__device__ __forceinline__ double pair_loss(const PrefArgs& a, double h, double& slope) {
    const double z = a.beta * h - a.margin;
    if (a.kind == IE_PREF_SIGMOID) {
        slope = a.beta * (a.smoothing / (1.0 + exp(-z)) - (1.0 - a.smoothing) / (1.0 + exp(z)));
        const double right = -(1.0 - a.smoothing) * log_sigmoid(z);
        return a.smoothing > 0.0 ? right - a.smoothing * log_sigmoid(-z) : right;   // (0 * inf would turn a pair that is infinitely right into NaN)
    }
    if (a.kind == IE_PREF_HINGE) {
        slope = z < 1.0 ? -a.beta : z == z ? 0.0 : z;
        return z == z ? fmax(0.0, 1.0 - z) : z;
    }
    const double q = h - 0.5 / a.beta;
    slope = 2.0 * q;
    return q * q;
}

struct PrefRows {
    const float *logp, *low;   // log-probability = logp + low
    const int64_t* labels;
    const int32_t* cu;
    const float* ref;
    int64_t rows, pairs, ignore_index;
    int vocab;
    float *rewards, *seq_logps, *coef;
};

__device__ __forceinline__ bool pref_label(const PrefRows& p, int64_t t) {
    int lab;
    return row_label(p.labels, t, p.ignore_index, p.vocab, lab);
}

// Sequence s by G waves, of which this is number `sub`: the wave's share of its rows' log-probabilities, summed in 64 bits (masked rows hold 0), and of their number.
template <int G>
__device__ __forceinline__ void pref_sums(const PrefRows& r, int64_t s, int sub, double& sum, double& cnt) {
    int64_t begin, end;
    seq_range(r.cu, s, r.rows, begin, end);
    double l = 0.0;
    int n = 0;
#pragma unroll 4
    for (int64_t t = begin + sub * 64 + (threadIdx.x & 63); t < end; t += G * 64) {
        l += (double)r.logp[t] + (double)r.low[t];
        n += pref_label(r, t) ? 1 : 0;
    }
    sum = wave_sum_d(l);
    cnt = wave_sum_d((double)n);
}

// the pair that sequence s belongs to, from its two sums and counts: its loss and d loss / d logp of a row of s
__device__ __forceinline__ double pref_pair(const PrefRows& r, const PrefArgs& a, int64_t s, double l[2], double n[2], bool write, float& w) {
    double gain[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int64_t q = (s & ~(int64_t)1) + c;
        n[c] = fmax(n[c], 1.0);
        if (a.average) l[c] /= n[c];
        gain[c] = l[c] - (r.ref ? (double)r.ref[q] : 0.0);
        if (write && q == s) {
            r.seq_logps[s] = (float)l[c];
            r.rewards[s] = (float)(a.beta * gain[c]);
        }
    }
    double slope;
    const double loss = pair_loss(a, gain[0] - gain[1], slope);
    w = (float)((s & 1 ? -slope : slope) / ((double)r.pairs * (a.average ? n[s & 1] : 1.0)));
    return loss;
}

template <int G>
__device__ __forceinline__ void pref_coef(const PrefRows& r, int64_t s, int sub, float w) {
    int64_t begin, end;
    seq_range(r.cu, s, r.rows, begin, end);
#pragma unroll 4
    for (int64_t t = begin + sub * 64 + (threadIdx.x & 63); t < end; t += G * 64)
        if (pref_label(r, t)) r.coef[t] = w;
}

// Up to 16 / G sequences, G waves each, in one workgroup: MANY false: the whole batch and its mean loss; true: one pair a workgroup (G = 8), its loss for the mean.
constexpr int kOnePairs = 8;          // one workgroup finishes a batch of up to this many pairs ...
constexpr int64_t kOneRows = 32768;   // ... of up to this many rows in all: 16 384 rows, 8 pairs: 14 us, a workgroup a pair and the mean apart 17

template <int G, bool MANY>
__global__ __launch_bounds__(1024) void preference_pairs_k(PrefRows r, PrefArgs a, float* __restrict__ loss, double* __restrict__ losses) {
    __shared__ double sum[16], cnt[16], each[kOnePairs];
    const int w = threadIdx.x >> 6, sub = w % G, first = w / G * G, other = (w / G ^ 1) * G;
    const int64_t s = (MANY ? 2 * (int64_t)blockIdx.x : 0) + w / G;
    const bool on = s < 2 * r.pairs;
    if (on) {
        double l, n;
        pref_sums<G>(r, s, sub, l, n);
        if ((threadIdx.x & 63) == 0) { sum[w] = l; cnt[w] = n; }
    }
    __syncthreads();
    if (on) {
        double l[2] = {0.0, 0.0}, n[2] = {0.0, 0.0};
        const int c0 = s & 1 ? other : first, c1 = s & 1 ? first : other;
        for (int i = 0; i < G; ++i) { l[0] += sum[c0 + i]; n[0] += cnt[c0 + i]; l[1] += sum[c1 + i]; n[1] += cnt[c1 + i]; }
        float c;
        const double v = pref_pair(r, a, s, l, n, sub == 0 && (threadIdx.x & 63) == 0, c);
        if (!(s & 1) && sub == 0 && (threadIdx.x & 63) == 0) {
            if (MANY) losses[blockIdx.x] = v;
            else each[s >> 1] = v;
        }
        pref_coef<G>(r, s, sub, c);
    }
    if (MANY) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        double v = 0.0;
        for (int i = 0; i < (int)r.pairs; ++i) v += each[i];
        loss[0] = (float)(v / (double)r.pairs);
    }
}

__global__ __launch_bounds__(256) void preference_mean_k(const double* __restrict__ losses, int64_t pairs, float* __restrict__ loss) {
    __shared__ double scratch[4];
    double v = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < pairs; i += 256) v += losses[i];
    v = block_sum_d<4>(v, scratch);
    if (threadIdx.x == 0) loss[0] = (float)(v / (double)pairs);
}

// ------------------------------------------------------------------------------------------ policy loss
constexpr int kCountRows = 4;      // labels a thread looks at where a row's own workgroup counts
constexpr int kSmallRows = 4096;
constexpr int kSmallSeqs = 1024;   // one workgroup finishes a forward pass of up to kSmallRows rows in up to this many sequences

struct PolicyArgs {
    const int64_t* labels;
    const int32_t* cu;      // null: one mean over all tokens
    const float *old_logps, *adv, *ref;   // ref null: no KL term
    const int32_t* counts;  // tokens of every sequence, or of the whole batch; null: the rows' own workgroups count
    float4* terms;          // [rows]: weighted surrogate, KL, clipped
    float* coef;
    int64_t rows, seqs, ignore_index;
    int vocab;
    float low, high, kl_coef;
};

// tokens with a label, per sequence (cu) or in all (cu null, one workgroup)
template <int NT>
__global__ __launch_bounds__(NT) void policy_counts_k(PolicyArgs a, int32_t* __restrict__ counts) {
    __shared__ double scratch[NT / 64];
    int64_t begin = 0, end = a.rows;
    if (a.cu) seq_range(a.cu, blockIdx.x, a.rows, begin, end);
    int n = 0;
#pragma unroll 8
    for (int64_t t = begin + threadIdx.x; t < end; t += NT) {
        int lab;
        n += row_label(a.labels, t, a.ignore_index, a.vocab, lab) ? 1 : 0;
    }
    const double total = block_sum_d<NT / 64>((double)n, scratch);
    if (threadIdx.x == 0) counts[blockIdx.x] = (int32_t)total;
}

// Rows [begin, end) that row t's mean runs over, s their sequence; false outside every sequence.  Called by whole waves with one t.
__device__ __forceinline__ bool policy_range(const PolicyArgs& a, int64_t t, int64_t& s, int64_t& begin, int64_t& end) {
    s = 0; begin = 0; end = a.rows;
    if (!a.cu) return true;
    int64_t left = a.seqs;   // how many of cu[1..S] are <= t: halved down to a wave's width, then one look
    while (left > 64) {
        const int64_t half = left >> 1;
        if ((int64_t)a.cu[s + half] <= t) { s += half; left -= half; } else left = half;
    }
    const int64_t lane = threadIdx.x & 63;
    s += __popcll(__ballot(lane < left && (int64_t)a.cu[s + min(lane, left - 1) + 1] <= t));
    if (s >= a.seqs) return false;
    seq_range(a.cu, s, a.rows, begin, end);
    return t >= begin && t < end;
}

// weight of a row's term: 1 / N, or 1 / (S n_s); 0 outside every sequence
__device__ __forceinline__ float policy_weight(const PolicyArgs& a, bool inside, int n) {
    return inside ? (float)(1.0 / ((a.cu ? (double)a.seqs : 1.0) * (double)max(n, 1))) : 0.f;
}

struct PolicyRow {
    float old, adv, ref;
};
__device__ __forceinline__ PolicyRow policy_row(const PolicyArgs& a, int64_t t) { return {a.old_logps[t], a.adv[t], a.ref ? a.ref[t] : 0.f}; }

// terms of one row and d loss / d logp; the log-ratios are differences of 64-bit values, so that they alone are rounded
__device__ __forceinline__ float policy_term(const PolicyArgs& a, const PolicyRow& in, double logp, float w, float4& term) {
    term = make_float4(0.f, 0.f, 0.f, 0.f);
    if (w == 0.f) return 0.f;
    const float ratio = expf((float)(logp - (double)in.old));
    const bool clipped = (in.adv > 0.f && ratio > 1.f + a.high) || (in.adv < 0.f && ratio < 1.f - a.low);
    const float bound = in.adv > 0.f ? 1.f + a.high : 1.f - a.low;
    const float gain = ratio == INFINITY && in.adv == 0.f ? 0.f : ratio * in.adv;   // (a ratio past fp32 without an advantage adds nothing)
    const float s = -(clipped ? bound * in.adv : gain);
    float d = clipped ? 0.f : -gain, kl = 0.f;
    if (a.ref) {
        const float q = (float)((double)in.ref - logp), e = expm1f(q);
        kl = e == INFINITY ? e : e - q;   // (a label of logit -inf: q is inf too, and inf - inf is NaN)
        if (a.kl_coef > 0.f) d -= a.kl_coef * e;   // (0 * inf would turn a mere report into NaN)
    }
    term = make_float4(w * s, w * kl, clipped ? w : 0.f, 0.f);
    return w * d;
}

// one wave per row: terms and coefficients from finished log-probabilities
__global__ __launch_bounds__(256) void policy_terms_k(PolicyArgs a, const float* __restrict__ logp) {
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.rows) return;
    int lab;
    const bool valid = row_label(a.labels, t, a.ignore_index, a.vocab, lab);
    int64_t s = 0, begin, end;
    const bool inside = valid && policy_range(a, t, s, begin, end);
    if ((threadIdx.x & 63) == 0) a.coef[t] = policy_term(a, policy_row(a, t), (double)logp[t], policy_weight(a, inside, inside ? a.counts[s] : 0), a.terms[t]);
}

// sums of the three terms over a workgroup of 1024 threads (scratch: 48 doubles) -> loss, surrogate, KL, clipped share
__device__ __forceinline__ void write_stats(double* v, float kl_coef, float* stats, double* scratch) {
    __syncthreads();   // (scratch may hold an earlier sum that other waves still read)
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        v[c] = wave_sum_d(v[c]);
        if ((threadIdx.x & 63) == 0) scratch[c * 16 + (threadIdx.x >> 6)] = v[c];
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        v[c] = 0.0;
        for (int w = 0; w < 16; ++w) v[c] += scratch[c * 16 + w];
    }
    stats[0] = (float)(kl_coef > 0.f ? v[0] + (double)kl_coef * v[1] : v[0]);
    stats[1] = (float)v[0];
    stats[2] = (float)v[1];
    stats[3] = (float)v[2];
}

// Counts, terms, coefficients and sums of a short batch in one workgroup: a launch less for each, which is all such a call costs.
__global__ __launch_bounds__(1024) void policy_small_k(PolicyArgs a, const float* __restrict__ logp, float* __restrict__ stats) {
    __shared__ int cnt[kSmallSeqs], cu[kSmallSeqs + 1];
    __shared__ double scratch[48];
    constexpr int R = kSmallRows / 1024;
    int seq[R];   // sequence of each of the thread's rows, -1: no label or outside
    if (a.cu) {
        for (int i = threadIdx.x; i <= a.seqs; i += 1024) {
            cu[i] = a.cu[i];
            if (i < a.seqs) cnt[i] = 0;
        }
        __syncthreads();
    }
    int n = 0;
#pragma unroll
    for (int q = 0; q < R; ++q) {
        const int64_t t = (int64_t)q * 1024 + threadIdx.x;
        int lab;
        seq[q] = t < a.rows && row_label(a.labels, t, a.ignore_index, a.vocab, lab) ? 0 : -1;
        if (a.cu && seq[q] == 0) {
            int lo = 0, hi = (int)a.seqs;   // how many of cu[1..S] are <= t
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if ((int64_t)cu[mid + 1] <= t) lo = mid + 1; else hi = mid;
            }
            int64_t begin = 0, end = 0;
            if (lo < (int)a.seqs) seq_range(cu, lo, a.rows, begin, end);
            seq[q] = t >= begin && t < end ? lo : -1;
            if (seq[q] >= 0) atomicAdd(&cnt[lo], 1);   // (whole numbers: the order does not matter)
        }
        n += seq[q] == 0;
    }
    if (a.cu) __syncthreads();
    else n = (int)block_sum_d<16>((double)n, scratch);
    double v[3] = {0.0, 0.0, 0.0};
#pragma unroll
    for (int q = 0; q < R; ++q) {
        const int64_t t = (int64_t)q * 1024 + threadIdx.x;
        if (t >= a.rows) continue;
        float4 term = make_float4(0.f, 0.f, 0.f, 0.f);
        a.coef[t] = seq[q] < 0 ? 0.f : policy_term(a, policy_row(a, t), (double)logp[t], policy_weight(a, true, a.cu ? cnt[seq[q]] : n), term);
        v[0] += (double)term.x; v[1] += (double)term.y; v[2] += (double)term.z;
    }
    write_stats(v, a.kl_coef, stats, scratch);
}

// Forward and backward of one row: its coefficient needs nothing but the row itself, so the logits are read once.  NV vectors a thread wait in
// registers, as exponentials in 32 bits; what a longer row has beyond them (REST) is read again, from the caches.
template <bool BF, int NT, int NV, bool REST, bool S>
__global__ __launch_bounds__(NT, NT >= 512 ? 4 : 1) void policy_fused_k(PolicyArgs a, const void* logits, int64_t ld, void* dlogits, int64_t ldd, float* __restrict__ logp_out,
                                                     float* __restrict__ lse_out, const float* __restrict__ dloss, float dloss_mul, Scale sc, int64_t row0) {
    typedef typename Elem<BF>::T T;
    constexpr int N = Elem<BF>::N;
    __shared__ float sh[NT / 32];
    __shared__ int counted[NT / 64];
    __shared__ float coef_sh;
    const int64_t row = row0 + blockIdx.x;
    const int vocab = a.vocab;
    T* d = (T*)dlogits + row * ldd;
    int lab;
    if (!row_label(a.labels, row, a.ignore_index, vocab, lab)) {
        if (threadIdx.x == 0) { logp_out[row] = 0.f; lse_out[row] = 0.f; a.coef[row] = 0.f; a.terms[row] = make_float4(0.f, 0.f, 0.f, 0.f); }
        row_zero<BF, NT, S>(d, vocab);
        return;
    }
    // everything the coefficient will need is asked for before the row's own loads, which it would otherwise wait behind
    const PolicyRow in = policy_row(a, row);
    const float scale = dloss_mul * dloss[0] * (float)sc.inv_tau;
    int64_t seq, begin, end;
    const bool inside = policy_range(a, row, seq, begin, end);
    int n = 0;
    unsigned live = 0;
    if (a.counts) {
        n = inside ? a.counts[seq] : 0;
    } else {   // no counts (rows <= kCountRows NT): this workgroup's threads look at all labels
#pragma unroll
        for (int q = 0; q < kCountRows; ++q) {
            const int64_t t = (int64_t)q * NT + threadIdx.x;
            int other;
            if (t < end && row_label(a.labels, t, a.ignore_index, vocab, other) && t >= begin) live |= 1u << q;
        }
    }
    const T* x = (const T*)logits + row * ld;
    const float xl = Elem<BF>::get(x + lab);
    const float k = sc.mine();
    const int nv = vocab / N;
    float ex[NV * N], ex_last = -INFINITY;
    {
        u32x4 v[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = threadIdx.x + j * NT;
            v[j] = Elem<BF>::ninf();
            if (i < nv) v[j] = ldv<true>(x + (int64_t)i * N);
        }
        if (nv * N + (int)threadIdx.x < vocab) ex_last = Elem<BF>::get(x + nv * N + threadIdx.x);
#pragma unroll
        for (int j = 0; j < NV; ++j) Elem<BF>::unpack(v[j], ex + j * N);
    }
    float m = ex_last, s = 0.f;
#pragma unroll
    for (int q = 0; q < NV * N; ++q) m = fmaxf(m, ex[q]);
    if (REST) {
        float rm = m;
        for (int i = NV * NT + threadIdx.x; i < nv; i += NT) {
            float e[N];
            Elem<BF>::unpack(ldv<false>(x + (int64_t)i * N), e);
            add_values<N>(e, k, rm, s);
        }
        m = rm;
    }
    float own = ref(m, k);   // reference of the thread's terms
    s += ex_last = term<true>(ex_last, k, own);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int q = 0; q < N; ++q) ex[j * N + q] = term<true>(ex[j * N + q], k, own);
        s += tree_sum<N>(ex + j * N);
    }
    RowStat st = join_stats<NT>(m, s, k, sc, sh);
    own = usable(m, k) ? to_max(m, k, st.m, sc) : 0.f;   // now: the factor of the thread's terms
    if (!st.fast) st = row_stat_again<BF, NT>(x, vocab, st.m, sc.lo, sh);
    if (!a.counts) {
#pragma unroll
        for (int q = 0; q < kCountRows; ++q) n += __popcll(__ballot(live >> q & 1u));
        if ((threadIdx.x & 63) == 0) counted[threadIdx.x >> 6] = n;
        __syncthreads();
        n = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) n += counted[w];
    }
    if (threadIdx.x == 0) {
        const double logp = st.logp(xl, sc.inv_tau);
        logp_out[row] = (float)logp;
        lse_out[row] = (float)st.lse(sc.inv_tau);
        coef_sh = a.coef[row] = policy_term(a, in, logp, policy_weight(a, inside, n), a.terms[row]);
    }
    __syncthreads();
    const float g = coef_sh * scale;
    if (g == 0.f) { row_zero<BF, NT, S>(d, vocab); return; }
    const float g_p = g / st.s;
    if (!st.fast) {
        row_grad_again<BF, NT>(x, d, vocab, sc.lo, max_ref(st.m), g, g_p, lab, xl);
        return;
    }
    const float f = -g_p * own;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * NT;
        float e[N];
#pragma unroll
        for (int q = 0; q < N; ++q) e[q] = f * ex[j * N + q];
        if (i < nv) stv<S>(d + (int64_t)i * N, Elem<BF>::pack(e));
    }
    const float r = st.m * sc.lo, g_r = g_p * exp2_(__builtin_fmaf(-st.m, sc.lo, r));   // for what is raised again
    if (REST)
        for (int i = NV * NT + threadIdx.x; i < nv; i += NT) stv<S>(d + (int64_t)i * N, grad_vector<BF, true>(ldv<false>(x + (int64_t)i * N), sc.lo, r, g_r));
    if (nv * N + (int)threadIdx.x < vocab) Elem<BF>::put(d + nv * N + threadIdx.x, f * ex_last);
    if (owns<BF, NT>(lab, vocab)) Elem<BF>::put(d + lab, g - g_r * term<true>(xl, sc.lo, r));
}

// stats = {loss, surrogate, KL, clipped share}
__global__ __launch_bounds__(1024) void policy_stats_k(const float4* __restrict__ terms, int64_t rows, float kl_coef, float* __restrict__ stats) {
    __shared__ double scratch[48];
    double v[3] = {0.0, 0.0, 0.0};
#pragma unroll 8
    for (int64_t t = threadIdx.x; t < rows; t += 1024) {
        const float4 q = terms[t];
        v[0] += (double)q.x; v[1] += (double)q.y; v[2] += (double)q.z;
    }
    write_stats(v, kl_coef, stats, scratch);
}

constexpr int64_t kMaxVocab = int64_t(1) << 30;   // in-row indices are 32-bit
constexpr int64_t kMaxRows = (int64_t(1) << 26) - 4;   // (a launch of a wave a row, four a workgroup, has fewer than 2^32 threads)
constexpr int64_t kMaxSeqs = (int64_t(1) << 22) - 1;   // ... and one of 1024 threads a pair fewer than half of that

#define IE_CHECK_LOGITS(fn)                                                                                                                              \
    IE_CHECK_ARG(dtype == IE_BF16 || dtype == IE_F32, fn ": bad dtype");                                                                                 \
    IE_CHECK_ARG(rows >= 0 && rows <= kMaxRows && vocab > 0 && vocab <= kMaxVocab && ld >= vocab, fn ": bad shape");                                     \
    IE_CHECK_ARG(inv_temperature >= 1e-30 && inv_temperature <= 1e30, fn ": the temperature must be positive and finite")

// dlogits is either the logits (same address, same stride) or does not touch them
bool overlap_ok(const void* x, int64_t ld, const void* d, int64_t ldd, int64_t rows, int64_t vocab, int dtype) {
    if (rows == 0 || (x == d && ld == ldd)) return true;
    const int64_t es = dtype == IE_BF16 ? 2 : 4;
    const char *xb = (const char*)x, *db = (const char*)d;
    return xb + ((rows - 1) * ld + vocab) * es <= db || db + ((rows - 1) * ldd + vocab) * es <= xb;
}

// Past the 256 MB of the last-level cache: loads of logits beyond 192 MB, stores where the call touches more than that in all.  30 % of the rows masked, logits just
// written, forward and backward, loads and stores cached | loads alone | neither: 92 544 bf16 columns, 128 MB in place 53 us | 56 | 58, into other memory 71 | 57 | 59;
// 192 MB 79 | 80 | 82 and 87 | 81 | 82; 256 MB 120 | 113 | 103 and 120 | 110 | 106; 768 MB 355 | 340 | 276.
bool beyond(int64_t rows, int64_t vocab, int dtype, bool twice) { return (rows * vocab * (dtype == IE_BF16 ? 2 : 4) << (twice ? 1 : 0)) > (int64_t(192) << 20); }

inline int vectors(int64_t vocab, int dtype) { return (int)(vocab / (dtype == IE_BF16 ? 8 : 4)); }

// rows in slices, so that no launch has 2^32 threads; the kernel's last argument is the slice's first row, before it the workgroups a row if there are several
struct Launch {
    hipStream_t st;
    int64_t rows;
    template <int NT, typename F, typename... A> void go(F f, A... args) const {
        const int64_t most = (int64_t(1) << 32) / NT - 1;
        for (int64_t row0 = 0; row0 < rows; row0 += most) hipLaunchKernelGGL(f, dim3((unsigned)std::min(most, rows - row0)), dim3(NT), 0, st, args..., row0);
    }
    template <int NT, typename F, typename... A> void parts(F f, int parts, A... args) const {
        const int64_t most = ((int64_t(1) << 32) / NT - 1) / parts;
        for (int64_t row0 = 0; row0 < rows; row0 += most)
            hipLaunchKernelGGL(f, dim3((unsigned)(std::min(most, rows - row0) * parts)), dim3(NT), 0, st, args..., Divisor((unsigned)parts), row0);
    }
};

// Threads a row.  Forward, 8000 x 4000 bf16: 64 threads 17.3 us, 256 17.8, 512 31; 2000 x 32 000 bf16: 256 22.0, 512 22.6, 1024 24.0; 3001 x 32 003 fp32: 256 54, 512 49,
// 1024 48; 16 384 x 92 544 bf16: 256 266, 512 259, 1024 260; with fewer rows than two a CU the widest workgroup is the shortest wait.
template <bool BF, bool S>
void launch_fwd(const Launch& l, int nv, const void* logits, int64_t ld, const int64_t* labels, float* logp, float* lse, float* coef, float* low, int vocab, int64_t ignore_index,
                const Scale& sc) {
    if (nv <= 256) l.go<64>(logprob_fwd_k<BF, 64, S>, logits, ld, labels, logp, lse, coef, low, vocab, ignore_index, sc);
    else if (nv <= 4096 && (l.rows >= 512 || nv <= 1024)) l.go<256>(logprob_fwd_k<BF, 256, S>, logits, ld, labels, logp, lse, coef, low, vocab, ignore_index, sc);
    else l.go<1024>(logprob_fwd_k<BF, 1024, S>, logits, ld, labels, logp, lse, coef, low, vocab, ignore_index, sc);
}

template <bool BF, bool L, bool S>
void launch_bwd(const Launch& l, int nv, const BwdArgs& a, const Scale& sc) {
    if (nv <= 128) l.parts<64>(logprob_bwd_k<BF, 64, L, S>, std::max((nv + 63) / 64, 1), a, sc);
    else l.parts<256>(logprob_bwd_k<BF, 256, L, S>, (nv + 255) / 256, a, sc);
}

// Threads and vectors a thread of the fused kernel, so that the row fills most of them and two workgroups share a CU while they can.  bf16, rows x vocabulary:
// 8000 x 4000: 256 x 4 26 us, 64 x 8 27; 8000 x 16 000: 256 x 8 93, 512 x 8 98; 8000 x 20 000: 512 x 8 105, 1024 x 4 156, 256 x 8 + rest 110; 4000 x 50 000:
// 512 x 10 + rest 141, 1024 x 8 149; 4000 x 60 000: 1024 x 8 180, 512 x 10 + rest 186; 16 384 x 92 544: 1024 x 10 + rest 942, x 8 993, x 12 (spills) 1063, 512 x 10 993.  fp32, 4000 x 92 544: 1024 x 16 + rest 494, x 10 542, x 20 513.
inline int fused_threads(int nv) { return nv <= 256 ? 64 : nv <= 2048 ? 256 : nv <= 6656 ? 512 : 1024; }

template <bool BF, bool S>
void launch_fused(const Launch& l, int nv, const PolicyArgs& a, const void* logits, int64_t ld, void* dlogits, int64_t ldd, float* logp, float* lse, const float* dloss, float dloss_mul,
                  const Scale& sc) {
    if (nv <= 128) l.go<64>(policy_fused_k<BF, 64, 2, false, S>, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, sc);
    else if (nv <= 256) l.go<64>(policy_fused_k<BF, 64, 4, false, S>, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, sc);
    else if (nv <= 1024) l.go<256>(policy_fused_k<BF, 256, 4, false, S>, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, sc);
    else if (nv <= 2048) l.go<256>(policy_fused_k<BF, 256, 8, false, S>, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, sc);
    else if (nv <= 4096) l.go<512>(policy_fused_k<BF, 512, 8, false, S>, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, sc);
    else if (nv <= 6656) l.go<512>(policy_fused_k<BF, 512, 10, true, S>, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, sc);
    else if (nv <= 8192) l.go<1024>(policy_fused_k<BF, 1024, 8, false, S>, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, sc);
    else l.go<1024>(policy_fused_k<BF, 1024, BF ? 10 : 16, true, S>, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, sc);
}

// fn<type, past>(args...)
#define IE_ROWS(fn, past, ...)                                                          \
    do {                                                                          \
        const bool s_ = past;                                                     \
        const Launch l_ = {(hipStream_t)stream, rows};                            \
        const int nv_ = vectors(vocab, dtype);                                    \
        if (dtype == IE_BF16) {                                                   \
            if (s_) fn<true, true>(l_, nv_, __VA_ARGS__);                         \
            else fn<true, false>(l_, nv_, __VA_ARGS__);                           \
        } else {                                                                  \
            if (s_) fn<false, true>(l_, nv_, __VA_ARGS__);                        \
            else fn<false, false>(l_, nv_, __VA_ARGS__);                          \
        }                                                                         \
    } while (0)

}  // namespace

extern "C" int ie_logprob_fwd(const void* logits, int dtype, int64_t ld, const int64_t* labels, float* logp, float* lse, int64_t rows, int64_t vocab,
                              int64_t ignore_index, double inv_temperature, void* stream) {
    IE_CHECK_ARG(logits && labels && logp && lse, "ie_logprob_fwd: null pointer");
    IE_CHECK_LOGITS("ie_logprob_fwd");
    if (rows == 0) return IE_OK;
    IE_ROWS(launch_fwd, beyond(rows, vocab, dtype, false), logits, ld, labels, logp, lse, (float*)nullptr, (float*)nullptr, (int)vocab, ignore_index, Scale(inv_temperature));
    return ie_launch_status("ie_logprob_fwd launch");
}

extern "C" int ie_logprob_bwd(const void* logits, int dtype, int64_t ld, void* dlogits, int64_t ldd, const int64_t* labels, const float* lse, const float* coef,
                              const float* dloss, float dloss_mul, int64_t rows, int64_t vocab, int64_t ignore_index, double inv_temperature, void* stream) {
    IE_CHECK_ARG(logits && dlogits && labels && lse && coef, "ie_logprob_bwd: null pointer");
    IE_CHECK_LOGITS("ie_logprob_bwd");
    IE_CHECK_ARG(ldd >= vocab && overlap_ok(logits, ld, dlogits, ldd, rows, vocab, dtype), "ie_logprob_bwd: dlogits must be the logits themselves or lie apart from them");
    if (rows == 0) return IE_OK;
    const Scale sc(inv_temperature);
    const BwdArgs a = {logits, dlogits, ld, ldd, labels, lse, coef, dloss ? dloss : lse, ignore_index, (double)sc.lo / inv_temperature, dloss_mul * (float)inv_temperature,
                       dloss ? 0.f : 1.f, (int)vocab};
    const bool loads = beyond(rows, vocab, dtype, false), stores = beyond(rows, vocab, dtype, dlogits != logits);
    const Launch l = {(hipStream_t)stream, rows};
    const int nv = vectors(vocab, dtype);
    if (dtype == IE_BF16) loads ? launch_bwd<true, true, true>(l, nv, a, sc) : stores ? launch_bwd<true, false, true>(l, nv, a, sc) : launch_bwd<true, false, false>(l, nv, a, sc);
    else loads ? launch_bwd<false, true, true>(l, nv, a, sc) : stores ? launch_bwd<false, false, true>(l, nv, a, sc) : launch_bwd<false, false, false>(l, nv, a, sc);
    return ie_launch_status("ie_logprob_bwd launch");
}

// the pairs' losses in 64 bits, then what the log-probabilities lose in 32
extern "C" int64_t ie_preference_loss_workspace(int64_t rows, int64_t pairs) { return rows >= 0 && pairs > 0 ? pairs * 8 + rows * 4 : 0; }

extern "C" int ie_preference_loss_fwd(const void* logits, int dtype, int64_t ld, const int64_t* labels, const int32_t* cu_seqlens, const float* ref_logps, int kind,
                                      double beta, double label_smoothing, double margin, int average, float* loss, float* rewards, float* seq_logps, float* logp,
                                      float* lse, float* coef, void* workspace, int64_t rows, int64_t vocab, int64_t pairs, int64_t ignore_index, double inv_temperature,
                                      void* stream) {
    IE_CHECK_ARG(logits && labels && cu_seqlens && loss && rewards && seq_logps && logp && lse && coef && workspace, "ie_preference_loss_fwd: null pointer");
    IE_CHECK_ARG(((uintptr_t)workspace & 7) == 0, "ie_preference_loss_fwd: the workspace must be 8-byte aligned");
    IE_CHECK_LOGITS("ie_preference_loss_fwd");
    IE_CHECK_ARG(pairs > 0 && pairs <= kMaxSeqs / 2, "ie_preference_loss_fwd: at least one pair");
    IE_CHECK_ARG(kind == IE_PREF_SIGMOID || kind == IE_PREF_HINGE || kind == IE_PREF_IPO, "ie_preference_loss_fwd: unknown kind");
    IE_CHECK_ARG(beta > 0.0 && beta <= 1e30, "ie_preference_loss_fwd: beta must be positive and finite");
    IE_CHECK_ARG(label_smoothing >= 0.0 && label_smoothing <= 0.5 && (kind == IE_PREF_SIGMOID || label_smoothing == 0.0),
                 "ie_preference_loss_fwd: label smoothing lies in [0, 0.5] and belongs to the sigmoid form");
    IE_CHECK_ARG(margin >= -1e30 && margin <= 1e30 && (kind != IE_PREF_IPO || margin == 0.0), "ie_preference_loss_fwd: the squared form takes no margin");
    hipStream_t st = (hipStream_t)stream;
    double* losses = (double*)workspace;
    float* low = (float*)(losses + pairs);
    if (rows > 0) IE_ROWS(launch_fwd, beyond(rows, vocab, dtype, false), logits, ld, labels, logp, lse, coef, low, (int)vocab, ignore_index, Scale(inv_temperature));
    const PrefArgs a = {kind, average, beta, label_smoothing, margin};
    const PrefRows r = {logp, low, labels, cu_seqlens, ref_logps, rows, pairs, ignore_index, (int)vocab, rewards, seq_logps, coef};
    if (pairs <= kOnePairs && rows <= kOneRows) {
        if (pairs == 1) hipLaunchKernelGGL((preference_pairs_k<8, false>), dim3(1), dim3(1024), 0, st, r, a, loss, losses);
        else if (pairs == 2) hipLaunchKernelGGL((preference_pairs_k<4, false>), dim3(1), dim3(1024), 0, st, r, a, loss, losses);
        else if (pairs <= 4) hipLaunchKernelGGL((preference_pairs_k<2, false>), dim3(1), dim3(1024), 0, st, r, a, loss, losses);
        else hipLaunchKernelGGL((preference_pairs_k<1, false>), dim3(1), dim3(1024), 0, st, r, a, loss, losses);
    } else {
        hipLaunchKernelGGL((preference_pairs_k<8, true>), dim3((unsigned)pairs), dim3(1024), 0, st, r, a, loss, losses);
        hipLaunchKernelGGL(preference_mean_k, dim3(1), dim3(256), 0, st, (const double*)losses, pairs, loss);
    }
    return ie_launch_status("ie_preference_loss_fwd launch");
}

// terms [rows] of four floats, then the counts
extern "C" int64_t ie_policy_loss_workspace(int64_t rows, int64_t seqs) { return rows < 0 || seqs < 0 ? 0 : (4 * rows + (seqs > 0 ? seqs : 1)) * 4; }

extern "C" int ie_policy_loss(const void* logits, int dtype, int64_t ld, void* dlogits, int64_t ldd, const int64_t* labels, const float* old_logps, const float* advantages,
                              const float* ref_logps, const int32_t* cu_seqlens, int64_t seqs, float clip_low, float clip_high, float kl_coef, const float* dloss,
                              float dloss_mul, float* stats, float* logp, float* lse, float* coef, void* workspace, int64_t rows, int64_t vocab, int64_t ignore_index,
                              double inv_temperature, void* stream) {
    IE_CHECK_ARG(logits && labels && old_logps && advantages && stats && logp && lse && coef && workspace, "ie_policy_loss: null pointer");
    IE_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "ie_policy_loss: the workspace must be 16-byte aligned");
    IE_CHECK_LOGITS("ie_policy_loss");
    IE_CHECK_ARG((dlogits != nullptr) == (dloss != nullptr), "ie_policy_loss: dlogits and dloss come together");
    IE_CHECK_ARG(!dlogits || (ldd >= vocab && overlap_ok(logits, ld, dlogits, ldd, rows, vocab, dtype)),
                 "ie_policy_loss: dlogits must be the logits themselves or lie apart from them");
    IE_CHECK_ARG(cu_seqlens ? seqs > 0 && seqs <= kMaxSeqs : seqs == 0, "ie_policy_loss: cu_seqlens and the number of sequences come together");
    IE_CHECK_ARG(clip_low >= 0.f && clip_low <= 1.f && clip_high >= 0.f && clip_high <= 1e30f, "ie_policy_loss: clip range");
    IE_CHECK_ARG(kl_coef >= 0.f && kl_coef <= 1e30f && (ref_logps || kl_coef == 0.f), "ie_policy_loss: a KL term needs the reference log-probabilities");
    hipStream_t st = (hipStream_t)stream;
    int32_t* counts = (int32_t*)((float*)workspace + 4 * rows);
    PolicyArgs a;
    a.labels = labels; a.cu = cu_seqlens; a.old_logps = old_logps; a.adv = advantages; a.ref = ref_logps;
    a.counts = counts; a.terms = (float4*)workspace;
    a.coef = coef; a.rows = rows; a.seqs = seqs; a.ignore_index = ignore_index; a.vocab = (int)vocab;
    a.low = clip_low; a.high = clip_high; a.kl_coef = kl_coef;
    if (!dlogits && rows <= kSmallRows && seqs <= kSmallSeqs) {
        if (rows > 0) IE_ROWS(launch_fwd, beyond(rows, vocab, dtype, false), logits, ld, labels, logp, lse, (float*)nullptr, (float*)nullptr, (int)vocab, ignore_index, Scale(inv_temperature));
        hipLaunchKernelGGL(policy_small_k, dim3(1), dim3(1024), 0, st, a, (const float*)logp, stats);
        return ie_launch_status("ie_policy_loss launch");
    }
    if (dlogits && rows <= (int64_t)kCountRows * fused_threads(vectors(vocab, dtype))) a.counts = nullptr;
    else if (cu_seqlens) hipLaunchKernelGGL((policy_counts_k<256>), dim3((unsigned)seqs), dim3(256), 0, st, a, counts);
    else hipLaunchKernelGGL((policy_counts_k<1024>), dim3(1), dim3(1024), 0, st, a, counts);
    if (rows > 0 && dlogits) {
        IE_ROWS(launch_fused, beyond(rows, vocab, dtype, dlogits != logits), a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, Scale(inv_temperature));
    } else if (rows > 0) {
        IE_ROWS(launch_fwd, beyond(rows, vocab, dtype, false), logits, ld, labels, logp, lse, (float*)nullptr, (float*)nullptr, (int)vocab, ignore_index, Scale(inv_temperature));
        hipLaunchKernelGGL(policy_terms_k, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, (const float*)logp);
    }
    hipLaunchKernelGGL(policy_stats_k, dim3(1), dim3(1024), 0, st, (const float4*)workspace, rows, kl_coef, stats);
    return ie_launch_status("ie_policy_loss launch");
}

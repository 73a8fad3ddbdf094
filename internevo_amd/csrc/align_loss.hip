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

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));   // 16 bytes at any element's address: rows of an odd vocabulary start anywhere

template <bool BF> struct Elem;
template <> struct Elem<true> {
    typedef bf16_t T;
    static constexpr int N = 8;
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

constexpr float kLog2e = 1.44269504088896341f;

// Maximum m of a row and s = sum 2^((x - m) k), k = log2(e) / tau, in one pass: 2^((m_old - m_new) k) rescales what was summed before a new maximum.  The difference
// is taken before the product: it is exact next to the maximum, and logits masked by the type's lowest value cannot overflow into inf - inf.  While nothing but
// -inf has been seen the reference is 0, so that such logits add 0; NaN and +inf make s NaN.
__device__ __forceinline__ float max_ref(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ float rescale(float m_old, float m_new, float k) { return m_old == -INFINITY ? 0.f : exp2_((m_old - max_ref(m_new)) * k); }

struct RowStat {
    float m, s;
    float log_sum;     // log sum exp((x - m) / tau)
    __device__ __forceinline__ float lse(float inv_tau) const { return fmaf(m, inv_tau, log_sum); }
};

template <bool BF, int NT>
__device__ RowStat row_stat(const typename Elem<BF>::T* __restrict__ x, int vocab, float k, float* scratch) {
    constexpr int N = Elem<BF>::N;
    float m = -INFINITY, s = 0.f;
    const int nv = vocab / N;
    for (int i = threadIdx.x; i < nv; i += NT) {
        float v[N];
        Elem<BF>::unpack(*(const u32x4_any*)(x + (int64_t)i * N), v);
        float cm = v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) cm = fmaxf(cm, v[e]);
        if (cm > m) { s *= rescale(m, cm, k); m = cm; }
        const float r = max_ref(m);
#pragma unroll
        for (int e = 0; e < N; ++e) s += exp2_((v[e] - r) * k);
    }
    for (int i = nv * N + threadIdx.x; i < vocab; i += NT) {
        const float v = Elem<BF>::get(x + i);
        if (v > m) { s *= rescale(m, v, k); m = v; }
        s += exp2_((v - max_ref(m)) * k);
    }
    RowStat st;
    st.m = block_max<NT / 64>(m, scratch);
    st.s = block_sum<NT / 64>(s * rescale(m, st.m, k), scratch);
    st.log_sum = logf(st.s);
    return st;
}

__device__ __forceinline__ bool row_label(const int64_t* labels, int64_t row, int64_t ignore_index, int vocab, int& lab) {
    const int64_t l = labels[row];
    lab = (int)l;
    return l != ignore_index && l >= 0 && l < vocab;
}

// d = g 1[j = label] - g_p 2^((x - m) k) for the whole row: with the row's maximum and sum g_p = g / s, with its log-sum-exp in m's place g_p = g.  The label's own
// element is written last by the thread that owns it, from the logit it read before: dlogits may be the logits themselves.
template <bool BF, int NT>
__device__ void row_grad(const typename Elem<BF>::T* x, typename Elem<BF>::T* d, int vocab, float k, float m, float g, float g_p, int lab) {
    constexpr int N = Elem<BF>::N;
    const int nv = vocab / N;
    const int owner = lab < nv * N ? (lab / N) % NT : (lab - nv * N) % NT;
    float xl = 0.f;
    if ((int)threadIdx.x == owner) xl = Elem<BF>::get(x + lab);
    for (int i = threadIdx.x; i < nv; i += NT) {
        float v[N];
        Elem<BF>::unpack(*(const u32x4_any*)(x + (int64_t)i * N), v);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = -g_p * exp2_((v[e] - m) * k);
        *(u32x4_any*)(d + (int64_t)i * N) = Elem<BF>::pack(v);
    }
    for (int i = nv * N + threadIdx.x; i < vocab; i += NT) Elem<BF>::put(d + i, -g_p * exp2_((Elem<BF>::get(x + i) - m) * k));
    if ((int)threadIdx.x == owner) Elem<BF>::put(d + lab, g - g_p * exp2_((xl - m) * k));
}

template <bool BF, int NT>
__device__ void row_zero(typename Elem<BF>::T* d, int vocab) {
    constexpr int N = Elem<BF>::N;
    const int nv = vocab / N;
    const u32x4 z = {0, 0, 0, 0};
    for (int i = threadIdx.x; i < nv; i += NT) *(u32x4_any*)(d + (int64_t)i * N) = z;
    for (int i = nv * N + threadIdx.x; i < vocab; i += NT) Elem<BF>::put(d + i, 0.f);
}

// ------------------------------------------------------------------------------------------ log-probabilities
// coef (may be null) is cleared: the loss kernels behind this one set it for the rows of their sequences only.
template <bool BF, int NT>
__global__ __launch_bounds__(NT) void logprob_fwd_k(const void* __restrict__ logits, int64_t ld, const int64_t* __restrict__ labels, float* __restrict__ logp,
                                                    float* __restrict__ lse, float* __restrict__ coef, int vocab, int64_t ignore_index, float inv_tau) {
    __shared__ float scratch[NT / 64];
    const int64_t row = blockIdx.x;
    int lab;
    if (!row_label(labels, row, ignore_index, vocab, lab)) {
        if (threadIdx.x == 0) { logp[row] = 0.f; lse[row] = 0.f; if (coef) coef[row] = 0.f; }
        return;
    }
    const typename Elem<BF>::T* x = (const typename Elem<BF>::T*)logits + row * ld;
    const RowStat st = row_stat<BF, NT>(x, vocab, inv_tau * kLog2e, scratch);
    if (threadIdx.x == 0) {
        lse[row] = st.lse(inv_tau);
        logp[row] = (Elem<BF>::get(x + lab) - st.m) * inv_tau - st.log_sum;
        if (coef) coef[row] = 0.f;
    }
}

template <bool BF, int NT>
__global__ __launch_bounds__(NT) void logprob_bwd_k(const void* logits, int64_t ld, void* dlogits, int64_t ldd, const int64_t* __restrict__ labels,
                                                    const float* __restrict__ lse, const float* __restrict__ coef, const float* __restrict__ dloss, float dloss_mul,
                                                    int vocab, int64_t ignore_index, float inv_tau) {
    __shared__ float scratch[NT / 64];
    const int64_t row = blockIdx.x;
    int lab;
    typename Elem<BF>::T* d = (typename Elem<BF>::T*)dlogits + row * ldd;
    const bool valid = row_label(labels, row, ignore_index, vocab, lab);
    float g = valid ? coef[row] * dloss_mul * inv_tau : 0.f;
    if (dloss) g *= dloss[0];
    if (!valid || g == 0.f) { row_zero<BF, NT>(d, vocab); return; }
    const float k = inv_tau * kLog2e;
    const typename Elem<BF>::T* x = (const typename Elem<BF>::T*)logits + row * ld;
    float m = lse[row] / inv_tau, g_p = g;
    if (m < -1e30f) {   // every logit at the type's lowest value or below: there the log-sum-exp cannot hold the sum beside the maximum
        const RowStat st = row_stat<BF, NT>(x, vocab, k, scratch);
        __syncthreads();
        m = st.m;
        g_p = g / st.s;
    }
    row_grad<BF, NT>(x, d, vocab, k, m, g, g_p, lab);
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
        return -(1.0 - a.smoothing) * log_sigmoid(z) - a.smoothing * log_sigmoid(-z);
    }
    if (a.kind == IE_PREF_HINGE) {
        slope = z < 1.0 ? -a.beta : z == z ? 0.0 : z;
        return z == z ? fmax(0.0, 1.0 - z) : z;
    }
    const double q = h - 0.5 / a.beta;
    slope = 2.0 * q;
    return q * q;
}

// One workgroup per pair (sequences 2p, 2p + 1): sums of the log-probabilities in 64 bits, the pair's loss, and the coefficient of every row of the pair.
__global__ __launch_bounds__(256) void preference_pair_k(const float* __restrict__ logp, const int64_t* __restrict__ labels, const int32_t* __restrict__ cu,
                                                         const float* __restrict__ ref, int64_t rows, int64_t pairs, int64_t ignore_index, int vocab, PrefArgs a,
                                                         double* __restrict__ losses, float* __restrict__ rewards, float* __restrict__ seq_logps,
                                                         float* __restrict__ coef) {
    __shared__ double scratch[4];
    const int64_t p = blockIdx.x;
    int64_t begin[2], end[2];
    double l[2], n[2], gain[2];
    for (int c = 0; c < 2; ++c) {
        const int64_t s = 2 * p + c;
        seq_range(cu, s, rows, begin[c], end[c]);
        double sum = 0.0, cnt = 0.0;
        for (int64_t t = begin[c] + threadIdx.x; t < end[c]; t += 256) {
            int lab;
            if (row_label(labels, t, ignore_index, vocab, lab)) { sum += (double)logp[t]; cnt += 1.0; }
        }
        l[c] = block_sum_d<4>(sum, scratch);
        n[c] = block_sum_d<4>(cnt, scratch);
        if (a.average) l[c] /= fmax(n[c], 1.0);
        gain[c] = l[c] - (ref ? (double)ref[s] : 0.0);
        if (threadIdx.x == 0) {
            seq_logps[s] = (float)l[c];
            rewards[s] = (float)(a.beta * gain[c]);
        }
    }
    double slope;
    const double loss = pair_loss(a, gain[0] - gain[1], slope);
    if (threadIdx.x == 0) losses[p] = loss;
    for (int c = 0; c < 2; ++c) {
        const float w = (float)((c ? -slope : slope) / (double)pairs / (a.average ? fmax(n[c], 1.0) : 1.0));
        for (int64_t t = begin[c] + threadIdx.x; t < end[c]; t += 256) {
            int lab;
            if (row_label(labels, t, ignore_index, vocab, lab)) coef[t] = w;
        }
    }
}

__global__ __launch_bounds__(256) void preference_mean_k(const double* __restrict__ losses, int64_t pairs, float* __restrict__ loss) {
    __shared__ double scratch[4];
    double v = 0.0;
    for (int64_t i = threadIdx.x; i < pairs; i += 256) v += losses[i];
    v = block_sum_d<4>(v, scratch);
    if (threadIdx.x == 0) loss[0] = (float)(v / (double)pairs);
}

// ------------------------------------------------------------------------------------------ policy loss
struct PolicyArgs {
    const int64_t* labels;
    const int32_t* cu;      // null: one mean over all tokens
    const float *old_logps, *adv, *ref;   // ref null: no KL term
    const int32_t* counts;  // tokens of every sequence, or of the whole batch
    float* terms;           // [3][rows]: weighted surrogate, KL, clipped
    float* coef;
    int64_t rows, seqs, ignore_index;
    int vocab;
    float low, high, kl_coef;
};

// tokens with a label, per sequence (cu) or in all (cu null, one workgroup)
__global__ __launch_bounds__(1024) void policy_counts_k(PolicyArgs a, int32_t* __restrict__ counts) {
    __shared__ double scratch[16];
    int64_t begin = 0, end = a.rows;
    if (a.cu) seq_range(a.cu, blockIdx.x, a.rows, begin, end);
    double n = 0.0;
    for (int64_t t = begin + threadIdx.x; t < end; t += 1024) {
        int lab;
        n += row_label(a.labels, t, a.ignore_index, a.vocab, lab) ? 1.0 : 0.0;
    }
    n = block_sum_d<16>(n, scratch);
    if (threadIdx.x == 0) counts[blockIdx.x] = (int32_t)n;
}

// weight of row t's term: 1 / N, or 1 / (S n_s); 0 outside every sequence.  Called by whole waves with one t.
__device__ __forceinline__ float policy_weight(const PolicyArgs& a, int64_t t) {
    if (!a.cu) return 1.f / (float)max(a.counts[0], 1);
    int64_t s = 0;   // how many of cu[1..S] are <= t
    for (int64_t i = threadIdx.x & 63; i - (int64_t)(threadIdx.x & 63) < a.seqs; i += 64) s += __popcll(__ballot(i < a.seqs && (int64_t)a.cu[i + 1] <= t));
    if (s >= a.seqs || t < (int64_t)a.cu[0]) return 0.f;
    return 1.f / ((float)a.seqs * (float)max(a.counts[s], 1));
}

// terms of one row and d loss / d logp
__device__ __forceinline__ float policy_term(const PolicyArgs& a, int64_t t, float logp, float w) {
    const float adv = a.adv[t];
    const float ratio = expf(logp - a.old_logps[t]);
    const bool clipped = (adv > 0.f && ratio > 1.f + a.high) || (adv < 0.f && ratio < 1.f - a.low);
    const float bound = adv > 0.f ? 1.f + a.high : 1.f - a.low;
    const float s = -(clipped ? bound : ratio) * adv;
    float d = clipped ? 0.f : -ratio * adv, kl = 0.f;
    if (a.ref) {
        const float q = a.ref[t] - logp, e = expm1f(q);
        kl = e - q;
        if (a.kl_coef > 0.f) d -= a.kl_coef * e;   // (0 * inf would turn a mere report into NaN)
    }
    if (w == 0.f) { a.terms[t] = 0.f; a.terms[a.rows + t] = 0.f; a.terms[2 * a.rows + t] = 0.f; return 0.f; }
    a.terms[t] = w * s;
    a.terms[a.rows + t] = w * kl;
    a.terms[2 * a.rows + t] = clipped ? w : 0.f;
    return w * d;
}

// one wave per row: terms and coefficients from finished log-probabilities
__global__ __launch_bounds__(256) void policy_terms_k(PolicyArgs a, const float* __restrict__ logp) {
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.rows) return;
    int lab;
    const bool valid = row_label(a.labels, t, a.ignore_index, a.vocab, lab);
    const float w = valid ? policy_weight(a, t) : 0.f;
    if ((threadIdx.x & 63) == 0) {
        if (valid) a.coef[t] = policy_term(a, t, logp[t], w);
        else { a.terms[t] = 0.f; a.terms[a.rows + t] = 0.f; a.terms[2 * a.rows + t] = 0.f; a.coef[t] = 0.f; }
    }
}

// forward and backward of one row: the coefficient needs nothing but the row itself
template <bool BF, int NT>
__global__ __launch_bounds__(NT) void policy_fused_k(PolicyArgs a, const void* logits, int64_t ld, void* dlogits, int64_t ldd, float* __restrict__ logp_out,
                                                     float* __restrict__ lse_out, const float* __restrict__ dloss, float dloss_mul, float inv_tau) {
    __shared__ float scratch[NT / 64];
    __shared__ float coef_sh;
    const int64_t row = blockIdx.x;
    typename Elem<BF>::T* d = (typename Elem<BF>::T*)dlogits + row * ldd;
    int lab;
    if (!row_label(a.labels, row, a.ignore_index, a.vocab, lab)) {
        if (threadIdx.x == 0) {
            logp_out[row] = 0.f; lse_out[row] = 0.f; a.coef[row] = 0.f;
            a.terms[row] = 0.f; a.terms[a.rows + row] = 0.f; a.terms[2 * a.rows + row] = 0.f;
        }
        row_zero<BF, NT>(d, a.vocab);
        return;
    }
    const typename Elem<BF>::T* x = (const typename Elem<BF>::T*)logits + row * ld;
    const float k = inv_tau * kLog2e;
    const RowStat st = row_stat<BF, NT>(x, a.vocab, k, scratch);
    const float w = policy_weight(a, row);
    if (threadIdx.x == 0) {
        const float logp = (Elem<BF>::get(x + lab) - st.m) * inv_tau - st.log_sum;
        logp_out[row] = logp;
        lse_out[row] = st.lse(inv_tau);
        coef_sh = a.coef[row] = policy_term(a, row, logp, w);
    }
    __syncthreads();
    const float g = coef_sh * dloss_mul * dloss[0] * inv_tau;
    if (g == 0.f) row_zero<BF, NT>(d, a.vocab);
    else row_grad<BF, NT>(x, d, a.vocab, k, st.m, g, g / st.s, lab);
}

// stats = {loss, surrogate, KL, clipped share}
__global__ __launch_bounds__(1024) void policy_stats_k(const float* __restrict__ terms, int64_t rows, float kl_coef, float* __restrict__ stats) {
    __shared__ double scratch[16];
    double v[3];
    for (int c = 0; c < 3; ++c) {
        double s = 0.0;
        for (int64_t t = threadIdx.x; t < rows; t += 1024) s += (double)terms[c * rows + t];
        v[c] = block_sum_d<16>(s, scratch);
    }
    if (threadIdx.x == 0) {
        stats[0] = (float)(kl_coef > 0.f ? v[0] + (double)kl_coef * v[1] : v[0]);
        stats[1] = (float)v[0];
        stats[2] = (float)v[1];
        stats[3] = (float)v[2];
    }
}

constexpr int64_t kMaxVocab = int64_t(1) << 30;   // in-row indices are 32-bit
constexpr int64_t kMaxRows = 0x7fffffff;          // one workgroup per row

#define IE_CHECK_LOGITS(fn)                                                                                                                              \
    IE_CHECK_ARG(dtype == IE_BF16 || dtype == IE_F32, fn ": bad dtype");                                                                                 \
    IE_CHECK_ARG(rows >= 0 && rows <= kMaxRows && vocab > 0 && vocab <= kMaxVocab && ld >= vocab, fn ": bad shape");                                     \
    IE_CHECK_ARG(inv_temperature > 0.f && inv_temperature <= 3.0e38f, fn ": the temperature must be positive and finite")

// dlogits is either the logits (same address, same stride) or does not touch them
bool overlap_ok(const void* x, int64_t ld, const void* d, int64_t ldd, int64_t rows, int64_t vocab, int dtype) {
    if (rows == 0 || (x == d && ld == ldd)) return true;
    const int64_t es = dtype == IE_BF16 ? 2 : 4;
    const char *xb = (const char*)x, *db = (const char*)d;
    return xb + ((rows - 1) * ld + vocab) * es <= db || db + ((rows - 1) * ldd + vocab) * es <= xb;
}

int launch_logprob_fwd(const void* logits, int dtype, int64_t ld, const int64_t* labels, float* logp, float* lse, float* coef, int64_t rows, int64_t vocab,
                       int64_t ignore_index, float inv_temperature, hipStream_t st) {
    if (rows == 0) return IE_OK;
    if (dtype == IE_BF16)
        hipLaunchKernelGGL((logprob_fwd_k<true, 256>), dim3((unsigned)rows), dim3(256), 0, st, logits, ld, labels, logp, lse, coef, (int)vocab, ignore_index, inv_temperature);
    else
        hipLaunchKernelGGL((logprob_fwd_k<false, 256>), dim3((unsigned)rows), dim3(256), 0, st, logits, ld, labels, logp, lse, coef, (int)vocab, ignore_index, inv_temperature);
    return ie_launch_status("log-probability launch");
}

}  // namespace

extern "C" int ie_logprob_fwd(const void* logits, int dtype, int64_t ld, const int64_t* labels, float* logp, float* lse, int64_t rows, int64_t vocab,
                              int64_t ignore_index, float inv_temperature, void* stream) {
    IE_CHECK_ARG(logits && labels && logp && lse, "ie_logprob_fwd: null pointer");
    IE_CHECK_LOGITS("ie_logprob_fwd");
    return launch_logprob_fwd(logits, dtype, ld, labels, logp, lse, nullptr, rows, vocab, ignore_index, inv_temperature, (hipStream_t)stream);
}

extern "C" int ie_logprob_bwd(const void* logits, int dtype, int64_t ld, void* dlogits, int64_t ldd, const int64_t* labels, const float* lse, const float* coef,
                              const float* dloss, float dloss_mul, int64_t rows, int64_t vocab, int64_t ignore_index, float inv_temperature, void* stream) {
    IE_CHECK_ARG(logits && dlogits && labels && lse && coef, "ie_logprob_bwd: null pointer");
    IE_CHECK_LOGITS("ie_logprob_bwd");
    IE_CHECK_ARG(ldd >= vocab && overlap_ok(logits, ld, dlogits, ldd, rows, vocab, dtype), "ie_logprob_bwd: dlogits must be the logits themselves or lie apart from them");
    if (rows == 0) return IE_OK;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == IE_BF16)
        hipLaunchKernelGGL((logprob_bwd_k<true, 256>), dim3((unsigned)rows), dim3(256), 0, st, logits, ld, dlogits, ldd, labels, lse, coef, dloss, dloss_mul, (int)vocab,
                           ignore_index, inv_temperature);
    else
        hipLaunchKernelGGL((logprob_bwd_k<false, 256>), dim3((unsigned)rows), dim3(256), 0, st, logits, ld, dlogits, ldd, labels, lse, coef, dloss, dloss_mul, (int)vocab,
                           ignore_index, inv_temperature);
    return ie_launch_status("ie_logprob_bwd launch");
}

extern "C" int64_t ie_preference_loss_workspace(int64_t pairs) { return pairs > 0 ? pairs * 8 : 0; }

extern "C" int ie_preference_loss_fwd(const void* logits, int dtype, int64_t ld, const int64_t* labels, const int32_t* cu_seqlens, const float* ref_logps, int kind,
                                      double beta, double label_smoothing, double margin, int average, float* loss, float* rewards, float* seq_logps, float* logp,
                                      float* lse, float* coef, void* workspace, int64_t rows, int64_t vocab, int64_t pairs, int64_t ignore_index, float inv_temperature,
                                      void* stream) {
    IE_CHECK_ARG(logits && labels && cu_seqlens && loss && rewards && seq_logps && logp && lse && coef && workspace, "ie_preference_loss_fwd: null pointer");
    IE_CHECK_LOGITS("ie_preference_loss_fwd");
    IE_CHECK_ARG(pairs > 0 && pairs <= kMaxRows / 2, "ie_preference_loss_fwd: at least one pair");
    IE_CHECK_ARG(kind == IE_PREF_SIGMOID || kind == IE_PREF_HINGE || kind == IE_PREF_IPO, "ie_preference_loss_fwd: unknown kind");
    IE_CHECK_ARG(beta > 0.0 && beta <= 1e30, "ie_preference_loss_fwd: beta must be positive and finite");
    IE_CHECK_ARG(label_smoothing >= 0.0 && label_smoothing <= 0.5 && (kind == IE_PREF_SIGMOID || label_smoothing == 0.0),
                 "ie_preference_loss_fwd: label smoothing lies in [0, 0.5] and belongs to the sigmoid form");
    IE_CHECK_ARG(margin >= -1e30 && margin <= 1e30 && (kind != IE_PREF_IPO || margin == 0.0), "ie_preference_loss_fwd: the squared form takes no margin");
    hipStream_t st = (hipStream_t)stream;
    const int rc = launch_logprob_fwd(logits, dtype, ld, labels, logp, lse, coef, rows, vocab, ignore_index, inv_temperature, st);
    if (rc != IE_OK) return rc;
    const PrefArgs a = {kind, average, beta, label_smoothing, margin};
    hipLaunchKernelGGL(preference_pair_k, dim3((unsigned)pairs), dim3(256), 0, st, logp, labels, cu_seqlens, ref_logps, rows, pairs, ignore_index, (int)vocab, a,
                       (double*)workspace, rewards, seq_logps, coef);
    hipLaunchKernelGGL(preference_mean_k, dim3(1), dim3(256), 0, st, (const double*)workspace, pairs, loss);
    return ie_launch_status("ie_preference_loss_fwd launch");
}

// terms [3][rows] floats, then the counts
extern "C" int64_t ie_policy_loss_workspace(int64_t rows, int64_t seqs) { return rows < 0 || seqs < 0 ? 0 : (3 * rows + (seqs > 0 ? seqs : 1)) * 4; }

extern "C" int ie_policy_loss(const void* logits, int dtype, int64_t ld, void* dlogits, int64_t ldd, const int64_t* labels, const float* old_logps, const float* advantages,
                              const float* ref_logps, const int32_t* cu_seqlens, int64_t seqs, float clip_low, float clip_high, float kl_coef, const float* dloss,
                              float dloss_mul, float* stats, float* logp, float* lse, float* coef, void* workspace, int64_t rows, int64_t vocab, int64_t ignore_index,
                              float inv_temperature, void* stream) {
    IE_CHECK_ARG(logits && labels && old_logps && advantages && stats && logp && lse && coef && workspace, "ie_policy_loss: null pointer");
    IE_CHECK_LOGITS("ie_policy_loss");
    IE_CHECK_ARG((dlogits != nullptr) == (dloss != nullptr), "ie_policy_loss: dlogits and dloss come together");
    IE_CHECK_ARG(!dlogits || (ldd >= vocab && overlap_ok(logits, ld, dlogits, ldd, rows, vocab, dtype)),
                 "ie_policy_loss: dlogits must be the logits themselves or lie apart from them");
    IE_CHECK_ARG(cu_seqlens ? seqs > 0 && seqs <= kMaxRows : seqs == 0, "ie_policy_loss: cu_seqlens and the number of sequences come together");
    IE_CHECK_ARG(clip_low >= 0.f && clip_low <= 1.f && clip_high >= 0.f && clip_high <= 1e30f, "ie_policy_loss: clip range");
    IE_CHECK_ARG(kl_coef >= 0.f && kl_coef <= 1e30f && (ref_logps || kl_coef == 0.f), "ie_policy_loss: a KL term needs the reference log-probabilities");
    hipStream_t st = (hipStream_t)stream;
    PolicyArgs a;
    a.labels = labels; a.cu = cu_seqlens; a.old_logps = old_logps; a.adv = advantages; a.ref = ref_logps;
    a.terms = (float*)workspace; a.counts = (const int32_t*)((float*)workspace + 3 * rows);
    a.coef = coef; a.rows = rows; a.seqs = seqs; a.ignore_index = ignore_index; a.vocab = (int)vocab;
    a.low = clip_low; a.high = clip_high; a.kl_coef = kl_coef;
    hipLaunchKernelGGL(policy_counts_k, dim3((unsigned)(cu_seqlens ? seqs : 1)), dim3(1024), 0, st, a, (int32_t*)((float*)workspace + 3 * rows));
    if (rows > 0 && dlogits) {
        if (dtype == IE_BF16)
            hipLaunchKernelGGL((policy_fused_k<true, 256>), dim3((unsigned)rows), dim3(256), 0, st, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, inv_temperature);
        else
            hipLaunchKernelGGL((policy_fused_k<false, 256>), dim3((unsigned)rows), dim3(256), 0, st, a, logits, ld, dlogits, ldd, logp, lse, dloss, dloss_mul, inv_temperature);
    } else if (rows > 0) {
        const int rc = launch_logprob_fwd(logits, dtype, ld, labels, logp, lse, nullptr, rows, vocab, ignore_index, inv_temperature, st);
        if (rc != IE_OK) return rc;
        hipLaunchKernelGGL(policy_terms_k, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, (const float*)logp);
    }
    hipLaunchKernelGGL(policy_stats_k, dim3(1), dim3(1024), 0, st, (const float*)workspace, rows, kl_coef, stats);
    return ie_launch_status("ie_policy_loss launch");
}

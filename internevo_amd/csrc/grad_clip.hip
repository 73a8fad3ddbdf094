// L2 norm over a list of gradient tensors, and the clipped gradients.
//   norm = sqrt(sum_i g_i^2),  g_i <- g_i min(1, max_norm / (norm + 1e-6))
// The list travels as launch arguments (4 KB of them: 192 tensors a launch of the norm, 136 of the clip), so that nothing is copied to the device first and a captured
// graph holds all it needs.  Every tensor is cut into chunks; a workgroup finds its chunk's tensor in the launch's table.
// HBM-bound: the norm reads every gradient once, the clip reads it again and writes it.
#include "ie_common.h"

#include <math.h>

#include <algorithm>
#include <vector>

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));   // 16 bytes at any element's address
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

constexpr int kNormTensors = 192, kClipTensors = 136;
constexpr int kNormBlocks = 2048;                // 8 workgroups of 256 threads a CU: one round of the chip
constexpr int kJoined = 1024;                    // up to this many partial sums every clip workgroup adds them up itself: a launch less
constexpr int kMinShift = 11, kMaxShift = 15;    // chunks of 2048 (one 8-element step of every thread) to 32768 elements
constexpr int64_t kBf = int64_t(1) << 62, kOutBf = int64_t(1) << 61, kLen = kOutBf - 1;

struct NormList {
    const void* in[kNormTensors];
    int64_t len[kNormTensors];                   // elements, | kBf
    int first[kNormTensors + 1];                 // first chunk of tensor i; first[n] = all chunks
    int n, shift;
};
struct ClipList {
    const void* in[kClipTensors];
    void* out[kClipTensors];
    int64_t len[kClipTensors];                   // elements, | kBf | kOutBf
    int first[kClipTensors + 1];                 // first workgroup of tensor i
    int n, u, rounds;                            // a workgroup takes u rounds steps of its threads
};

// tensor that chunk c belongs to (first[] grows strictly: tensors without elements are not in the table)
template <typename L>
__device__ __forceinline__ int find_tensor(const L& l, int c) {
    int lo = 0, hi = l.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.first[mid] <= c) lo = mid; else hi = mid;
    }
    return lo;
}

template <bool S> __device__ __forceinline__ u32x4 ldv(const void* p) { return S ? __builtin_nontemporal_load((const u32x4_any*)p) : *(const u32x4_any*)p; }
template <bool S> __device__ __forceinline__ void stv(void* p, const u32x4& v) {
    if (S) __builtin_nontemporal_store(v, (u32x4_any*)p);
    else *(u32x4_any*)p = v;
}

// Squares in 64 bits: the product of two bf16 or fp32 values is exact there, and no gradient that fits its type overflows.
__device__ __forceinline__ void add_square(float x, double& acc) { acc = fma((double)x, (double)x, acc); }

template <bool BF, bool S>
__device__ __forceinline__ void chunk_squares(const void* in, int64_t base, int n, double& acc) {
    constexpr int N = BF ? 8 : 4, U = 4;
    const char* p = (const char*)in + base * (BF ? 2 : 4);
    auto add = [&](const u32x4& v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (BF) { add_square(bflo(v[e]), acc); add_square(bfhi(v[e]), acc); }
            else add_square(__uint_as_float(v[e]), acc);
        }
    };
    const int nv = n / N;
    int i = threadIdx.x;
    for (; i + (U - 1) * 256 < nv; i += U * 256) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = ldv<S>(p + (int64_t)(i + u * 256) * 16);
#pragma unroll
        for (int u = 0; u < U; ++u) add(w[u]);
    }
    for (; i < nv; i += 256) add(ldv<S>(p + (int64_t)i * 16));
    if (nv * N + (int)threadIdx.x < n) add_square(BF ? bf2f(((const bf16_t*)p)[nv * N + threadIdx.x]) : ((const float*)p)[nv * N + threadIdx.x], acc);
}

template <bool S>
__global__ __launch_bounds__(256) void grad_norm_k(NormList l, double* __restrict__ partial) {
    __shared__ double scratch[4];
    double acc = 0.0;
    const int total = l.first[l.n];
    int t = find_tensor(l, blockIdx.x);
    for (int c = blockIdx.x; c < total; c += gridDim.x) {
        while (l.first[t + 1] <= c) ++t;
        const int64_t base = (int64_t)(c - l.first[t]) << l.shift, len = l.len[t];
        const int n = (int)min((len & kLen) - base, (int64_t)1 << l.shift);
        if (len & kBf) chunk_squares<true, S>(l.in[t], base, n, acc);
        else chunk_squares<false, S>(l.in[t], base, n, acc);
    }
    acc = wave_sum_d(acc);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// norm from the partial sums, in a fixed order; every thread returns it
template <int NT>
__device__ __forceinline__ float join_norm(const double* __restrict__ partial, int n, double* scratch) {
    double acc = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += NT) acc += partial[i];
    acc = wave_sum_d(acc);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = acc;
    __syncthreads();
    acc = 0.0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) acc += scratch[w];
    return (float)sqrt(acc);
}

__global__ __launch_bounds__(256) void grad_norm_finish_k(const double* __restrict__ partial, int n, float* __restrict__ norm) {
    __shared__ double scratch[4];
    const float v = join_norm<256>(partial, n, scratch);
    if (threadIdx.x == 0) norm[0] = v;
}

// N elements at element i of a tensor: the step of one thread.  Its store is never wider than 16 bytes, so that a wave's stores lie side by side (8 fp32 values a
// thread, two stores 32 bytes apart, took 1673 us where this takes 1223: 0.87e9 bf16 gradients into fp32).
template <bool BF, int N, bool S> struct Step;
template <bool S> struct Step<true, 8, S> {
    u32x4 v;
    __device__ __forceinline__ void load(const bf16_t* p) { v = ldv<S>(p); }
    __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[2 * e] = bflo(v[e]); f[2 * e + 1] = bfhi(v[e]); }
    }
    __device__ __forceinline__ static void store(bf16_t* p, const float* f) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = pack2bf(f[2 * e], f[2 * e + 1]);
        stv<S>(p, w);
    }
};
template <bool S> struct Step<true, 4, S> {
    u32x2 v;
    __device__ __forceinline__ void load(const bf16_t* p) { v = S ? __builtin_nontemporal_load((const u32x2_any*)p) : *(const u32x2_any*)p; }
    __device__ __forceinline__ void unpack(float* f) const { f[0] = bflo(v[0]); f[1] = bfhi(v[0]); f[2] = bflo(v[1]); f[3] = bfhi(v[1]); }
    __device__ __forceinline__ static void store(bf16_t* p, const float* f) {
        const u32x2 w = {pack2bf(f[0], f[1]), pack2bf(f[2], f[3])};
        if (S) __builtin_nontemporal_store(w, (u32x2_any*)p);
        else *(u32x2_any*)p = w;
    }
};
template <bool S> struct Step<false, 4, S> {
    u32x4 v;
    __device__ __forceinline__ void load(const float* p) { v = ldv<S>(p); }
    __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(v[e]);
    }
    __device__ __forceinline__ static void store(float* p, const float* f) {
        const u32x4 w = {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
        stv<S>(p, w);
    }
};
template <bool BF> struct Type;
template <> struct Type<true> {
    typedef bf16_t T;
    static __device__ __forceinline__ float get(T x) { return bf2f(x); }
    static __device__ __forceinline__ T put(float x) { return f2bf(x); }
};
template <> struct Type<false> {
    typedef float T;
    static __device__ __forceinline__ float get(T x) { return x; }
    static __device__ __forceinline__ T put(float x) { return x; }
};

constexpr int kClipThreads = 1024;
inline __host__ __device__ int step_of(bool in_bf, bool out_bf) { return in_bf && out_bf ? 8 : 4; }

// U rounds of kClipThreads steps, from step `first` of a tensor of n elements on: all loads, then all stores
template <bool IB, bool OB, int U, bool S>
__device__ __forceinline__ void scale_steps(const void* in, void* out, int64_t n, int64_t first, float f) {
    constexpr int N = IB && OB ? 8 : 4;
    const typename Type<IB>::T* p = (const typename Type<IB>::T*)in;
    typename Type<OB>::T* o = (typename Type<OB>::T*)out;
    const int64_t steps = n / N, i = first + threadIdx.x;
    auto scaled = [&](const Step<IB, N, S>& q, int64_t k) {
        float v[N];
        q.unpack(v);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= f;
        Step<OB, N, S>::store(o + k * N, v);
    };
    if (U > 1 && first + U * kClipThreads <= steps) {   // (the same for all threads: no step needs a look at the end)
        Step<IB, N, S> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u].load(p + (i + u * kClipThreads) * N);
#pragma unroll
        for (int u = 0; u < U; ++u) scaled(q[u], i + u * kClipThreads);
        return;
    }
    for (int u = 0; u < U; ++u) {
        const int64_t k = i + u * kClipThreads;
        if (k < steps) {
            Step<IB, N, S> q;
            q.load(p + k * N);
            scaled(q, k);
        } else if (k - steps < n - steps * N) {   // the elements behind the last whole step, one a thread
            const int64_t j = steps * N + (k - steps);
            o[j] = Type<OB>::put(Type<IB>::get(p[j]) * f);
        }
    }
}

// min(1, max_norm / (norm + 1e-6)); NaN stays NaN
__device__ __forceinline__ float clip_factor(float norm, double max_norm) {
    const double q = max_norm / ((double)norm + 1e-6);
    return q >= 1.0 ? 1.f : (float)q;
}

__global__ __launch_bounds__(256) void grad_clip_finish_k(const double* __restrict__ partial, int n, double max_norm, float* __restrict__ norm, float* __restrict__ factor) {
    __shared__ double scratch[4];
    const float v = join_norm<256>(partial, n, scratch);
    if (threadIdx.x == 0) { norm[0] = v; factor[0] = clip_factor(v, max_norm); }
}

// Partial sums given: norm and factor are formed here (and the norm kept by the first workgroup if norm_out is given); otherwise `factor` holds it.
// What a launch touches at one time should lie close together: HBM then serves mixed reads and writes at 6 TB/s and more.  0.87e9 bf16 gradients into fp32, this kernel
// alone: 1024 threads with 8 steps each, loads before stores: 862 us; 256 threads with 32 steps, 4 at a time: 953; one step a thread would take 790 but for this
// kernel's start (table, factor), which makes it 1212.
template <int U, bool S>
__global__ __launch_bounds__(kClipThreads) void grad_clip_k(ClipList l, const double* __restrict__ partial, int parts, const float* __restrict__ factor, float* norm_out,
                                                            double max_norm, int in_place) {
    __shared__ double scratch[kClipThreads / 64];
    float f;
    if (partial) {
        const float nrm = join_norm<kClipThreads>(partial, parts, scratch);
        if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = nrm;
        f = clip_factor(nrm, max_norm);
    } else {
        f = factor[0];
    }
    if (in_place && f == 1.f) return;
    const int t = find_tensor(l, blockIdx.x);
    const int64_t len = l.len[t], n = len & kLen;
    const int rounds = l.rounds;   // (1 unless one tensor alone needs more workgroups than a launch has)
    int64_t first = (int64_t)((int)blockIdx.x - l.first[t]) * rounds * (U * kClipThreads);
    for (int q = 0; q < rounds; ++q, first += U * kClipThreads) {
        if (len & kBf) {
            if (len & kOutBf) scale_steps<true, true, U, S>(l.in[t], l.out[t], n, first, f);
            else scale_steps<true, false, U, S>(l.in[t], l.out[t], n, first, f);
        } else {
            if (len & kOutBf) scale_steps<false, true, U, S>(l.in[t], l.out[t], n, first, f);
            else scale_steps<false, false, U, S>(l.in[t], l.out[t], n, first, f);
        }
    }
}

inline int64_t esize(int dtype) { return dtype == IE_BF16 ? 2 : 4; }

struct Lists {
    const void* const* ptrs;
    const int64_t* numels;
    const int* dtypes;
    void* const* outs;
    const int* out_dtypes;
    int64_t n, elems, bytes;
    int shift;
    bool stream;   // beyond the 256 MB of the last-level cache: past it
};

constexpr int64_t kMostBlocks = (int64_t(1) << 22) - 1;   // workgroups of 1024 threads a launch: fewer than 2^32 threads

int check_list(const char* msg, Lists& l) {
    if (l.n < 0 || l.n > (int64_t(1) << 24) || (l.n > 0 && (!l.ptrs || !l.numels || !l.dtypes))) { ie_set_error(msg); return IE_ERR_INVALID; }
    l.elems = l.bytes = 0;
    for (int64_t i = 0; i < l.n; ++i) {
        if (l.numels[i] < 0 || l.numels[i] > (int64_t(1) << 38) || (l.numels[i] > 0 && !l.ptrs[i]) || (l.dtypes[i] != IE_BF16 && l.dtypes[i] != IE_F32)) {
            ie_set_error(msg);
            return IE_ERR_INVALID;
        }
        l.elems += l.numels[i];
        l.bytes += l.numels[i] * esize(l.dtypes[i]);
        if (l.elems > (int64_t(1) << 48)) { ie_set_error(msg); return IE_ERR_INVALID; }
    }
    // 4096 chunks or more, where the list is long enough for it; longer ones where one tensor stands in it so often that a launch could not hold all its tensors' chunks
    // (the workspace is made for launches of kNormTensors)
    l.shift = kMinShift;
    while ((l.shift < kMaxShift && (l.elems >> l.shift) > 4096) || (l.elems >> l.shift) > kMostBlocks - kNormTensors) ++l.shift;
    l.stream = l.bytes > (int64_t(256) << 20);
    return IE_OK;
}

inline int64_t blocks_of(const NormList& t, const Lists& l, int64_t i) { return (l.numels[i] + (int64_t(1) << t.shift) - 1) >> t.shift; }
inline int64_t blocks_of(const ClipList& t, const Lists& l, int64_t i) {
    const bool in = l.dtypes[i] == IE_BF16, out = l.outs ? l.out_dtypes[i] == IE_BF16 : in;
    const int64_t steps = l.numels[i] / step_of(in, out) + l.numels[i] % step_of(in, out), per = (int64_t)kClipThreads * t.u * t.rounds;   // (whole steps, then elements)
    return (steps + per - 1) / per;
}
inline void fit(NormList&, const Lists&, int64_t) {}   // (the whole list's chunks fit one launch)
inline void fit(ClipList& t, const Lists& l, int64_t i) {
    while (blocks_of(t, l, i) > kMostBlocks) t.rounds *= 2;
}
inline void put_out(NormList&, int, const Lists&, int64_t) {}
inline void put_out(ClipList& t, int k, const Lists& l, int64_t i) {
    t.out[k] = l.outs ? l.outs[i] : (void*)l.ptrs[i];
    if ((l.outs ? l.out_dtypes[i] : l.dtypes[i]) == IE_BF16) t.len[k] |= kOutBf;
}

// the next launch's tensors, from i on; returns where the one after it starts.  A tensor that needs more workgroups alone than a launch has gets several rounds each.
template <int CAP, typename L>
int64_t fill(L& t, int64_t i, const Lists& l) {
    t.n = 0;
    int64_t total = 0;
    for (; i < l.n && t.n < CAP; ++i) {
        if (l.numels[i] == 0) continue;
        if (t.n == 0) fit(t, l, i);
        const int64_t chunks = blocks_of(t, l, i);
        if (total + chunks > kMostBlocks) break;
        t.in[t.n] = l.ptrs[i];
        t.len[t.n] = l.numels[i] | (l.dtypes[i] == IE_BF16 ? kBf : 0);
        put_out(t, t.n, l, i);
        t.first[t.n++] = (int)total;
        total += chunks;
    }
    t.first[t.n] = (int)total;
    return i;
}

// partial sums of the whole list; returns how many
int launch_norm(const Lists& l, double* partial, hipStream_t st) {
    NormList t;
    int used = 0;
    for (int64_t i = 0; i < l.n;) {
        t.shift = l.shift;
        i = fill<kNormTensors>(t, i, l);
        if (t.n == 0) continue;
        const int blocks = std::min(t.first[t.n], kNormBlocks);
        if (l.stream) hipLaunchKernelGGL((grad_norm_k<true>), dim3((unsigned)blocks), dim3(256), 0, st, t, partial + used);
        else hipLaunchKernelGGL((grad_norm_k<false>), dim3((unsigned)blocks), dim3(256), 0, st, t, partial + used);
        used += blocks;
    }
    return used;
}

// every written range is disjoint from every other range, except from the one it is made of (same address, same type)
int check_overlap(const Lists& l) {
    struct Range { const char *a, *b; bool written; };
    std::vector<Range> rs;
    try {
        rs.reserve((size_t)l.n * 2);
        for (int64_t i = 0; i < l.n; ++i) {
            if (l.numels[i] == 0) continue;
            const char* p = (const char*)l.ptrs[i];
            const bool same = !l.outs || (l.outs[i] == l.ptrs[i] && l.out_dtypes[i] == l.dtypes[i]);
            rs.push_back({p, p + l.numels[i] * esize(l.dtypes[i]), same});
            if (same) continue;
            IE_CHECK_ARG(l.outs[i] && (l.out_dtypes[i] == IE_BF16 || l.out_dtypes[i] == IE_F32), "ie_grad_clip: bad output list");
            const char* o = (const char*)l.outs[i];
            rs.push_back({o, o + l.numels[i] * esize(l.out_dtypes[i]), true});
        }
        std::sort(rs.begin(), rs.end(), [](const Range& x, const Range& y) { return x.a < y.a; });
    } catch (...) {
        ie_set_error("ie_grad_clip: out of host memory");
        return IE_ERR_INVALID;
    }
    const char *end_any = nullptr, *end_written = nullptr;   // ends of the ranges before, read or written
    for (const Range& r : rs) {
        IE_CHECK_ARG(!(r.a < end_written || (r.written && r.a < end_any)), "ie_grad_clip: tensors overlap");
        end_any = std::max(end_any, r.b);
        if (r.written) end_written = std::max(end_written, r.b);
    }
    return IE_OK;
}

}  // namespace

extern "C" int64_t ie_grad_norm_workspace(int64_t n) { return n < 0 ? 0 : (n / kNormTensors + 1) * kNormBlocks * 8 + 8; }

extern "C" int ie_grad_norm(const void* const* ptrs, const int64_t* numels, const int* dtypes, int64_t n, void* workspace, float* norm, void* stream) {
    IE_CHECK_ARG(workspace && norm, "ie_grad_norm: null pointer");
    IE_CHECK_ARG(((uintptr_t)workspace & 7) == 0, "ie_grad_norm: the workspace must be 8-byte aligned");
    Lists l = {ptrs, numels, dtypes, nullptr, nullptr, n, 0, 0, 0, false};
    const int rc = check_list("ie_grad_norm: bad tensor list", l);
    if (rc != IE_OK) return rc;
    const int parts = launch_norm(l, (double*)workspace, (hipStream_t)stream);
    hipLaunchKernelGGL(grad_norm_finish_k, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)workspace, parts, norm);
    return ie_launch_status("ie_grad_norm launch");
}

extern "C" int ie_grad_clip(const void* const* ptrs, const int64_t* numels, const int* dtypes, void* const* outs, const int* out_dtypes, int64_t n, double max_norm,
                            void* workspace, float* norm, void* stream) {
    IE_CHECK_ARG(workspace && norm, "ie_grad_clip: null pointer");
    IE_CHECK_ARG(((uintptr_t)workspace & 7) == 0, "ie_grad_clip: the workspace must be 8-byte aligned");
    IE_CHECK_ARG(max_norm >= 0.0, "ie_grad_clip: max_norm must not be negative");
    Lists l = {ptrs, numels, dtypes, outs, out_dtypes, n, 0, 0, 0, false};
    int rc = check_list("ie_grad_clip: bad tensor list", l);
    if (rc != IE_OK) return rc;
    IE_CHECK_ARG(!outs || out_dtypes || n == 0, "ie_grad_clip: null pointer");
    rc = check_overlap(l);
    if (rc != IE_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    double* partial = (double*)workspace;
    const int parts = launch_norm(l, partial, st);
    const bool joined = parts <= kJoined && parts > 0;
    float* factor = (float*)(partial + ie_grad_norm_workspace(n) / 8 - 1);   // behind the partial sums
    if (!joined) hipLaunchKernelGGL(grad_clip_finish_k, dim3(1), dim3(256), 0, st, (const double*)partial, parts, max_norm, norm, factor);
    ClipList t;
    float* norm_out = joined ? norm : nullptr;
    const double* from = joined ? partial : nullptr;
    for (int64_t i = 0; i < n;) {
        // 8 steps a thread where they leave every CU at least 4 workgroups
        t.u = l.elems >= int64_t(8) * 4 * kClipThreads * 1024 ? 8 : 1;
        t.rounds = 1;
        i = fill<kClipTensors>(t, i, l);
        if (t.n == 0) continue;
        const dim3 grid((unsigned)t.first[t.n]);
        const int in_place = outs == nullptr;
        if (t.u == 8) {
            if (l.stream) hipLaunchKernelGGL((grad_clip_k<8, true>), grid, dim3(kClipThreads), 0, st, t, from, parts, (const float*)factor, norm_out, max_norm, in_place);
            else hipLaunchKernelGGL((grad_clip_k<8, false>), grid, dim3(kClipThreads), 0, st, t, from, parts, (const float*)factor, norm_out, max_norm, in_place);
        } else {
            if (l.stream) hipLaunchKernelGGL((grad_clip_k<1, true>), grid, dim3(kClipThreads), 0, st, t, from, parts, (const float*)factor, norm_out, max_norm, in_place);
            else hipLaunchKernelGGL((grad_clip_k<1, false>), grid, dim3(kClipThreads), 0, st, t, from, parts, (const float*)factor, norm_out, max_norm, in_place);
        }
        norm_out = nullptr;
    }
    return ie_launch_status("ie_grad_clip launch");
}

// L2 norm over a list of gradient tensors, and the clipped gradients.  The list travels as launch arguments, a fixed number of tensors a launch.
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

constexpr int kTensors = 96;                     // per launch: 96 x 28 bytes of arguments, well inside the 4 KB a launch carries
constexpr int64_t kChunk = 1 << 15;              // elements a workgroup takes at a time
constexpr int kNormBlocks = 2048;

struct TensorList {
    const void* in[kTensors];
    void* out[kTensors];
    int64_t numel[kTensors];
    int first[kTensors + 1];                     // first chunk of tensor i; first[n] = all chunks
    unsigned char in_bf[kTensors], out_bf[kTensors];
    int n;
};

// tensor that chunk c belongs to (first[] is sorted; tensors without elements own no chunk)
__device__ __forceinline__ int find_tensor(const TensorList& l, int c) {
    int lo = 0, hi = l.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (l.first[mid] <= c) lo = mid; else hi = mid;
    }
    return lo;
}

// Squares in 64 bits: a bf16 or fp32 product is exact there, and no gradient that fits its type overflows.
__global__ __launch_bounds__(256) void grad_norm_k(TensorList l, double* __restrict__ partial) {
    __shared__ double scratch[4];
    double acc = 0.0;
    for (int c = blockIdx.x; c < l.first[l.n]; c += gridDim.x) {
        const int t = find_tensor(l, c);
        const int64_t base = (int64_t)(c - l.first[t]) * kChunk;
        const int n = (int)min(l.numel[t] - base, kChunk);
        if (l.in_bf[t]) {
            const bf16_t* p = (const bf16_t*)l.in[t] + base;
            for (int i = threadIdx.x; i < n / 8; i += 256) {
                const u32x4 v = *(const u32x4_any*)(p + i * 8);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double a = (double)bflo(v[e]), b = (double)bfhi(v[e]);
                    acc = fma(a, a, acc);
                    acc = fma(b, b, acc);
                }
            }
            for (int i = n / 8 * 8 + threadIdx.x; i < n; i += 256) { const double a = (double)bf2f(p[i]); acc = fma(a, a, acc); }
        } else {
            const float* p = (const float*)l.in[t] + base;
            for (int i = threadIdx.x; i < n / 4; i += 256) {
                const u32x4 v = *(const u32x4_any*)(p + i * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) { const double a = (double)__uint_as_float(v[e]); acc = fma(a, a, acc); }
            }
            for (int i = n / 4 * 4 + threadIdx.x; i < n; i += 256) { const double a = (double)p[i]; acc = fma(a, a, acc); }
        }
    }
    acc = wave_sum_d(acc);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

__global__ __launch_bounds__(256) void grad_norm_finish_k(const double* __restrict__ partial, int64_t n, float* __restrict__ norm) {
    __shared__ double scratch[4];
    double acc = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) acc += partial[i];
    acc = wave_sum_d(acc);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) norm[0] = (float)sqrt(scratch[0] + scratch[1] + scratch[2] + scratch[3]);
}

__global__ __launch_bounds__(256) void grad_clip_k(TensorList l, const float* __restrict__ norm, double max_norm, int in_place) {
    const double q = max_norm / ((double)norm[0] + 1e-6);
    const float f = q < 1.0 ? (float)q : q == q ? 1.f : (float)q;
    if (in_place && f == 1.f) return;
    const int c = blockIdx.x, t = find_tensor(l, c);
    const int64_t base = (int64_t)(c - l.first[t]) * kChunk;
    const int n = (int)min(l.numel[t] - base, kChunk);
    if (l.in_bf[t]) {
        const bf16_t* p = (const bf16_t*)l.in[t] + base;
        if (l.out_bf[t]) {
            bf16_t* o = (bf16_t*)l.out[t] + base;
            for (int i = threadIdx.x; i < n / 8; i += 256) {
                u32x4 v = *(const u32x4_any*)(p + i * 8);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = pack2bf(bflo(v[e]) * f, bfhi(v[e]) * f);
                *(u32x4_any*)(o + i * 8) = v;
            }
            for (int i = n / 8 * 8 + threadIdx.x; i < n; i += 256) o[i] = f2bf(bf2f(p[i]) * f);
        } else {
            float* o = (float*)l.out[t] + base;
            for (int i = threadIdx.x; i < n / 4; i += 256) {   // 4 elements a thread: the stores are 16 bytes
                const u32x2 v = *(const u32x2_any*)(p + i * 4);
                u32x4 w;
                w[0] = __float_as_uint(bflo(v[0]) * f); w[1] = __float_as_uint(bfhi(v[0]) * f);
                w[2] = __float_as_uint(bflo(v[1]) * f); w[3] = __float_as_uint(bfhi(v[1]) * f);
                *(u32x4_any*)(o + i * 4) = w;
            }
            for (int i = n / 4 * 4 + threadIdx.x; i < n; i += 256) o[i] = bf2f(p[i]) * f;
        }
    } else {
        const float* p = (const float*)l.in[t] + base;
        if (l.out_bf[t]) {
            bf16_t* o = (bf16_t*)l.out[t] + base;
            for (int i = threadIdx.x; i < n / 4; i += 256) {
                const u32x4 v = *(const u32x4_any*)(p + i * 4);
                u32x2 w;
                w[0] = pack2bf(__uint_as_float(v[0]) * f, __uint_as_float(v[1]) * f);
                w[1] = pack2bf(__uint_as_float(v[2]) * f, __uint_as_float(v[3]) * f);
                *(u32x2_any*)(o + i * 4) = w;
            }
            for (int i = n / 4 * 4 + threadIdx.x; i < n; i += 256) o[i] = f2bf(p[i] * f);
        } else {
            float* o = (float*)l.out[t] + base;
            for (int i = threadIdx.x; i < n / 4; i += 256) {
                u32x4 v = *(const u32x4_any*)(p + i * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                *(u32x4_any*)(o + i * 4) = v;
            }
            for (int i = n / 4 * 4 + threadIdx.x; i < n; i += 256) o[i] = p[i] * f;
        }
    }
}

int check_list(const char* fn, const void* const* ptrs, const int64_t* numels, const int* dtypes, int64_t n) {
    if (n < 0 || n > (int64_t(1) << 24) || (n > 0 && (!ptrs || !numels || !dtypes))) { ie_set_error(fn); return IE_ERR_INVALID; }
    for (int64_t i = 0; i < n; ++i)
        if (numels[i] < 0 || numels[i] > (int64_t(1) << 40) || (numels[i] > 0 && !ptrs[i]) || (dtypes[i] != IE_BF16 && dtypes[i] != IE_F32)) { ie_set_error(fn); return IE_ERR_INVALID; }
    return IE_OK;
}

inline int64_t esize(int dtype) { return dtype == IE_BF16 ? 2 : 4; }
inline int64_t chunks(int64_t numel) { return (numel + kChunk - 1) / kChunk; }

// the next launch's tensors, starting at i: at most kTensors of them and fewer than 2^30 chunks in all
int64_t fill(TensorList& l, int64_t i, const void* const* ptrs, const int64_t* numels, const int* dtypes, void* const* outs, const int* out_dtypes, int64_t n) {
    l.n = 0;
    int64_t total = 0;
    for (; i < n && l.n < kTensors; ++i) {
        if (numels[i] == 0) continue;
        if (total + chunks(numels[i]) > (int64_t(1) << 30)) break;
        l.in[l.n] = ptrs[i];
        l.out[l.n] = outs ? outs[i] : (void*)ptrs[i];
        l.numel[l.n] = numels[i];
        l.in_bf[l.n] = dtypes[i] == IE_BF16;
        l.out_bf[l.n] = outs ? out_dtypes[i] == IE_BF16 : l.in_bf[l.n];
        l.first[l.n++] = (int)total;
        total += chunks(numels[i]);
    }
    l.first[l.n] = (int)total;
    return i;
}

inline int norm_blocks(const TensorList& l) { return std::min(l.first[l.n], kNormBlocks); }

}  // namespace

// launches of kTensors tensors each (one tensor at least), kNormBlocks partial sums each
extern "C" int64_t ie_grad_norm_workspace(int64_t n) { return n < 0 ? 0 : (n / kTensors + 1) * kNormBlocks * 8; }

extern "C" int ie_grad_norm(const void* const* ptrs, const int64_t* numels, const int* dtypes, int64_t n, void* workspace, float* norm, void* stream) {
    IE_CHECK_ARG(workspace && norm, "ie_grad_norm: null pointer");
    const int rc = check_list("ie_grad_norm: bad tensor list", ptrs, numels, dtypes, n);
    if (rc != IE_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    TensorList l;
    int64_t used = 0;
    for (int64_t i = 0; i < n;) {
        i = fill(l, i, ptrs, numels, dtypes, nullptr, nullptr, n);
        if (l.n == 0) continue;
        const int blocks = norm_blocks(l);
        hipLaunchKernelGGL(grad_norm_k, dim3((unsigned)blocks), dim3(256), 0, st, l, (double*)workspace + used);
        used += blocks;
    }
    hipLaunchKernelGGL(grad_norm_finish_k, dim3(1), dim3(256), 0, st, (const double*)workspace, used, norm);
    return ie_launch_status("ie_grad_norm launch");
}

extern "C" int ie_grad_clip(const void* const* ptrs, const int64_t* numels, const int* dtypes, void* const* outs, const int* out_dtypes, int64_t n,
                            const float* norm, double max_norm, void* stream) {
    IE_CHECK_ARG(norm, "ie_grad_clip: null pointer");
    IE_CHECK_ARG(max_norm >= 0.0, "ie_grad_clip: max_norm must not be negative");
    const int rc = check_list("ie_grad_clip: bad tensor list", ptrs, numels, dtypes, n);
    if (rc != IE_OK) return rc;
    IE_CHECK_ARG(!outs || out_dtypes || n == 0, "ie_grad_clip: null pointer");
    // every written range is disjoint from every other range, except from the one it is made of (same address, same type)
    struct Range { const char *a, *b; int64_t owner; bool written; };
    std::vector<Range> rs;
    try {
        rs.reserve((size_t)n * 2);
        for (int64_t i = 0; i < n; ++i) {
            if (numels[i] == 0) continue;
            const char* p = (const char*)ptrs[i];
            const bool same = !outs || (outs[i] == ptrs[i] && out_dtypes[i] == dtypes[i]);
            rs.push_back({p, p + numels[i] * esize(dtypes[i]), i, same});
            if (same) continue;
            IE_CHECK_ARG(outs[i] && (out_dtypes[i] == IE_BF16 || out_dtypes[i] == IE_F32), "ie_grad_clip: bad output list");
            const char* o = (const char*)outs[i];
            rs.push_back({o, o + numels[i] * esize(out_dtypes[i]), i, true});
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
    hipStream_t st = (hipStream_t)stream;
    TensorList l;
    for (int64_t i = 0; i < n;) {
        i = fill(l, i, ptrs, numels, dtypes, outs, out_dtypes, n);
        if (l.n == 0) continue;
        hipLaunchKernelGGL(grad_clip_k, dim3((unsigned)l.first[l.n]), dim3(256), 0, st, l, norm, max_norm, (int)(outs == nullptr));
    }
    return ie_launch_status("ie_grad_clip launch");
}

// Global norm over many tensors, and clipping by it:
//     n = (sum over all tensors of g^2)^(1/2)   or   max |g|            c = min(1, max_norm / (n + 1e-6))            g <- c g
//
// What bounds it: memory.  The norm reads every gradient once; clipping reads it again (from the 256 MB cache where the whole set
// fits there) and writes it.  Tensors are given as a list of pointers, so one launch serves as many of them as fit the kernel's
// 4 KB argument block; they are cut into chunks of kChunk elements and the blocks walk the chunks with a binary search in the
// argument block, so a list of a few large and many tiny tensors keeps every CU busy.
//
// Sums are float64 from the first square on: bfloat16 and float32 gradients reach 1e38, whose square float32 cannot hold, and a
// sum over 1e9 values would lose 2^-24 per step.  (A double-precision fma runs at half the float32 rate here, far above what
// the memory delivers.)  Every block writes one partial, and the partials are summed in a fixed order: the same list gives the same bits.
// The blocks of the clipping pass each sum the (at most 1024 per launch) partials again, from L2, instead of waiting for a
// launch that does it.  When c = 1 and the result goes back in place there is nothing to write and the pass ends there: g * 1 is g.
#include "mmfe_internal.h"

#include <algorithm>
#include <cmath>
#include <new>

namespace mmfe {
namespace {

constexpr int kThreads = 256;
// Elements of a chunk, and blocks (and partials) of one launch: 4 blocks a CU.  200 bfloat16 tensors of 6.5 million: norm 434 us (6.0 TB/s) and
// clipping 1467 us (5.4), with 2048 blocks 464 and 1527; 96 tensors of up to 590 thousand float32: clipping 20.9 us, with chunks of 4096 25.4,
// of 65536 19.7; two small tensors: 5.9 us, 5.4 and 7.5.
constexpr int kChunk = 16384;
constexpr int kMaxBlocks = 1024;
constexpr int kMaxNorm = 160;            // tensors of one launch: 24 bytes each in the argument block
constexpr int kMaxScale = 112;           // 32 bytes each

struct NormArgs {
    const void* x[kMaxNorm];
    int64_t n[kMaxNorm];
    uint32_t first[kMaxNorm];            // first chunk of the tensor
    uint8_t dtype[kMaxNorm];
    uint32_t n_tensors, n_chunks;
    double* partial;
    int max_kind;
};

struct ScaleArgs {
    const void* x[kMaxScale];
    void* y[kMaxScale];
    int64_t n[kMaxScale];
    uint32_t first[kMaxScale];
    uint8_t dtype[kMaxScale];            // of x, and of y << 4
    uint32_t n_tensors, n_chunks;
    const double* partial;
    uint32_t n_partial;
    int max_kind, store;                 // store: this launch's block 0 writes the norm
    float max_norm;
    float* norm;
};
static_assert(sizeof(NormArgs) <= 4000 && sizeof(ScaleArgs) <= 4000, "kernel arguments");

template <typename E>
struct Vec {
    static constexpr int V = 16 / sizeof(E);
    E v[V];
};
template <typename E>
__device__ __forceinline__ Vec<E> load_vec(const E* p) {      // any alignment
    Vec<E> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}

// max that keeps a NaN, as a comparison-based maximum would lose it
__device__ __forceinline__ double max_nan(double a, double b) { return (a > b || a != a) ? a : b; }

__device__ __forceinline__ double wave_reduce(double v, int max_kind) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const double w = __shfl_xor(v, o);
        v = max_kind ? max_nan(v, w) : v + w;
    }
    return v;
}
// the block's total in every thread
__device__ __forceinline__ double block_reduce(double v, int max_kind, double* lds) {
    v = wave_reduce(v, max_kind);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = lds[0];
    for (int w = 1; w < kThreads / 64; ++w) t = max_kind ? max_nan(t, lds[w]) : t + lds[w];
    __syncthreads();
    return t;
}

// last tensor whose first chunk is <= c (tensors without elements have no chunk: their successor has the same first one)
__device__ __forceinline__ int find(const uint32_t* first, int n, uint32_t c) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename E, bool MAX>
__device__ __forceinline__ double chunk_norm(const E* x, int n) {
    constexpr int V = Vec<E>::V;
    double a0 = 0, a1 = 0, a2 = 0, a3 = 0;
    float m = 0;
    bool bad = false;
    auto take = [&](const Vec<E>& v, double& s, double& t) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float f = (float)v.v[j];
            if constexpr (MAX) { m = fmaxf(m, fabsf(f)); bad |= f != f; }
            else {
                const double d = f;
                if (j & 1) t = fma(d, d, t);
                else s = fma(d, d, s);
            }
        }
    };
    int i = threadIdx.x * V;
    const int step = kThreads * V;
    for (; i + 3 * step + V <= n; i += 4 * step) {               // four loads in flight
        const Vec<E> u = load_vec(x + i), v = load_vec(x + i + step), w = load_vec(x + i + 2 * step), z = load_vec(x + i + 3 * step);
        take(u, a0, a1); take(v, a2, a3); take(w, a0, a1); take(z, a2, a3);
    }
    for (; i + V <= n; i += step) take(load_vec(x + i), a0, a1);
    for (; i < n; ++i) {                                         // at most one thread has a part of a vector left
        const float f = (float)x[i];
        if constexpr (MAX) { m = fmaxf(m, fabsf(f)); bad |= f != f; }
        else a0 = fma((double)f, (double)f, a0);
    }
    if constexpr (MAX) return bad ? (double)__builtin_nanf("") : (double)m;
    return (a0 + a1) + (a2 + a3);
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) norm_kernel(const NormArgs p) {
    __shared__ double lds[kThreads / 64];
    double acc = 0;
    for (uint32_t c = blockIdx.x; c < p.n_chunks; c += gridDim.x) {
        const int t = find(p.first, p.n_tensors, c);
        const int64_t at = (int64_t)(c - p.first[t]) * kChunk;
        const int n = (int)(p.n[t] - at < kChunk ? p.n[t] - at : kChunk);
        double v;
        if (p.dtype[t] == MMFE_OUT_F32) v = chunk_norm<float, MAX>(static_cast<const float*>(p.x[t]) + at, n);
        else if (p.dtype[t] == MMFE_OUT_F16) v = chunk_norm<_Float16, MAX>(static_cast<const _Float16*>(p.x[t]) + at, n);
        else v = chunk_norm<__bf16, MAX>(static_cast<const __bf16*>(p.x[t]) + at, n);
        acc = MAX ? max_nan(acc, v) : acc + v;
    }
    acc = block_reduce(acc, MAX, lds);
    if (threadIdx.x == 0) p.partial[blockIdx.x] = acc;
}

// Norm from the partials, in every thread.
__device__ __forceinline__ double total_norm(const double* partial, uint32_t n, int max_kind, double* lds) {
    double v = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) v = max_kind ? max_nan(v, partial[i]) : v + partial[i];
    v = block_reduce(v, max_kind, lds);
    return max_kind ? v : sqrt(v);
}

__global__ void __launch_bounds__(kThreads) total_kernel(const double* partial, uint32_t n, int max_kind, float* norm) {
    __shared__ double lds[kThreads / 64];
    const double v = total_norm(partial, n, max_kind, lds);
    if (threadIdx.x == 0) *norm = (float)v;
}

template <typename E, typename F>
__device__ __forceinline__ void chunk_scale(const E* x, F* y, int n, float c) {
    constexpr int V = Vec<E>::V;
    auto put = [&](const Vec<E>& v, int i) {
        F r[V];
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = (F)((float)v.v[j] * c);
        __builtin_memcpy(y + i, r, sizeof(r));
    };
    int i = threadIdx.x * V;
    const int step = kThreads * V;
    for (; i + step + V <= n; i += 2 * step) {
        const Vec<E> u = load_vec(x + i), v = load_vec(x + i + step);
        put(u, i); put(v, i + step);
    }
    for (; i + V <= n; i += step) put(load_vec(x + i), i);
    for (; i < n; ++i) y[i] = (F)((float)x[i] * c);
}
template <typename E>
__device__ __forceinline__ void chunk_scale_to(const E* x, void* y, int64_t at, int n, float c, int dtype) {
    if (dtype == MMFE_OUT_F32) chunk_scale(x, static_cast<float*>(y) + at, n, c);
    else if (dtype == MMFE_OUT_F16) chunk_scale(x, static_cast<_Float16*>(y) + at, n, c);
    else chunk_scale(x, static_cast<__bf16*>(y) + at, n, c);
}

__global__ void __launch_bounds__(kThreads) scale_kernel(const ScaleArgs p) {
    __shared__ double lds[kThreads / 64];
    const double norm = total_norm(p.partial, p.n_partial, p.max_kind, lds);
    if (p.store && blockIdx.x == 0 && threadIdx.x == 0) *p.norm = (float)norm;
    // rounded once, and the product once; a norm that float32 does not hold counts as the infinity it is returned as: a factor of 0, or NaN where the
    // limit is infinite too
    const float held = (float)norm;
    float c = isinf(held) ? p.max_norm / held : (float)(p.max_norm / (norm + 1e-6));
    if (c > 1.f) c = 1.f;                                        // a NaN norm stays a NaN and reaches every gradient
    for (uint32_t k = blockIdx.x; k < p.n_chunks; k += gridDim.x) {
        const int t = find(p.first, p.n_tensors, k);
        if (c == 1.f && p.x[t] == p.y[t]) continue;
        const int64_t at = (int64_t)(k - p.first[t]) * kChunk;
        const int n = (int)(p.n[t] - at < kChunk ? p.n[t] - at : kChunk);
        const int din = p.dtype[t] & 15, dout = p.dtype[t] >> 4;
        if (din == MMFE_OUT_F32) chunk_scale_to(static_cast<const float*>(p.x[t]) + at, p.y[t], at, n, c, dout);
        else if (din == MMFE_OUT_F16) chunk_scale_to(static_cast<const _Float16*>(p.x[t]) + at, p.y[t], at, n, c, dout);
        else chunk_scale_to(static_cast<const __bf16*>(p.x[t]) + at, p.y[t], at, n, c, dout);
    }
}

int esize(int dtype) { return dtype == MMFE_OUT_F32 ? 4 : 2; }

struct Range {
    uintptr_t lo, hi;
};

}  // namespace
}  // namespace mmfe

using namespace mmfe;

extern "C" {

int64_t mmfe_grad_partials(int64_t n_tensors) {
    if (n_tensors < 0) return 0;
    return ((n_tensors + kMaxNorm - 1) / kMaxNorm + 1) * kMaxBlocks;
}

int mmfe_grad_clip(int64_t n_tensors, const void* const* x, const int64_t* numel, const int32_t* dtype, void* const* out, const int32_t* out_dtype,
                   int32_t norm_kind, float max_norm, double* partials, float* norm, int device, void* hip_stream) {
    if (n_tensors < 0 || partials == nullptr || norm == nullptr || (n_tensors > 0 && (x == nullptr || numel == nullptr || dtype == nullptr))) { set_error("grad_clip: bad argument"); return MMFE_EINVAL; }
    if (norm_kind != MMFE_NORM_2 && norm_kind != MMFE_NORM_MAX) { set_error("grad_clip: unknown norm"); return MMFE_EINVAL; }
    if (out != nullptr && (out_dtype == nullptr || std::isnan(max_norm) || max_norm < 0.f)) { set_error("grad_clip: the limit must be a number >= 0"); return MMFE_EINVAL; }
    for (int64_t i = 0; i < n_tensors; ++i) {
        if (numel[i] < 0 || numel[i] > (1ll << 44) || dtype[i] < MMFE_OUT_F32 || dtype[i] > MMFE_OUT_BF16 || (numel[i] > 0 && x[i] == nullptr)) { set_error("grad_clip: tensor %lld: bad size, type or pointer", (long long)i); return MMFE_EINVAL; }
        if (reinterpret_cast<uintptr_t>(x[i]) % esize(dtype[i]) != 0) { set_error("grad_clip: tensor %lld is not aligned to its elements", (long long)i); return MMFE_EINVAL; }
        if (out != nullptr) {
            if (out_dtype[i] < MMFE_OUT_F32 || out_dtype[i] > MMFE_OUT_BF16 || (numel[i] > 0 && out[i] == nullptr) || reinterpret_cast<uintptr_t>(out[i]) % esize(out_dtype[i]) != 0) { set_error("grad_clip: output %lld: bad type, pointer or alignment", (long long)i); return MMFE_EINVAL; }
            if (numel[i] > 0 && out[i] == x[i] && out_dtype[i] != dtype[i]) { set_error("grad_clip: output %lld overwrites its input with another type", (long long)i); return MMFE_EINVAL; }
        }
    }
    if (out != nullptr && n_tensors > 0) {
        // what is written must not be written or read by another tensor's chunks: the same gradient given twice would be scaled twice
        Range* r = new (std::nothrow) Range[2 * (size_t)n_tensors];
        if (r == nullptr) { set_error("out of host memory"); return MMFE_ENOMEM; }
        size_t k = 0;
        for (int64_t i = 0; i < n_tensors; ++i) {
            if (numel[i] == 0) continue;
            const uintptr_t o = reinterpret_cast<uintptr_t>(out[i]), in = reinterpret_cast<uintptr_t>(x[i]);
            r[k++] = Range{o, o + (uintptr_t)numel[i] * esize(out_dtype[i])};
            if (out[i] != x[i]) r[k++] = Range{in, in + (uintptr_t)numel[i] * esize(dtype[i])};
        }
        std::sort(r, r + k, [](const Range& a, const Range& b) { return a.lo < b.lo; });
        bool overlap = false;
        for (size_t i = 1; i < k; ++i) overlap |= r[i].lo < r[i - 1].hi;
        delete[] r;
        if (overlap) { set_error("grad_clip: two of the tensors share memory (the same gradient given twice?)"); return MMFE_EINVAL; }
    }
    OnDevice on(device);
    if (on.rc) return on.rc;
    hipStream_t stream = reinterpret_cast<hipStream_t>(hip_stream);
    uint32_t n_partial = 0;
    for (int64_t i = 0; i < n_tensors;) {
        NormArgs a;
        a.n_tensors = 0; a.n_chunks = 0; a.max_kind = norm_kind == MMFE_NORM_MAX;
        for (; i < n_tensors && a.n_tensors < (uint32_t)kMaxNorm; ++i) {
            const int64_t chunks = (numel[i] + kChunk - 1) / kChunk;
            if (chunks == 0) continue;
            if (chunks > 0x7fffffffll - a.n_chunks) break;
            const uint32_t t = a.n_tensors++;
            a.x[t] = x[i]; a.n[t] = numel[i]; a.dtype[t] = (uint8_t)dtype[i]; a.first[t] = a.n_chunks;
            a.n_chunks += (uint32_t)chunks;
        }
        if (a.n_chunks == 0) continue;
        const uint32_t grid = a.n_chunks < (uint32_t)kMaxBlocks ? a.n_chunks : kMaxBlocks;
        a.partial = partials + n_partial;
        if (a.max_kind) hipLaunchKernelGGL(norm_kernel<true>, dim3(grid), dim3(kThreads), 0, stream, a);
        else hipLaunchKernelGGL(norm_kernel<false>, dim3(grid), dim3(kThreads), 0, stream, a);
        n_partial += grid;
    }
    bool stored = false;
    if (out != nullptr)
        for (int64_t i = 0; i < n_tensors;) {
            ScaleArgs a;
            a.n_tensors = 0; a.n_chunks = 0; a.max_kind = norm_kind == MMFE_NORM_MAX;
            for (; i < n_tensors && a.n_tensors < (uint32_t)kMaxScale; ++i) {
                const int64_t chunks = (numel[i] + kChunk - 1) / kChunk;
                if (chunks == 0) continue;
                if (chunks > 0x7fffffffll - a.n_chunks) break;
                const uint32_t t = a.n_tensors++;
                a.x[t] = x[i]; a.y[t] = out[i]; a.n[t] = numel[i]; a.dtype[t] = (uint8_t)(dtype[i] | out_dtype[i] << 4); a.first[t] = a.n_chunks;
                a.n_chunks += (uint32_t)chunks;
            }
            if (a.n_chunks == 0) continue;
            a.partial = partials; a.n_partial = n_partial; a.norm = norm; a.max_norm = max_norm; a.store = stored ? 0 : 1;
            stored = true;
            const uint32_t grid = a.n_chunks < (uint32_t)kMaxBlocks ? a.n_chunks : kMaxBlocks;
            hipLaunchKernelGGL(scale_kernel, dim3(grid), dim3(kThreads), 0, stream, a);
        }
    if (!stored) hipLaunchKernelGGL(total_kernel, dim3(1), dim3(kThreads), 0, stream, partials, n_partial, norm_kind == MMFE_NORM_MAX ? 1 : 0, norm);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) { set_error("grad_clip launch failed: %s", hipGetErrorString(e)); return MMFE_EHIP; }
    return MMFE_OK;
}

}  // extern "C"

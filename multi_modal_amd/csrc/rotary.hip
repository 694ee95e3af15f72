// Rotary positions with several axes.  A token carries one position per axis (frequency and time of a spectrogram patch; time,
// height and width of a video patch); pair i of a head turns by the angle  phi = position[axis(i)] * theta_i :
//     (x, y) -> (x cos phi - y sin phi, y cos phi + x sin phi)
// and the elements behind the last pair pass through.  The backward pass is the same map with -phi (it is a rotation).
//
// What bounds it: memory.  Every element is read once and written once with 4 flops in between, so the only arithmetic that
// could show is the angle: it is formed in float64 as a number of TURNS (theta / 2 pi is tabulated in float64), reduced to
// [-1/2, 1/2] and only then rounded to float32, so that positions in the millions keep their phase; float32 products would be
// off by 2^-24 * position radians.  One angle serves the pair in all query and key heads of its token, so a block computes the
// angles of its tokens once, keeps their cosines and sines in LDS, and walks the heads of q and k over them in one launch.
// Rounding: inputs are widened to float32, the result is rounded once to the tensors' type (the fused products are written out, so that
// every path through the kernel gives the same bits).
#include "mmfe_internal.h"

#include <cmath>
#include <new>

namespace mmfe {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;
constexpr int kMaxDim = 1024;
constexpr int kMaxTokens = 16;           // tokens of a block

// n / d for 0 <= n < 2^31 by multiplication; m = ceil(2^(31 + s) / d) with 2^s >= d
struct FastDiv {
    uint32_t d, s;
    uint64_t m;
};
FastDiv fast_div(uint32_t d) {
    FastDiv f{d, 0, 0};
    while ((1ull << f.s) < d) ++f.s;
    f.m = ((1ull << (31 + f.s)) + d - 1) / d;          // <= 2^32
    return f;
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) { return (uint32_t)((n * f.m) >> (31 + f.s)); }

struct Side {                            // q or k
    const void* in;
    void* out;
    int64_t ib, in_, ih, ob, on, oh;     // batch, token and head strides in elements
    int heads;
};

struct RotaryArgs {
    Side side[2];
    const void* pos;
    int64_t pa, pb, pn;                  // axis, batch and token strides of the positions
    const double* turns;                 // R: theta / (2 pi)
    const int* axis;                     // R
    int64_t tokens;                      // B * N
    int N, D, R, T;                      // T: tokens of a block
    int chunks;                          // vectors of a head
    int again;                           // elements may be computed twice (not in place)
    float sign;
    FastDiv dN, dR, dItems, dChunks;     // items of a token = (heads of q + heads of k) * chunks
};

template <typename E>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<_Float16> {
    static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};
template <>
struct Elem<__bf16> {
    static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};

// V elements = 16 bytes, read and written as one instruction whatever their alignment (device memory allows it; an odd section
// size or an odd stride then costs some bandwidth, not a scalar loop)
template <typename E>
struct Vec {
    static constexpr int V = 16 / sizeof(E);
    E v[V];
};
template <typename E>
__device__ __forceinline__ Vec<E> load_vec(const E* p) {
    Vec<E> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
template <typename E>
__device__ __forceinline__ void store_vec(E* p, const Vec<E>& r) { __builtin_memcpy(p, &r, 16); }

// 64 x 192 tokens, 24 heads of 64, float16, out of a packed projection: 15 us (4.9 TB/s); 25088 tokens, 20 heads of 128, bfloat16: 48 us (5.4 TB/s),
// with sections of 15 + 21 + 27 pairs 67.
//
// HALVES: the pair of element i is element i + R; otherwise pairs are (2 i, 2 i + 1).
// Item = one vector of pairs of one head (HALVES: a vector of first and a vector of second elements).  Where the elements do not fill their last
// vector, it is moved back over the one before it, and both compute the same values; in place, or with less than a vector, the elements
// are read one by one, all of them before the first is written (one at a time, each waited for, the sections of 15 + 21 + 27 took 152 us).
template <typename E, typename P, bool HALVES>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int64_t* base = reinterpret_cast<int64_t*>(smem);                        // [T][4]: offsets of a token in q, q out, k, k out
    float2* cs = reinterpret_cast<float2*>(smem + kMaxTokens * 4 * 8);       // [T][R]
    constexpr int V = Vec<E>::V;
    const int64_t first = (int64_t)blockIdx.x * p.T;
    const int T = (int)(p.tokens - first < p.T ? p.tokens - first : p.T);
    const P* pos = static_cast<const P*>(p.pos);
    for (int i = threadIdx.x; i < T * 4; i += kThreads) {
        const uint32_t tok = (uint32_t)(first + (i >> 2));
        const int64_t b = div_by(tok, p.dN), n = tok - (uint32_t)b * (uint32_t)p.N;
        const Side& s = p.side[(i >> 1) & 1];
        base[i] = (i & 1) ? b * s.ob + n * s.on : b * s.ib + n * s.in_;
    }
    for (int i = threadIdx.x; i < T * p.R; i += kThreads) {
        const uint32_t t = div_by((uint32_t)i, p.dR), j = i - t * p.R;
        const uint32_t tok = (uint32_t)first + t;
        const int64_t b = div_by(tok, p.dN), n = tok - (uint32_t)b * (uint32_t)p.N;
        double turn = (double)pos[p.axis[j] * p.pa + b * p.pb + n * p.pn] * p.turns[j];
        turn -= rint(turn);
        float s, c;
        sincospif(2.f * (float)turn, &s, &c);
        cs[i] = make_float2(c, p.sign * s);
    }
    __syncthreads();
    const uint32_t items = (uint32_t)(p.side[0].heads + p.side[1].heads) * (uint32_t)p.chunks;
    for (uint32_t i = threadIdx.x; i < (uint32_t)T * items; i += kThreads) {
        const uint32_t t = div_by(i, p.dItems), r = i - t * items;
        uint32_t h = div_by(r, p.dChunks);
        const int c = (int)(r - h * (uint32_t)p.chunks);
        const int which = h >= (uint32_t)p.side[0].heads;
        if (which) h -= p.side[0].heads;
        const Side& s = p.side[which];
        const E* x = static_cast<const E*>(s.in) + base[4 * t + 2 * which] + h * s.ih;
        E* y = static_cast<E*>(s.out) + base[4 * t + 2 * which + 1] + h * s.oh;
        const float2* a = cs + t * p.R;
        const int n_rot = HALVES ? (p.R + V - 1) / V : (2 * p.R + V - 1) / V;
        if (c >= n_rot) {                                        // the elements without a pair
            const int e = p.again && p.D - 2 * p.R >= V ? min(2 * p.R + (c - n_rot) * V, p.D - V) : 2 * p.R + (c - n_rot) * V;
            if (e + V <= p.D) store_vec(y + e, load_vec(x + e));
            else {
                E u[V];
#pragma unroll
                for (int j = 0; j < V; ++j) u[j] = x[e + j < p.D ? e + j : e];
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (e + j < p.D) y[e + j] = u[j];
            }
        } else if constexpr (HALVES) {
            const int e = p.again && p.R >= V ? min(c * V, p.R - V) : c * V;
            if (e + V <= p.R) {
                Vec<E> u = load_vec(x + e), w = load_vec(x + e + p.R);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 k = a[e + j];
                    const float xu = Elem<E>::get(u.v[j]), xw = Elem<E>::get(w.v[j]);
                    u.v[j] = Elem<E>::put(fmaf(xu, k.x, -(xw * k.y)));
                    w.v[j] = Elem<E>::put(fmaf(xw, k.x, xu * k.y));
                }
                store_vec(y + e, u);
                store_vec(y + e + p.R, w);
            } else {
                E u[V], w[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int i = e + j < p.R ? e + j : e;
                    u[j] = x[i];
                    w[j] = x[i + p.R];
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (e + j >= p.R) continue;
                    const float2 k = a[e + j];
                    const float xu = Elem<E>::get(u[j]), xw = Elem<E>::get(w[j]);
                    y[e + j] = Elem<E>::put(fmaf(xu, k.x, -(xw * k.y)));
                    y[e + j + p.R] = Elem<E>::put(fmaf(xw, k.x, xu * k.y));
                }
            }
        } else {
            const int e = p.again && 2 * p.R >= V ? min(c * V, 2 * p.R - V) : c * V;
            if (e + V <= 2 * p.R) {
                Vec<E> u = load_vec(x + e);
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    const float2 k = a[(e + j) >> 1];
                    const float xu = Elem<E>::get(u.v[j]), xw = Elem<E>::get(u.v[j + 1]);
                    u.v[j] = Elem<E>::put(fmaf(xu, k.x, -(xw * k.y)));
                    u.v[j + 1] = Elem<E>::put(fmaf(xw, k.x, xu * k.y));
                }
                store_vec(y + e, u);
            } else {
                E u[V];
#pragma unroll
                for (int j = 0; j < V; ++j) u[j] = x[e + j < 2 * p.R ? e + j : e];
#pragma unroll
                for (int j = 0; j < V; j += 2) {
                    if (e + j >= 2 * p.R) continue;
                    const float2 k = a[(e + j) >> 1];
                    const float xu = Elem<E>::get(u[j]), xw = Elem<E>::get(u[j + 1]);
                    y[e + j] = Elem<E>::put(fmaf(xu, k.x, -(xw * k.y)));
                    y[e + j + 1] = Elem<E>::put(fmaf(xw, k.x, xu * k.y));
                }
            }
        }
    }
}

typedef void (*kernel_fn)(const RotaryArgs);
template <typename E>
kernel_fn pick(bool wide, bool halves) {
    if (wide) return halves ? &rotary_kernel<E, int64_t, true> : &rotary_kernel<E, int64_t, false>;
    return halves ? &rotary_kernel<E, int32_t, true> : &rotary_kernel<E, int32_t, false>;
}

struct Rotary {
    int device = -1, axes = 0, R = 0;
    bool halves = true;
    double* d_turns = nullptr;
    int* d_axis = nullptr;
};

}  // namespace
}  // namespace mmfe

using namespace mmfe;

extern "C" {

int mmfe_rotary_create(int32_t n_axes, const int32_t* sections, int32_t ladder, int32_t pairing, double base, int device, mmfe_rotary** out_handle) {
    if (out_handle == nullptr) { set_error("out_handle is NULL"); return MMFE_EINVAL; }
    *out_handle = nullptr;
    if (n_axes < 1 || n_axes > kMaxAxes || sections == nullptr) { set_error("rotary: 1 to %d axes, got %d", kMaxAxes, n_axes); return MMFE_EINVAL; }
    if ((ladder != MMFE_ROTARY_SHARED && ladder != MMFE_ROTARY_PER_AXIS) || (pairing != MMFE_ROTARY_HALVES && pairing != MMFE_ROTARY_ADJACENT)) {
        set_error("rotary: unknown ladder or pairing"); return MMFE_EINVAL;
    }
    if (!(base > 0.0) || !std::isfinite(base)) { set_error("rotary: base must be a positive number"); return MMFE_EINVAL; }
    int R = 0;
    for (int a = 0; a < n_axes; ++a) {
        if (sections[a] < 0 || sections[a] > kMaxDim / 2) { set_error("rotary: section %d has %d pairs (0 to %d)", a, sections[a], kMaxDim / 2); return MMFE_EINVAL; }
        R += sections[a];
    }
    if (R < 1 || R > kMaxDim / 2) { set_error("rotary: the sections hold %d pairs (1 to %d)", R, kMaxDim / 2); return MMFE_EINVAL; }
    const int ndev = mmfe_device_count();
    if (ndev <= 0) { set_error("no HIP device available: this library has no CPU path"); return MMFE_ENODEVICE; }
    if (device < 0 || device >= ndev) { set_error("device %d out of range (%d devices)", device, ndev); return MMFE_ENODEVICE; }
    double turns[kMaxDim / 2];
    int axis[kMaxDim / 2];
    for (int a = 0, i = 0; a < n_axes; ++a)
        for (int j = 0; j < sections[a]; ++j, ++i) {
            const double e = ladder == MMFE_ROTARY_SHARED ? (double)i / R : (double)j / sections[a];
            turns[i] = std::pow(base, -e) / (2.0 * M_PI);
            axis[i] = a;
        }
    Rotary* h = new (std::nothrow) Rotary();
    if (h == nullptr) { set_error("out of host memory"); return MMFE_ENOMEM; }
    h->device = device; h->axes = n_axes; h->R = R; h->halves = pairing == MMFE_ROTARY_HALVES;
    OnDevice on(device);
    int rc = on.rc;
    if (rc == MMFE_OK && (hipMalloc((void**)&h->d_turns, R * sizeof(double)) != hipSuccess || hipMalloc((void**)&h->d_axis, R * sizeof(int)) != hipSuccess ||
        hipMemcpy(h->d_turns, turns, R * sizeof(double), hipMemcpyHostToDevice) != hipSuccess ||
        hipMemcpy(h->d_axis, axis, R * sizeof(int), hipMemcpyHostToDevice) != hipSuccess || hipDeviceSynchronize() != hipSuccess)) {
        set_error("rotary: uploading the frequencies failed");
        rc = MMFE_EHIP;
    }
    if (rc) { (void)hipFree(h->d_turns); (void)hipFree(h->d_axis); delete h; return rc; }
    *out_handle = reinterpret_cast<mmfe_rotary*>(h);
    return MMFE_OK;
}

int mmfe_rotary_destroy(mmfe_rotary* handle) {
    Rotary* h = reinterpret_cast<Rotary*>(handle);
    if (h == nullptr) return MMFE_OK;
    OnDevice on(h->device);
    (void)hipFree(h->d_turns); (void)hipFree(h->d_axis);
    delete h;
    return MMFE_OK;
}

int mmfe_rotary_run(const mmfe_rotary* handle, const mmfe_rotary_args* a, void* hip_stream) {
    const Rotary* h = reinterpret_cast<const Rotary*>(handle);
    if (h == nullptr || a == nullptr || a->struct_size != (int32_t)sizeof(mmfe_rotary_args)) { set_error("rotary: NULL handle or arguments of another version"); return MMFE_EINVAL; }
    if (a->dtype < MMFE_OUT_F32 || a->dtype > MMFE_OUT_BF16) { set_error("rotary: unknown dtype"); return MMFE_EINVAL; }
    if (a->n_batch < 0 || a->n_tokens < 0 || a->heads_q < 0 || a->heads_k < 0) { set_error("rotary: negative size"); return MMFE_EINVAL; }
    if (a->dim < 2 * h->R || a->dim > kMaxDim) { set_error("rotary: head size %d, the sections need %d to %d", a->dim, 2 * h->R, kMaxDim); return MMFE_EINVAL; }
    if (a->heads_q > 65536 || a->heads_k > 65536) { set_error("rotary: too many heads"); return MMFE_EINVAL; }
    if (a->n_batch == 0 || a->n_tokens == 0 || a->heads_q + a->heads_k == 0) return MMFE_OK;
    if (a->n_tokens > 0x7fffff00ll || a->n_batch > 0x7fffff00ll / a->n_tokens) { set_error("rotary: more than 2^31 tokens in one call"); return MMFE_EINVAL; }
    if (a->positions == nullptr || (a->heads_q > 0 && (a->q == nullptr || a->q_out == nullptr)) || (a->heads_k > 0 && (a->k == nullptr || a->k_out == nullptr))) {
        set_error("rotary: NULL data pointer"); return MMFE_EINVAL;
    }
    RotaryArgs p{};
    p.side[0] = Side{a->q, a->q_out, a->q_stride[0], a->q_stride[1], a->q_stride[2], a->q_out_stride[0], a->q_out_stride[1], a->q_out_stride[2], a->heads_q};
    p.side[1] = Side{a->k, a->k_out, a->k_stride[0], a->k_stride[1], a->k_stride[2], a->k_out_stride[0], a->k_out_stride[1], a->k_out_stride[2], a->heads_k};
    p.pos = a->positions; p.pa = a->pos_stride[0]; p.pb = a->pos_stride[1]; p.pn = a->pos_stride[2];
    p.turns = h->d_turns; p.axis = h->d_axis;
    p.tokens = a->n_batch * a->n_tokens; p.N = (int)a->n_tokens; p.D = a->dim; p.R = h->R; p.sign = a->inverse ? -1.f : 1.f;
    const int V = a->dtype == MMFE_OUT_F32 ? 4 : 8;
    const bool copy_rest = !(a->q == a->q_out && a->k == a->k_out);      // in place, the elements without a pair stay where they are
    p.again = !((a->heads_q > 0 && a->q == a->q_out) || (a->heads_k > 0 && a->k == a->k_out));
    p.chunks = ((h->halves ? h->R : 2 * h->R) + V - 1) / V + (copy_rest ? (a->dim - 2 * h->R + V - 1) / V : 0);
    const int64_t items = (int64_t)(a->heads_q + a->heads_k) * p.chunks;
    // A block takes as many tokens as give its threads 4 items each, within the LDS image of the angles (16 KB) and within what
    // leaves two blocks for every CU.  One token a block: 20000 tokens, 12 heads of 64: 21.6 us in place of 12.6; one new token of 8 streams in one block:
    // 4.0 us, in 8 blocks 3.0; 8 items a thread: 20000 tokens, 12 heads of 128, float32: 49 us, with 4 42.
    int64_t T = (4 * kThreads + items - 1) / items;
    if (T > kMaxTokens) T = kMaxTokens;
    if (T > 2048 / h->R) T = 2048 / h->R;
    if (T > p.tokens / 512) T = p.tokens / 512;
    if (T < 1) T = 1;
    p.T = (int)T;
    p.dN = fast_div((uint32_t)p.N); p.dR = fast_div((uint32_t)p.R); p.dItems = fast_div((uint32_t)items); p.dChunks = fast_div((uint32_t)p.chunks);
    if (too_many_blocks((p.tokens + p.T - 1) / p.T, kThreads)) { set_error("rotary: too many tokens in one call"); return MMFE_EINVAL; }
    OnDevice on(h->device);
    if (on.rc) return on.rc;
    const size_t lds = kMaxTokens * 4 * 8 + (size_t)p.T * p.R * 8;
    const kernel_fn fn = a->dtype == MMFE_OUT_F32 ? pick<float>(a->pos_64, h->halves) : a->dtype == MMFE_OUT_F16 ? pick<_Float16>(a->pos_64, h->halves) : pick<__bf16>(a->pos_64, h->halves);
    hipLaunchKernelGGL(fn, dim3((uint32_t)((p.tokens + p.T - 1) / p.T)), dim3(kThreads), lds, reinterpret_cast<hipStream_t>(hip_stream), p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) { set_error("rotary launch failed: %s", hipGetErrorString(e)); return MMFE_EHIP; }
    return MMFE_OK;
}

}  // extern "C"

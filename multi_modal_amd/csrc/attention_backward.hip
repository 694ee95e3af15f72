// Gradients of attention (attention.hip), from q, k, v, the output o, its gradient g and the saved lse:
//     p_ij = e^(s_ij - lse_i)      delta_i = g_i . o_i      dp_ij = g_i . v_j      ds_ij = p_ij (dp_ij - delta_i) (1 - tanh^2 of a capped score)
//     dv_j = sum_i p_ij g_i        dk_j = scale sum_i ds_ij q_i                     dq_i = scale sum_j ds_ij k_j
// the sums over i running over all query heads that share the key head.
//
// Two passes, each recomputing the scores: one block per 128 keys walks the rows (dk, dv), one block per 128 rows walks the keys (dq).
// That is 7 matrix products where one pass with atomic additions into dq would need 5, but every sum has one owner and a fixed
// order: the same call gives the same bits.  As in the forward pass, products are arranged so that a result is the next operand: the key pass
// forms scores as rows x keys (a lane has one key), the row pass as keys x rows (a lane has one row); sums over the lane's own index stay in
// registers for the whole walk.
//
// What is rounded: p and ds to the 16-bit type, for the second products; dp and all sums are float32, and delta is formed from o and
// the rest that its rounding lost.  Short documents add second products with what the rounding of p and ds lost, as the forward pass does.  float16 has 5
// exponent bits, which products p (dp - delta) of long rows and small gradients fall out of.  Its values are therefore scaled by
// powers of two, exactly: p by 2^8, and (dp - delta) by phi = 2^(6 - ceil(log2(max |g_i| max |v_j|))) per document and key head, with which
// |dp| phi <= 2^6 by Cauchy and Schwarz, |delta| phi too (o is a mean of v), and |ds| <= 2^15: nothing overflows, and values down to
// 2^-29 of the largest possible are normal numbers.  bfloat16 needs none of this (phi = 1, p as it is).
#include "attention_tiles.h"

#include <cmath>

namespace mmfe {
using namespace attn;

namespace attn {
int padded_dim(int dim);
bool bad_rows(const char* name, const void* ptr, const int64_t* s);
int make_problem(const mmfe_attention_args* a, Problem& p);
int64_t count_tiles(Problem& p, int64_t rows, int tile_rows);
int launched(const char* what);
}  // namespace attn

namespace {

struct BackwardArgs {
    Problem p;
    Rows out, g, dq, dk, dv;
    const char* rest;                 // like out: what its rounding lost, or NULL
    const float* lse;
    float *lse2, *delta;              // like lse: lse in log2 units (less the shift of p; +inf for rows without keys), g . o
    int64_t lse_b, lse_h;
    unsigned *norm_g, *norm_v;        // float16: largest squared row norms, per document and key head (bit patterns of floats >= 0)
};

template <bool BF>
constexpr float kShift = BF ? 0.f : 8.f;

__device__ __forceinline__ void block_max(float v, unsigned* to) {
    __shared__ float m[kWaves];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) m[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) atomicMax(to, __float_as_uint(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))));     // a maximum has no order
}

// delta and lse2 of 128 rows of one head; float16: and the rows' largest gradient norm.  DP / 8 lanes share a row.
template <bool BF, int DP>
__global__ void __launch_bounds__(kThreads) delta_kernel(const BackwardArgs a) {
    const Problem& p = a.p;
    Doc d;
    if (!find_doc<true>(p, blockIdx.x / p.heads, kRows, d)) return;
    const int head = blockIdx.x % p.heads;
    constexpr int kLanes = DP / 8;
    const int e = (threadIdx.x & (kLanes - 1)) * 8;
    float biggest = 0.f;
    for (int r = threadIdx.x / kLanes; r < kRows; r += kThreads / kLanes) {
        const int row = d.tile * kRows + r;
        float dot = 0.f, sq = 0.f;
        if (row < d.nq && e < p.dim) {
            const int64_t at = 2 * (d.batch * a.out.b + (d.q0 + row) * a.out.n + head * a.out.h + e);
            const u32x4 o = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.out.p) + at);
            u32x4 rest{0, 0, 0, 0};
            if (a.rest != nullptr) rest = *reinterpret_cast<const u32x4*>(a.rest + at);
            const u32x4 g = *reinterpret_cast<const u32x4*>(row_base(a.g, d, d.q0 + row, head) + 2 * e);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = widen<BF>(g[i >> 1], i & 1);
                dot = fmaf(x, widen<BF>(o[i >> 1], i & 1) + widen<BF>(rest[i >> 1], i & 1), dot);
                if constexpr (!BF) sq = fmaf(x, x, sq);
            }
        }
#pragma unroll
        for (int m = 1; m < kLanes; m <<= 1) {
            dot += __shfl_xor(dot, m);
            if constexpr (!BF) sq += __shfl_xor(sq, m);
        }
        biggest = fmaxf(biggest, sq);
        if (row < d.nq && e == 0) {
            const int64_t at = d.batch * a.lse_b + head * a.lse_h + d.q0 + row;
            const float l = a.lse[at];
            a.lse2[at] = l == -INFINITY ? INFINITY : l * kLog2e - kShift<BF>;
            a.delta[at] = l == -INFINITY ? 0.f : dot;
        }
    }
    if constexpr (!BF)
        if (d.index >= 0) block_max(biggest, a.norm_g + (int64_t)d.index * p.kv_heads + head / p.group);
}

// float16: largest squared norm of 128 rows of v
template <int DP>
__global__ void __launch_bounds__(kThreads) norm_kernel(const BackwardArgs a) {
    const Problem& p = a.p;
    Doc d;
    if (!find_doc<false>(p, blockIdx.x / p.kv_heads, kRows, d) || d.index < 0) return;
    const int head = blockIdx.x % p.kv_heads;
    constexpr int kLanes = DP / 8;
    const int e = (threadIdx.x & (kLanes - 1)) * 8;
    float biggest = 0.f;
    for (int r = threadIdx.x / kLanes; r < kRows; r += kThreads / kLanes) {
        const int row = d.tile * kRows + r;
        float sq = 0.f;
        if (row < d.nk && e < p.dim) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(row_base(p.v, d, d.k0 + row, head) + 2 * e);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = widen<false>(v[i >> 1], i & 1);
                sq = fmaf(x, x, sq);
            }
        }
#pragma unroll
        for (int m = 1; m < kLanes; m <<= 1) sq += __shfl_xor(sq, m);
        biggest = fmaxf(biggest, sq);
    }
    block_max(biggest, a.norm_v + (int64_t)d.index * p.kv_heads + head);
}

template <bool BF>
__device__ __forceinline__ float find_phi(const BackwardArgs& a, const Doc& d, int kvh) {
    if constexpr (BF) return 1.f;
    else {
        if (d.index < 0) return 1.f;
        const int64_t i = (int64_t)d.index * a.p.kv_heads + kvh;
        const float bound = sqrtf(__uint_as_float(a.norm_g[i])) * sqrtf(__uint_as_float(a.norm_v[i]));
        if (!(bound > 0.f) || !(bound < 3e38f)) return 1.f;
        int e;
        (void)frexpf(bound, &e);                       // bound < 2^e
        return ldexpf(1.f, 6 - e);
    }
}

// How scores leave the linear form, in log2 units.
struct Shape {
    bool cap, bias;
    float c, slope, cap_in, cap_out;
    __device__ __forceinline__ Shape(const Problem& p, int head) {
        cap = p.cap > 0.f;
        bias = p.slopes != nullptr;
        c = p.scale * kLog2e;
        slope = bias ? p.slopes[head] * kLog2e : 0.f;
        cap_in = cap ? p.scale / p.cap : 0.f;
        cap_out = p.cap * kLog2e;
    }
};

// rows [0, dim) of result registers to 16-bit memory, times `by`
template <bool BF, int DP>
__device__ __forceinline__ void store_rows(char* to, const f32x16 (&o)[DP / 32], int dim, float by, bool some) {
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = 32 * i + 8 * g;
            if (e < dim) {
                u32x2 w{0, 0};
                if (some) w = u32x2{pack2<BF>(o[i][4 * g] * by, o[i][4 * g + 1] * by), pack2<BF>(o[i][4 * g + 2] * by, o[i][4 * g + 3] * by)};
                *reinterpret_cast<u32x2*>(to + 2 * (e + 4 * half)) = w;
            }
        }
}

template <bool BF, int DP>
__device__ __forceinline__ void load_rows(u32x4 (&f)[DP / 16], const char* row, int dim, bool some) {
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        f[s] = u32x4{0, 0, 0, 0};
        if (some && 16 * s + 8 * half < dim) f[s] = *reinterpret_cast<const u32x4*>(row + 32 * s + 16 * half);
    }
}

// dk and dv of 128 keys, 32 per wave.  Head sizes up to 64: 8 waves, the second four taking the second 32 rows of every tile, whose sums join
// the first four's through LDS at the end; a block then takes half as long, and the longest one (4096 keys of a causal document,
// three heads' rows behind it) bounds the launch: FIXME.  Head size 128 has no registers for that.
template <int DP>
constexpr int kKeyWaves = DP == 128 ? 4 : 8;

template <bool BF, int DP>
__global__ void __launch_bounds__(64 * kKeyWaves<DP>, 1) keys_kernel(const BackwardArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];       // 2 x [q tile][g tile][lse2][delta]
    const Problem& p = a.p;
    constexpr int kTileBytes = kTile * DP * 2;
    constexpr int kBuf = 2 * kTileBytes + 2 * kTile * 4;
    constexpr int kW = kKeyWaves<DP>;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int part = wave >> 2;                                       // which of the tile's 32 rows (8 waves)
    const int kvh = blockIdx.x % p.kv_heads;
    Doc d;
    if (!find_doc<false>(p, blockIdx.x / p.kv_heads, kRows, d)) return;
    const int key0 = d.tile * kRows, w0 = key0 + 32 * (wave & 3), key = w0 + col;
    const int nq = d.nq, nk = d.nk, off = nk - nq;
    // rows [first, nq) see key j: all of them, or those from j - off on
    auto first_row = [&](int j) { return p.causal && j >= d.prefix ? max(0, j - off) : 0; };
    const int block_first = key0 < nk ? first_row(key0) : nq;
    const int wave_first = w0 < nk ? first_row(w0) : nq;
    const int wave_full = first_row(min(w0 + 31, nk - 1));            // from here on every row sees all keys of the wave
    const int my_first = first_row(key);
    const int t_first = block_first / kTile, t_end = block_first < nq ? (nq + kTile - 1) / kTile : t_first;
    const int per_head = t_end - t_first, steps = per_head * p.group;

    Loader<DP, kTile, kW> lq, lg;
    lq.init(p.dim, p.q.n, wave);
    lg.init(p.dim, a.g.n, wave);
    const unsigned lds0 = lds_address(smem);
    auto stage = [&](int g, int t, int buf) {
        const int head = kvh * p.group + g, r0 = t * kTile;
        const unsigned dst = uniform(lds0 + buf * kBuf);
        lq.load(row_base(p.q, d, d.q0 + r0, head), nq - r0, p.dim, p.q.n, dst, wave);
        lg.load(row_base(a.g, d, d.q0 + r0, head), nq - r0, p.dim, a.g.n, dst + kTileBytes, wave);
        const int64_t at = d.batch * a.lse_b + head * a.lse_h + d.q0 + r0;
        const unsigned mine = 4 * min(lane, nq - 1 - r0);
        if (wave == 0) dma4(a.lse2 + at, mine, dst + 2 * kTileBytes);
        if (wave == 1) dma4(a.delta + at, mine, dst + 2 * kTileBytes + kTile * 4);
    };
    if (steps > 0) stage(0, t_first, 0);
    u32x4 kf[DP / 16], vf[DP / 16];
    {
        const int r = max(0, min(key, nk - 1));
        load_rows<BF, DP>(kf, row_base(p.k, d, d.k0 + r, kvh), p.dim, nk > 0);
        load_rows<BF, DP>(vf, row_base(p.v, d, d.k0 + r, kvh), p.dim, nk > 0);
    }
    const float phi = find_phi<BF>(a, d, kvh);
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = f32x16{};

    wait_all();
    arrived(kf);
    arrived(vf);
    int g = 0, t = t_first;
    for (int step = 0; step < steps; ++step) {
        wait_all();
        block_sync();
        int gn = g, tn = t + 1;
        if (tn == t_end) { tn = t_first; ++gn; }
        if (step + 1 < steps) stage(gn, tn, (step + 1) & 1);
        const char* qt = smem + (step & 1) * kBuf;
        const char* gt = qt + kTileBytes;
        const float* lse2 = reinterpret_cast<const float*>(gt + kTileBytes);
        const float* delta = lse2 + kTile;
        const Shape sh(p, kvh * p.group + g);
#pragma unroll 1
        for (int b = kW == 8 ? part : 0; b < (kW == 8 ? part + 1 : 2); ++b) {
            const int i0 = t * kTile + 32 * b;
            if (i0 + 32 <= wave_first || i0 >= nq) continue;
            f32x16 x{}, dp{};
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) x = mfma<BF>(read_rows<DP>(qt, 32 * b, s), kf[s], x);
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) dp = mfma<BF>(read_rows<DP>(gt, 32 * b, s), vf[s], dp);
            f32x16 th{};
            if (sh.cap) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    th[i] = tanh_fast(x[i] * sh.cap_in);
                    x[i] = sh.cap_out * th[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] *= sh.c;
            }
            if (sh.bias) {
                const float at = (float)(i0 + 4 * half + off - key);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] -= sh.slope * fabsf(at + (float)reg_row(i));
            }
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const float4 l4 = *reinterpret_cast<const float4*>(lse2 + 32 * b + 8 * q4 + 4 * half);
                const float4 d4 = *reinterpret_cast<const float4*>(delta + 32 * b + 8 * q4 + 4 * half);
                const float l[4] = {l4.x, l4.y, l4.z, l4.w}, de[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 4 * q4 + r;
                    x[i] = exp2_fast(x[i] - l[r]);
                    dp[i] = fmaf(dp[i], phi, -de[r] * phi);
                }
            }
            if (i0 < wave_full || i0 + 32 > nq) {
                const int lo = my_first - i0 - 4 * half, hi = nq - i0 - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = reg_row(i) >= lo && reg_row(i) < hi ? x[i] : 0.f;
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const u32x4 pf = operand<BF>(x, s);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) dv[i] = mfma<BF>(read_cols<DP>(gt, 32 * b + 16 * s, 32 * i), pf, dv[i]);
                if (nk <= kShortKeys) {
                    const u32x4 rf = operand_rest<BF>(x, s, pf);
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) dv[i] = mfma<BF>(read_cols<DP>(gt, 32 * b + 16 * s, 32 * i), rf, dv[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= dp[i];
            if (sh.cap) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] *= 1.f - th[i] * th[i];
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const u32x4 df = operand<BF>(x, s);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) dk[i] = mfma<BF>(read_cols<DP>(qt, 32 * b + 16 * s, 32 * i), df, dk[i]);
                if (nk <= kShortKeys) {
                    const u32x4 rf = operand_rest<BF>(x, s, df);
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) dk[i] = mfma<BF>(read_cols<DP>(qt, 32 * b + 16 * s, 32 * i), rf, dk[i]);
                }
            }
        }
        g = gn;
        t = tn;
    }
    if constexpr (kW == 8) {
        wait_all();
        block_sync();
        float* meet = reinterpret_cast<float*>(smem) + (wave & 3) * (DP / 32) * 2 * 16 * 64 + lane;
        if (part == 1)
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    meet[(i * 32 + r) * 64] = dk[i][r];
                    meet[(i * 32 + 16 + r) * 64] = dv[i][r];
                }
        __syncthreads();
        if (part == 1) return;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dk[i][r] += meet[(i * 32 + r) * 64];
                dv[i][r] += meet[(i * 32 + 16 + r) * 64];
            }
    }
    if (key >= d.rows) return;
    const float back = __builtin_amdgcn_exp2f(-kShift<BF>);
    store_rows<BF, DP>(const_cast<char*>(row_base(a.dk, d, d.k0 + key, kvh)), dk, p.dim, p.scale * back / phi, key < nk && steps > 0 && nk > 1);      // a softmax over one key is constant
    store_rows<BF, DP>(const_cast<char*>(row_base(a.dv, d, d.k0 + key, kvh)), dv, p.dim, back, key < nk && steps > 0);
}

// dq of 128 rows (32 per wave)
template <bool BF, int DP>
__global__ void __launch_bounds__(kThreads, 2) rows_kernel(const BackwardArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];       // 2 x [k tile][v tile]
    const Problem& p = a.p;
    constexpr int kTileBytes = kTile * DP * 2;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    Doc d;
    if (!find_doc<true>(p, blockIdx.x / p.heads, kRows, d)) return;
    const int head = head_of(p, blockIdx.x % p.heads), kvh = head / p.group;
    const int row0 = d.tile * kRows, w0 = row0 + 32 * wave, row = w0 + col;
    const int nq = d.nq, nk = d.nk, off = nk - nq;
    auto limit = [&](int r) {
        if (r >= nq) r = nq - 1;
        return p.causal ? min(nk, max(d.prefix, r + off + 1)) : nk;
    };
    const int block_lim = row0 < nq ? limit(row0 + kRows - 1) : 0;
    const int wave_lim = w0 < nq ? limit(w0 + 31) : 0;
    const int full_lim = w0 < nq ? limit(w0) : 0;
    const int lim = row < nq ? limit(row) : 0;
    const int n_tiles = block_lim > 0 ? (block_lim + kTile - 1) / kTile : 0;

    Loader<DP, kTile, kWaves> lk, lv;
    lk.init(p.dim, p.k.n, wave);
    lv.init(p.dim, p.v.n, wave);
    const unsigned lds0 = lds_address(smem);
    auto stage = [&](int t, int buf) {
        const unsigned dst = uniform(lds0 + buf * 2 * kTileBytes);
        lk.load(row_base(p.k, d, d.k0 + (int64_t)t * kTile, kvh), nk - t * kTile, p.dim, p.k.n, dst, wave);
        lv.load(row_base(p.v, d, d.k0 + (int64_t)t * kTile, kvh), nk - t * kTile, p.dim, p.v.n, dst + kTileBytes, wave);
    };
    if (n_tiles > 0) stage(0, 0);
    u32x4 qf[DP / 16], gf[DP / 16];
    const int r = max(0, min(row, nq - 1));
    load_rows<BF, DP>(qf, row_base(p.q, d, d.q0 + r, head), p.dim, nq > 0);
    load_rows<BF, DP>(gf, row_base(a.g, d, d.q0 + r, head), p.dim, nq > 0);
    const int64_t at = d.batch * a.lse_b + head * a.lse_h + d.q0 + r;
    const float phi = find_phi<BF>(a, d, kvh);
    const float lse2 = nq > 0 ? a.lse2[at] : 0.f;
    const float delta = nq > 0 ? -a.delta[at] * phi : 0.f;
    const Shape sh(p, head);
    f32x16 dq[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dq[i] = f32x16{};

    wait_all();
    arrived(qf);
    arrived(gf);
    for (int t = 0; t < n_tiles; ++t) {
        wait_all();
        block_sync();
        if (t + 1 < n_tiles) stage(t + 1, (t + 1) & 1);
        const char* kt = smem + (t & 1) * 2 * kTileBytes;
        const char* vt = kt + kTileBytes;
#pragma unroll 1
        for (int b = 0; b < 2; ++b) {
            const int j0 = t * kTile + 32 * b;
            if (j0 >= wave_lim) break;
            f32x16 x{}, dp{};
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) x = mfma<BF>(read_rows<DP>(kt, 32 * b, s), qf[s], x);
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) dp = mfma<BF>(read_rows<DP>(vt, 32 * b, s), gf[s], dp);
            f32x16 th{};
            if (sh.cap) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    th[i] = tanh_fast(x[i] * sh.cap_in);
                    x[i] = sh.cap_out * th[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] *= sh.c;
            }
            if (sh.bias) {
                const float far = (float)(row + off - j0 - 4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] -= sh.slope * fabsf(far - (float)reg_row(i));
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = exp2_fast(x[i] - lse2);
                dp[i] = fmaf(dp[i], phi, delta);
            }
            if (j0 + 32 > full_lim) {
                const int left = lim - j0 - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = reg_row(i) < left ? x[i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= dp[i];
            if (sh.cap) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] *= 1.f - th[i] * th[i];
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const u32x4 df = operand<BF>(x, s);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) dq[i] = mfma<BF>(read_cols<DP>(kt, 32 * b + 16 * s, 32 * i), df, dq[i]);
                if (nk <= kShortKeys) {
                    const u32x4 rf = operand_rest<BF>(x, s, df);
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) dq[i] = mfma<BF>(read_cols<DP>(kt, 32 * b + 16 * s, 32 * i), rf, dq[i]);
                }
            }
        }
    }
    if (row >= d.rows) return;
    store_rows<BF, DP>(const_cast<char*>(row_base(a.dq, d, d.q0 + row, head)), dq, p.dim, p.scale * __builtin_amdgcn_exp2f(-kShift<BF>) / phi, lim > 1);       // a softmax over one key is constant
}

template <bool BF, int DP>
int launch(BackwardArgs& b, int64_t q_rows, int64_t k_rows, hipStream_t stream) {
    Problem& p = b.p;
    int rc = MMFE_OK, blocks = 1, cus = 256;
    const size_t tiles_lds = 4 * (size_t)kTile * DP * 2, meet_lds = 4 * (size_t)(DP / 32) * 2 * 16 * 64 * 4;
    const size_t keys_lds = kKeyWaves<DP> == 8 && meet_lds > tiles_lds + 4 * kTile * 4 ? meet_lds : tiles_lds + 4 * kTile * 4;
    if ((rc = kernel_prepare(reinterpret_cast<const void*>(&keys_kernel<BF, DP>), 64 * kKeyWaves<DP>, keys_lds, &blocks, &cus)) != MMFE_OK) return rc;
    if ((rc = kernel_prepare(reinterpret_cast<const void*>(&rows_kernel<BF, DP>), kThreads, tiles_lds, &blocks, &cus)) != MMFE_OK) return rc;
    const int64_t tq = count_tiles(p, q_rows, kRows);
    const int q_tiles = p.tiles;
    if (tq > 0) hipLaunchKernelGGL((delta_kernel<BF, DP>), dim3((uint32_t)(tq * p.heads)), dim3(kThreads), 0, stream, b);
    const int64_t tk = count_tiles(p, k_rows, kRows);
    if (tk > 0) {
        if constexpr (!BF) hipLaunchKernelGGL((norm_kernel<DP>), dim3((uint32_t)(tk * p.kv_heads)), dim3(kThreads), 0, stream, b);
        hipLaunchKernelGGL((keys_kernel<BF, DP>), dim3((uint32_t)(tk * p.kv_heads)), dim3(64 * kKeyWaves<DP>), keys_lds, stream, b);
    }
    p.tiles = q_tiles;
    if (tq > 0) hipLaunchKernelGGL((rows_kernel<BF, DP>), dim3((uint32_t)(tq * p.heads)), dim3(kThreads), tiles_lds, stream, b);
    return launched("attention backward");
}

}  // namespace
}  // namespace mmfe

using namespace mmfe;

extern "C" {

int mmfe_attention_backward(const mmfe_attention_args* a, const mmfe_attention_grads* g, int device, void* hip_stream) {
    BackwardArgs b{};
    int rc = make_problem(a, b.p);
    if (rc) return rc;
    if (g == nullptr || g->struct_size != (int32_t)sizeof(mmfe_attention_grads)) { set_error("attention: gradients NULL or of another version"); return MMFE_EINVAL; }
    const bool any_q = a->q_rows > 0 && (a->packed || a->n_docs > 0), any_k = a->k_rows > 0 && (a->packed || a->n_docs > 0);
    if (any_q && (a->out == nullptr || a->lse == nullptr || g->grad_out == nullptr || g->grad_q == nullptr || g->scratch == nullptr)) { set_error("attention: NULL data pointer"); return MMFE_EINVAL; }
    if (any_k && (g->grad_k == nullptr || g->grad_v == nullptr)) { set_error("attention: NULL data pointer"); return MMFE_EINVAL; }
    if (a->dtype == MMFE_OUT_F16 && (any_q || any_k) && a->n_docs > 0 && g->norms == nullptr) { set_error("attention: NULL norms"); return MMFE_EINVAL; }
    if ((reinterpret_cast<uintptr_t>(a->out_rest) & 15) != 0) { set_error("attention: out_rest: 16-byte aligned"); return MMFE_EINVAL; }
    if (bad_rows("out", a->out, a->out_stride) || bad_rows("grad_out", g->grad_out, g->grad_out_stride) || bad_rows("grad_q", g->grad_q, g->grad_q_stride) ||
        bad_rows("grad_k", g->grad_k, g->grad_k_stride) || bad_rows("grad_v", g->grad_v, g->grad_v_stride)) return MMFE_EINVAL;
    if (count_tiles(b.p, a->q_rows, kRows) * a->heads > 0x7fffffffll || count_tiles(b.p, a->k_rows, kRows) * a->kv_heads > 0x7fffffffll) {
        set_error("attention: too many rows and heads in one call"); return MMFE_EINVAL;
    }
    auto rows = [](const void* ptr, const int64_t* s) { return Rows{ptr, s[0], s[1], s[2]}; };
    b.out = rows(a->out, a->out_stride); b.rest = static_cast<const char*>(a->out_rest); b.g = rows(g->grad_out, g->grad_out_stride);
    b.dq = rows(g->grad_q, g->grad_q_stride); b.dk = rows(g->grad_k, g->grad_k_stride); b.dv = rows(g->grad_v, g->grad_v_stride);
    b.lse = a->lse; b.lse_b = a->lse_stride[0]; b.lse_h = a->lse_stride[1];
    const int64_t n = (a->packed ? 1 : (int64_t)a->n_docs) * a->heads * a->q_rows;
    b.lse2 = g->scratch; b.delta = g->scratch + n;
    b.norm_g = g->norms; b.norm_v = g->norms ? g->norms + (int64_t)a->n_docs * a->kv_heads : nullptr;
    OnDevice on(device);
    if (on.rc) return on.rc;
    hipStream_t stream = reinterpret_cast<hipStream_t>(hip_stream);
    const int dp = padded_dim(a->dim);
    if (a->dtype == MMFE_OUT_BF16) return dp == 32 ? launch<true, 32>(b, a->q_rows, a->k_rows, stream) : dp == 64 ? launch<true, 64>(b, a->q_rows, a->k_rows, stream) : launch<true, 128>(b, a->q_rows, a->k_rows, stream);
    return dp == 32 ? launch<false, 32>(b, a->q_rows, a->k_rows, stream) : dp == 64 ? launch<false, 64>(b, a->q_rows, a->k_rows, stream) : launch<false, 128>(b, a->q_rows, a->k_rows, stream);
}

}  // extern "C"

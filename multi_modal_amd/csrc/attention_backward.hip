// Gradients of attention (attention.hip), from q, k, v, the output o, its gradient g and the saved lse:
//     p_ij = e^(s_ij - lse_i)      delta_i = g_i . o_i      dp_ij = g_i . v_j      ds_ij = p_ij (dp_ij - delta_i) (1 - tanh^2 of a capped score)
//     dv_j = sum_i p_ij g_i        dk_j = scale sum_i ds_ij q_i                     dq_i = scale sum_j ds_ij k_j
// the sums over i running over all query heads that share the key head.
//
// Two passes, each recomputing the scores: one block per 128 keys walks the rows (dk, dv), one block per 128 rows walks the keys (dq).
// That is 7 matrix products where one pass with atomic additions into dq would need 5, but every sum has one owner and a fixed
// order: the same call gives the same bits.  As in the forward pass, products are arranged so that a result is the next operand: the key pass
// forms scores as rows x keys (a lane has one key), the row pass as keys x rows (a lane has one row); sums over the lane's own index stay in
// registers for the whole walk.  Where there are few blocks with long walks, the walks are cut into parts that another launch adds up in order.
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
int64_t in_all(const mmfe_attention_args* a, int64_t rows);
int walk_cuts(const mmfe_attention_args* a, int64_t rows, int heads, int64_t partners, int64_t want);
}  // namespace attn

namespace {

struct BackwardArgs {
    Problem p;
    Rows out, g, dq, dk, dv;
    const char* rest;                 // like out: what its rounding lost, or NULL
    const float* lse;
    float *lse2, *delta;              // like lse: lse in log2 units (less the shift of p; +inf for rows without keys), g . o
    u32x4* aux;                       // like lse, 16 bytes: both again in the form keys_kernel takes (see there)
    float *part, *part_v;             // walks cut into parts: their gradients in float32, keys_kernel's (key heads, cuts, keys, dim) of k and then of v,
                                      // rows_kernel's (cuts, heads, rows, dim)
    bool whole;                       // whole_kernel serves the call
    int k_cuts, q_cuts;               // parts of keys_kernel's walk over the rows, and of rows_kernel's over the keys
    int64_t lse_b, lse_h;
    float *norm_g, *norm_v;           // float16: largest squared row norm of each 128-row tile, (heads, q_slots) and (kv_heads, k_slots)
    int q_slots, k_slots, q_tiles, k_tiles, q_blocks;
};

template <bool BF>
constexpr float kShift = BF ? 0.f : 8.f;

// Place of a document's tile among the norms: one place per tile, in a document's order, without a table.  Packed documents may share
// a 128-row stretch with their neighbours, one place is added per document before them.
__device__ __forceinline__ int64_t slot(const Problem& p, const Doc& d, bool qside, int tile) {
    if (p.packed) return ((qside ? d.q0 : d.k0) >> 7) + d.index + tile;
    return (int64_t)d.batch * (((qside ? p.q_rows : p.k_rows) + kRows - 1) / kRows) + tile;
}

__device__ __forceinline__ float block_max(float v, float* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max2(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float m = lds[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) m = max2(m, lds[w]);
    __syncthreads();
    return m;
}

// A float32 as three bfloat16 values that add up to it (8 bits each; a fourth place is zero).
__device__ __forceinline__ u32x2 thirds(float v) {
    const unsigned a = pack2<true>(v, 0.f);
    const float r = v - widen<true>(a, 0);
    const unsigned b = pack2<true>(r, 0.f);
    const unsigned c = pack2<true>(r - widen<true>(b, 0), 0.f);
    return u32x2{(a & 0xffffu) | b << 16, c & 0xffffu};
}

// What a score's form lacks to log2 p beside the row's lse (see Shape).
__device__ __forceinline__ float lacks(const Problem& p) { return p.cap > 0.f && p.cap <= kUsualCap ? p.cap * kLog2e : 0.f; }
// What keys_kernel adds to a row's products: in log2 units beside a capped score, in the products' own otherwise.  -1e30: p = 0
__device__ __forceinline__ float row_add(const Problem& p, float lse2) {
    const float add = p.cap > 0.f ? lacks(p) - lse2 : -lse2 / (p.scale * kLog2e);
    return add < -1e30f ? -1e30f : add;                // a NaN stays one
}

// 2^(6 - ceil(log2(bound)))
__device__ __forceinline__ float phi_of(float bound) {
    if (!(bound > 0.f) || !(bound < 3e38f)) return 1.f;
    int e;
    (void)frexpf(bound, &e);                           // bound < 2^e
    return ldexpf(1.f, 6 - e);
}

// Memory bound: 17 thousand rows of 12 heads of 64, 4 tensors' rows read: 16 us.
// What both passes need of every row: delta and lse2 (blocks below q_blocks, 128 rows of one head each), and for float16 the tiles' largest
// squared norms of g and, in the blocks behind, of v.  One lane has 8 elements of a row.
template <bool BF, int DP>
__global__ void __launch_bounds__(kThreads) prepare_kernel(const BackwardArgs a) {
    __shared__ float lds[kWaves];
    Problem p = a.p;
    constexpr int kLanes = kPitch<DP> / 8;
    const int e = (threadIdx.x & (kLanes - 1)) * 8;
    Doc d;
    float biggest = 0.f;
    if ((int)blockIdx.x < a.q_blocks) {
        p.tiles = a.q_tiles;
        if (!find_doc<true>(p, blockIdx.x / p.heads, kRows, d)) return;
        const int head = blockIdx.x % p.heads;
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
            biggest = max2(biggest, sq);
            if (row < d.nq && e == 0) {
                const int64_t at = d.batch * a.lse_b + head * a.lse_h + d.q0 + row;
                const float l = a.lse[at];
                const float l2 = l == -INFINITY ? INFINITY : l * kLog2e - kShift<BF>;
                if (l == -INFINITY) dot = 0.f;
                a.lse2[at] = l2;
                a.delta[at] = dot;
                const u32x2 x = thirds(row_add(p, l2)), y = thirds(-dot);
                a.aux[at] = u32x4{x.x, x.y, y.x, y.y};
            }
        }
        if constexpr (!BF) {
            biggest = block_max(biggest, lds);
            if (d.index >= 0 && threadIdx.x == 0) a.norm_g[(int64_t)head * a.q_slots + slot(p, d, true, d.tile)] = biggest;
        }
    } else if constexpr (!BF) {
        p.tiles = a.k_tiles;
        const int block = blockIdx.x - a.q_blocks;
        if (!find_doc<false>(p, block / p.kv_heads, kRows, d) || d.index < 0) return;
        const int head = block % p.kv_heads;
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
            biggest = max2(biggest, sq);
        }
        biggest = block_max(biggest, lds);
        if (threadIdx.x == 0) a.norm_v[(int64_t)head * a.k_slots + slot(p, d, false, d.tile)] = biggest;
    }
}

// phi of a document and key head, from its tiles' norms; called by the whole block.
template <bool BF>
__device__ __forceinline__ float find_phi(const BackwardArgs& a, const Doc& d, int kvh, float* lds) {
    if constexpr (BF) return 1.f;
    else {
        if (d.index < 0) return 1.f;
        float g = 0.f, v = 0.f;
        const int tq = (d.nq + kRows - 1) / kRows, tk = (d.nk + kRows - 1) / kRows;
        const float* ng = a.norm_g + slot(a.p, d, true, 0) + (int64_t)kvh * a.p.group * a.q_slots;
        for (int h = 0; h < a.p.group; ++h)
            for (int i = threadIdx.x; i < tq; i += blockDim.x) g = max2(g, ng[(int64_t)h * a.q_slots + i]);
        const float* nv = a.norm_v + slot(a.p, d, false, 0) + (int64_t)kvh * a.k_slots;
        for (int i = threadIdx.x; i < tk; i += blockDim.x) v = max2(v, nv[i]);
        return phi_of(sqrtf(block_max(g, lds)) * sqrtf(block_max(v, lds)));
    }
}

// Scores in log2 units from the products, and the factor that a capped score's gradient has.  In kExpCap's form a score is
// cap tanh(z) = cap (1 - 2 r) with r = 1 / (e^(2 z) + 1), and 1 - tanh^2 = 4 (r - r^2): one exponential and one reciprocal; the 4
// is left to the gradients' final factor.
template <int CAP>
struct Shape {
    bool bias;
    float c, slope, cap_in, cap_out;
    AnyCap any;
    __device__ __forceinline__ void set(const Problem& p, int head) {
        bias = p.slopes != nullptr;
        c = p.scale * kLog2e;
        slope = bias ? p.slopes[head] * kLog2e : 0.f;
        cap_in = CAP == kExpCap ? 2.f * kLog2e * p.scale / p.cap : 0.f;
        cap_out = CAP == kExpCap ? 2.f * p.cap * kLog2e : 0.f;
        if constexpr (CAP == kAnyCap) any.set(p);
    }
    // x -> score + add, w -> the factor.  at: distance of register row 0, step: its sign per row.  FOLDED: the products hold `add` already
    template <bool FOLDED, typename ADD>
    __device__ __forceinline__ void apply(f32x16& x, f32x16& w, ADD add, float at, float step) const {
        if constexpr (CAP == kAnyCap) any.apply<true>(x, &w);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (CAP == kExpCap) {
                const float r = __builtin_amdgcn_rcpf(exp2_fast(x[i] * cap_in) + 1.f);
                x[i] = fmaf(-cap_out, r, add(i));
                w[i] = fmaf(-r, r, r);
            } else if constexpr (FOLDED && !CAP) x[i] *= c;
            else x[i] = fmaf(x[i], c, add(i));
        }
        if (bias) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fmaf(-slope, fabsf(at + step * (float)reg_row(i)), x[i]);
        }
    }
    __device__ __forceinline__ float factor() const { return CAP ? 4.f : 1.f; }
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
            if (e >= dim) continue;
            if (some) store4<BF>(to + 2 * (e + 4 * half), nullptr, o[i][4 * g] * by, o[i][4 * g + 1] * by, o[i][4 * g + 2] * by, o[i][4 * g + 3] * by);
            else store4<BF>(to + 2 * (e + 4 * half), nullptr, 0.f, 0.f, 0.f, 0.f);
        }
}

// the same in float32
template <int DP>
__device__ __forceinline__ void store_part(float* to, const f32x16 (&o)[DP / 32], int dim, float by, bool some) {
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = 32 * i + 8 * g;
            if (e >= dim) continue;
            *reinterpret_cast<float4*>(to + e + 4 * half) = some ? make_float4(o[i][4 * g] * by, o[i][4 * g + 1] * by, o[i][4 * g + 2] * by, o[i][4 * g + 3] * by) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
}

template <int DP>
__device__ __forceinline__ void load_rows(u32x4 (&f)[DP / 16], const char* row, int dim, bool some) {
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        f[s] = u32x4{0, 0, 0, 0};
        if (some && 16 * s + 8 * half < dim) f[s] = *reinterpret_cast<const u32x4*>(row + 32 * s + 16 * half);
    }
}

// acc += columns of a tile's 32 rows from row0 on, times x: what the short documents' rounding lost goes in as a second product
template <bool BF, int DP>
__device__ __forceinline__ void accumulate(f32x16 (&acc)[DP / 32], const char* tile, int row0, const f32x16& x, bool both) {
    u32x4 f[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        f[s] = operand<BF>(x, s);
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) acc[i] = mfma<BF>(read_cols<DP>(tile, row0 + 16 * s, 32 * i), f[s], acc[i]);
    }
    if (both)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const u32x4 r = operand_rest<BF>(x, s, f[s]);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) acc[i] = mfma<BF>(read_cols<DP>(tile, row0 + 16 * s, 32 * i), r, acc[i]);
        }
}

constexpr int kRing = 4;              // tiles in LDS: the one in use, the next one's scores, two on their way
template <int DP>
constexpr int kKeysTile = DP == 96 ? 32 : 64;          // rows of keys_kernel's tiles
constexpr int kStatBytes = 64 * 16;                    // of a tile's row statistics (one DMA)

// Row statistics come as a third kind of operand: prepare_kernel leaves -lse and -delta of each row as three bfloat16 values that add
// up to the float32, and a product with ones adds them to a row's scores and dp, over all keys at once.  Read as numbers they
// would be 8 broadcast reads of 1 KB per 32 rows and wave, a third of all LDS traffic, which is what bounds this kernel; so
// they are one read of 16 bytes a row and two products more (16 to 18, head size 64).
//
// dk and dv of 128 keys, 32 per wave, over tiles of 64 rows.  Step u turns the scores of its rows (computed a step earlier) into p and
// ds beside the products of the next rows, then adds them to dv and dk; its tiles stay until then, and it asks for those of step u + 3.
// Head size 128 has one wave per SIMD (357 registers), 64 and less two.  At 96, with half the tile and without the overlap, two blocks fit a CU, and one's
// products run beside the other's exponentials: 8192 rows, 12 heads on 4, 987 -> 636 us, causal 518 -> 337 (4096 rows, 12 heads of 72: 356 -> 209).
// The same at 128 leaves 41 registers in memory: 744 -> 673 us for 8 heads of 8192 rows, but causal 403 -> 413 with the walks cut and 636 without.
template <bool BF, int DP, int CAP>
__global__ void __launch_bounds__(kThreads, DP == 128 ? 1 : 2) keys_kernel(const BackwardArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];       // kRing x [q tile][g tile][row statistics]
    const Problem& p = a.p;
    constexpr int kTile = kKeysTile<DP>;
    constexpr int kTileBytes = kTile * kPitch<DP> * 2;
    constexpr int kBuf = 2 * kTileBytes + kStatBytes;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int lot = blockIdx.x % (p.kv_heads * a.k_cuts), kvh = lot % p.kv_heads, cut = lot / p.kv_heads;
    Doc d;
    if (!find_doc<false>(p, blockIdx.x / (p.kv_heads * a.k_cuts), kRows, d)) return;
    const int head0 = kvh * p.group;
    const int key0 = d.tile * kRows, w0 = key0 + 32 * wave, key = w0 + col;
    const int nq = d.nq, nk = d.nk, off = nk - nq;
    // rows [first, nq) see key j: all of them, or those from j - off on
    auto first_row = [&](int j) { return p.causal && j >= d.prefix ? max(0, j - off) : 0; };
    const int block_first = key0 < nk ? first_row(key0) : nq;
    const int wave_first = w0 < nk ? first_row(w0) : nq;
    const int wave_full = first_row(min(w0 + 31, nk - 1));            // from here on every row sees all keys of the wave
    const int my_first = first_row(key);
    const int t_first = block_first / kTile, t_end = block_first < nq ? (nq + kTile - 1) / kTile : t_first;
    // the tiles of all query heads, one head after the other, and this block's part of them
    const int all_steps = (t_end - t_first) * p.group, part_steps = (all_steps + a.k_cuts - 1) / a.k_cuts;
    const int first_step = min(cut * part_steps, all_steps), steps = min(part_steps, all_steps - first_step);
    const int first_g = steps > 0 ? first_step / (t_end - t_first) : 0;

    typedef Loader<DP, kTile, kWaves> Load;
    Load lq, lg;
    lq.init(p.dim, p.q.n, wave);
    lg.init(p.dim, a.g.n, wave);
    const unsigned lds0 = lds_address(smem);
    int g = first_g, t = t_first + (steps > 0 ? first_step - first_g * (t_end - t_first) : 0);
    int ask_g = g, ask_t = t, ask = 0;                                // the next tile to ask for
    auto stage = [&]() {
        const int head = head0 + ask_g, r0 = ask_t * kTile;
        const unsigned dst = uniform(lds0 + (ask % kRing) * kBuf);
        lq.load(row_base(p.q, d, d.q0 + r0, head), nq - r0, p.dim, p.q.n, dst, wave);
        lg.load(row_base(a.g, d, d.q0 + r0, head), nq - r0, p.dim, a.g.n, dst + kTileBytes, wave);
        const int64_t at = d.batch * a.lse_b + head * a.lse_h + d.q0 + r0;
        if (wave == 0) dma16(a.aux + at, 16 * min(lane, nq - 1 - r0), dst + 2 * kTileBytes);
        ++ask;
        if (++ask_t == t_end) { ask_t = t_first; ++ask_g; }
    };
    u32x4 kf[DP / 16], vf[DP / 16];
    {
        const int r = max(0, min(key, nk - 1));
        load_rows<DP>(kf, row_base(p.k, d, d.k0 + r, kvh), p.dim, nk > 0);
        load_rows<DP>(vf, row_base(p.v, d, d.k0 + r, kvh), p.dim, nk > 0);
    }
    const float phi = find_phi<BF>(a, d, kvh, reinterpret_cast<float*>(smem));
    for (int i = 0; i < kRing - 1 && i < steps; ++i) stage();
    f32x16 dk[DP / 32], dv[DP / 32], x{}, dp{};
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = f32x16{};
    const u32x4 ones = half == 0 ? u32x4{0x3f803f80u, 0x00003f80u, 0u, 0u} : u32x4{0u, 0u, 0u, 0u};       // of the three places
    auto statistics = [&](const char* qt, int b) { return *reinterpret_cast<const u32x4*>(qt + 2 * kTileBytes + (32 * b + col) * 16); };
    // scores and dp - delta of 32 rows: register rows are rows, a lane has one key
    auto products = [&](const char* qt, int b, f32x16& sx, f32x16& sd) {
        const u32x4 st = statistics(qt, b);
        if constexpr (CAP) sx = f32x16{};
        else sx = mfma<true>(u32x4{st.x, st.y, 0u, 0u}, ones, f32x16{});
        sd = mfma<true>(u32x4{st.z, st.w, 0u, 0u}, ones, f32x16{});
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) sx = mfma<BF>(read_rows<DP>(qt, 32 * b, s), kf[s], sx);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) sd = mfma<BF>(read_rows<DP>(qt + kTileBytes, 32 * b, s), vf[s], sd);
    };
    wait_all();
    block_sync();
    arrived(kf);
    arrived(vf);
    Shape<CAP> sh;
    sh.set(p, head0 + g);
    // p and ds of 32 rows, from their scores and dp - delta, into dv and dk
    auto before = [&](const char* qt, int b, f32x16& x, f32x16& w) {
        const int i0 = t * kTile + 32 * b;
        f32x16 add;
        if constexpr (CAP) {
            const u32x4 st = statistics(qt, b);
            add = mfma<true>(u32x4{st.x, st.y, 0u, 0u}, ones, f32x16{});
        }
        sh.template apply<true>(x, w, [&](int i) { return add[i]; }, (float)(i0 + 4 * half + off - key), 1.f);
        if (i0 < wave_full || i0 + 32 > nq) {
            const int lo = my_first - i0 - 4 * half, hi = nq - i0 - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = reg_row(i) >= lo && reg_row(i) < hi ? x[i] : -INFINITY;
        }
    };
    auto behind = [&](const char* qt, int b, f32x16& x, f32x16& dp, const f32x16& w) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = exp2_fast(x[i]);
            dp[i] *= x[i];
            if constexpr (!BF) dp[i] *= phi;
            if constexpr (CAP) dp[i] *= w[i];
        }
        accumulate<BF, DP>(dv, qt + kTileBytes, 32 * b, x, nk <= kShortKeys);
        accumulate<BF, DP>(dk, qt, 32 * b, dp, nk <= kShortKeys);
    };
    auto live = [&](int b) {
        const int i0 = t * kTile + 32 * b;
        return i0 + 32 > wave_first && i0 < nq;
    };
    if constexpr (kTile == 64) {
        if (steps > 0) products(smem, 0, x, dp);
    }
    for (int step = 0; step < steps; ++step) {
        // one step ahead, tile step + 1 is there, and what step - 1 asked for may be on its way; otherwise tile step, and two
        if (step + kRing - 2 < steps) wait_but<(kTile == 64 ? 2 : 4) * Load::kCount>();
        else wait_all();
        block_sync();
        if (step + kRing - 1 < steps) stage();
        const char* qt = smem + (step % kRing) * kBuf;
        f32x16 w;
        if constexpr (kTile == 64) {
            const char* next = smem + ((step + 1) % kRing) * kBuf;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bool on = live(b);
                if (on) before(qt, b, x, w);
                f32x16 nx, nd;
                products(b == 0 ? qt : next, 1 - b, nx, nd);
                if (on) behind(qt, b, x, dp, w);
                x = nx;
                dp = nd;
            }
        } else if (live(0)) {
            products(qt, 0, x, dp);
            before(qt, 0, x, w);
            behind(qt, 0, x, dp, w);
        }
        if (++t == t_end) {
            t = t_first;
            if (++g < p.group) sh.set(p, head0 + g);
        }
    }
    if (key >= d.rows) return;
    const float back = __builtin_amdgcn_exp2f(-kShift<BF>), fk = p.scale * back / phi * sh.factor();
    const bool any = key < nk && steps > 0, any_k = any && nk > 1;    // a softmax over one key is constant
    if (a.k_cuts == 1) {
        store_rows<BF, DP>(const_cast<char*>(row_base(a.dk, d, d.k0 + key, kvh)), dk, p.dim, fk, any_k);
        store_rows<BF, DP>(const_cast<char*>(row_base(a.dv, d, d.k0 + key, kvh)), dv, p.dim, back, any);
        return;
    }
    const int64_t rows = p.packed ? p.k_rows : p.k_rows * p.n_docs;
    const int64_t at = (((int64_t)kvh * a.k_cuts + cut) * rows + (p.packed ? d.k0 : d.batch * p.k_rows) + key) * p.dim;
    store_part<DP>(a.part + at, dk, p.dim, fk, any_k);
    store_part<DP>(a.part_v + at, dv, p.dim, back, any);
}

// Sums of the parts of one or two gradients, 4 elements a thread; memory bound (17 thousand keys, 4 key heads of 64 in two parts: 15 us).
struct Sum {
    const float* part[2];
    Rows to[2];
    int64_t rows, batch_rows;         // of a head, and of a batch entry (all of them where documents are packed)
    int64_t head_step, part_step;     // from one head's first part, and one part, to the next
    int heads, parts, pieces, tensors;
};
template <bool BF>
__global__ void __launch_bounds__(kThreads) sum_kernel(const Sum a) {
    const int64_t n = a.rows * a.heads * a.pieces;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n * a.tensors; i += (int64_t)gridDim.x * kThreads) {
        const int which = i >= n;
        const int64_t j = i - which * n, hr = j / a.pieces;
        const int e = 4 * (int)(j - hr * a.pieces), head = (int)(hr / a.rows);
        const int64_t row = hr - head * a.rows;
        const float* part = a.part[which] + head * a.head_step + row * (4 * a.pieces) + e;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < a.parts; ++c) {
            const float4 v = *reinterpret_cast<const float4*>(part + c * a.part_step);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        const Rows& to = a.to[which];
        const int64_t b = row / a.batch_rows;
        store4<BF>(static_cast<char*>(const_cast<void*>(to.p)) + 2 * (b * to.b + (row - b * a.batch_rows) * to.n + head * to.h + e), nullptr, s.x, s.y, s.z, s.w);
    }
}

// dq of 128 rows, 32 per wave, over tiles of 32 keys; steps overlap as in keys_kernel.  Head size 64 is held to 168 registers for three waves
// a SIMD (6 of them spilled): 8192 rows, 12 heads, 840 -> 954 TFLOP/s without a mask, 871 -> 830 under a causal one.
// CUT: the walk is cut into parts (as an argument that any call could have, 4 to 25 % slower where it is not).
template <bool BF, int DP, int CAP, bool CUT>
__global__ void __launch_bounds__(kThreads, DP == 64 ? 3 : 2) rows_kernel(const BackwardArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];       // kRing x [k tile][v tile]
    const Problem& p = a.p;
    constexpr int kKeys = 32;
    constexpr int kTileBytes = kKeys * kPitch<DP> * 2;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    Doc d;
    const int cuts = CUT ? a.q_cuts : 1, lot = blockIdx.x % (p.heads * cuts), cut = CUT ? lot / p.heads : 0;
    if (!find_doc<true>(p, blockIdx.x / (p.heads * cuts), kRows, d)) return;
    const int head = head_of(p, lot % p.heads), kvh = head / p.group;
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
    const int all = block_lim > 0 ? (block_lim + kKeys - 1) / kKeys : 0, part = CUT ? (all + cuts - 1) / cuts : all;
    const int t0 = CUT ? min(cut * part, all) : 0, n = CUT ? min(t0 + part, all) : all;       // this block's tiles

    typedef Loader<DP, kKeys, kWaves> Load;
    Load lk, lv;
    lk.init(p.dim, p.k.n, wave);
    lv.init(p.dim, p.v.n, wave);
    const unsigned lds0 = lds_address(smem);
    auto stage = [&](int t) {
        const unsigned dst = uniform(lds0 + (t % kRing) * 2 * kTileBytes);
        lk.load(row_base(p.k, d, d.k0 + (int64_t)t * kKeys, kvh), nk - t * kKeys, p.dim, p.k.n, dst, wave);
        lv.load(row_base(p.v, d, d.k0 + (int64_t)t * kKeys, kvh), nk - t * kKeys, p.dim, p.v.n, dst + kTileBytes, wave);
    };
    u32x4 qf[DP / 16], gf[DP / 16];
    const int r = max(0, min(row, nq - 1));
    load_rows<DP>(qf, row_base(p.q, d, d.q0 + r, head), p.dim, nq > 0);
    load_rows<DP>(gf, row_base(a.g, d, d.q0 + r, head), p.dim, nq > 0);
    const int64_t at = d.batch * a.lse_b + head * a.lse_h + d.q0 + r;
    const float phi = find_phi<BF>(a, d, kvh, reinterpret_cast<float*>(smem));
    float add = nq > 0 ? lacks(p) - a.lse2[at] : 0.f;                         // what the scores' log2 form lacks to log2 p
    float delta = nq > 0 ? -a.delta[at] * phi : 0.f;
    Shape<CAP> sh;
    sh.set(p, head);
    for (int i = t0; i < t0 + kRing - 1 && i < n; ++i) stage(i);
    f32x16 dq[DP / 32], x{}, dp{};
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dq[i] = f32x16{};
    auto products = [&](const char* kt, f32x16& sx, f32x16& sd) {
        sx = f32x16{};
        sd = f32x16{};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) sx = mfma<BF>(read_rows<DP>(kt, 0, s), qf[s], sx);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) sd = mfma<BF>(read_rows<DP>(kt + kTileBytes, 0, s), gf[s], sd);
    };
    wait_all();
    block_sync();
    arrived(qf);
    arrived(gf);
    asm volatile("" : "+v"(add), "+v"(delta));
    if (t0 < n && t0 * kKeys < wave_lim) products(smem + (t0 % kRing) * 2 * kTileBytes, x, dp);
    for (int t = t0; t < n; ++t) {
        if (t + kRing - 2 < n) wait_but<2 * Load::kCount>();
        else wait_all();
        block_sync();
        if (t + kRing - 1 < n) stage(t + kRing - 1);
        const int j0 = t * kKeys;
        if (j0 >= wave_lim) continue;
        const char* kt = smem + (t % kRing) * 2 * kTileBytes;
        f32x16 w;
        sh.template apply<false>(x, w, [&](int) { return add; }, (float)(row + off - j0 - 4 * half), -1.f);
        if (j0 + kKeys > full_lim) {
            const int left = lim - j0 - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = reg_row(i) < left ? x[i] : -INFINITY;
        }
        f32x16 nx, nd;
        products(smem + ((t + 1) % kRing) * 2 * kTileBytes, nx, nd);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            dp[i] = (BF ? dp[i] + delta : fmaf(dp[i], phi, delta)) * exp2_fast(x[i]);
            if constexpr (CAP) dp[i] *= w[i];
        }
        accumulate<BF, DP>(dq, kt, 0, dp, nk <= kShortKeys);
        x = nx;
        dp = nd;
    }
    wait_all();
    if (row >= d.rows) return;
    const float by = p.scale * __builtin_amdgcn_exp2f(-kShift<BF>) / phi * sh.factor();
    const bool some = lim > 1;                                        // a softmax over one key is constant
    if constexpr (!CUT) {
        store_rows<BF, DP>(const_cast<char*>(row_base(a.dq, d, d.q0 + row, head)), dq, p.dim, by, some);
        return;
    }
    const int64_t rows = p.packed ? p.q_rows : p.q_rows * p.n_docs;
    store_part<DP>(a.part + (((int64_t)cut * p.heads + head) * rows + (p.packed ? d.q0 : d.batch * p.q_rows) + row) * p.dim, dq, p.dim, by, some);
}

// ---- short documents ----
//
// Documents of up to 256 rows and keys (a clip's 192 patches and class token) with a key head per query head and a head size up to 64: one block
// does all of a head's gradients, with q, k, v and g in LDS, a wave for every 32 rows and then for the 32 keys of the same numbers.  Eight
// waves and one block per CU; documents of up to 128 take four, and two blocks share a CU.  The tensors are read from memory once, delta is
// the sum of p dp over the keys, taken in a first walk over them, and neither o nor what its rounding lost is read, or has to be stored by the
// forward pass.  Neither pipe is full (vector instructions 47 % of a CU's cycles, products 24 %): one block a CU brings its tensors, waits, and computes with nothing beside
// it, and 193 rows take the products of 224.  64 clips of 193 rows, 12 heads of 64, float16: 84 to 88 us (in four waves with two groups of rows each, two blocks a CU and q and g brought after
// k and v, 92; by the two passes above and the launch before them, whose blocks wait for their first tiles most of the time, 105), and the
// forward pass 29 in place of 34 us.
constexpr int kWholeRows = 256;
template <int DP, int WAVES>
constexpr int kWholeLoad = WAVES * 512 / DP;           // rows that one DMA of each wave brings

template <bool BF, int DP, int CAP, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 2) whole_kernel(const BackwardArgs a, int padded_rows) {
    extern __shared__ __attribute__((aligned(16))) char smem[];       // k, v, q, g of padded_rows rows each, statistics of the rows, WAVES floats
    const Problem& p = a.p;
    constexpr int kTileBytes = 32 * DP * 2;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int head = blockIdx.x % p.heads;
    Doc d;
    (void)find_doc<true>(p, blockIdx.x / p.heads, kWholeRows, d);     // one tile per document
    const int nq = d.nq, nk = d.nk, off = nk - nq;
    const int tq = (nq + 31) / 32;
    const bool any = nq > 0 && nk > 0;
    const int part = padded_rows * DP * 2;
    const char *lk = smem, *lv = lk + part, *lq = lv + part, *lg = lq + part;
    u32x4* stats = reinterpret_cast<u32x4*>(smem + 4 * part);
    float* scratch = reinterpret_cast<float*>(stats + padded_rows);
    const unsigned lds0 = lds_address(smem);
    auto limit = [&](int r) { return p.causal ? min(nk, max(d.prefix, min(r, nq - 1) + off + 1)) : nk; };
    auto first_row = [&](int j) { return p.causal && j >= d.prefix ? max(0, j - off) : 0; };
    constexpr int kLoad = kWholeLoad<DP, WAVES>;
    typedef Loader<DP, kLoad, WAVES> Load;
    auto load = [&](const Rows& x, const Rows& y, int rows, unsigned lds) {
        Load lx, ly;
        lx.init(p.dim, x.n, wave);
        ly.init(p.dim, y.n, wave);
        for (int r = 0; r < rows; r += kLoad) {
            lx.load(row_base(x, d, r, head), rows - r, p.dim, x.n, uniform(lds + r * DP * 2), wave);
            ly.load(row_base(y, d, r, head), rows - r, p.dim, y.n, uniform(lds + part + r * DP * 2), wave);
        }
    };
    if (any) {
        load(p.k, p.v, nk, lds0);
        load(p.q, a.g, nq, lds0 + 2 * part);
    }
    Shape<CAP> sh;
    sh.set(p, head);
    const float back = __builtin_amdgcn_exp2f(-kShift<BF>);
    const int w0 = 32 * wave, mine = w0 + col;                        // a wave's rows, and then its keys
    float lse = any ? a.lse[d.batch * a.lse_b + head * a.lse_h + min(mine, nq - 1)] : 0.f;
    wait_all();
    block_sync();
    asm volatile("" : "+v"(lse));

    // dq
    u32x4 qf[DP / 16], gf[DP / 16];
    const int own = any ? min(wave, tq - 1) * kTileBytes : 0;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        qf[s] = read_rows<DP>(lq + own, 0, s);
        gf[s] = read_rows<DP>(lg + own, 0, s);
    }
    float phi = 1.f;
    if constexpr (!BF) {
        float g = 0.f, v = 0.f;
        if (any) {
            const int t = min(wave, (nk - 1) / 32);
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                const u32x4 vf = read_rows<DP>(lv + t * kTileBytes, 0, s);               // rows past the last repeat it; pieces past the head
                if (16 * s + 8 * half < p.dim)                                           // size repeat the first, and are left out
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x = widen<BF>(gf[s][e >> 1], e & 1), y = widen<BF>(vf[e >> 1], e & 1);
                        g = fmaf(x, x, g);
                        v = fmaf(y, y, v);
                    }
            }
            g = both_sum(g);
            v = both_sum(v);
        }
        phi = phi_of(sqrtf(block_max(g, scratch)) * sqrtf(block_max(v, scratch)));
    }
    // pieces past the head size: zero on one side of each product (k and v there repeat others)
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
        if (16 * s + 8 * half >= p.dim) qf[s] = gf[s] = u32x4{0u, 0u, 0u, 0u};
    auto products = [&](const char* a, const char* b, const u32x4 (&f)[DP / 16], const u32x4 (&h)[DP / 16], f32x16& sx, f32x16& sd) {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) sx = mfma<BF>(read_rows<DP>(a, 0, s), f[s], sx);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) sd = mfma<BF>(read_rows<DP>(b, 0, s), h[s], sd);
    };
    if (w0 < p.q_rows) {
        const int lim = any && mine < nq ? limit(mine) : 0, wave_lim = any && w0 < nq ? limit(w0 + 31) : 0, full_lim = any && w0 < nq ? limit(w0) : 0;
        const float l2 = lse == -INFINITY ? INFINITY : lse * kLog2e - kShift<BF>;
        const float add = lacks(p) - l2;
        f32x16 dq[DP / 32];
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) dq[e] = f32x16{};
        auto probabilities = [&](int t, f32x16& x, f32x16& dp, f32x16& w) {
            const int j0 = 32 * t;
            x = dp = f32x16{};
            products(lk + t * kTileBytes, lv + t * kTileBytes, qf, gf, x, dp);
            sh.template apply<false>(x, w, [&](int) { return add; }, (float)(mine + off - j0 - 4 * half), -1.f);
            if (j0 + 32 > full_lim) {
                const int left = lim - j0 - 4 * half;
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = reg_row(e) < left ? x[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = exp2_fast(x[e]);
        };
        float sum = 0.f;
        for (int t = 0; 32 * t < wave_lim; ++t) {
            f32x16 x, dp, w;
            probabilities(t, x, dp, w);
#pragma unroll
            for (int e = 0; e < 16; ++e) sum = fmaf(x[e], dp[e], sum);
        }
        const float delta = lim > 0 ? both_sum(sum) * back : 0.f;
        for (int t = 0; 32 * t < wave_lim; ++t) {
            f32x16 x, dp, w;
            probabilities(t, x, dp, w);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                dp[e] = (dp[e] - delta) * x[e];
                if constexpr (!BF) dp[e] *= phi;
                if constexpr (CAP) dp[e] *= w[e];
            }
            accumulate<BF, DP>(dq, lk + t * kTileBytes, 0, dp, nk <= kShortKeys);
        }
        if (mine < p.q_rows)
            store_rows<BF, DP>(const_cast<char*>(row_base(a.dq, d, mine, head)), dq, p.dim, p.scale * back / phi * sh.factor(), lim > 1);     // a softmax over one key is constant
        if (half == 0 && mine < nq) {
            const u32x2 u = thirds(row_add(p, l2)), v = thirds(-delta);
            stats[mine] = u32x4{u.x, u.y, v.x, v.y};
        }
    }
    wait_but<63>();                                                   // the statistics are written; stores may go on
    block_sync();

    // dk and dv
    if (w0 < p.k_rows) {
        u32x4 kf[DP / 16], vf[DP / 16];
        const int at = any ? min(wave, (nk - 1) / 32) * kTileBytes : 0;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const bool in = 16 * s + 8 * half < p.dim;
            kf[s] = in ? read_rows<DP>(lk + at, 0, s) : u32x4{0u, 0u, 0u, 0u};
            vf[s] = in ? read_rows<DP>(lv + at, 0, s) : u32x4{0u, 0u, 0u, 0u};
        }
        const u32x4 ones = half == 0 ? u32x4{0x3f803f80u, 0x00003f80u, 0u, 0u} : u32x4{0u, 0u, 0u, 0u};
        const int wave_first = any && w0 < nk ? first_row(w0) : nq, wave_full = first_row(min(w0 + 31, nk - 1)), my_first = first_row(mine);
        f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) dk[e] = dv[e] = f32x16{};
        for (int t = wave_first / 32; t < tq && wave_first < nq; ++t) {
            const int i0 = 32 * t;
            const u32x4 st = stats[min(i0 + col, nq - 1)];
            f32x16 x{}, dp, w, add;
            const f32x16 lo = mfma<true>(u32x4{st.x, st.y, 0u, 0u}, ones, f32x16{});
            if constexpr (CAP) add = lo;
            else x = lo;
            dp = mfma<true>(u32x4{st.z, st.w, 0u, 0u}, ones, f32x16{});
            products(lq + t * kTileBytes, lg + t * kTileBytes, kf, vf, x, dp);
            sh.template apply<true>(x, w, [&](int e) { return add[e]; }, (float)(i0 + 4 * half + off - mine), 1.f);
            if (i0 < wave_full || i0 + 32 > nq) {
                const int from = my_first - i0 - 4 * half, to = nq - i0 - 4 * half;
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = reg_row(e) >= from && reg_row(e) < to ? x[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[e] = exp2_fast(x[e]);
                dp[e] *= x[e];
                if constexpr (!BF) dp[e] *= phi;
                if constexpr (CAP) dp[e] *= w[e];
            }
            accumulate<BF, DP>(dv, lg + t * kTileBytes, 0, x, nk <= kShortKeys);
            accumulate<BF, DP>(dk, lq + t * kTileBytes, 0, dp, nk <= kShortKeys);
        }
        if (mine < p.k_rows) {
            const bool some = mine < nk && wave_first < nq;
            store_rows<BF, DP>(const_cast<char*>(row_base(a.dk, d, mine, head)), dk, p.dim, p.scale * back / phi * sh.factor(), some && nk > 1);
            store_rows<BF, DP>(const_cast<char*>(row_base(a.dv, d, mine, head)), dv, p.dim, back, some);
        }
    }
}

template <bool BF>
void launch_sum(const Sum& s, hipStream_t stream) {
    const int64_t need = (s.rows * s.heads * s.pieces * s.tensors + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(sum_kernel<BF>, dim3((uint32_t)(need < 8192 ? need : 8192)), dim3(kThreads), 0, stream, s);
}

template <bool BF, int DP, int CAP, int WAVES>
int launch_whole(BackwardArgs& b, hipStream_t stream) {
    Problem& p = b.p;
    constexpr int kLoad = kWholeLoad<DP, WAVES>;
    const int rows = (int)((p.q_rows > p.k_rows ? p.q_rows : p.k_rows) + kLoad - 1) / kLoad * kLoad;
    const auto fn = &whole_kernel<BF, DP, CAP, WAVES>;
    const size_t lds = (size_t)rows * (4 * DP * 2 + 16) + WAVES * 4;
    int rc, blocks = 1, cus = 256;
    if ((rc = kernel_prepare(reinterpret_cast<const void*>(fn), 64 * WAVES, lds, &blocks, &cus)) != MMFE_OK) return rc;
    p.tiles = 1;
    hipLaunchKernelGGL(fn, dim3((uint32_t)(p.n_docs * p.heads)), dim3(64 * WAVES), lds, stream, b, rows);
    return launched("attention backward");
}

template <bool BF, int DP, int CAP>
int launch(BackwardArgs& b, hipStream_t stream) {
    Problem& p = b.p;
    int rc = MMFE_OK, blocks = 1, cus = 256;
    if constexpr (DP <= 64)
        if (b.whole) return p.q_rows <= kWholeRows / 2 && p.k_rows <= kWholeRows / 2 ? launch_whole<BF, DP, CAP, 4>(b, stream) : launch_whole<BF, DP, CAP, 8>(b, stream);
    const int64_t tk = count_tiles(p, p.k_rows, kRows);
    b.k_tiles = p.tiles;
    const int64_t tq = count_tiles(p, p.q_rows, kRows);
    b.q_tiles = p.tiles;
    b.q_blocks = (int)(tq * p.heads);
    const int64_t norms = BF ? 0 : tk * p.kv_heads;
    if (b.q_blocks + norms > 0) hipLaunchKernelGGL((prepare_kernel<BF, DP>), dim3((uint32_t)(b.q_blocks + norms)), dim3(kThreads), 0, stream, b);
    if (tk > 0) {
        p.tiles = b.k_tiles;
        const auto fn = &keys_kernel<BF, DP, CAP>;
        const size_t lds = kRing * (2 * (size_t)kKeysTile<DP> * kPitch<DP> * 2 + kStatBytes);
        if ((rc = kernel_prepare(reinterpret_cast<const void*>(fn), kThreads, lds, &blocks, &cus)) != MMFE_OK) return rc;
        hipLaunchKernelGGL(fn, dim3((uint32_t)(tk * p.kv_heads * b.k_cuts)), dim3(kThreads), lds, stream, b);
        if (b.k_cuts > 1) {
            const int64_t rows = p.packed ? p.k_rows : p.k_rows * p.n_docs;
            launch_sum<BF>(Sum{{b.part, b.part_v}, {b.dk, b.dv}, rows, p.k_rows, b.k_cuts * rows * p.dim, rows * p.dim, p.kv_heads, b.k_cuts, p.dim / 4, 2}, stream);
        }
    }
    if (tq > 0) {
        p.tiles = b.q_tiles;
        const auto fn = b.q_cuts > 1 ? &rows_kernel<BF, DP, CAP, true> : &rows_kernel<BF, DP, CAP, false>;
        const size_t lds = kRing * 2 * (size_t)32 * kPitch<DP> * 2;
        if ((rc = kernel_prepare(reinterpret_cast<const void*>(fn), kThreads, lds, &blocks, &cus)) != MMFE_OK) return rc;
        hipLaunchKernelGGL(fn, dim3((uint32_t)(tq * p.heads * b.q_cuts)), dim3(kThreads), lds, stream, b);
        if (b.q_cuts > 1) {
            const int64_t rows = p.packed ? p.q_rows : p.q_rows * p.n_docs;
            launch_sum<BF>(Sum{{b.part, nullptr}, {b.dq, Rows{}}, rows, p.q_rows, rows * p.dim, rows * p.heads * p.dim, p.heads, b.q_cuts, p.dim / 4, 1}, stream);
        }
    }
    return launched("attention backward");
}

template <bool BF, int CAP>
int launch_dim(BackwardArgs& b, hipStream_t stream) {
    const int dp = padded_dim(b.p.dim);
    return dp == 32 ? launch<BF, 32, CAP>(b, stream) : dp == 64 ? launch<BF, 64, CAP>(b, stream) : dp == 96 ? launch<BF, 96, CAP>(b, stream) : launch<BF, 128, CAP>(b, stream);
}

template <bool BF>
int launch_cap(BackwardArgs& b, hipStream_t stream) {
    return b.p.cap > kUsualCap ? launch_dim<BF, kAnyCap>(b, stream) : b.p.cap > 0.f ? launch_dim<BF, kExpCap>(b, stream) : launch_dim<BF, kUncapped>(b, stream);
}

// places of the norms' tiles (see slot)
int64_t slots(const mmfe_attention_args* a, int64_t rows) {
    const int64_t tiles = (rows + kRows - 1) / kRows;
    return a->packed ? tiles + a->n_docs + 1 : tiles * a->n_docs;
}
bool is_whole(const mmfe_attention_args* a) {
    return !a->packed && a->n_docs > 0 && a->heads == a->kv_heads && a->dim <= 64 && a->q_rows <= kWholeRows && a->k_rows <= kWholeRows && a->q_rows + a->k_rows > 0;
}

// parts of the two walks; a causal mask leaves a key min(rows, keys) rows
int key_cuts(const mmfe_attention_args* a) {
    const int64_t seen = a->causal && a->prefix == nullptr && a->k_rows < a->q_rows ? a->k_rows : a->q_rows;
    return walk_cuts(a, a->k_rows, a->kv_heads, seen * (a->heads / a->kv_heads), a->dim > 96 ? 512 : 768);
}
int row_cuts(const mmfe_attention_args* a) { return walk_cuts(a, a->q_rows, a->heads, a->k_rows, 768); }
int64_t key_parts(const mmfe_attention_args* a) { return key_cuts(a) > 1 ? key_cuts(a) * in_all(a, a->k_rows) * a->kv_heads * a->dim : 0; }
int64_t parts(const mmfe_attention_args* a) {          // the two passes use them one after the other
    const int64_t q = row_cuts(a) > 1 ? row_cuts(a) * in_all(a, a->q_rows) * a->heads * a->dim : 0;
    return 2 * key_parts(a) > q ? 2 * key_parts(a) : q;
}
int64_t lse_size(const mmfe_attention_args* a) { return (a->packed ? 1 : (int64_t)a->n_docs) * a->heads * a->q_rows; }

}  // namespace
}  // namespace mmfe

using namespace mmfe;

extern "C" {

int64_t mmfe_attention_backward_workspace(const mmfe_attention_args* a) {
    Problem p{};
    if (make_problem(a, p)) return -1;
    if (is_whole(a)) return 0;
    const int64_t norms = a->dtype == MMFE_OUT_F16 ? a->heads * slots(a, a->q_rows) + a->kv_heads * slots(a, a->k_rows) : 0;
    return (6 * lse_size(a) + parts(a) + norms + 4) * (int64_t)sizeof(float);
}

int mmfe_attention_backward(const mmfe_attention_args* a, const mmfe_attention_grads* g, void* workspace, int device, void* hip_stream) {
    BackwardArgs b{};
    int rc = make_problem(a, b.p);
    if (rc) return rc;
    if (g == nullptr || g->struct_size != (int32_t)sizeof(mmfe_attention_grads)) { set_error("attention: gradients NULL or of another version"); return MMFE_EINVAL; }
    const bool any_q = a->q_rows > 0 && (a->packed || a->n_docs > 0), any_k = a->k_rows > 0 && (a->packed || a->n_docs > 0);
    const bool whole = is_whole(a);
    if (any_q && ((a->out == nullptr && !whole) || a->lse == nullptr || g->grad_out == nullptr || g->grad_q == nullptr)) { set_error("attention: NULL data pointer"); return MMFE_EINVAL; }
    if (any_k && (g->grad_k == nullptr || g->grad_v == nullptr)) { set_error("attention: NULL data pointer"); return MMFE_EINVAL; }
    if ((any_q || any_k) && !whole && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)) { set_error("attention: this call needs a 16-byte aligned workspace"); return MMFE_EINVAL; }
    if ((reinterpret_cast<uintptr_t>(a->out_rest) & 15) != 0) { set_error("attention: out_rest: 16-byte aligned"); return MMFE_EINVAL; }
    // the workspace's statistics are addressed as lse is
    if (any_q && ((a->heads > 1 && a->lse_stride[1] != a->q_rows) || (!a->packed && a->n_docs > 1 && a->lse_stride[0] != a->heads * a->q_rows))) { set_error("attention: lse must be dense"); return MMFE_EINVAL; }
    if (bad_rows("out", a->out, a->out_stride) || bad_rows("grad_out", g->grad_out, g->grad_out_stride) || bad_rows("grad_q", g->grad_q, g->grad_q_stride) ||
        bad_rows("grad_k", g->grad_k, g->grad_k_stride) || bad_rows("grad_v", g->grad_v, g->grad_v_stride)) return MMFE_EINVAL;
    const int64_t tq = count_tiles(b.p, a->q_rows, kRows), tk = count_tiles(b.p, a->k_rows, kRows);
    if (whole ? too_many_blocks((int64_t)a->n_docs * a->heads, 512)
              : too_many_blocks(tq * a->heads + tk * a->kv_heads, kThreads) || too_many_blocks(tq * a->heads * row_cuts(a), kThreads) || too_many_blocks(tk * a->kv_heads * key_cuts(a), kThreads)) {
        set_error("attention: too many rows and heads in one call"); return MMFE_EINVAL;
    }
    auto rows = [](const void* ptr, const int64_t* s) { return Rows{ptr, s[0], s[1], s[2]}; };
    b.out = rows(a->out, a->out_stride); b.rest = static_cast<const char*>(a->out_rest); b.g = rows(g->grad_out, g->grad_out_stride);
    b.dq = rows(g->grad_q, g->grad_q_stride); b.dk = rows(g->grad_k, g->grad_k_stride); b.dv = rows(g->grad_v, g->grad_v_stride);
    b.lse = a->lse; b.lse_b = a->lse_stride[0]; b.lse_h = a->lse_stride[1];
    b.whole = whole;
    b.k_cuts = key_cuts(a); b.q_cuts = row_cuts(a);
    b.aux = static_cast<u32x4*>(workspace);
    b.part = reinterpret_cast<float*>(b.aux + lse_size(a)); b.part_v = b.part + key_parts(a);
    b.lse2 = b.part + parts(a); b.delta = b.lse2 + lse_size(a);
    b.q_slots = (int)slots(a, a->q_rows); b.k_slots = (int)slots(a, a->k_rows);
    b.norm_g = b.delta + lse_size(a); b.norm_v = b.norm_g + (int64_t)a->heads * b.q_slots;
    OnDevice on(device);
    if (on.rc) return on.rc;
    hipStream_t stream = reinterpret_cast<hipStream_t>(hip_stream);
    return a->dtype == MMFE_OUT_BF16 ? launch_cap<true>(b, stream) : launch_cap<false>(b, stream);
}

}  // extern "C"

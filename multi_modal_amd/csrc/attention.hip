// Attention over the tokens of documents (clips of a batch, recordings packed one behind the other):
//     s_ij = scale q_i . k_j          capped: cap tanh(s / cap)          with distance bias: s - slope_h |i + (len_k - len_q) - j|
//     p = softmax over the keys j of the row's document that it may see          o_i = sum_j p_ij v_j          lse_i = log sum_j e^s_ij
// A row sees key j when  not causal, or j <= i + len_k - len_q, or j < prefix of its document.  Rows that see nothing give zeros
// and lse = -inf.
//
// One pass over the keys per block of 128 rows, with the running maximum and sum of the softmax: scores never leave the registers.
// A wave owns 32 rows and computes the TRANSPOSED scores of 32 keys x 32 rows at a time (keys as the first operand), so that a
// lane holds scores of one row only: maximum and sum are register arithmetic plus one exchange between the wave's halves, the
// running state is one value per lane, and the scores, rounded to the 16-bit type, are the second operand of the next product
// (o^T += v^T p^T) as they stand.  Keys and values come by LDS-DMA, in tiles of 32 rows that the 4 waves share, several steps ahead.
//
// What is rounded: p to the tensors' 16-bit type for the second product (half a step each, independent, so the error of o is that
// of its own rounding again); the sums of p are taken before that rounding, in float32, as are maximum, sum and both accumulators.
// Documents of at most kShortKeys keys add a second product with what the rounding of p lost: there an error has few others to average
// with, in o and through delta = g . o in the gradients (grad_q of 3-key documents was 2.0 times as far from the exact one as a
// float32 computation rounded once), and their time is launch and latency.
// A call whose gradients will be wanted also stores the rest of o, what its rounding to 16 bits lost, for delta.
//
// Few rows over many keys (new tokens over what a stream has kept) would leave most of the machine idle in that form: split_kernel
// below cuts the keys into chunks, one block each, and join_kernel puts the chunks' results together.
// The running maximum is raised only when a row's scores exceed it by more than 8 (in log2 units): p stays below 2^8, which both
// types hold, and most tiles skip the rescaling of o.
#include "attention_tiles.h"

#include <algorithm>
#include <cmath>

namespace mmfe {
using namespace attn;

namespace attn {
int64_t in_all(const mmfe_attention_args* a, int64_t rows);
int walk_cuts(const mmfe_attention_args* a, int64_t rows, int heads, int64_t partners, int64_t want);
}  // namespace attn

namespace {

constexpr int kSplitTile = 32;         // keys of a wave's tile in split_kernel
constexpr int kSplitWaves = 2;

struct ForwardArgs {
    Problem p;
    Rows out;
    char* rest;                       // like out: what its rounding lost; NULL: not wanted
    float* lse;                       // (batch, heads, rows) or (heads, rows); NULL: not wanted
    int64_t lse_b, lse_h;
    int cuts;                         // parts of forward_kernel's walk over the keys; more than one: (cuts, heads, rows) results over their own
    float* part;                      // maximum, in float32, and that maximum and sum
    float2* part_ml;
};

// How scores leave the linear form (bits); kBias and kCap take them to log2 units before the maximum.  kCap is kExpCap's form, kWide kAnyCap's.
enum { kPlain = 0, kBias = 1, kCap = 2, kWide = 4 };

template <int SHAPE>
struct Shape {
    float c, slope, cap_in, cap_out;
    AnyCap any;
    __device__ __forceinline__ Shape(const Problem& p, int head) {
        c = p.scale * kLog2e;
        slope = SHAPE & kBias ? __uint_as_float(uniform(__float_as_uint(p.slopes[head] * kLog2e))) : 0.f;
        cap_in = SHAPE & kCap ? 2.f * kLog2e * p.scale / p.cap : 0.f;
        cap_out = SHAPE & kCap ? 2.f * p.cap * kLog2e : 0.f;
        if constexpr (SHAPE & kWide) any.set(p);
    }
    // x: products of 32 keys; at: distance from the lane's row back to its first key (row + off - j0 - 4 * half); side 1: all keys stand at
    // or before all rows of the wave, -1: all behind them, 0: some of each.  Returns what the scores lack: on one side, -slope * |at - r|
    // is a number of the row's plus a number that all lanes share, and only the shared one is added here (one instruction a score, not three).
    // A capped score is cap tanh(z) = cap - 2 cap / (e^(2 z) + 1).
    __device__ __forceinline__ float apply(f32x16& x, float at, int side) const {
        if constexpr (SHAPE & kWide) any.apply<false>(x, nullptr);
        if constexpr (SHAPE & kCap)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fmaf(-cap_out, __builtin_amdgcn_rcpf(exp2_fast(x[i] * cap_in) + 1.f), 0.5f * cap_out);
        if constexpr (SHAPE & kBias) {
            if (side == 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float far = slope * fabsf(at - (float)reg_row(i));
                    x[i] = SHAPE & kCap ? x[i] - far : fmaf(x[i], c, -far);
                }
                return 0.f;
            }
            const float s = side > 0 ? slope : -slope;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float shared = __uint_as_float(uniform(__float_as_uint(s * (float)reg_row(i))));
                x[i] = SHAPE & kCap ? x[i] + shared : fmaf(x[i], c, shared);
            }
            return -s * at;
        }
        return 0.f;
    }
    // factor from the units the maximum is kept in to log2 units
    __device__ __forceinline__ float unit() const { return SHAPE & (kBias | kCap) ? 1.f : c; }
};

// Softmax state of a lane's row, and what 32 keys do to it.
struct State {
    float m = -INFINITY, l = 0.f;
    __device__ __forceinline__ static float largest(const f32x16& a, float lack) {      // lack: the lane's own, before the halves meet
        float m = a[0], k = a[1];
#pragma unroll
        for (int i = 2; i < 16; i += 4) {
            m = max2(max2(m, a[i]), a[i + 1]);
            if (i + 2 < 16) k = max2(max2(k, a[i + 2]), a[i + 3]);
        }
        return both_max(max2(m, k) + lack);
    }
    // raises the running maximum when scores exceed it by more than 8 log2 units; true: o and l have to be scaled by alpha
    __device__ __forceinline__ bool raise(float mx, float unit, float& alpha) {
        if (!__any((mx - m) * unit > 8.f)) return false;
        const float up = max2(m, mx);
        alpha = exp2_fast(up == -INFINITY ? 0.f : (m - up) * unit);
        m = up;
        l *= alpha;
        return true;
    }
    // lack: what the scores lack, in log2 units
    __device__ __forceinline__ void exponentials(f32x16& x, float unit, float lack) {
        const float mc = (m == -INFINITY ? 0.f : m * unit) - lack;
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            x[i] = exp2_fast(fmaf(x[i], unit, -mc));
            x[i + 1] = exp2_fast(fmaf(x[i + 1], unit, -mc));
            s0 += x[i];
            s1 += x[i + 1];
        }
        l += s0 + s1;
    }
};

__device__ __forceinline__ void hide(f32x16& x, int left) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = reg_row(i) < left ? x[i] : -INFINITY;
}

// Bound by the matrix and the vector instructions of a SIMD, which overlap only in part: 8192 rows, 16 heads of 128: 533 us, 1031 TFLOP/s, causal 288; 12 heads of
// 64: 254 us, 812 TFLOP/s (fewer products per exponential).
//
// Keys of a step, and tiles of keys (and of values) in LDS.
constexpr int kStepKeys = 32;
constexpr int kRing = 4;
constexpr float kLowest = -__FLT_MAX__;      // maximum of keys that are seen and have scores of -infinity, which no keys at all have
static_assert(kStepKeys * kRing >= kShortKeys, "a short document's keys are in LDS at once");

// CUT: the walk is cut into parts (as an argument that any call could have, 3 % slower where it is not)
// Head sizes up to 64 are held to 128 registers, four waves a SIMD (64 x 193 rows, 12 heads: 28 us, with three 29; 16 x 577: 32 and 35).
template <bool BF, int DP, int SHAPE, bool CUT>
__global__ void __launch_bounds__(kThreads, DP <= 64 ? 4 : 2) forward_kernel(const ForwardArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];               // [kRing k tiles][kRing v tiles]
    const Problem& p = a.p;
    constexpr int kTileBytes = kStepKeys * kPitch<DP> * 2;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int cuts = CUT ? a.cuts : 1, lot = blockIdx.x % (p.heads * cuts), cut = CUT ? lot / p.heads : 0;
    Doc d;
    if (!find_doc<true>(p, blockIdx.x / (p.heads * cuts), kRows, d)) return;
    const int head = head_of(p, lot % p.heads), kvh = head / p.group;
    const int row0 = d.tile * kRows, w0 = row0 + 32 * wave, row = w0 + col;
    const int nq = d.nq, nk = d.nk, off = nk - nq;
    // keys [0, limit of the block / the wave / the row) are visible
    auto limit = [&](int r) {
        if (r >= nq) r = nq - 1;
        return p.causal ? min(nk, max(d.prefix, r + off + 1)) : nk;
    };
    const int block_lim = row0 < nq ? limit(row0 + kRows - 1) : 0;
    const int wave_lim = w0 < nq ? limit(w0 + 31) : 0;
    const int full_lim = w0 < nq ? limit(w0) : 0;                             // keys that all rows of the wave see
    const int lim = row < nq ? limit(row) : 0;
    const bool at_once = nk <= kShortKeys;                                    // at most kRing tiles: all of them are asked for at the start
    const int all = block_lim > 0 ? (block_lim + kStepKeys - 1) / kStepKeys : 0, share = !CUT || at_once ? all : (all + cuts - 1) / cuts;
    const int t0 = CUT ? min(cut * share, all) : 0, n = min(t0 + share, all); // this block's steps

    typedef Loader<DP, kStepKeys, kWaves> Load;
    Load lk, lv;
    lk.init(p.dim, p.k.n, wave);
    lv.init(p.dim, p.v.n, wave);
    const unsigned lds0 = lds_address(smem);
    auto load_k = [&](int t) {
        lk.load(row_base(p.k, d, d.k0 + (int64_t)t * kStepKeys, kvh), nk - t * kStepKeys, p.dim, p.k.n, uniform(lds0 + (t % kRing) * kTileBytes), wave);
    };
    auto load_v = [&](int t) {
        lv.load(row_base(p.v, d, d.k0 + (int64_t)t * kStepKeys, kvh), nk - t * kStepKeys, p.dim, p.v.n, uniform(lds0 + (kRing + t % kRing) * kTileBytes), wave);
    };
    // in the order in which the steps need them
    if (t0 < n) load_k(t0);
    if (t0 + 1 < n) load_k(t0 + 1);
#pragma unroll
    for (int i = 0; i < kRing - 2; ++i) {
        if (t0 + i < n) load_v(t0 + i);
        if (t0 + i + 2 < n) load_k(t0 + i + 2);
    }

    u32x4 qf[DP / 16];
    {
        const int r = row < nq ? row : nq - 1;
        const char* q = row_base(p.q, d, d.q0 + (r > 0 ? r : 0), head);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            qf[s] = u32x4{0, 0, 0, 0};
            if (nq > 0 && 16 * s + 8 * half < p.dim) qf[s] = *reinterpret_cast<const u32x4*>(q + 32 * s + 16 * half);
        }
    }
    const Shape<SHAPE> sh(p, head);
    const float unit = sh.unit();
    f32x16 o[DP / 32], x{};
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = f32x16{};
    State st;

    auto scores = [&](int t) {
        const char* kt = smem + (t % kRing) * kTileBytes;
        f32x16 y{};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) y = mfma<BF>(read_rows<DP>(kt, 0, s), qf[s], y);
        return y;
    };
    auto values = [&](int t, int s, u32x4 pf) {
        const char* vt = smem + (kRing + t % kRing) * kTileBytes;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) o[i] = mfma<BF>(read_cols<DP>(vt, 16 * s, 32 * i), pf, o[i]);
    };
    auto shape_and_hide = [&](f32x16& x, int t) {
        const int j0 = t * kStepKeys;
        float lack = 0.f;
        if constexpr (SHAPE != kPlain) lack = sh.apply(x, (float)(row + off - j0 - 4 * half), j0 + kStepKeys - 1 <= w0 + off ? 1 : j0 >= w0 + 31 + off ? -1 : 0);
        if (j0 + kStepKeys > full_lim) hide(x, lim - j0 - 4 * half);
        return lack;
    };
    auto rescale = [&](float mx) {
        float alpha;
        if (st.raise(mx, unit, alpha)) {
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[i] *= alpha;
        }
    };

    if (at_once)
#pragma unroll
        for (int t = kRing - 2; t < kRing; ++t)
            if (t0 == 0 && t < n) load_v(t);
    wait_all();
    block_sync();
    arrived(qf);
    if (at_once) {
        for (int t = t0; t < n && t * kStepKeys < wave_lim; ++t) {
            x = scores(t);
            const float lack = shape_and_hide(x, t);
            rescale(State::largest(x, lack));
            st.exponentials(x, unit, lack);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const u32x4 pf = operand<BF>(x, s);
                values(t, s, pf);
                values(t, s, operand_rest<BF>(x, s, pf));
            }
        }
    } else if (t0 < n) {
        // Products of one step run beside the softmax of another: step t turns the scores of its 32 keys, computed a step earlier, into p,
        // while the matrix pipe adds step t - 1 to o (beside the maximum) and forms the scores of step t + 1 (beside the exponentials).
        // So step t needs k of t + 1 and v of t - 1; their buffers' former tiles were used up in step t - 1 at the latest, and it asks for
        // k of t + kRing and v of t + kRing - 2: kRing - 1 steps ahead of their use.
        constexpr int kAhead = (kRing - 2) * 2 * Load::kCount;
        u32x4 pf[2];
        if (t0 * kStepKeys < wave_lim) x = scores(t0);
        auto step = [&](int t) {           // every wave's parts have arrived, and its reads of the buffers that are asked for now are done
            if (t - 1 + kRing < n) wait_but<kAhead>();     // the last kRing - 2 steps asked for a whole tile of each
            else wait_all();
            block_sync();
            if (t + kRing < n) load_k(t + kRing);
            if (t + kRing - 2 < n) load_v(t + kRing - 2);
        };
        // this wave's steps end before `mine`; it only keeps step with the others behind them
        const int mine = max(t0, min(n, (wave_lim + kStepKeys - 1) / kStepKeys));
        auto walk = [&](int t, f32x16& x, f32x16& y) {
            step(t);
            const float lack = shape_and_hide(x, t);
            const float mx = State::largest(x, lack);
            if (t > t0) {
                values(t - 1, 0, pf[0]);
                values(t - 1, 1, pf[1]);
            }
            rescale(mx);
            y = scores(t + 1);                       // past the last step: of whatever the buffer holds, and dropped
            st.exponentials(x, unit, lack);
            pf[0] = operand<BF>(x, 0);
            pf[1] = operand<BF>(x, 1);
        };
        // by twos, as the next step's scores would else be copied over this one's: 8 instructions of about 100 (8192 rows, 16 heads of 128: 553 -> 533 us;
        // 12 heads of 64: 266 -> 254)
        f32x16 y;
        for (int t = t0; t < mine; t += 2) {
            walk(t, x, y);
            if (t + 1 < mine) walk(t + 1, y, x);
        }
        if (mine < n) step(mine);
        else {
            wait_all();
            block_sync();
        }
        if (mine > t0) {
            values(mine - 1, 0, pf[0]);
            values(mine - 1, 1, pf[1]);
        }
        for (int t = mine + 1; t < n; ++t) step(t);
        if (mine < n) {
            wait_all();
            block_sync();
        }
    }
    const float l = both_sum(st.l);
    if (row >= d.rows) return;
    if constexpr (CUT) {
        const int64_t place = ((int64_t)cut * p.heads + head) * (p.packed ? p.q_rows : p.q_rows * p.n_docs) + (p.packed ? d.q0 : d.batch * p.q_rows) + row;
        const bool sees = lim > t0 * kStepKeys && t0 < n;
        if (half == 0) a.part_ml[place] = sees ? make_float2(st.m == -INFINITY ? kLowest : st.m * unit, l) : make_float2(-INFINITY, 0.f);
        if (!sees) return;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (32 * i + 8 * g < p.dim)
                    *reinterpret_cast<float4*>(a.part + place * p.dim + 32 * i + 8 * g + 4 * half) = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
        return;
    }
    const bool some = lim > 0;
    const float inv = some ? 1.f / l : 0.f;
    const int64_t at = 2 * (d.batch * a.out.b + (d.q0 + row) * a.out.n + head * a.out.h);
    char* out = static_cast<char*>(const_cast<void*>(a.out.p)) + at;
    char* rest = a.rest ? a.rest + at : nullptr;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = 32 * i + 8 * g;
            if (e >= p.dim) continue;
            const int to = 2 * (e + 4 * half);
            if (some) store4<BF>(out + to, rest ? rest + to : nullptr, o[i][4 * g] * inv, o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv);
            else store4<BF>(out + to, rest ? rest + to : nullptr, 0.f, 0.f, 0.f, 0.f);
        }
    if (a.lse != nullptr && half == 0)
        a.lse[d.batch * a.lse_b + head * a.lse_h + d.q0 + row] = some ? (st.m * unit + __builtin_amdgcn_logf(l)) * (1.f / kLog2e) : -INFINITY;
}

// The parts of cut walks, 4 elements of a row a thread; memory bound (8192 rows, 16 heads of 128 in two parts: 31 us, 5.4 TB/s).
template <bool BF>
__global__ void __launch_bounds__(kThreads) gather_kernel(const ForwardArgs a) {
    const Problem& p = a.p;
    const int pieces = p.dim / 4;
    const int64_t rows = p.packed ? p.q_rows : p.q_rows * p.n_docs, step = rows * p.heads, n = step * pieces;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
        const int64_t hr = i / pieces;
        const int e = 4 * (int)(i - hr * pieces), head = (int)(hr / rows);
        const int64_t row = hr - head * rows;
        float top = -INFINITY;
        for (int c = 0; c < a.cuts; ++c) top = max2(top, a.part_ml[c * step + hr].x);
        const bool some = top != -INFINITY;
        float total = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < a.cuts; ++c) {
            const float2 ml = a.part_ml[c * step + hr];
            if (ml.x == -INFINITY) continue;                          // sees none of these keys
            const float k = exp2_fast(ml.x - top);
            const float4 u = *reinterpret_cast<const float4*>(a.part + (c * step + hr) * p.dim + e);
            total += k * ml.y;
            v.x += k * u.x; v.y += k * u.y; v.z += k * u.z; v.w += k * u.w;
        }
        const int64_t b = p.packed ? 0 : row / p.q_rows, r = row - b * p.q_rows;
        const int64_t at = 2 * (b * a.out.b + r * a.out.n + head * a.out.h + e);
        const float inv = some ? 1.f / total : 0.f;
        char* out = static_cast<char*>(const_cast<void*>(a.out.p)) + at;
        if (some) store4<BF>(out, a.rest ? a.rest + at : nullptr, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        else store4<BF>(out, a.rest ? a.rest + at : nullptr, 0.f, 0.f, 0.f, 0.f);
        if (e == 0 && a.lse != nullptr) a.lse[b * a.lse_b + head * a.lse_h + r] = some ? (top + __builtin_amdgcn_logf(total)) * (1.f / kLog2e) : -INFINITY;
    }
}

// ---- few rows over many keys ----
//
// The rows of one key head are its query heads' rows, row r = (token r / group, query head r % group), so that a group reads its keys
// once; a block takes 32 of them and one chunk of the keys.  Its 2 waves work on tiles of 32 keys of their own (every other one), each
// with its own double-buffered LDS tiles and no barrier, and meet once at the end.  Bound by reading k and v: the products run at
// 32 rows whatever the number of valid ones, and p enters with both halves (hi + rest), which costs nothing here.  16 streams of 1000 to 30001 keys, 4 key
// heads of 128: 90 us for 385 MB, 4.3 TB/s.

struct SplitArgs {
    ForwardArgs f;
    int chunk, n_splits, n_units, row_tiles;
    float* part;                      // (unit, split, 32, dim) partial results over their own maximum; (unit, split, 32, 2) maximum and sum behind them
    float* part_ml;
};

// Row r of a unit.
struct SplitRow {
    int token, head;
    bool valid;
    __device__ __forceinline__ SplitRow(const Problem& p, int r, int kvh, int nq) {
        token = r / p.group;
        head = kvh * p.group + r - token * p.group;
        valid = token < nq;
    }
};

template <bool BF>
__device__ __forceinline__ void finish_row(const ForwardArgs& f, int doc, const SplitRow& r, int e, bool some, float m, float l, float4 v) {
    const int64_t at = 2 * (doc * f.out.b + r.token * f.out.n + r.head * f.out.h + e);
    const float inv = some ? 1.f / l : 0.f;
    char* out = static_cast<char*>(const_cast<void*>(f.out.p)) + at;
    if (some) store4<BF>(out, f.rest ? f.rest + at : nullptr, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    else store4<BF>(out, f.rest ? f.rest + at : nullptr, 0.f, 0.f, 0.f, 0.f);
    if (e == 0 && f.lse != nullptr)
        f.lse[doc * f.lse_b + r.head * f.lse_h + r.token] = some ? (m + __builtin_amdgcn_logf(l)) * (1.f / kLog2e) : -INFINITY;
}

template <bool BF, int DP>
__global__ void __launch_bounds__(64 * kSplitWaves, 1) split_kernel(const SplitArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];       // per wave: 2 x [k tile][v tile]
    const Problem& p = a.f.p;
    constexpr int kTileBytes = kSplitTile * kPitch<DP> * 2;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    // Chunk by chunk, the units of a chunk turned by the chunk's number: neighbouring blocks go to different XCDs, and a document's chunks
    // (long documents have many, short ones one) then spread over all of them, while the key heads of a chunk's keys, which lie
    // interleaved in memory, are read at the same time.
    const int split = blockIdx.x / a.n_units, place = blockIdx.x - split * a.n_units;
    const int unit = (place + split) % a.n_units, part = unit * a.n_splits + split;
    const int kvh = unit % p.kv_heads, rt = (unit / p.kv_heads) % a.row_tiles;
    const int b = unit / p.kv_heads / a.row_tiles;
    Doc d;
    (void)find_doc<true>(p, b, kRows, d);                             // padded, one "tile" per document
    const int nq = d.nq, nk = d.nk, off = nk - nq;
    const int n_rows = min(32, (int)p.q_rows * p.group - 32 * rt);    // rows that exist, valid or not
    auto limit = [&](int token) { return token >= nq ? 0 : p.causal ? min(nk, max(d.prefix, token + off + 1)) : nk; };
    const int last_token = min((32 * rt + n_rows - 1) / p.group, nq - 1);
    const int max_lim = last_token >= 0 && 32 * rt / p.group < nq ? limit(last_token) : 0;
    const int full_lim = limit(32 * rt / p.group);
    const int s0 = split * a.chunk, s1 = min(s0 + a.chunk, max_lim);
    float2* ml = reinterpret_cast<float2*>(a.part_ml) + (int64_t)part * 32;
    if (s0 >= s1 && a.n_splits > 1) {                                 // nothing of this chunk is visible to these rows
        if (threadIdx.x < n_rows) ml[threadIdx.x] = make_float2(-INFINITY, 0.f);
        return;
    }
    const SplitRow mine(p, 32 * rt + col, kvh, nq);
    const int lim = col < n_rows ? limit(mine.token) : 0;
    const int n_tiles = s1 > s0 ? (s1 - s0 + kSplitTile - 1) / kSplitTile : 0;

    Loader<DP, kSplitTile, 1> lk, lv;
    lk.init(p.dim, p.k.n, 0);
    lv.init(p.dim, p.v.n, 0);
    const unsigned lds0 = uniform(lds_address(smem) + wave * 4 * kTileBytes);
    auto stage = [&](int t, int buf) {
        const int j0 = s0 + t * kSplitTile;
        const unsigned dst = uniform(lds0 + buf * 2 * kTileBytes);
        lk.load(row_base(p.k, d, j0, kvh), nk - j0, p.dim, p.k.n, dst, 0);
        lv.load(row_base(p.v, d, j0, kvh), nk - j0, p.dim, p.v.n, dst + kTileBytes, 0);
    };
    u32x4 qf[DP / 16];
    {
        const bool ok = mine.valid && col < n_rows;
        const char* q = row_base(p.q, d, ok ? mine.token : 0, ok ? mine.head : 0);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            qf[s] = u32x4{0, 0, 0, 0};
            if (ok && 16 * s + 8 * half < p.dim) qf[s] = *reinterpret_cast<const u32x4*>(q + 32 * s + 16 * half);
        }
    }
    const float c = p.slopes ? 1.f : p.scale * kLog2e;
    const float slope = p.slopes && col < n_rows ? p.slopes[mine.head] * kLog2e : 0.f;
    AnyCap cap{};
    if (p.cap > 0.f) cap.set(p);
    if (wave < n_tiles) stage(wave, 0);

    f32x16 o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.f;
    int buf = 0;
    wait_all();
    arrived(qf);
    for (int t = wave; t < n_tiles; t += kSplitWaves, buf ^= 1) {
        if (t + kSplitWaves < n_tiles) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the other buffer has been read
            stage(t + kSplitWaves, buf ^ 1);
            asm volatile("s_waitcnt vmcnt(%0)" :: "n"(2 * Loader<DP, kSplitTile, 1>::kCount) : "memory");      // all but the tile just asked for
        } else wait_all();
        const int j0 = s0 + t * kSplitTile;
        const char* kt = smem + (wave * 2 + buf) * 2 * kTileBytes;
        const char* vt = kt + kTileBytes;
        f32x16 x{};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) x = mfma<BF>(read_rows<DP>(kt, 0, s), qf[s], x);
        if (p.cap > 0.f) cap.apply<false>(x, nullptr);
        if (p.slopes) {
            const float at = (float)(mine.token + off - j0 - 4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fmaf(x[i], p.scale * kLog2e, -slope * fabsf(at - (float)reg_row(i)));
        }
        if (j0 + kSplitTile > full_lim || j0 + kSplitTile > s1) {
            const int left = min(lim, s1) - j0 - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = reg_row(i) < left ? x[i] : -INFINITY;
        }
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
        mx = both_max(mx);
        if (__any((mx - m) * c > 8.f)) {
            const float up = fmaxf(m, mx);
            const float alpha = exp2_fast(up == -INFINITY ? 0.f : (m - up) * c);
            m = up;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[i] *= alpha;
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = exp2_fast(fmaf(x[i], c, -mc));
            sum += x[i];
        }
        l += sum;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const u32x4 pf = operand<BF>(x, s), rf = operand_rest<BF>(x, s, pf);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const u32x4 vf = read_cols<DP>(vt, 16 * s, 32 * i);
                o[i] = mfma<BF>(vf, pf, o[i]);
                o[i] = mfma<BF>(vf, rf, o[i]);
            }
        }
    }
    l = both_sum(l);
    m = m * c;                                                        // log2 units (c > 0; -inf stays)
    // the waves' results meet in LDS: [wave][row][DP + 4] values, [wave][row] maximum and sum
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    block_sync();
    constexpr int kMeet = DP + 4;
    float* wo = reinterpret_cast<float*>(smem);
    float2* wml = reinterpret_cast<float2*>(wo + kSplitWaves * 32 * kMeet);
    if (col < n_rows) {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4*>(wo + (wave * 32 + col) * kMeet + 32 * i + 8 * g + 4 * half) = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
        if (half == 0) wml[wave * 32 + col] = make_float2(m, l);
    }
    __syncthreads();
    const int pieces = p.dim / 4;
    for (int i = threadIdx.x; i < n_rows * pieces; i += 64 * kSplitWaves) {
        const int r = i / pieces, e = 4 * (i - r * pieces);
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kSplitWaves; ++w) top = fmaxf(top, wml[w * 32 + r].x);
        float total = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kSplitWaves; ++w) {
            const float2 s = wml[w * 32 + r];
            if (s.y == 0.f) continue;                                 // saw no key
            const float k = exp2_fast(s.x - top);
            const float4 u = *reinterpret_cast<const float4*>(wo + (w * 32 + r) * kMeet + e);
            total += k * s.y;
            v.x += k * u.x; v.y += k * u.y; v.z += k * u.z; v.w += k * u.w;
        }
        const SplitRow row(p, 32 * rt + r, kvh, nq);
        if (a.n_splits == 1) finish_row<BF>(a.f, b, row, e, limit(row.token) > 0, top, total, v);
        else {
            *reinterpret_cast<float4*>(a.part + ((int64_t)part * 32 + r) * p.dim + e) = v;
            if (e == 0) ml[r] = make_float2(top, total);
        }
    }
}

// One block per row: kThreads / (dim / 4) chunks at a time, then the chunks' sums in LDS.  256 rows of 128 in up to 32 chunks: 7.5 us, launch and latency.
template <bool BF>
__global__ void __launch_bounds__(kThreads) join_kernel(const SplitArgs a) {
    __shared__ float4 lds_v[kThreads];
    __shared__ float2 lds_ml[kThreads];
    const Problem& p = a.f.p;
    const int unit = blockIdx.x >> 5, r = blockIdx.x & 31;
    const int kvh = unit % p.kv_heads, rt = (unit / p.kv_heads) % a.row_tiles;
    const int b = unit / p.kv_heads / a.row_tiles;
    if (32 * rt + r >= (int)p.q_rows * p.group) return;
    Doc d;
    (void)find_doc<true>(p, b, kRows, d);
    const int pieces = p.dim / 4, groups = kThreads / pieces;
    const int g = threadIdx.x / pieces, e = 4 * (threadIdx.x - g * pieces);
    float top = -INFINITY, total = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (g < groups)
        for (int s = g; s < a.n_splits; s += groups) {
            const int64_t at = (int64_t)(unit * a.n_splits + s) * 32 + r;
            const float2 ml = reinterpret_cast<const float2*>(a.part_ml)[at];
            if (ml.y == 0.f) continue;
            const float4 u = *reinterpret_cast<const float4*>(a.part + at * p.dim + e);
            const float up = fmaxf(top, ml.x);
            const float k0 = exp2_fast(top - up), k1 = exp2_fast(ml.x - up);
            top = up;
            total = total * k0 + ml.y * k1;
            v.x = v.x * k0 + u.x * k1; v.y = v.y * k0 + u.y * k1; v.z = v.z * k0 + u.z * k1; v.w = v.w * k0 + u.w * k1;
        }
    lds_v[threadIdx.x] = v;
    lds_ml[threadIdx.x] = make_float2(top, total);
    __syncthreads();
    if (g != 0) return;
    for (int o = 1; o < groups; ++o) top = fmaxf(top, lds_ml[o * pieces + threadIdx.x].x);
    total = 0.f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int o = 0; o < groups; ++o) {
        const float2 ml = lds_ml[o * pieces + threadIdx.x];
        if (ml.y == 0.f) continue;
        const float k = exp2_fast(ml.x - top);
        const float4 u = lds_v[o * pieces + threadIdx.x];
        total += k * ml.y;
        v.x += k * u.x; v.y += k * u.y; v.z += k * u.z; v.w += k * u.w;
    }
    const SplitRow row(p, 32 * rt + r, kvh, d.nq);
    const int lim = !row.valid ? 0 : p.causal ? min(d.nk, max(d.prefix, row.token + d.nk - d.nq + 1)) : d.nk;
    finish_row<BF>(a.f, b, row, e, lim > 0, top, total, v);
}

typedef void (*forward_fn)(const ForwardArgs);
typedef void (*split_fn)(const SplitArgs);
template <bool BF, int SHAPE, bool CUT>
forward_fn pick_dim(int dim) {
    return dim <= 32 ? &forward_kernel<BF, 32, SHAPE, CUT> : dim <= 64 ? &forward_kernel<BF, 64, SHAPE, CUT> : dim <= 96 ? &forward_kernel<BF, 96, SHAPE, CUT> : &forward_kernel<BF, 128, SHAPE, CUT>;
}
template <bool BF, bool CUT>
forward_fn pick_forward(int dim, bool bias, float cap) {
    if (cap > kUsualCap) return bias ? pick_dim<BF, kBias | kWide, CUT>(dim) : pick_dim<BF, kWide, CUT>(dim);
    if (bias) return cap > 0.f ? pick_dim<BF, kBias | kCap, CUT>(dim) : pick_dim<BF, kBias, CUT>(dim);
    return cap > 0.f ? pick_dim<BF, kCap, CUT>(dim) : pick_dim<BF, kPlain, CUT>(dim);
}
template <bool BF>
split_fn pick_split(int dim) {
    return dim <= 32 ? &split_kernel<BF, 32> : dim <= 64 ? &split_kernel<BF, 64> : dim <= 96 ? &split_kernel<BF, 96> : &split_kernel<BF, 128>;
}

// How a call's keys are cut: chunks of split_kernel (n_splits > 0), or parts of forward_kernel's walks.
//
// A unit's block takes about 8 us to start and end and 16 (head size 64: 15) per 1000 keys, a block of the row kernel 19 for the four times as many
// rows it shares its keys among.  So split_kernel pays for units of few rows, above all where query heads share their keys, which the row
// kernel reads once per query head.  Measured over 1 to 8000 rows, 1 to 128 documents of 200 to 32000 keys, 12 heads, 16 on 4 and smaller sets, of 64 and 128,
// documents as long as their room and of lengths from 1 to 30 in 32:
//   - up to 512 keys, and up to 2048 where 256 units fill the CUs: no chunks; the row kernel, unless units share keys and its blocks do not all run
//     at once (128 streams of 500 keys, one row, 16 heads on 4: 26.6 us, row kernel 61.4; 32 of them 17.3 and 18.3; 64 rows of 32 documents
//     of 1000 keys, 12 heads of 64: 27, in chunks of 512 keys 75)
//   - more than 64 units, nearly as many as the row kernel's blocks or more: the row kernel, its walks cut (8000 keys, 16 heads on 4 of 128, 512 rows: 61 us,
//     uncut 172, in chunks 120; 128 rows, 64 units: 39 in chunks, 173 uncut; 8 documents of 32 rows, 6000 keys, 16 heads on 4 of 128: 49 cut, 63 in
//     chunks; of 9 rows, half as many units as blocks: 47 cut, 44 in chunks)
//     Several documents with lengths of their own may be much shorter than their room: up to 128 rows of each are then cut into parts of 2048 keys as
//     long as that makes no more than four times the blocks (16 documents of 32 rows over 1000 to 30001 keys in 32768, 16 heads on 4 of 128: 356 us
//     without, 183 with; 8192 rows of one, 16 heads: 370 without, 415 with)
//   - else chunks that make 512 blocks, two on each CU, of 256 keys at least, and of 1024 at most (documents shorter than their room leave chunks
//     empty) unless that makes more than 2048: 16 streams of 1000 to 30001 keys in 32768, 4 key heads of 128: 109 / 93 / 100 / 113 us with 512 /
//     1024 / 2048 / 4096 keys; 32 streams of 2000 keys, one row, 4 key heads of 128: 39 / 34 / 33 with 256 / 512 / 1024.
// Over 486 shapes of 1 to 32 documents, 1 to 2048 rows and 500 to 32000 keys (profiles/token_ops_cuts.csv) a call takes 4.6 % longer on average than with the
// best of these choices for it (documents as long as their room 3.7 %, of uneven lengths 6.2 %), half of them at most 1.3 %; the worst are 8 documents of 512 rows and
// 1000 to 30001 keys in 32000, 16 heads on 4 of 64, in two parts: 500 us, in six 302.
struct Cut {
    int row_tiles = 0, chunk = 0, n_splits = 0, cuts = 1;
    int64_t units = 0;
};
Cut cut_keys(const mmfe_attention_args* a) {
    Cut c;
    const int64_t keys = a->k_rows, row_tiles = (a->q_rows * (a->heads / a->kv_heads) + 31) / 32, units = a->n_docs * row_tiles * a->kv_heads;
    const int64_t blocks = a->n_docs * ((a->q_rows + kRows - 1) / kRows) * a->heads;       // of the row kernel, of padded documents
    const int want = a->dim > 64 ? 512 : 768;
    c.cuts = std::min(12, walk_cuts(a, a->q_rows, a->heads, keys, want));
    if (a->packed || a->q_rows < 1 || a->n_docs < 1) return c;
    if (a->k_len != nullptr && a->n_docs > 1 && a->q_rows <= kRows) c.cuts = (int)std::max<int64_t>(c.cuts, std::min<int64_t>(16, std::min(keys / 2048, 4 * want / blocks)));
    if (keys <= kShortKeys) return c;
    const bool whole = keys <= 512 || (keys <= 2048 && units >= 256);
    if (whole ? units >= blocks || blocks <= 512 : units > 64 && 5 * units >= 4 * blocks) return c;
    const int64_t all = keys * units;
    int64_t chunk = (all + 511) / 512, most = (all + 2047) / 2048;
    if (most < 1024) most = 1024;
    chunk = chunk < 256 ? 256 : chunk > most ? most : chunk;
    chunk = whole ? keys : (chunk + 127) / 128 * 128;
    c.cuts = 1;
    c.row_tiles = (int)row_tiles;
    c.units = units;
    c.chunk = (int)chunk;
    c.n_splits = (int)((keys + chunk - 1) / chunk);
    return c;
}

}  // namespace

namespace attn {

int64_t in_all(const mmfe_attention_args* a, int64_t rows) { return a->packed ? rows : rows * a->n_docs; }
// Parts that the walks of `rows` (the rows, or for the gradients of k and v the keys) over `partners` are cut into, whose float32 sums another
// launch adds: as many as fill the machine, about `want` blocks in all (768; 512 where a CU holds fewer, at head size 128), each of 256 partners or
// more.  Walks of less than 1000 are not worth that launch, nor of 2000 where half of the blocks are there.  Of packed documents only the mean
// is known here; the long ones are taken to have three times as many partners.  Forward and backward, causal, head size 64: 4000 rows, 4 query
// heads on one key head: 548 us uncut, 126 so; 64 rows over 8000 keys, 6 heads: 234 and 62; 32 documents of 400, 12 heads on 4, which 512 blocks
// serve: 132, and 151 if cut.  Forward alone: 4000 rows, 2 key heads of 128 and 4 query heads: 104 and 46; one recording of 4000 among 12 of 50, 6 heads: 86
// and 40.  Over 87 shapes of 1 to 32 documents of 64 to 8000 rows (profiles/token_ops_cuts.csv) forward and backward take 3.1 % longer on average than with the best
// number of parts for the keys' walks, 1.2 % for the rows'; the worst are 2 documents of 300 rows and 3000 keys, 16 heads on 4 of 128: 214 us, uncut 178.
int walk_cuts(const mmfe_attention_args* a, int64_t rows, int heads, int64_t partners, int64_t want) {
    if (a->n_docs < 1 || rows < 1) return 1;
    const int64_t tiles = (rows + kRows - 1) / kRows, blocks = (a->packed ? tiles : tiles * a->n_docs) * heads;
    if (a->packed && a->n_docs > 3) partners = partners * 3 / a->n_docs;
    if (partners < (2 * blocks < want ? 1000 : 2000)) return 1;
    int64_t n = (want + blocks / 2) / blocks;
    if (n > partners / 256) n = partners / 256;
    return n < 1 ? 1 : (int)n;
}

int padded_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128; }
int pitch(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

bool bad_rows(const char* name, const void* ptr, const int64_t* s) {
    // 16-byte pieces; a tile's rows are reached by 32-bit byte offsets
    if ((reinterpret_cast<uintptr_t>(ptr) & 15) != 0 || (s[0] & 7) != 0 || (s[1] & 7) != 0 || (s[2] & 7) != 0 || s[0] < 0 || s[1] < 0 || s[2] < 0 || s[1] > (1 << 24)) {
        set_error("attention: %s: 16-byte aligned rows (strides multiples of 8 elements, row stride up to 2^24)", name);
        return true;
    }
    return false;
}

// Checks what can be checked on the host and fills the kernels' view of the call.
int make_problem(const mmfe_attention_args* a, Problem& p) {
    if (a == nullptr || a->struct_size != (int32_t)sizeof(mmfe_attention_args)) { set_error("attention: arguments NULL or of another version"); return MMFE_EINVAL; }
    if (a->dtype != MMFE_OUT_F16 && a->dtype != MMFE_OUT_BF16) { set_error("attention: float16 or bfloat16 tensors"); return MMFE_EINVAL; }
    if (a->dim < 8 || a->dim > 128 || a->dim % 8 != 0) { set_error("attention: head size %d: a multiple of 8 up to 128", a->dim); return MMFE_EINVAL; }
    if (a->n_docs < 0 || a->q_rows < 0 || a->k_rows < 0) { set_error("attention: negative size"); return MMFE_EINVAL; }
    if (a->heads < 1 || a->kv_heads < 1 || a->heads > 4096 || a->heads % a->kv_heads != 0) { set_error("attention: %d query heads cannot share %d key heads", a->heads, a->kv_heads); return MMFE_EINVAL; }
    if (a->q_rows > (1 << 30) || a->k_rows > (1 << 30) || a->n_docs > (1 << 24)) { set_error("attention: too many rows"); return MMFE_EINVAL; }
    if (a->slopes != nullptr && (a->q_rows > (1 << 24) || a->k_rows > (1 << 24))) { set_error("attention: distances are float32: at most 2^24 rows with slopes"); return MMFE_EINVAL; }
    // the least scale takes the gradients' mark of rows without keys, -1e30 in the products' units, to -1200 in log2 units: p = 0
    if (!(a->scale >= 0x1p-90f) || a->scale > 0x1p126f || !(a->cap >= 0.f) || !std::isfinite(a->cap)) { set_error("attention: scale must lie between 2^-90 and 2^126, cap >= 0 be finite"); return MMFE_EINVAL; }
    if (a->cap > 0.f && !std::isfinite(4.f * a->scale / a->cap)) { set_error("attention: cap is too small against scale"); return MMFE_EINVAL; }
    if (a->packed && (a->q_off == nullptr || a->k_off == nullptr)) { set_error("attention: packed documents need offsets"); return MMFE_EINVAL; }
    if (a->prefix != nullptr && !a->causal) { set_error("attention: a prefix belongs to a causal mask"); return MMFE_EINVAL; }
    const bool any_q = a->q_rows > 0 && (a->packed || a->n_docs > 0), any_k = a->k_rows > 0 && (a->packed || a->n_docs > 0);
    if ((any_q && a->q == nullptr) || (any_k && (a->k == nullptr || a->v == nullptr))) { set_error("attention: NULL data pointer"); return MMFE_EINVAL; }
    if (bad_rows("q", a->q, a->q_stride) || bad_rows("k", a->k, a->k_stride) || bad_rows("v", a->v, a->v_stride)) return MMFE_EINVAL;
    p.q = Rows{a->q, a->q_stride[0], a->q_stride[1], a->q_stride[2]};
    p.k = Rows{a->k, a->k_stride[0], a->k_stride[1], a->k_stride[2]};
    p.v = Rows{a->v, a->v_stride[0], a->v_stride[1], a->v_stride[2]};
    p.q_len = a->packed ? nullptr : a->q_len; p.k_len = a->packed ? nullptr : a->k_len;
    p.q_off = a->q_off; p.k_off = a->k_off; p.prefix = a->prefix; p.slopes = a->slopes;
    p.q_rows = a->q_rows; p.k_rows = a->k_rows; p.n_docs = a->n_docs; p.heads = a->heads; p.kv_heads = a->kv_heads; p.group = a->heads / a->kv_heads; p.dim = a->dim;
    p.packed = a->packed; p.causal = a->causal; p.scale = a->scale; p.cap = a->cap; p.tiles = 0;
    return MMFE_OK;
}

// Row tiles of a launch: exact for padded documents, for packed ones the most that the offsets can make (one partial tile per
// document, and the rows before and behind them).
int64_t count_tiles(Problem& p, int64_t rows, int tile_rows) {
    const int64_t n = (rows + tile_rows - 1) / tile_rows;
    p.tiles = (int)(p.packed ? n + p.n_docs + 2 : n);
    return p.packed ? (rows > 0 ? n + p.n_docs + 2 : 0) : n * p.n_docs;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return MMFE_OK;
    set_error("%s launch failed: %s", what, hipGetErrorString(e));
    return MMFE_EHIP;
}

}  // namespace attn
}  // namespace mmfe

using namespace mmfe;

extern "C" {

int64_t mmfe_attention_workspace(const mmfe_attention_args* a) {
    Problem p{};
    if (make_problem(a, p)) return -1;
    const Cut c = cut_keys(a);
    const int64_t rows = c.n_splits > 1 ? c.units * c.n_splits * 32 : c.cuts > 1 ? c.cuts * a->heads * in_all(a, a->q_rows) : 0;
    return rows * (a->dim + 2) * (int64_t)sizeof(float);
}

int mmfe_attention_forward(const mmfe_attention_args* a, void* workspace, int device, void* hip_stream) {
    ForwardArgs f{};
    int rc = make_problem(a, f.p);
    if (rc) return rc;
    const int64_t tiles = count_tiles(f.p, a->q_rows, kRows);
    if (tiles == 0) return MMFE_OK;
    if (a->out == nullptr) { set_error("attention: NULL data pointer"); return MMFE_EINVAL; }
    if (bad_rows("out", a->out, a->out_stride)) return MMFE_EINVAL;
    f.out = Rows{a->out, a->out_stride[0], a->out_stride[1], a->out_stride[2]};
    f.rest = static_cast<char*>(a->out_rest);
    if ((reinterpret_cast<uintptr_t>(a->out_rest) & 15) != 0) { set_error("attention: out_rest: 16-byte aligned"); return MMFE_EINVAL; }
    f.lse = a->lse; f.lse_b = a->lse_stride[0]; f.lse_h = a->lse_stride[1];
    const Cut c = cut_keys(a);
    if ((c.n_splits > 1 || c.cuts > 1) && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)) { set_error("attention: this call needs a 16-byte aligned workspace"); return MMFE_EINVAL; }
    // (keys are cut into several chunks below 2048 units only, so that the joining launch is always small)
    if (c.n_splits > 0 ? too_many_blocks(c.units * c.n_splits, 64 * kSplitWaves) : too_many_blocks(tiles * a->heads * c.cuts, kThreads)) { set_error("attention: too many rows and heads in one call"); return MMFE_EINVAL; }
    OnDevice on(device);
    if (on.rc) return on.rc;
    const bool bf = a->dtype == MMFE_OUT_BF16;
    if (c.n_splits > 0) {
        SplitArgs s{};
        s.f = f;
        s.f.p.tiles = 1;
        s.chunk = c.chunk; s.n_splits = c.n_splits; s.n_units = (int)c.units; s.row_tiles = c.row_tiles;
        s.part = static_cast<float*>(workspace);
        s.part_ml = c.n_splits > 1 ? s.part + c.units * c.n_splits * 32 * a->dim : nullptr;
        const split_fn fn = bf ? pick_split<true>(a->dim) : pick_split<false>(a->dim);
        const size_t tiles = (size_t)kSplitWaves * 4 * kSplitTile * pitch(a->dim) * 2, meet = (size_t)kSplitWaves * 32 * ((padded_dim(a->dim) + 4) * 4 + 8);
        const size_t lds = tiles > meet ? tiles : meet;
        int blocks = 1, cus = 256;
        rc = kernel_prepare(reinterpret_cast<const void*>(fn), 64 * kSplitWaves, lds, &blocks, &cus);
        if (rc) return rc;
        hipLaunchKernelGGL(fn, dim3((uint32_t)(c.units * c.n_splits)), dim3(64 * kSplitWaves), lds, reinterpret_cast<hipStream_t>(hip_stream), s);
        if (c.n_splits > 1) hipLaunchKernelGGL(bf ? &join_kernel<true> : &join_kernel<false>, dim3((uint32_t)(c.units * 32)), dim3(kThreads), 0, reinterpret_cast<hipStream_t>(hip_stream), s);
        return launched("attention");
    }
    const bool bias = a->slopes != nullptr;
    const forward_fn fn = c.cuts > 1 ? (bf ? pick_forward<true, true>(a->dim, bias, a->cap) : pick_forward<false, true>(a->dim, bias, a->cap))
                                     : (bf ? pick_forward<true, false>(a->dim, bias, a->cap) : pick_forward<false, false>(a->dim, bias, a->cap));
    const size_t lds = 2 * (size_t)kRing * kStepKeys * pitch(a->dim) * 2;
    int blocks = 1, cus = 256;
    rc = kernel_prepare(reinterpret_cast<const void*>(fn), kThreads, lds, &blocks, &cus);
    if (rc) return rc;
    f.cuts = c.cuts;
    const int64_t rows = a->heads * in_all(a, a->q_rows);
    f.part = static_cast<float*>(workspace);
    f.part_ml = c.cuts > 1 ? reinterpret_cast<float2*>(f.part + c.cuts * rows * a->dim) : nullptr;
    hipLaunchKernelGGL(fn, dim3((uint32_t)(tiles * a->heads * c.cuts)), dim3(kThreads), lds, reinterpret_cast<hipStream_t>(hip_stream), f);
    if (c.cuts > 1) {
        const int64_t need = (rows * (a->dim / 4) + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(bf ? &gather_kernel<true> : &gather_kernel<false>, dim3((uint32_t)(need < 8192 ? need : 8192)), dim3(kThreads), 0, reinterpret_cast<hipStream_t>(hip_stream), f);
    }
    return launched("attention");
}

}  // extern "C"

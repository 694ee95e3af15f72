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
// (o^T += v^T p^T) as they stand.  Keys and values come by LDS-DMA into double-buffered tiles of 64 rows that the 4 waves share.
//
// What is rounded: p to the tensors' 16-bit type for the second product (half a step each, independent, so the error of o is that
// of its own rounding again); the sums of p are taken before that rounding, in float32, as are maximum, sum and both accumulators.
// The running maximum is raised only when a row's scores exceed it by more than 8 (in log2 units): p stays below 2^8, which both
// types hold, and most tiles skip the rescaling of o.
#include "attention_tiles.h"

#include <cmath>

namespace mmfe {
using namespace attn;
namespace {

struct ForwardArgs {
    Problem p;
    Rows out;
    float* lse;                       // (batch, heads, rows) or (heads, rows); NULL: not wanted
    int64_t lse_b, lse_h;
    int grid_tiles;
};

template <bool BF, int DP>
__global__ void __launch_bounds__(kThreads, 2) forward_kernel(const ForwardArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const Problem& p = a.p;
    constexpr int kTileBytes = kTile * DP * 2;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    const int j = blockIdx.x % p.heads;
    const int t0 = blockIdx.x / p.heads;
    Doc d;
    if (!find_doc<true>(p, a.grid_tiles - 1 - t0, kRows, d)) return;          // last tiles first: under a causal mask they are the long ones
    const int head = head_of(p, j), kvh = head / p.group;
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
    const bool shaped = p.cap > 0.f || p.slopes != nullptr;                    // scores leave the linear form: they are taken to log2 units first
    const float c = shaped ? 1.f : p.scale * kLog2e;
    const float slope = p.slopes ? p.slopes[head] * kLog2e : 0.f;
    const float cap_in = p.cap > 0.f ? p.scale / p.cap : 0.f, cap_out = p.cap * kLog2e;

    f32x16 o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.f;

    for (int t = 0; t < n_tiles; ++t) {
        wait_all();                    // this wave's part of tile t is there, and its reads of the other buffer are done
        block_sync();                  // ... and so for every wave
        if (t + 1 < n_tiles) stage(t + 1, (t + 1) & 1);
        const int j0 = t * kTile;
        if (j0 >= wave_lim) continue;
        const char* kt = smem + (t & 1) * 2 * kTileBytes;
        const char* vt = kt + kTileBytes;
        f32x16 x[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            x[b] = f32x16{};
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) x[b] = mfma<BF>(read_rows<DP>(kt, 32 * b, s), qf[s], x[b]);
        }
        if (shaped) {
            const float at = (float)(row + off - j0 - 4 * half);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float v = p.cap > 0.f ? cap_out * tanh_fast(x[b][i] * cap_in) : x[b][i] * (p.scale * kLog2e);
                    if (p.slopes) v -= slope * fabsf(at - (float)(32 * b + reg_row(i)));
                    x[b][i] = v;
                }
        }
        if (j0 + kTile > full_lim) {
            const int left = lim - j0 - 4 * half;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[b][i] = 32 * b + reg_row(i) < left ? x[b][i] : -INFINITY;
        }
        float mx = fmaxf(x[0][0], x[1][0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, fmaxf(x[0][i], x[1][i]));
        mx = fmaxf(mx, other_half(mx));
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
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[b][i] = exp2_fast(fmaf(x[b][i], c, -mc));
                sum += x[b][i];
            }
        l += sum;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const u32x4 pf = operand<BF>(x[s >> 1], s & 1);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[i] = mfma<BF>(read_cols<DP>(vt, 16 * s, 32 * i), pf, o[i]);
        }
    }
    l += other_half(l);
    if (row >= d.rows) return;
    const bool some = lim > 0;
    const float inv = some ? 1.f / l : 0.f;
    char* out = const_cast<char*>(row_base(a.out, d, d.q0 + row, head));
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int e = 32 * i + 8 * g;
            if (e < p.dim) {
                u32x2 w{0, 0};
                if (some) w = u32x2{pack2<BF>(o[i][4 * g] * inv, o[i][4 * g + 1] * inv), pack2<BF>(o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv)};
                *reinterpret_cast<u32x2*>(out + 2 * (e + 4 * half)) = w;
            }
        }
    if (a.lse != nullptr && half == 0)
        a.lse[d.batch * a.lse_b + head * a.lse_h + d.q0 + row] = some ? (m * c + __builtin_amdgcn_logf(l)) * (1.f / kLog2e) : -INFINITY;
}

typedef void (*forward_fn)(const ForwardArgs);
template <bool BF>
forward_fn pick_forward(int dim) {
    return dim <= 32 ? &forward_kernel<BF, 32> : dim <= 64 ? &forward_kernel<BF, 64> : &forward_kernel<BF, 128>;
}

}  // namespace

namespace attn {

int padded_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

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
    if (!(a->scale > 0.f) || !std::isfinite(a->scale) || !(a->cap >= 0.f) || !std::isfinite(a->cap)) { set_error("attention: scale > 0 and cap >= 0 must be finite"); return MMFE_EINVAL; }
    if (a->packed && a->n_docs > 0 && (a->q_off == nullptr || a->k_off == nullptr)) { set_error("attention: packed documents need offsets"); return MMFE_EINVAL; }
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

int mmfe_attention_forward(const mmfe_attention_args* a, int device, void* hip_stream) {
    ForwardArgs f{};
    int rc = make_problem(a, f.p);
    if (rc) return rc;
    const int64_t tiles = count_tiles(f.p, a->q_rows, kRows);
    if (tiles == 0) return MMFE_OK;
    if (a->out == nullptr) { set_error("attention: NULL data pointer"); return MMFE_EINVAL; }
    if (bad_rows("out", a->out, a->out_stride)) return MMFE_EINVAL;
    if (tiles * a->heads > 0x7fffffffll) { set_error("attention: too many rows and heads in one call"); return MMFE_EINVAL; }
    f.out = Rows{a->out, a->out_stride[0], a->out_stride[1], a->out_stride[2]};
    f.lse = a->lse; f.lse_b = a->lse_stride[0]; f.lse_h = a->lse_stride[1];
    f.grid_tiles = (int)tiles;
    OnDevice on(device);
    if (on.rc) return on.rc;
    const forward_fn fn = a->dtype == MMFE_OUT_BF16 ? pick_forward<true>(a->dim) : pick_forward<false>(a->dim);
    const size_t lds = 4 * (size_t)kTile * padded_dim(a->dim) * 2;
    int blocks = 1, cus = 256;
    rc = kernel_prepare(reinterpret_cast<const void*>(fn), kThreads, lds, &blocks, &cus);
    if (rc) return rc;
    hipLaunchKernelGGL(fn, dim3((uint32_t)(tiles * a->heads)), dim3(kThreads), lds, reinterpret_cast<hipStream_t>(hip_stream), f);
    return launched("attention");
}

}  // extern "C"

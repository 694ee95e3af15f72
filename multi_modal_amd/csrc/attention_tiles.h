// Shared device code of the attention kernels (attention.hip, attention_backward.hip): which rows a block works on, how tiles get
// into LDS, and how matrix operands are read out of them.
//
// All products use v_mfma_f32_32x32x16 (32 x 32 results, 16 terms per instruction, float32 accumulation).  A lane (c = lane & 31,
// h = lane >> 5) holds of the operands 8 consecutive terms k = 8 h .. 8 h + 7 of row (column) c, and of the result column c,
// rows 8 (i / 4) + 4 h + i % 4 in register i = 0 .. 15.  Products are arranged so that a result is the next product's operand as it
// stands: the result's registers 8 s .. 8 s + 7 hold rows {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3} of its 16-row step s, and since the order of
// terms is free as long as both operands agree, the partner operand is fetched in that order (two transposing reads of 4 rows each).
//
// Tiles of rows lie in LDS as they lie in memory, in 16-byte pieces, piece c of row r at position c ^ swizzle(r): the reads of 16
// rows' pieces of one column, and the transposing reads of 4 rows x 32 bytes, then spread over all banks.  They arrive by LDS-DMA
// (global_load_lds_dwordx4: 64 pieces per instruction to consecutive LDS addresses, each lane naming its source), so that no
// register or vector instruction is spent on staging; the swizzle is applied to the source addresses.
#pragma once

#include "mmfe_internal.h"

namespace mmfe {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kRows = 128;            // rows of a block: 32 per wave
constexpr int kTile = 64;             // rows of a streamed tile
constexpr int kShortKeys = 128;       // documents of at most so many keys: 16-bit operands made of float32 values enter with their rest
constexpr float kLog2e = 1.4426950408889634f;

// A tensor of (batch, row, head) vectors with unit stride inside; strides in elements, batch = 0 where documents are packed.
struct Rows {
    const void* p;
    int64_t b, n, h;
};

// What forward and backward share.  Documents: batch entries of the padded form (q_len / k_len valid rows of q_rows / k_rows), or the
// row ranges that offsets cut the packed rows into.
struct Problem {
    Rows q, k, v;
    const int32_t *q_len, *k_len;     // padded: per document, or NULL = all rows
    const int32_t *q_off, *k_off;     // packed: n_docs + 1 entries
    const int32_t* prefix;            // per document, or NULL
    const float* slopes;              // per query head, or NULL
    int64_t q_rows, k_rows;           // per document (padded) or in all (packed)
    int n_docs, heads, kv_heads, group, dim;
    int packed, causal;
    float scale, cap;
    int tiles;                        // padded: row tiles per document; packed: tiles in all (an upper bound)
};

// One document's rows, and which of them a block has.
struct Doc {
    int64_t q0, k0;                   // first row (packed: in all rows; padded: 0, with batch set)
    int batch;                        // batch entry (padded), 0 when packed
    int index;                        // document, or -1: rows that belong to none
    int nq, nk;                       // valid rows
    int rows;                         // rows to produce, from the tiled side (padded: all of them, whatever their length)
    int tile;                         // tile inside the document
    int prefix;
};

__device__ __forceinline__ int clamp_int(int64_t v, int64_t lo, int64_t hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Sum over a wave's lanes, in every lane.
__device__ __forceinline__ int wave_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);           // row_shr 1, 2, 4, 8: sums of 16 lanes in their last one
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    return __builtin_amdgcn_readlane(v, 15) + __builtin_amdgcn_readlane(v, 31) + __builtin_amdgcn_readlane(v, 47) + __builtin_amdgcn_readlane(v, 63);
}

// Document and tile of tile number t, on the query side (QSIDE) or the key side.  False: there is no such tile.
// Packed rows that no document holds (before the first offset, behind the last) form tiles of their own, of a document without
// partners: their results are zeros.  Offsets are clamped into the rows, so that no entry can lead out of the tensors.
//
// Blocks start in the order of their numbers, and a block's time goes with the partners its tile has, so tiles are numbered from the
// longest to the shortest: under a causal mask the last row tile and the first key tile of a document have the most.  Packed
// documents are sorted that way up to 64 of them (one lane each: under a causal mask by the tile's distance from the short end, found by
// bisection over the counts; otherwise by the partners' number); of more documents a single one matters less, and they are taken in
// reverse.  16 recordings of 1 to 4096 tokens, causal, forward: 155 us sorted, 200 in reverse.
template <bool QSIDE>
__device__ __forceinline__ bool find_doc(const Problem& p, int t, int tile_rows, Doc& d) {
    if (!p.packed) {
        int b = t / p.tiles, tile = t - b * p.tiles;
        if (p.causal) {                                   // all documents' longest tiles first
            tile = t / p.n_docs;
            b = t - tile * p.n_docs;
            if (QSIDE) tile = p.tiles - 1 - tile;
        }
        d.batch = d.index = b;
        d.tile = tile;
        d.q0 = d.k0 = 0;
        d.nq = p.q_len ? clamp_int(uniform(p.q_len[b]), 0, p.q_rows) : (int)p.q_rows;
        d.nk = p.k_len ? clamp_int(uniform(p.k_len[b]), 0, p.k_rows) : (int)p.k_rows;
        d.rows = QSIDE ? (int)p.q_rows : (int)p.k_rows;
        d.prefix = p.prefix ? uniform(p.prefix[b]) : 0;
        return true;
    }
    const int32_t* off = QSIDE ? p.q_off : p.k_off;
    const int32_t* other = QSIDE ? p.k_off : p.q_off;
    const int64_t all = QSIDE ? p.q_rows : p.k_rows, other_all = QSIDE ? p.k_rows : p.q_rows;
    const int lane = threadIdx.x & 63;
    d.batch = 0;
    d.index = -1;
    d.nq = d.nk = 0;
    d.q0 = d.k0 = 0;
    d.prefix = 0;
    auto found = [&](int index, int tile, int start, int rows) {
        d.index = index;
        d.tile = tile;
        d.rows = rows;
        const int os = clamp_int(uniform(other[index]), 0, other_all);
        const int oe = clamp_int(uniform(other[index + 1]), os, other_all);
        if (QSIDE) { d.q0 = start; d.nq = rows; d.k0 = os; d.nk = oe - os; }
        else { d.k0 = start; d.nk = rows; d.q0 = os; d.nq = oe - os; }
        if (p.prefix) d.prefix = uniform(p.prefix[index]);
        return true;
    };
    const int first = clamp_int(uniform(off[0]), 0, all);
    int last = first;
    if (p.n_docs <= 64) {
        int s = 0, e = 0, partners = 0;
        if (lane < p.n_docs) {
            s = clamp_int(off[lane], 0, all);
            e = clamp_int(off[lane + 1], s, all);
            const int os = clamp_int(other[lane], 0, other_all);
            partners = clamp_int(other[lane + 1], os, other_all) - os;
        }
        if (p.n_docs > 0) last = __builtin_amdgcn_readlane(e, p.n_docs - 1);
        const int n = (e - s + tile_rows - 1) / tile_rows;
        const int total = wave_sum(n);
        if (t < total) {
            int w, tile;
            if (p.causal) {
                int lo = 0, hi = total;                   // tiles of level >= lo: more than t; of level >= hi: not more
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (wave_sum(max(0, n - mid)) > t) lo = mid;
                    else hi = mid;
                }
                int rank = t - wave_sum(max(0, n - lo - 1));
                unsigned long long has = __ballot(n > lo);
                for (; rank > 0; --rank) has &= has - 1;
                w = __ffsll(has) - 1;
                tile = QSIDE ? lo : __builtin_amdgcn_readlane(n, w) - 1 - lo;
            } else {
                int before = 0;
                for (int i = 0; i < p.n_docs; ++i) {
                    const int m = __builtin_amdgcn_readlane(partners, i);
                    if (m > partners || (m == partners && i < lane)) before += __builtin_amdgcn_readlane(n, i);
                }
                w = __ffsll(__ballot(before <= t && t < before + n)) - 1;
                tile = t - __builtin_amdgcn_readlane(before, w);
            }
            const int ds = __builtin_amdgcn_readlane(s, w);
            return found(w, uniform(tile), ds, __builtin_amdgcn_readlane(e, w) - ds);
        }
        t -= total;
        const int lead = (first + tile_rows - 1) / tile_rows;
        if (t < lead) {
            d.tile = t;
            d.rows = first;
            return true;
        }
        t -= lead;
    } else {
        // Stretch 0 is the rows before the first document, 1 .. n_docs the documents, then the rows behind them.  Tile k of a stretch that
        // starts at row s has number (s >> 7) + stretch + k: distinct, rising, and below the launch's bound, so that the stretch is found by
        // search (64 places at a time) without counting the tiles before it.
        static_assert(kRows == 128, "");
        t = p.tiles - 1 - t;
        auto start = [&](int i) { return i == 0 ? 0 : clamp_int(off[min(i, p.n_docs + 1) - 1], 0, all); };
        int lo = 0, len = p.n_docs + 2;
        while (len > 1) {
            const int step = (len + 63) >> 6, i = lane * step;
            const bool at_or_before = i < len && (start(lo + i) >> 7) + lo + i <= t;
            const int n = max(1, __popcll(__ballot(at_or_before)));
            len = min(step, len - (n - 1) * step);
            lo += (n - 1) * step;
        }
        const int s = uniform(start(lo)), e = lo == p.n_docs + 1 ? (int)all : max(s, uniform(start(lo + 1)));
        const int tile = t - (s >> 7) - lo;
        if (tile < 0 || tile >= (e - s + tile_rows - 1) / tile_rows) return false;
        if (lo >= 1 && lo <= p.n_docs) return found(lo - 1, tile, s, e - s);
        d.tile = tile;
        d.rows = e - s;
        if (QSIDE) d.q0 = s;
        else d.k0 = s;
        return true;
    }
    const int rest = (int)all - last;
    if (t >= (rest + tile_rows - 1) / tile_rows) return false;
    d.tile = t;
    d.rows = rest;
    if (QSIDE) d.q0 = last;
    else d.k0 = last;
    return true;
}

__device__ __forceinline__ const char* row_base(const Rows& r, const Doc& d, int64_t row0, int head) {
    return static_cast<const char*>(r.p) + 2 * (d.batch * r.b + row0 * r.n + head * r.h);
}

// ---- LDS tiles ----

// DP, the head size that the products run over, is 32, 64, 96 or 128; a row of 96 lies in the place of 128.  4096 rows, 12 heads of 72, bfloat16: forward
// 124 us, gradients 209 + 137; as 128: 141, 419 + 176.
template <int DP>
constexpr int kPitch = DP == 96 ? 128 : DP;

template <int DP>
__device__ __forceinline__ constexpr int swizzle(int row) {
    if constexpr (kPitch<DP> == 128) return ((row & 3) << 2) | ((row >> 2) & 3);        // 16 pieces a row
    else if constexpr (DP == 64) return (row & 7) ^ ((row >> 3) & 1);           // 8
    else return (row >> 2) & 3;                                                 // 4
}

// 16 bytes per lane: from base + voff to LDS byte lds_dst + 16 * lane.  M0 holds the destination for the instruction; it is the
// compiler's register, so it is saved and restored.  The compiler does not count these; their completion is waited for by hand.
__device__ __forceinline__ void dma16(const void* base, unsigned voff, unsigned lds_dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(base), "s"(lds_dst) : "memory");
}
// two of them
__device__ __forceinline__ void dma16x2(const void* base0, unsigned voff0, unsigned dst0, const void* base1, unsigned voff1, unsigned dst1) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %6\n\ts_nop 0\n\t"
                 "global_load_lds_dwordx4 %3, %4\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff0), "s"(base0), "v"(voff1), "s"(base1), "s"(dst0), "s"(dst1) : "memory");
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// Tile of ROWS rows brought in by WAVES waves.  Rows past the last valid one repeat it and pieces past the head size repeat the
// first: their products are masked, dropped or multiplied by zeros, and they hold no other document's (or no one's) values.
template <int DP, int ROWS, int WAVES>
struct Loader {
    static constexpr int kPieces = kPitch<DP> / 8;
    static constexpr int kAll = ROWS * kPieces / 64;                // DMA instructions
    static constexpr int kCount = kAll > WAVES ? kAll / WAVES : 1;  // of a wave (where there are fewer than waves, some bring the same pieces)
    static constexpr int kStep = 64 * WAVES / kPieces;              // rows from one of them to the next
    static constexpr int kKept = kStep % 16 == 0 ? 1 : kCount;      // the swizzle repeats every 16 rows
    static_assert(kAll * 64 == ROWS * kPieces && (kAll % WAVES == 0 || WAVES % kAll == 0), "whole instructions");
    unsigned off[kKept];                                            // byte offsets from the tile's first row
    __device__ __forceinline__ static int number(int i, int wave) { return (i * WAVES + wave) % kAll; }
    __device__ __forceinline__ static int piece(int i, int wave) { return number(i, wave) * 64 + (int)(threadIdx.x & 63); }
    __device__ __forceinline__ static unsigned offset(int ci, int rows, int dim, unsigned stride) {
        const int r0 = ci / kPieces;
        const int c = (ci & (kPieces - 1)) ^ swizzle<DP>(r0);
        const int r = r0 < rows ? r0 : rows - 1;
        return (unsigned)r * stride + (c * 8 < dim ? c * 16 : 0);
    }
    __device__ __forceinline__ void init(int dim, int64_t stride, int wave) {
#pragma unroll
        for (int i = 0; i < kKept; ++i) off[i] = offset(piece(i, wave), ROWS, dim, (unsigned)(2 * stride));
    }
    // base: the tile's first row; rows >= 1: valid rows from there on
    __device__ __forceinline__ void load(const char* base, int rows, int dim, int64_t stride, unsigned lds, int wave) const {
        if (rows >= ROWS && kCount % 2 == 0) {
#pragma unroll
            for (int i = 0; i + 1 < kCount; i += 2)
                dma16x2(kKept == 1 ? base + i * kStep * 2 * stride : base, off[kKept == 1 ? 0 : i], lds + number(i, wave) * 1024,
                        kKept == 1 ? base + (i + 1) * kStep * 2 * stride : base, off[kKept == 1 ? 0 : i + 1], lds + number(i + 1, wave) * 1024);
        } else if (rows >= ROWS) {
#pragma unroll
            for (int i = 0; i < kCount; ++i)
                dma16(kKept == 1 ? base + i * kStep * 2 * stride : base, off[kKept == 1 ? 0 : i], lds + number(i, wave) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < kCount; ++i) dma16(base, offset(piece(i, wave), rows, dim, (unsigned)(2 * stride)), lds + number(i, wave) * 1024);
        }
    }
};

__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
// all but the youngest N of this wave's DMAs have arrived; its LDS reads are done
template <int N>
__device__ __forceinline__ void wait_but() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory"); }
__device__ __forceinline__ void block_sync() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Operands loaded from memory before a loop, once they have been waited for: says so to the compiler, which would otherwise wait for
// them (and so for every DMA in flight) at their first use in every pass of the loop.
template <int N>
__device__ __forceinline__ void arrived(u32x4 (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// Operand with one row per lane (row0 + c), step s of 16 columns.
template <int DP>
__device__ __forceinline__ u32x4 read_rows(const char* tile, int row0, int s) {
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    return *reinterpret_cast<const u32x4*>(tile + (row0 + r) * (2 * kPitch<DP>) + (((2 * s + h) ^ swizzle<DP>(r)) << 4));
}

// Transposed operand: lane c gets column col0 + c of the rows row0 + {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3} (row0 a multiple of 16).  A
// transposing read serves 16 lanes: lane i names 8 bytes (4 columns) of row i / 4 and receives column i of the 4 rows.
template <int DP>
__device__ __forceinline__ u32x4 read_cols(const char* tile, int row0, int col0) {
    const int lane = threadIdx.x & 63, i = lane & 15, h = lane >> 5;
    const int c = (col0 >> 3) + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
    const int r = 4 * h + (i >> 2);
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const char* a = tile + (row0 + r) * (2 * kPitch<DP>) + ((c ^ swizzle<DP>(r)) << 4) + 8 * (i & 1);
    const char* b = tile + (row0 + r + 8) * (2 * kPitch<DP>) + ((c ^ swizzle<DP>(r + 8)) << 4) + 8 * (i & 1);
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)a));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)b));
    return u32x4{lo.x, lo.y, hi.x, hi.y};
}

template <bool BF>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// two float32 to one word of 16-bit values, round to nearest even
template <bool BF>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    if constexpr (BF) return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, f16x2));
}
// result registers 8 s .. 8 s + 7 as an operand
template <bool BF>
__device__ __forceinline__ u32x4 operand(const f32x16& v, int s) {
    return u32x4{pack2<BF>(v[8 * s], v[8 * s + 1]), pack2<BF>(v[8 * s + 2], v[8 * s + 3]), pack2<BF>(v[8 * s + 4], v[8 * s + 5]), pack2<BF>(v[8 * s + 6], v[8 * s + 7])};
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// The larger one, NaN if either is: v_maximum_f32 and, of three, v_maximum3_f32, without the canonicalising moves that fmaxf takes
// along (51 of 59 instructions of a tile's row maximum were those).
__device__ __forceinline__ float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// over the two lanes (half 0 and 1) of a column
__device__ __forceinline__ float both_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return max2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <bool BF>
__device__ __forceinline__ float widen(unsigned w, int hi) {
    if constexpr (BF) return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
    else return (float)__builtin_bit_cast(_Float16, (unsigned short)(hi ? w >> 16 : w));
}
// what operand(v, s), given as `hi`, lost to rounding, as another operand
template <bool BF>
__device__ __forceinline__ u32x4 operand_rest(const f32x16& v, int s, u32x4 hi) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<BF>(v[8 * s + 2 * i] - widen<BF>(hi[i], 0), v[8 * s + 2 * i + 1] - widen<BF>(hi[i], 1));
    return r;
}
// four results (4 consecutive columns of a lane's row) to 16-bit memory, and what that rounding lost next to it
template <bool BF>
__device__ __forceinline__ void store4(char* to, char* rest, float a, float b, float c, float d) {
    const u32x2 w{pack2<BF>(a, b), pack2<BF>(c, d)};
    *reinterpret_cast<u32x2*>(to) = w;
    if (rest != nullptr)
        *reinterpret_cast<u32x2*>(rest) = u32x2{pack2<BF>(a - widen<BF>(w.x, 0), b - widen<BF>(w.x, 1)), pack2<BF>(c - widen<BF>(w.y, 0), d - widen<BF>(w.y, 1))};
}

// tanh(z) / z for |z| <= 1/2, u = (z / 2)^2: minimax in z^2 with the constant term held at 1 (fitted in float64), off by 2^-26 relative; the coefficients hold
// the powers of 4.
__device__ __forceinline__ float tanh_ratio(float u) {
    return fmaf(fmaf(fmaf(fmaf(0.01724148727953434f * 256.f, u, -0.05304549261927605f * 64.f), u, 0.13325878977775574f * 16.f), u, -0.333331435918808f * 4.f), u, 1.f);
}

// How scores are capped (0: not).  1 - 2 / (e^(2 z) + 1) takes an exponential and a reciprocal, and its error is that of a number of size cap: 1.2e-7 cap,
// which up to kUsualCap stays below what the float32 products behind scores of that size are off by.  Any other cap takes kAnyCap, whose error is relative to the
// score (the exponential's form: 1.2e-3 at 1e4, 0.09 at 1e6).  It is a kernel of its own because it branches, which parts the products from the vector
// instructions beside them: 2 x 4096 rows, 12 heads on 4 of 64, bfloat16, causal, forward and backward 162 + 353 us, 130 + 345 with the exponential.  (split_kernel,
// which waits for memory, has kAnyCap only: 16 streams of 20 000 keys, 16 heads on 4 of 128: 136 us, 144 with the exponential.)
enum { kUncapped = 0, kExpCap = 1, kAnyCap = 2 };
constexpr float kUsualCap = 64.f;

// kAnyCap: the products x become those that an uncapped score of the same value has, cap / scale tanh(z) with z = scale x / cap.
// For |z| <= 1/2 that is x tanh(z) / z; beyond, cap / scale (1 - 2 r) with r = 1 / (e^(2 z) + 1), where the score is at least 0.46 cap.  Where all of a wave's
// 1024 products are of the first kind neither exponential nor reciprocal is taken.
struct AnyCap {
    float half, twice, most;          // scale / (2 cap), 2 log2(e) scale / cap, cap / scale
    __device__ __forceinline__ void set(const Problem& p) {
        half = 0.5f * p.scale / p.cap;
        twice = 2.f * kLog2e * p.scale / p.cap;
        most = fminf(p.cap / p.scale, 0.25f * __FLT_MAX__);
    }
    // w (WEIGHTS): (1 - tanh^2 z) / 4, which is r - r^2
    template <bool WEIGHTS>
    __device__ __forceinline__ void apply(f32x16& x, f32x16* w) const {
        float m = 0.f, k = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, fabsf(x[i])), fabsf(x[i + 1]));
            k = __builtin_elementwise_maximum(__builtin_elementwise_maximum(k, fabsf(x[i + 2])), fabsf(x[i + 3]));
        }
        if (__all(__builtin_elementwise_maximum(m, k) * half <= 0.25f)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float h = x[i] * half, t = tanh_ratio(h * h);
                if constexpr (WEIGHTS) (*w)[i] = fmaf(-(h * t), h * t, 0.25f);
                x[i] *= t;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float h = x[i] * half, t = tanh_ratio(h * h), r = __builtin_amdgcn_rcpf(exp2_fast(x[i] * twice) + 1.f);
            const bool small = fabsf(h) <= 0.25f;
            if constexpr (WEIGHTS) (*w)[i] = small ? fmaf(-(h * t), h * t, 0.25f) : fmaf(-r, r, r);
            x[i] = small ? x[i] * t : fmaf(-2.f * most, r, most);
        }
    }
};

// Row i of the result registers (see above).
__device__ __forceinline__ constexpr int reg_row(int i) { return 8 * (i >> 2) + (i & 3); }

__device__ __forceinline__ int head_of(const Problem& p, int j) {
    // neighbouring block numbers go to different XCDs: number the heads so that block j and j + 8 share key heads where they can
    return (j % p.kv_heads) * p.group + j / p.kv_heads;
}

}  // namespace attn
}  // namespace mmfe

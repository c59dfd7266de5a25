// attention_bwd.hip -- gradients of the fused attention (attention.hip) for gfx950.
//
// With S = scale Q K^T (+ mask), P = softmax(S) per query i and O = P V:
//   delta_i = sum_d dO_id O_id          (= sum_j P_ij dP_ij)
//   dP = dO V^T,   dS = P (dP - delta)
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO
// delta is taken from O as the caller has it. In fp16 that carries O's rounding, up to 2^-11 of |O|, into dS: nothing beside
// the rounding of dS where the rows of V differ as much as they are large, but where they share a mean of 5, 30 or 300 times
// their spread dQ and dK come out 1.5e-3, 7e-3 or 0.1 off. (The sum of exp2(s - m) (dP - delta), kept beside l, says what
// delta is off by; handed to the key kernel it mends dK alone, at 3% of 2x10x4096^2 and 2x20x1024x77, and dQ would take an
// eighth product, P K.)
// P is never stored: two kernels recompute it, one for queries, one for keys.
//
// attn_bwd_q_kernel: blocks of 128 queries of one (batch, head), 4 waves x 32, walk over 64-key tiles of K and V in
// LDS. S^T = K Q^T and dP^T = V dO^T leave a lane with one query and 32 keys, so the softmax is the forward pass's
// online one: with a running reference m, dQ accumulates exp2(s - m) (dP - delta) K and is rescaled with the row sum l
// when m rises (lazily); dQ = scale / l times that. Nothing but Q, K, V, O and dO is needed from the forward pass;
// m + log2 l and delta of each row go to the workspace for the other kernel.
// attn_bwd_k_kernel: blocks of 128 keys, 4 waves x 32, walk over 64-query tiles of Q and dO. S = Q K^T and dP = dO V^T
// leave a lane with one key and 32 queries; P = exp2(s - (m + log2 l)). dV^T = dO^T P and dK^T = Q^T dS take P and dS
// from the registers they are in (the MFMA's output order of the contracted index is the order in which the other
// operand is read).
// Every MFMA is v_mfma_f32_32x32x16_f16: seven products of Tq x Tk x 64 instead of five, for no atomic additions and
// no dQ partials in memory (results repeat bit for bit).
//
// Work is dealt in tiles: each workgroup (two per CU) takes as many whole blocks as there are for all, and the tiles of
// the blocks left, in order, are cut into equal shares, so that a grid of 640 blocks does not take two rounds of 512, and
// few blocks still fill the GPU. A workgroup whose share ends or begins inside a block writes its part of the block to
// the workspace; a second kernel adds the parts of such blocks in order.
//
// Each tile is staged row-major (64 rows x 64 columns fp16) by loads straight into LDS; 16-byte chunk c of row r lies at
// slot c ^ f(r), f the bit reversal of (r / 2) % 8. That makes both uses free of bank conflicts (counted: none): the
// 16-byte row fragments (16 rows of one chunk: every slot of either half once) and the transposing reads of
// ds_read_b64_tr_b16 (four rows of four chunks: the reversal puts rows r and r + 2 into different halves of a row).
//
// fp32 tensors, and fp16 ones whose rows are not 16-byte aligned or a multiple of 8 wide, are first packed into
// [batch, head][token][64] fp16 planes in the workspace (attn_bwd_pack_kernel). fp32 becomes pairs x = hi + lo and takes
// three MFMAs per product (hi hi + hi lo + lo hi), as in the forward pass; P and dS too. fp16's range is kept by powers
// of two, which are exact:
//   * in the query kernel, dS of a row by the row's largest |dO| (kRowExp), carried by exp2's argument;
//   * in the key kernel, P by 2^14 (weights of 2^-28 are normal numbers then), whatever V and dO are; dS by what keeps
//     2^14 (|dP| + |delta|) under 2^15, for the largest |delta| of the (batch, head) and the bound of |dP| that its rows of
//     dO and the block's of V give: fp32 64 max|dO| max|V|, fp16 the product of the largest rows' norms. dS cannot
//     overflow, and a weight of 2^-20 still has all its bits. fp16: that power of two is carried by V, whose largest
//     element stays in 2^-6 .. 2^12 (an element under 2^-8 of it may lose bits, 2^-19 of it at most), and by dS itself
//     beyond that, in a multiplication that only such blocks make: with the elements' bound N(0, 1) tensors made it
//     (2x10x4096^2 fp16 357 us, with the norms 351);
//   * dO of fp32, row by row, by its largest element, taken to 2^8.
//
// P and dS are rounded to fp16 for fp16 tensors (2^-11 of each, beside the result's own 2^-11; pairs as for fp32 would take 21
// products for seven).
//
// Measured (MI355X, us a call; a call of the kernels that its sizes take): fp16 2x10x4096^2 hd 64 358 (keys 207, queries 189,
// their merges 10 and 7, each timed alone; 840 TFLOP/s over the seven products), 2x20x1024x77 30 and fp32 causal 12x77 29
// (three launches of first loads and one or two tiles: latency), fp32 10x2304^2 189 (keys 99, queries 83, packing 11, merges
// 10 and 8; 760 TFLOP/s over its 21 products). What bounds the large calls: no unit is full. Of the cycles (1.7 to 1.8 GHz)
// MFMAs are busy 50% in the key and 39% in the query kernel, VALUs 42% and 55%, LDS 38% and 20% (fp32: 49 and 42, 32 and 42, 21
// and 15). A wave's scores, exponentials and products follow one another, and two or three waves a SIMD do not fill the gaps.
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace mi {
namespace {

constexpr int kB = 128;                  // queries (keys) per block
constexpr int kTile = 64;                // keys (queries) per staged tile
// A row's reference m rises when a lane's sum of exp2(s - m) passes 2^kLazy; kRowExp is the power of two that a row's
// largest |dO| is taken to in dS: exp2(s - m) (dP - delta) stays in fp16's range for |V| up to 32 even where 64 products
// agree in sign; where it would not, m rises further. A pair's low part is a subnormal number where dS is small, so fp32 takes it larger and rescales more often.
template <int NP>
constexpr int kLazy = NP == 2 ? 2 : 8;
template <int NP>
constexpr int kRowExp = NP == 2 ? 2 : -4;
constexpr int kPairExp = 8;              // fp32: the power of two that a row's largest |dO| is taken to in its pairs
constexpr int kPExp = 14;                // P's power of two in the key kernel
constexpr uint32_t kOob = 0x80000000u;   // a buffer offset past every record: the load returns zeros

struct Tensor {
    const void* p;
    uint64_t ld, s, sh;  // token, batch and head strides, elements
};
// An operand of the MFMA kernels: fp16 rows of whole 16-byte chunks, the head h of row t of batch b at
// p + b s + h sh + t ld; the plane of the pairs' low parts `lo` elements further.
struct Operand {
    const _Float16* p;
    uint64_t ld, s, sh, lo;
};
// How one kernel's blocks are dealt: NT tiles to a block (causal: fewer, see before()), nb blocks to a (batch, head),
// `per` tiles to those. Each of wgs workgroups takes `whole` blocks, and an equal share of the tiles of the blocks left.
struct Deal {
    uint32_t NT, nb, per, wgs, whole;
    uint32_t quo, rem, frac;  // the tiles dealt in shares are quo * wgs + rem (share_start), none or quo > 0
};
struct BwdArgs {
    Tensor q, k, v, o, g;     // g: dO
    Tensor dq, dk, dv;
    Operand xq, xk, xv, xg;
    uint32_t batch, Tq, Tk, heads, hd;
    int causal;
    const int32_t* kv_len;
    float c;                  // |scale| log2(e)
    float sgn, scale;         // the scale's sign, and itself
    // workspace: per (batch, head) rows of 128 ceil(Tq / 128): m + log2 l (+inf: no key), delta, and (packed) the row's
    // exponent in the pairs; then per 128 queries max|dO| and max|delta|; then the parts of shared blocks
    float *lse, *delta, *maxes, *part;
    int* rexp;
    uint32_t qblocks;
    Deal qd, kd;
    uint32_t ohd;             // columns of dq, dk and dv: hd, or 64 of planes in the workspace (unpacked by a kernel of its own)
    Tensor user[3];           // (unpack) the caller's dq, dk and dv
    uint32_t vin;             // (pack) the inputs take 16-byte loads
};

__device__ __forceinline__ uint32_t keys_of(const BwdArgs& a, uint32_t b) {
    if (!a.kv_len) return a.Tk;
    const int32_t l = a.kv_len[b];
    return l < 0 ? 0u : min(static_cast<uint32_t>(l), a.Tk);
}
template <typename T>
__device__ __forceinline__ T* head_of(const Tensor& t, uint32_t b, uint32_t h) {
    return static_cast<T*>(const_cast<void*>(t.p)) + b * t.s + h * t.sh;
}
__device__ __forceinline__ const _Float16* head_of(const Operand& x, uint32_t b, uint32_t h) { return x.p + b * x.s + h * x.sh; }

// ---- shares ------------------------------------------------------------------------------------------------------
//
// Tiles of the blocks before block i of a (batch, head). Causal: query block i sees keys up to its last query (2 i + 2
// tiles, NT at most), key block i the queries from its first key on (NT - 2 i tiles; past the queries one, without work).
template <bool KEYS>
__host__ __device__ inline uint32_t before(uint32_t i, uint32_t NT, bool causal) {
    if (!causal) return i * NT;
    if (KEYS) {
        const uint32_t half = (NT + 1) / 2, j = i < half ? i : half;
        return j * (NT + 1 - j) + (i - j);
    }
    const uint32_t half = NT / 2, j = i < half ? i : half;
    return j * (j + 1) + (i - j) * NT;
}
// The first tile of share w, counted from the first block that is dealt in shares: floor(w tiles / wgs), without a division
// (frac: 2^32 rem / wgs rounded up; off by one in places for more than 65535 shares, where that changes nothing but the
// balance); and the share of tile u.
__host__ __device__ inline uint32_t share_start(const Deal& d, uint32_t w) {
    return w * d.quo + static_cast<uint32_t>((static_cast<uint64_t>(w) * d.frac) >> 32);
}
__host__ __device__ inline uint32_t share_of(const Deal& d, uint32_t u) {
    const uint64_t total = static_cast<uint64_t>(d.quo) * d.wgs + d.rem;
    uint32_t w = static_cast<uint32_t>(static_cast<uint64_t>(u) * d.wgs / total);
    while (share_start(d, w) > u) --w;
    while (share_start(d, w + 1) <= u) ++w;
    return w;
}
__host__ __device__ inline uint32_t dealt_whole(const Deal& d) { return d.wgs * d.whole; }

// The pieces of a workgroup's work, one after the other: tiles [t0, t1) of block blk of (batch, head) bh.
template <bool KEYS>
struct Pieces {
    const Deal d;
    const bool causal;
    uint32_t base, at, end;  // tiles, counted from the first block of all
    uint32_t id, blocks;     // the next whole block and those left
    uint32_t bh, blk, t0, t1;
    bool whole, first;       // the whole block; the first piece of the share

    __device__ __forceinline__ Pieces(const Deal& d_, bool causal_, uint32_t w) : d(d_), causal(causal_) {
        id = w * d.whole;
        blocks = d.whole;
        base = at = end = 0;
        if (d.quo) {
            const uint32_t skip = dealt_whole(d) * d.NT;
            base = at = skip + share_start(d, w);
            end = skip + share_start(d, w + 1);
        }
    }
    __device__ __forceinline__ bool next() {
        if (blocks) {
            bh = id / d.nb;
            blk = id % d.nb;
            t0 = 0;
            t1 = d.NT;
            whole = true;
            ++id;
            --blocks;
            return true;
        }
        if (at >= end) return false;
        first = at == base;
        bh = at / d.per;
        const uint32_t r = at % d.per;
        uint32_t lo = 0, hi = d.nb;  // the last block with no more than r tiles before it
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (before<KEYS>(mid, d.NT, causal) <= r) lo = mid;
            else hi = mid;
        }
        blk = lo;
        const uint32_t b0 = before<KEYS>(blk, d.NT, causal), n = before<KEYS>(blk + 1, d.NT, causal) - b0;
        t0 = r - b0;
        t1 = min(n, t0 + (end - at));
        whole = t0 == 0 && t1 == n;
        at += t1 - t0;
        return true;
    }
};
// The parts of a shared block: workgroups w0 .. w1 (equal: not shared); each keeps its part in slot 0 if its share
// begins with it, else in slot 1.
template <bool KEYS>
struct Parts {
    uint32_t u0, w0, w1;
    __device__ __forceinline__ Parts(const Deal& d, bool causal, uint32_t bh, uint32_t blk) {
        u0 = w0 = w1 = 0;
        if (bh * d.nb + blk < dealt_whole(d)) return;
        u0 = bh * d.per + before<KEYS>(blk, d.NT, causal) - dealt_whole(d) * d.NT;
        w0 = share_of(d, u0);
        w1 = share_of(d, u0 + (before<KEYS>(blk + 1, d.NT, causal) - before<KEYS>(blk, d.NT, causal)) - 1);
    }
    __device__ __forceinline__ uint64_t slot(const Deal& d, uint32_t w) const { return 2ull * w + (share_start(d, w) >= u0 ? 0 : 1); }
};
constexpr uint32_t kQPart = kB * 64 + 2 * kB;  // floats of a query block's part: dQ rows, m, l
constexpr uint32_t kKPart = 2 * kB * 64;       // of a key block's: dK and dV rows

// ---- fragments ------------------------------------------------------------------------------------------------------

// bit reversal of (r / 2) % 8
__device__ __forceinline__ int swz(int r) { return ((r >> 3) & 1) | ((r >> 1) & 2) | ((r << 1) & 4); }
__device__ __forceinline__ half8 zero8() { return half8{0, 0, 0, 0, 0, 0, 0, 0}; }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
// The exponent e of a positive x in [2^e, 2^(e+1)); zero and subnormals -127.
__device__ __forceinline__ int exponent(float x) { return static_cast<int>(__float_as_uint(x) >> 23) - 127; }
__device__ __forceinline__ int clamp(int x, int lo, int hi) { return max(lo, min(hi, x)); }

// Row `t` of an operand's head, columns 16 s + 8 g .. + 7, both planes; zeros where !in or past hd.
template <int NP>
__device__ __forceinline__ void row_operand(const _Float16* head, const Operand& x, uint32_t t, int s, int g, bool in, int hd,
                                            half8 (&f)[NP]) {
    const int d = 16 * s + 8 * g;
    const _Float16* p = head + (in ? t : 0u) * x.ld + (d < hd ? d : 0);
#pragma unroll
    for (int pl = 0; pl < NP; ++pl) {
        f[pl] = zero8();
        if (in && d < hd) f[pl] = *reinterpret_cast<const half8*>(p + pl * x.lo);
    }
}

// Where a lane's fragments lie in a staged tile (halves), the same in every stage and plane.
struct Places {
    int row[4], col[2][2];
    __device__ __forceinline__ explicit Places(int lane) {
        const int l32 = lane & 31, g = lane >> 5, rk = (lane >> 2) & 3;
#pragma unroll
        for (int s = 0; s < 4; ++s) row[s] = l32 * 64 + (((2 * s + g) ^ swz(l32)) * 8);
        // lane i of a 16-lane group supplies row i / 4, columns 4 (i % 4) .. + 3 of the group's 16
#pragma unroll
        for (int rd = 0; rd < 2; ++rd)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int d = 32 * u + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                col[rd][u] = (4 * g + rk) * 64 + (((d >> 3) ^ swz(8 * rd + 4 * g + rk)) * 8) + (d & 7);
            }
    }
};

// One staged operand: 64 rows of up to 64 columns, NS LDS stages of NP planes. The stages are arrays of their own and known
// at compile time: the compiler then knows that reads of one do not wait for the loads into another.
template <int NP, int NS>
struct Stage {
    static constexpr int kPlane = kTile * 64, kHalves = NP * kPlane;
    _Float16* lds[NS];
    const _Float16* base;
    uint64_t ld, lo;
    uint32_t rows;  // rows of the tensor that are read; others are zeros
    int wave, lane;
    uint32_t off[2];

    __device__ __forceinline__ void set(const _Float16* head, const Operand& x, uint32_t rows_, int hd, int wave_, int lane_) {
        base = head;
        ld = x.ld;
        lo = x.lo;
        rows = rows_;
        wave = wave_;
        lane = lane_;
        // lane l brings slot l % 8 of row 8 piece + l / 8
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = 8 * (wave * 2 + i) + (lane >> 3), c = (lane & 7) ^ swz(row);
            off[i] = c * 8 < hd ? (row * static_cast<uint32_t>(ld) + c * 8) * 2u : kOob;
        }
        hd2 = hd;
    }
    int hd2;
    template <int ST>
    __device__ __forceinline__ void load(uint32_t row0) {
        const uint32_t n = row0 < rows ? min(rows - row0, static_cast<uint32_t>(kTile)) : 0u;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<_Float16*>(base + p * lo + static_cast<uint64_t>(n ? row0 : 0u) * ld), 0,
                n ? static_cast<int>(((n - 1) * ld + hd2) * 2) : 0, 0x00020000);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void*)(lds[ST] + p * kPlane + (wave * 2 + i) * 512), 16, off[i], 0, 0, 0);
        }
    }
    // rows 32 t + l32, columns 16 s + 8 g .. + 7
    template <int ST>
    __device__ __forceinline__ void row_frag(const Places& at, int t, int s, half8 (&f)[NP]) const {
#pragma unroll
        for (int p = 0; p < NP; ++p) f[p] = *reinterpret_cast<const half8*>(lds[ST] + p * kPlane + 32 * t * 64 + at.row[s]);
    }
    // column 32 u + l32, rows 32 t + 16 sp + 4 g + {0..3, 8..11}
    template <int ST>
    __device__ __forceinline__ void col_frag(const Places& at, int t, int sp, int u, half8 (&f)[NP]) const {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            half4 x[2];
#pragma unroll
            for (int rd = 0; rd < 2; ++rd) x[rd] = lds_read_tr16(lds[ST] + p * kPlane + (32 * t + 16 * sp + 8 * rd) * 64 + at.col[rd][u]);
            f[p] = half8{x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
        }
    }
};
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)

// acc += a b of one 16-deep slice: one MFMA, or three of the pairs' planes (those with a residual first).
template <int NP>
__device__ __forceinline__ floatx16 mma(const half8 (&x)[NP], const half8 (&y)[NP], floatx16 acc) {
    if constexpr (NP == 2) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[NP - 1], y[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[0], y[NP - 1], acc, 0, 0, 0);
    }
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x[0], y[0], acc, 0, 0, 0);
}
// Elements 8 sp .. 8 sp + 7 of x as an MFMA operand. The empty register constraint holds the fp32 value: the rounding to hi
// must not fuse into the multiplication that made it (a mixed-precision fma rounds the exact product), or lo, the rest of
// the fp32 value, would belong to another hi now and then (a row in a hundred off by 1e-4).
// neg1: residual2's.
template <int NP>
__device__ __forceinline__ void operand(const float (&x)[16], int sp, half8 (&f)[NP], float neg1) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float v = x[8 * sp + i], w = x[8 * sp + i + 1];
        if constexpr (NP == 2) asm volatile("" : "+v"(v), "+v"(w));
        const half2 hi = pack2(v, w);
        f[0][i] = hi[0];
        f[0][i + 1] = hi[1];
        if constexpr (NP == 2) {
            const half2 lo = residual2(hi, v, w, neg1);
            f[NP - 1][i] = lo[0];
            f[NP - 1][i + 1] = lo[1];
        }
    }
}

// Columns 32 u + 8 (r / 4) + 4 g + r % 4 of one row of T from two accumulator tiles, times f; hd is a multiple of 4, the row
// 4-element aligned (other gradients go through planes in the workspace).
template <typename T>
__device__ __forceinline__ void store_row(T* row, const floatx16 (&acc)[2], float f, int hd, int g) {
    typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * u + 8 * q + 4 * g;
            if (d < hd)
                *reinterpret_cast<T4*>(row + d) = T4{static_cast<T>(acc[u][4 * q] * f), static_cast<T>(acc[u][4 * q + 1] * f),
                                                     static_cast<T>(acc[u][4 * q + 2] * f), static_cast<T>(acc[u][4 * q + 3] * f)};
        }
}

// ---- packing --------------------------------------------------------------------------------------------------------

// q, k, v and dO (blockIdx.y) into fp16 planes [batch, head][token][64], columns past hd zero; for dO also delta of the
// row and its exponent. Eight lanes a row; keys past their row's length are not read and become zeros.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_pack_kernel(BwdArgs a) {
    constexpr bool kPair = sizeof(T) == 4;
    const uint32_t which = blockIdx.y;
    // (fields one by one: a choice between the structures would copy them to memory)
    auto of = [&](auto q, auto k, auto v, auto g) { return which == 0 ? q : which == 1 ? k : which == 2 ? v : g; };
    const Tensor t{of(a.q.p, a.k.p, a.v.p, a.g.p), of(a.q.ld, a.k.ld, a.v.ld, a.g.ld), of(a.q.s, a.k.s, a.v.s, a.g.s), a.hd};
    const Operand x{of(a.xq.p, a.xk.p, a.xv.p, a.xg.p), 64, of(a.xq.s, a.xk.s, a.xv.s, a.xg.s), of(a.xq.sh, a.xk.sh, a.xv.sh, a.xg.sh),
                    of(a.xq.lo, a.xk.lo, a.xv.lo, a.xg.lo)};
    const uint32_t len = which == 0 || which == 3 ? a.Tq : a.Tk;
    const uint64_t rows = static_cast<uint64_t>(a.batch) * len * a.heads;
    const uint64_t at = blockIdx.x * 32ull + (threadIdx.x >> 3);
    const uint64_t tok = at / a.heads;
    const uint32_t h = static_cast<uint32_t>(at % a.heads), b = static_cast<uint32_t>(tok / max(len, 1u)), i = static_cast<uint32_t>(tok % max(len, 1u));
    const int d = (threadIdx.x & 7) * 8, hd = static_cast<int>(a.hd);
    const bool in = at < rows && (which == 0 || which == 3 || i < keys_of(a, b));
    auto read = [&](const Tensor& y, float (&v)[8]) {
        const T* p = head_of<T>(y, in ? b : 0u, in ? h : 0u) + static_cast<uint64_t>(in ? i : 0u) * y.ld;
        typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int NV = 16 / sizeof(T);
        if (a.vin && in && d < hd) {
#pragma unroll
            for (int k = 0; k < 8 / NV; ++k) {
                const V w = reinterpret_cast<const V*>(p + d)[k];
#pragma unroll
                for (int e = 0; e < NV; ++e) v[k * NV + e] = static_cast<float>(w[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = in && d + e < hd ? static_cast<float>(p[d + e]) : 0.0f;
        }
    };
    float v[8];
    read(t, v);
    int re = 0;
    if (which == 3) {  // uniform in the workgroup
        float o[8], delta = 0.0f, mx = 0.0f;
        read(a.o, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            delta = __builtin_fmaf(v[e], o[e], delta);
            mx = fmaxf(mx, fabsf(v[e]));
        }
#pragma unroll
        for (int k = 1; k < 8; k <<= 1) {
            delta += __shfl_xor(delta, k);
            mx = fmaxf(mx, __shfl_xor(mx, k));
        }
        if (kPair) re = clamp(kPairExp - exponent(mx), -100, 100);
        if (in && d == 0) {
            const uint64_t row = (static_cast<uint64_t>(b) * a.heads + h) * a.qblocks * kB + i;
            a.delta[row] = delta;
            a.rexp[row] = re;
        }
    }
    if (at >= rows) return;
    _Float16* out = const_cast<_Float16*>(head_of(x, b, h)) + i * x.ld + d;
    half8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float w = kPair ? ldexpf(v[e], re) : v[e];
        hi[e] = static_cast<_Float16>(w);
        lo[e] = static_cast<_Float16>(w - static_cast<float>(hi[e]));
    }
    *reinterpret_cast<half8*>(out) = hi;
    if (kPair) *reinterpret_cast<half8*>(out + x.lo) = lo;
}

// ---- queries --------------------------------------------------------------------------------------------------------

// T: the type of O (read where !PACKED) and dQ.
template <typename T, bool PACKED>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 2 : 3) void attn_bwd_q_kernel(BwdArgs a) {
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    constexpr int NS = 2;
    // The fragments of a product are read from LDS ahead of the one before it: fp32 2x20x256^2 45.1 us with and 47.2 without.
    // fp16 has no registers for it at three waves per SIMD (2x10x4096x77 47.9 and 46.5).
    constexpr int kAhead = NP == 2 ? 1 : 0;
    static_assert(NP == 1 || PACKED, "fp32 is packed into pairs");
    typedef Stage<NP, NS> St;
    __shared__ __attribute__((aligned(16))) _Float16 ks0[St::kHalves], ks1[St::kHalves], vs0[St::kHalves], vs1[St::kHalves];
    __shared__ float wmax[2][4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, g = lane >> 5;
    const int hd = static_cast<int>(a.hd), ohd = static_cast<int>(a.ohd);
    St K, V;
    K.lds[0] = ks0;
    K.lds[1] = ks1;
    V.lds[0] = vs0;
    V.lds[1] = vs1;

    const Places places(lane);
    float neg1 = -1.0f;  // (residual2)
    asm volatile("" : "+v"(neg1));
    const uint32_t wg = xcd_swizzle(blockIdx.x, gridDim.x);
    Pieces<false> pc(a.qd, a.causal != 0, wg);
    while (pc.next()) {
        const uint32_t bh = pc.bh, h = bh % a.heads, b = bh / a.heads, qb = pc.blk;
        const uint32_t q0 = qb * kB, qi = q0 + wave * 32 + l32;
        // this lane's query: fragments of Q (with the scale's sign) and dO, delta, the row's power of two
        const bool in = qi < a.Tq;
        const uint64_t row = static_cast<uint64_t>(bh) * a.qblocks * kB + q0 + wave * 32 + l32;
        const uint32_t L = keys_of(a, b);  // (first: what is behind it waits for it alone)
        __builtin_amdgcn_sched_barrier(0);
        half8 qf[4][NP], gf[4][NP], of[PACKED ? 1 : 4];
        float delta = 0.0f, gmax = 0.0f, gsq = 0.0f;
        int re = 0;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            row_operand<NP>(head_of(a.xq, b, h), a.xq, qi, s, g, in, PACKED ? 64 : hd, qf[s]);
            row_operand<NP>(head_of(a.xg, b, h), a.xg, qi, s, g, in, PACKED ? 64 : hd, gf[s]);
            if constexpr (!PACKED) {
                const int d = 16 * s + 8 * g;
                const T* op = head_of<T>(a.o, b, h) + static_cast<uint64_t>(in ? qi : 0u) * a.o.ld;
                of[s] = zero8();
                if (in && d < hd) of[s] = *reinterpret_cast<const half8*>(op + d);
            }
        }
        if constexpr (PACKED) {
            if (in) {
                delta = a.delta[row];
                re = a.rexp[row];
            }
        }
        const uint32_t kend = a.causal ? min(L, q0 + kB) : L;
        // tiles that end at or before kfull need no mask for any query of this wave
        uint32_t kfull = L / kTile * kTile;
        if (a.causal) kfull = min(kfull, (q0 + wave * 32 + 1) / kTile * kTile);
        const uint32_t ntiles = min(pc.t1, (kend + kTile - 1) / kTile);
        K.set(head_of(a.xk, b, h), a.xk, kend, PACKED ? 64 : hd, wave, lane);
        V.set(head_of(a.xv, b, h), a.xv, kend, PACKED ? 64 : hd, wave, lane);
        uint32_t it = pc.t0;
        if (it < ntiles) {
            K.template load<0>(it * kTile);
            V.template load<0>(it * kTile);
        }

#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (!PACKED) delta = __builtin_fmaf(static_cast<float>(gf[s][0][e]), static_cast<float>(of[s][e]), delta);
                const float x = static_cast<float>(gf[s][0][e]);
                gmax = fmaxf(gmax, fabsf(x));
                if constexpr (NP == 1) gsq = __builtin_fmaf(x, x, gsq);
            }
            if (a.sgn < 0.0f) {
#pragma unroll
                for (int p = 0; p < NP; ++p) qf[s][p] = -qf[s][p];
            }
        }
        gmax = fmaxf(gmax, __shfl_xor(gmax, 32));
        if constexpr (NP == 1) gsq += __shfl_xor(gsq, 32);
        if constexpr (!PACKED) delta += __shfl_xor(delta, 32);
        // exp2(s - m) carries 2^ge; dP and delta carry 2^re
        const int ge = clamp(kRowExp<NP> - exponent(gmax), -100, 100);
        const float dl = ldexpf(delta, re);
        const float thr = ldexpf(1.0f, kLazy<NP> + ge);
        {
            // the block's largest |dO| (fp16: row of it, in the Euclidean norm) and |delta|, from its first part
            const float x = wave_max(NP == 1 ? sqrtf(gsq) : ldexpf(gmax, -re)), y = wave_max(fabsf(delta));
            if (lane == 0) {
                wmax[0][wave] = x;
                wmax[1][wave] = y;
            }
        }

        floatx16 acc[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[0][r] = acc[1][r] = 0.0f;
        float m = 0.0f, l = 0.0f;  // m: the reference less ge, so that exp2(s - m) carries 2^ge
        bool fresh = true;         // no reference yet
        wait_loads();
        __syncthreads();
        auto tile = [&](uint32_t j, auto ST) {
            constexpr int st = decltype(ST)::value;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                __builtin_amdgcn_sched_barrier(0);  // one half's values live at a time
                floatx16 s, dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
                half8 kf[kAhead + 1][NP], vf[kAhead + 1][NP];
                auto rows = [&](int i) {
                    K.template row_frag<st>(places, t, i, kf[i & kAhead]);
                    V.template row_frag<st>(places, t, i, vf[i & kAhead]);
                };
                if (kAhead) rows(0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i + kAhead < 4) rows(i + kAhead);
                    if (kAhead) __builtin_amdgcn_sched_barrier(0);
                    s = mma<NP>(kf[i & kAhead], qf[i], s);
                    dp = mma<NP>(vf[i & kAhead], gf[i], dp);
                }
                if (j * kTile >= kfull) {  // wave-uniform
                    const uint32_t k0 = j * kTile + 32 * t;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const uint32_t key = k0 + 8 * (r >> 2) + 4 * g + (r & 3);
                        if (key >= L || (a.causal && key > qi)) s[r] = -INFINITY;
                    }
                }
                auto largest = [&] {
                    float mx = s[0];
#pragma unroll
                    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
                    return fmaxf(mx, __shfl_xor(mx, 32)) * a.c;
                };
                // The first half of a piece sets the reference to its largest score (every query that sees a key of the
                // piece sees one there; the others keep l = 0). Later the lane's sum bounds each weight, so no maximum is
                // taken until it passes the threshold.
                if (fresh) {
                    const float mx = largest();
                    m = (mx == -INFINITY ? 0.0f : mx) - static_cast<float>(ge);
                    fresh = false;
                }
                float p[16], ts = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -m));
                    ts += p[r];
                }
                if (__any(ts > thr)) {
                    const float mx = largest() - static_cast<float>(ge);
                    const float mn = fmaxf(m, mx);
                    const float alpha = __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    l *= alpha;
                    ts = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        acc[0][r] *= alpha;
                        acc[1][r] *= alpha;
                        p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -m));
                        ts += p[r];
                    }
                }
                l += ts;
                float big = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[r] *= dp[r] - dl;
                    big = fmaxf(big, fabsf(p[r]));
                }
                // large values of V: the reference rises until the row's dS is under 2^15 (at 2^13 or more)
                if (__any(big > 32768.0f)) {
                    const float most = fmaxf(big, __shfl_xor(big, 32));
                    const int k = max(0, min(exponent(most), 100) - 13);
                    const float alpha = ldexpf(1.0f, -k);
                    m += static_cast<float>(k);
                    l *= alpha;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        acc[0][r] *= alpha;
                        acc[1][r] *= alpha;
                        p[r] *= alpha;
                    }
                }
                half8 df[2][NP], kt[kAhead + 1][NP];
                auto columns = [&](int n) { K.template col_frag<st>(places, t, n >> 1, n & 1, kt[n & kAhead]); };
                if (kAhead) columns(0);
                operand<NP>(p, 0, df[0], neg1);
                operand<NP>(p, 1, df[1], neg1);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    if (n + kAhead < 4) columns(n + kAhead);
                    if (kAhead) __builtin_amdgcn_sched_barrier(0);
                    acc[n & 1] = mma<NP>(kt[n & kAhead], df[n >> 1], acc[n & 1]);
                }
            }
        };
        auto step = [&](uint32_t j, auto ST) {
            constexpr int nx = decltype(ST)::value ^ 1;
            // (the last tile loads one past the piece, which is not used)
            K.template load<nx>((j + 1) * kTile);
            V.template load<nx>((j + 1) * kTile);
            tile(j, ST);
            wait_loads();
            __syncthreads();
        };
        for (; it < ntiles; it += 2) {
            step(it, std::integral_constant<int, 0>{});
            if (it + 1 < ntiles) step(it + 1, std::integral_constant<int, 1>{});
        }
        l += __shfl_xor(l, 32);
        if (pc.t0 == 0) {
            // (packed rows have theirs; those past Tq get zeros here)
            if (g == 0 && (!PACKED || !in)) a.delta[row] = in ? delta : 0.0f;
            if (PACKED && g == 0 && !in) a.rexp[row] = 0;
            if (tid < 2) {
                float x = wmax[tid][0];
#pragma unroll
                for (int w = 1; w < 4; ++w) x = fmaxf(x, wmax[tid][w]);
                a.maxes[(static_cast<uint64_t>(bh) * a.qblocks + qb) * 2 + tid] = x;
            }
        }
        __syncthreads();  // wmax and the stages are free for the next piece
        if (!pc.whole) {
            float* P = a.part + (2ull * wg + (pc.first ? 0 : 1)) * kQPart;
            const int r = wave * 32 + l32;
            store_row(P + r * 64, acc, 1.0f, 64, g);
            if (g == 0) {
                P[kB * 64 + r] = l > 0.0f ? m : -INFINITY;
                P[kB * 64 + kB + r] = l;
            }
            continue;
        }
        // a row without keys, or past Tq: its P is 0 in the key kernel whatever its scores
        if (g == 0) a.lse[row] = in && l > 0.0f ? m + __builtin_log2f(l) : INFINITY;
        if (in) {
            const float f = l > 0.0f ? ldexpf(a.scale / l, -re) : 0.0f;
            store_row(head_of<T>(a.dq, b, h) + static_cast<uint64_t>(qi) * a.dq.ld, acc, f, ohd, g);
        }
    }
}

// dQ and m + log2 l of the shared query blocks: sum_i 2^(m_i - M) part_i, M = max m_i, four parts at a time, in order. Four
// workgroups a block; thread t takes query t / 8 of its 32, columns 8 (t % 8).
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_q_merge_kernel(BwdArgs a) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const uint32_t id = blockIdx.x / 4, bh = id / a.qblocks, qb = id % a.qblocks;
    const Parts<false> ps(a.qd, a.causal != 0, bh, qb);
    if (ps.w0 == ps.w1) return;
    const int r = static_cast<int>(blockIdx.x % 4) * 32 + static_cast<int>(threadIdx.x >> 3), d = (threadIdx.x & 7) * 8;
    const uint32_t qi = qb * kB + r;
    const uint64_t row = static_cast<uint64_t>(bh) * a.qblocks * kB + qi;
    const bool in = qi < a.Tq;
    const int re = a.rexp && in ? a.rexp[row] : 0;
    float M = -INFINITY, l = 0.0f;
    floatx4 s0 = {0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
    for (uint32_t w = ps.w0; w <= ps.w1; w += 4) {
        float mi[4], li[4];
        floatx4 x0[4], x1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // every load first; past the last part it again, without weight
            const float* P = a.part + ps.slot(a.qd, min(w + i, ps.w1)) * kQPart;
            mi[i] = P[kB * 64 + r];
            li[i] = P[kB * 64 + kB + r];
            x0[i] = *reinterpret_cast<const floatx4*>(P + r * 64 + d);
            x1[i] = *reinterpret_cast<const floatx4*>(P + r * 64 + d + 4);
        }
        float mx = M;
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, mi[i]);
        const float keep = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - mx);
        M = mx;
        l *= keep;
        s0 *= keep;
        s1 *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (w + i > ps.w1 || mi[i] == -INFINITY) continue;
            const float f = __builtin_amdgcn_exp2f(mi[i] - M);
            l += f * li[i];
            s0 += f * x0[i];
            s1 += f * x1[i];
        }
    }
    if (d == 0) a.lse[row] = in && l > 0.0f ? M + __builtin_log2f(l) : INFINITY;
    const int ohd = static_cast<int>(a.ohd);
    const float f = l > 0.0f ? ldexpf(a.scale / l, -re) : 0.0f;
    T* out = head_of<T>(a.dq, bh / a.heads, bh % a.heads) + static_cast<uint64_t>(qi) * a.dq.ld + d;
    s0 *= f;
    s1 *= f;
    if (in && d < ohd) *reinterpret_cast<T4*>(out) = T4{static_cast<T>(s0[0]), static_cast<T>(s0[1]), static_cast<T>(s0[2]), static_cast<T>(s0[3])};
    if (in && d + 4 < ohd)
        *reinterpret_cast<T4*>(out + 4) = T4{static_cast<T>(s1[0]), static_cast<T>(s1[1]), static_cast<T>(s1[2]), static_cast<T>(s1[3])};
}

// ---- keys -----------------------------------------------------------------------------------------------------------

template <typename T, bool PACKED, bool CAUSAL>
__global__ __launch_bounds__(256, 2) void attn_bwd_k_kernel(BwdArgs a) {
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    constexpr int NS = 2;
    // The fragments of a product are read from LDS ahead of the one before it, where registers allow: fp16 2x20x1024^2 90.7 us
    // with and 92.1 without; fp32 would spill (1x8x2048^2 causal 105 and 103).
    constexpr int kAhead = NP == 1 ? 1 : 0;
    typedef Stage<NP, NS> St;
    __shared__ __attribute__((aligned(16))) _Float16 qs0[St::kHalves], qs1[St::kHalves], gs0[St::kHalves], gs1[St::kHalves];
    // per stage and query: m + log2 l less P's power of two, and -delta in the unit of dP
    __shared__ __attribute__((aligned(16))) float row0[2 * kTile], row1[2 * kTile];
    __shared__ float wmax[2][4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, g = lane >> 5;
    const int hd = static_cast<int>(a.hd), ohd = static_cast<int>(a.ohd);
    St Q, G;
    Q.lds[0] = qs0;
    Q.lds[1] = qs1;
    G.lds[0] = gs0;
    G.lds[1] = gs1;

    const Places places(lane);
    float neg1 = -1.0f;  // (residual2)
    asm volatile("" : "+v"(neg1));
    const uint32_t wg = xcd_swizzle(blockIdx.x, gridDim.x);
    Pieces<true> pc(a.kd, CAUSAL, wg);
    while (pc.next()) {
        const uint32_t bh = pc.bh, h = bh % a.heads, b = bh / a.heads;
        const uint32_t k0 = pc.blk * kB, kj = k0 + wave * 32 + l32;
        // query tiles of this piece; causal: counted from the first one with a query at or past the block's first key
        const uint32_t tiles = (a.Tq + kTile - 1) / kTile;
        const uint32_t first = CAUSAL ? min(k0 / kTile, tiles) : 0u;
        uint32_t it = first + pc.t0;
        const uint32_t tend = min(first + pc.t1, tiles);
        const uint32_t L = keys_of(a, b);
        Q.set(head_of(a.xq, b, h), a.xq, a.Tq, PACKED ? 64 : hd, wave, lane);
        G.set(head_of(a.xg, b, h), a.xg, a.Tq, PACKED ? 64 : hd, wave, lane);
        Q.template load<0>(it * kTile);
        G.template load<0>(it * kTile);

        // this lane's key: fragments of K (with the scale's sign) and V; zeros past the row's length
        half8 kf[4][NP], vf[4][NP];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            row_operand<NP>(head_of(a.xk, b, h), a.xk, kj, s, g, kj < a.Tk, PACKED ? 64 : hd, kf[s]);
            row_operand<NP>(head_of(a.xv, b, h), a.xv, kj, s, g, kj < a.Tk, PACKED ? 64 : hd, vf[s]);
        }
        // threads 0..63 bring m + log2 l, 64..127 delta (the others repeat them); the arrays hold 128 ceil(Tq / 128) rows, and
        // a tile past them is loaded from the last one and not used
        const bool second = (tid & kTile) != 0;
        const uint64_t rbase = static_cast<uint64_t>(bh) * a.qblocks * kB + (tid & (kTile - 1));
        const float* rows = (second ? a.delta : a.lse) + rbase;
        float rv;
        int rx = 0;
        auto load_rows = [&](uint32_t j) {
            const uint32_t o = min(j, 2 * a.qblocks - 1) * kTile;
            rv = rows[o];
            if constexpr (NP == 2) rx = a.rexp[rbase + o];
        };
        load_rows(it);
        // max|dO| (fp16: the largest row's norm) and max|delta| of the (batch, head)
        float gm = 0.0f, dm = 0.0f;
        for (uint32_t i = lane; i < a.qblocks; i += 64) {
            const float* x = a.maxes + (static_cast<uint64_t>(bh) * a.qblocks + i) * 2;
            gm = fmaxf(gm, x[0]);
            dm = fmaxf(dm, x[1]);
        }
        const bool in = kj < L;
        const uint32_t t1 = k0 < L ? tend : it;
        gm = wave_max(gm);
        dm = wave_max(dm);
        float vm = 0.0f, vsq = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                if (!in) kf[s][p] = vf[s][p] = zero8();
                if (a.sgn < 0.0f) kf[s][p] = -kf[s][p];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = static_cast<float>(vf[s][0][e]);
                vm = fmaxf(vm, fabsf(x));
                if constexpr (NP == 1) vsq = __builtin_fmaf(x, x, vsq);
            }
        }
        vm = wave_max(vm);
        if constexpr (NP == 1) vsq = wave_max(vsq + __shfl_xor(vsq, 32));
        if (lane == 0) {
            wmax[0][wave] = vm;
            wmax[1][wave] = vsq;
        }
        __syncthreads();
        auto largest = [&](int i) { return fmaxf(fmaxf(wmax[i][0], wmax[i][1]), fmaxf(wmax[i][2], wmax[i][3])); };
        vm = largest(0);
        // dS times 2^(kPExp + s0) stays under 2^15. fp16: V and delta carry 2^se (where the block has no values, delta
        // alone), V's largest element within 2^-6 .. 2^12, and dS what is left, 2^rest, by a multiplication of its own.
        // fp32: row i of dO carries 2^(e_i), P 2^(E - e_i) with E of the largest row, and the fma below the rest: se
        // is held where 2^(se - E) is finite (without values in the block, se goes by delta, E by dO).
        const int E = NP == 2 ? clamp(kPairExp - exponent(gm), -100, 100) : 0;
        const float bound = gm * (NP == 1 ? sqrtf(largest(1)) : 64.0f * vm) + dm;  // of |dP| and |delta|
        const int s0 = bound > 0.0f ? 15 - kPExp - 1 - exponent(bound) : 0;
        const int sv = NP == 1 && vm > 0.0f ? clamp(s0, -6 - exponent(vm), 12 - exponent(vm)) : s0;
        const int se = NP == 1 ? clamp(sv, -30, 30) : clamp(s0, -126, min(100, E + 100));
        const int rest = NP == 1 ? clamp(s0 - se, -100, 100) : 0;
        const float rsc = ldexpf(1.0f, rest);
        const float psc = ldexpf(1.0f, se - E);
        if constexpr (NP == 1) {
            const float up = ldexpf(1.0f, se);
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) vf[s][0][e] = static_cast<_Float16>(static_cast<float>(vf[s][0][e]) * up);
        }

        auto store_rows = [&](float* r) {
            const float v = second ? -ldexpf(rv, NP == 2 ? rx - E + se : se) : rv - static_cast<float>(kPExp) + static_cast<float>(NP == 2 ? rx - E : 0);
            if (tid < 2 * kTile) r[tid] = v;
        };

        floatx16 dk[2], dv[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[0][r] = dk[1][r] = dv[0][r] = dv[1][r] = 0.0f;
        store_rows(row0);
        wait_loads();
        __syncthreads();
        floatx16 s, dp;
        half8 pf[2][NP], df[2][NP];
        auto scores = [&](int t, auto ST) {
            constexpr int st = decltype(ST)::value;
            const float* rw = st ? row1 : row0;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
            // fp16: dP's sum starts from -delta
            if constexpr (NP == 1) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const floatx4 dq = *reinterpret_cast<const floatx4*>(&rw[kTile + 32 * t + 8 * q + 4 * g]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dp[4 * q + e] = dq[e];
                }
            }
            half8 qf[kAhead + 1][NP], gf[kAhead + 1][NP];
            auto rows = [&](int i) {
                Q.template row_frag<st>(places, t, i, qf[i & kAhead]);
                G.template row_frag<st>(places, t, i, gf[i & kAhead]);
            };
            if (kAhead) rows(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i + kAhead < 4) rows(i + kAhead);
                if (kAhead) __builtin_amdgcn_sched_barrier(0);
                s = mma<NP>(qf[i & kAhead], kf[i], s);
                dp = mma<NP>(gf[i & kAhead], vf[i], dp);
            }
        };
        auto weights = [&](uint32_t j, int t, auto ST) {
            constexpr int st = decltype(ST)::value;
            const float* rw = st ? row1 : row0;
            float p[16], ds[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const floatx4 lq = *reinterpret_cast<const floatx4*>(&rw[32 * t + 8 * q + 4 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) p[4 * q + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * q + e], a.c, -lq[e]));
                if constexpr (NP == 2) {
                    const floatx4 dq = *reinterpret_cast<const floatx4*>(&rw[kTile + 32 * t + 8 * q + 4 * g]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dp[4 * q + e] = __builtin_fmaf(dp[4 * q + e], psc, dq[e]);
                }
            }
            // causal: tiles that start at or past the wave's last key need no mask (wave-uniform)
            if constexpr (CAUSAL) {
                if (j * kTile < k0 + wave * 32 + 31) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (j * kTile + 32 * t + 8 * (r >> 2) + 4 * g + (r & 3) < kj) p[r] = 0.0f;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = p[r] * dp[r];
            if constexpr (NP == 1) {
                if (rest) {  // uniform in the workgroup
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] *= rsc;
                }
            }
#pragma unroll
            for (int sp = 0; sp < 2; ++sp) {
                operand<NP>(p, sp, pf[sp], neg1);
                operand<NP>(ds, sp, df[sp], neg1);
            }
        };
        auto products = [&](int t, auto ST) {
            constexpr int st = decltype(ST)::value;
            half8 gt[kAhead + 1][NP], qt[kAhead + 1][NP];
            auto columns = [&](int n) {
                G.template col_frag<st>(places, t, n >> 1, n & 1, gt[n & kAhead]);
                Q.template col_frag<st>(places, t, n >> 1, n & 1, qt[n & kAhead]);
            };
            if (kAhead) columns(0);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                if (n + kAhead < 4) columns(n + kAhead);
                if (kAhead) __builtin_amdgcn_sched_barrier(0);
                dv[n & 1] = mma<NP>(gt[n & kAhead], pf[n >> 1], dv[n & 1]);
                dk[n & 1] = mma<NP>(qt[n & kAhead], df[n >> 1], dk[n & 1]);
            }
        };
        auto tile = [&](uint32_t j, auto ST) {
            // one half's values live at a time (the scores of one half between the exponentials of the other: 225 us
            // against 212 at 2 x 10 x 4096^2)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                __builtin_amdgcn_sched_barrier(0);
                scores(t, ST);
                weights(j, t, ST);
                products(t, ST);
            }
        };
        auto step = [&](uint32_t j, auto ST) {
            constexpr int nx = decltype(ST)::value ^ 1;
            // (the last tile loads the one after it, which is not used)
            Q.template load<nx>((j + 1) * kTile);
            G.template load<nx>((j + 1) * kTile);
            load_rows(j + 1);
            tile(j, ST);
            store_rows(nx ? row1 : row0);
            wait_loads();
            __syncthreads();
        };
        for (; it < t1; it += 2) {
            step(it, std::integral_constant<int, 0>{});
            if (it + 1 < t1) step(it + 1, std::integral_constant<int, 1>{});
        }
        // keys past their row's length get zeros (their P is not: their scores are those of a zero key)
        const float fv = ldexpf(1.0f, -kPExp - E), fk = ldexpf(a.scale, -kPExp - se - rest);
        if (!in)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[0][r] = dk[1][r] = dv[0][r] = dv[1][r] = 0.0f;
        if (!pc.whole) {
            float* P = a.part + (2ull * wg + (pc.first ? 0 : 1)) * kKPart + (wave * 32 + l32) * 64;
            store_row(P, dk, fk, 64, g);
            store_row(P + kB * 64, dv, fv, 64, g);
        } else if (kj < a.Tk) {
            store_row(head_of<T>(a.dk, b, h) + static_cast<uint64_t>(kj) * a.dk.ld, dk, fk, ohd, g);
            store_row(head_of<T>(a.dv, b, h) + static_cast<uint64_t>(kj) * a.dv.ld, dv, fv, ohd, g);
        }
    }
}

// dK (blockIdx.y = 0) and dV (1) of the shared key blocks: the parts added in order, four loaded at a time. Eight
// workgroups a block; thread t takes key t / 16 of its 16, columns 4 (t % 16).
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_k_merge_kernel(BwdArgs a) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const uint32_t id = blockIdx.x / 8, bh = id / a.kd.nb, kb = id % a.kd.nb;
    const Parts<true> ps(a.kd, a.causal != 0, bh, kb);
    const int r = static_cast<int>(blockIdx.x % 8) * 16 + static_cast<int>(threadIdx.x >> 4), d = (threadIdx.x & 15) * 4;
    const uint32_t kj = kb * kB + r;
    if (ps.w0 == ps.w1 || kj >= a.Tk || d >= static_cast<int>(a.ohd)) return;
    const float* P = a.part + blockIdx.y * kB * 64 + r * 64 + d;
    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t w = ps.w0; w <= ps.w1; w += 4) {
        floatx4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const floatx4*>(P + ps.slot(a.kd, min(w + i, ps.w1)) * kKPart);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (w + i <= ps.w1) v += x[i];
    }
    const uint64_t ld = blockIdx.y ? a.dv.ld : a.dk.ld;
    T* out = (blockIdx.y ? head_of<T>(a.dv, bh / a.heads, bh % a.heads) : head_of<T>(a.dk, bh / a.heads, bh % a.heads)) + kj * ld + d;
    *reinterpret_cast<T4*>(out) = T4{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
}

// dq, dk and dv (blockIdx.y) from planes in the workspace into tensors that take no 4-element stores.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_unpack_kernel(BwdArgs a) {
    const uint32_t which = blockIdx.y, len = which ? a.Tk : a.Tq;
    const uint64_t rows = static_cast<uint64_t>(a.batch) * len * a.heads, n = rows * a.hd;
    const T* from = static_cast<const T*>(which == 0 ? a.dq.p : which == 1 ? a.dk.p : a.dv.p);
    T* to = static_cast<T*>(const_cast<void*>(which == 0 ? a.user[0].p : which == 1 ? a.user[1].p : a.user[2].p));
    const uint64_t ld = which == 0 ? a.user[0].ld : which == 1 ? a.user[1].ld : a.user[2].ld;
    const uint64_t sb = which == 0 ? a.user[0].s : which == 1 ? a.user[1].s : a.user[2].s;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += static_cast<uint64_t>(gridDim.x) * 256) {
        const uint64_t d = i % a.hd, at = i / a.hd, h = at % a.heads, tok = at / a.heads, b = tok / len, t = tok % len;
        to[b * sb + t * ld + h * a.hd + d] = from[((b * a.heads + h) * len + t) * 64 + d];
    }
}

// Zeros in dk and dv, for a call without queries.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_zero_kernel(BwdArgs a) {
    const uint64_t C = static_cast<uint64_t>(a.heads) * a.hd, n = static_cast<uint64_t>(a.batch) * a.Tk * C;
    const Tensor& t = blockIdx.y ? a.dv : a.dk;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += static_cast<uint64_t>(gridDim.x) * 256) {
        const uint64_t r = i / C;
        head_of<T>(t, 0, 0)[r / a.Tk * t.s + r % a.Tk * t.ld + i % C] = static_cast<T>(0.0f);
    }
}

// ---- plan -----------------------------------------------------------------------------------------------------------

constexpr uint32_t kSlots = 512;     // workgroups resident at once: two per CU
// Tiles of a share, at least, where blocks are shared. us with 4 / 2 / 1: fp16 2x20x1024x77 33.8 / 36.9 / 55, 2x20x256^2
// 23.8 / 34.3 / 42, fp32 2x20x1024x77 60.0 / 61.5 / 82 (and with 3: 38.4, 44, 63.6): smaller shares are mostly first loads, and
// their parts are written, read back and added.
constexpr uint32_t kMinShare = 4;

// Tiles that sharing has to take off the longest workgroup where there are more blocks than kSlots, to be worth its parts
// and their merge; without it the blocks of the second round start as those of the first end. us shared / whole: fp16
// 2x10x4096x256 66.6 / 56.4 (3 tiles off the queries' kernel), x1024 126 / 119 (12), x2048 212 / 205 (24), x4096 365 / 382
// (48), 2x18x2048^2 192 / 199 (28); fp32 2x10x4096x512 175 / 171 (6), x1024 278 / 277 (12), x2048 482 / 489 (24).
constexpr uint32_t kMinSaved[2] = {24, 12};  // fp16, fp32

// Whole blocks, a workgroup each, where they fill rounds of kSlots well enough; else kSlots workgroups, or as many as get
// kMinShare tiles.

template <bool KEYS>
Deal deal(uint32_t bhs, uint32_t T, uint32_t Tother, bool causal, bool f32) {
    Deal d{};
    d.NT = std::max(1u, ceil_div(Tother, kTile));
    d.nb = ceil_div(T, kB);
    d.per = before<KEYS>(d.nb, d.NT, causal);
    const uint32_t blocks = bhs * d.nb;
    const uint64_t total = static_cast<uint64_t>(bhs) * d.per;
    d.wgs = blocks;
    const bool alike = d.per == d.nb * d.NT;  // all blocks have NT tiles
    d.whole = alike ? 1 : 0;
    if (total >= 1ull << 31) {  // (the tiles are counted in 32 bits; the last of so many rounds matters little)
        d.wgs = blocks;
        d.whole = 1;
        return d;
    }
    const uint64_t rounds = (blocks + kSlots - 1) / kSlots;
    const uint32_t shares = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(kSlots, total / kMinShare)));
    const bool worth = !alike || rounds * d.NT > total / kSlots + kMinSaved[f32];
    if (blocks && blocks < rounds * kSlots * 9 / 10 && (blocks > kSlots ? worth : shares > blocks)) {
        d.wgs = shares;
        d.whole = alike ? blocks / shares : 0;
    }
    if (!d.wgs) return d;
    const uint32_t shared = static_cast<uint32_t>(total) - dealt_whole(d) * d.NT;
    if (shared && shared < d.wgs) {  // (alike: the parts of a block are of workgroups one after the other, none without a tile)
        d.wgs = blocks;
        d.whole = 1;
        return d;
    }
    d.quo = shared / d.wgs;
    d.rem = shared % d.wgs;
    d.frac = static_cast<uint32_t>(((static_cast<uint64_t>(d.rem) << 32) + d.wgs - 1) / d.wgs);
    return d;
}
// No block is shared.
bool all_whole(const Deal& d, uint32_t bhs) { return d.whole && dealt_whole(d) == bhs * d.nb; }

struct Layout {
    uint64_t delta, rexp, maxes, part, planes, outs, total;  // byte offsets
    uint64_t qplane, kplane;                           // elements of a plane
};
Layout layout(uint32_t batch, uint32_t heads, uint32_t Tq, uint32_t Tk, bool packed, bool f32, bool vout) {
    Layout l;
    const uint64_t bh = static_cast<uint64_t>(batch) * heads, qb = ceil_div(Tq, kB), rows = bh * qb * kB * 4;
    l.delta = rows;
    l.rexp = 2 * rows;
    l.maxes = l.rexp + (packed ? rows : 0);
    l.part = (l.maxes + bh * qb * 8 + 255) / 256 * 256;
    // (the same bytes for causal calls and others)
    uint64_t parts = 0;
    for (const bool causal : {false, true}) {
        const uint32_t n = static_cast<uint32_t>(bh);
        const Deal qd = deal<false>(n, Tq, Tk, causal, f32), kd = deal<true>(n, Tk, Tq, causal, f32);
        parts = std::max(parts, std::max<uint64_t>(all_whole(qd, n) ? 0 : 8ull * qd.wgs * kQPart, all_whole(kd, n) ? 0 : 8ull * kd.wgs * kKPart));
    }
    l.planes = l.part + (parts + 255) / 256 * 256;
    l.qplane = bh * Tq * 64;
    l.kplane = bh * Tk * 64;
    l.outs = l.planes + (packed ? (l.qplane + l.kplane) * 2 * 2 * (f32 ? 2 : 1) : 0);
    l.total = l.outs + (vout ? 0 : (l.qplane + 2 * l.kplane) * (f32 ? 4 : 2));
    return l;
}

template <typename T>
void unpack(const BwdArgs& a, hipStream_t s) {
    const uint64_t n = static_cast<uint64_t>(a.batch) * a.heads * std::max(a.Tq, a.Tk) * a.hd;
    attn_bwd_unpack_kernel<T><<<dim3(static_cast<unsigned>(std::min<uint64_t>(ceil_div(n, 256), 4096)), 3), 256, 0, s>>>(a);
}

template <typename T, bool PACKED>
void launch(const BwdArgs& a, hipStream_t s) {
    const uint32_t bh = a.batch * a.heads;
    if constexpr (PACKED) {
        const uint64_t rows = static_cast<uint64_t>(bh) * std::max(a.Tq, a.Tk);
        attn_bwd_pack_kernel<T><<<dim3(ceil_div(rows, 32), 4), 256, 0, s>>>(a);
    }
    attn_bwd_q_kernel<T, PACKED><<<a.qd.wgs, 256, 0, s>>>(a);
    if (!all_whole(a.qd, bh)) attn_bwd_q_merge_kernel<T><<<bh * a.qblocks * 4, 256, 0, s>>>(a);
    if (a.Tk == 0) {
        if (a.user[0].ld) unpack<T>(a, s);
        return;
    }
    if (a.causal) attn_bwd_k_kernel<T, PACKED, true><<<a.kd.wgs, 256, 0, s>>>(a);
    else attn_bwd_k_kernel<T, PACKED, false><<<a.kd.wgs, 256, 0, s>>>(a);
    if (!all_whole(a.kd, bh)) attn_bwd_k_merge_kernel<T><<<dim3(bh * a.kd.nb * 8, 2), 256, 0, s>>>(a);
    if (a.user[0].ld) unpack<T>(a, s);
}

struct Span {
    const void* p;
    uint64_t bytes;
};

// Two outputs whose byte spans overlap without sharing an element: column blocks of one matrix (the joint Q / K / V
// gradient [rows, 3C]), the same strides and C columns apart at least; the last row of a batch (the further block's, of Tx
// or Ty rows) ends before the next batch begins.
bool interleaved(const Tensor& x, const Tensor& y, uint64_t Tx, uint64_t Ty, uint64_t batch, uint64_t C, uint64_t e) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(x.p), q = reinterpret_cast<uintptr_t>(y.p);
    const uint64_t apart = (p > q ? p - q : q - p), T = p > q ? Tx : Ty;
    return x.ld == y.ld && x.s == y.s && apart >= C * e && apart + C * e <= x.ld * e &&
           (batch == 1 || apart + ((T - 1) * x.ld + C) * e <= x.s * e);
}

// Both kernels' shares; the launches' limits.
int plan(const mi_attn_args& f, Deal& qd, Deal& kd, const char* fn) {
    const uint64_t bh = static_cast<uint64_t>(f.batch) * f.heads;
    const uint64_t qb = ceil_div(f.Tq, kB), kb = ceil_div(f.Tk, kB), qt = ceil_div(f.Tq, kTile) + 1, kt = ceil_div(f.Tk, kTile) + 1;
    if (bh * std::max(qb, kb) >= (1u << 20) || qb * kt >= (1u << 31) || kb * qt >= (1u << 31))
        return fail(MI_ERR_UNSUPPORTED, "%s: batch * heads * tokens too large", fn);
    qd = deal<false>(static_cast<uint32_t>(bh), f.Tq, f.Tk, f.causal != 0, f.in_dtype == MI_F32);
    kd = deal<true>(static_cast<uint32_t>(bh), f.Tk, f.Tq, f.causal != 0, f.in_dtype == MI_F32);
    return MI_OK;
}

// Every row of the inputs in whole 16-byte chunks.
bool wide(const mi_attn_bwd_args& x) {
    const mi_attn_args& f = x.fwd;
    const uint64_t e = f.in_dtype == MI_F16 ? 2 : 4;
    const struct {
        const void* p;
        uint64_t ld, s;
    } in[5] = {{f.q, f.ldq, f.sq}, {f.k, f.ldk, f.sk}, {f.v, f.ldv, f.sv}, {f.out, f.ldo, f.so}, {x.dout, x.lddout, x.sdout}};
    bool w = f.C / f.heads % 8 == 0;
    for (const auto& t : in) w = w && aligned(t.p, 16) && (t.ld ? t.ld : f.C) * e % 16 == 0 && (f.batch == 1 || t.s * e % 16 == 0);
    return w;
}

// Gradients that take 4-element stores.
bool wide_out(const mi_attn_bwd_args& x) {
    const mi_attn_args& f = x.fwd;
    const uint64_t e = f.in_dtype == MI_F16 ? 2 : 4;
    const struct {
        const void* p;
        uint64_t ld, s;
    } out[3] = {{x.dq, x.lddq, x.sdq}, {x.dk, x.lddk, x.sdk}, {x.dv, x.lddv, x.sdv}};
    bool w = f.C / f.heads % 4 == 0;
    for (const auto& t : out) w = w && aligned(t.p, 4 * e) && (t.ld ? t.ld : f.C) % 4 == 0 && (f.batch == 1 || t.s % 4 == 0);
    return w;
}

int run(const mi_attn_bwd_args& x, void* ws, uint64_t ws_bytes, hipStream_t stream, const char* fn) {
    const mi_attn_args& f = x.fwd;
    if (f.in_dtype != MI_F32 && f.in_dtype != MI_F16) return fail(MI_ERR_INVALID_ARG, "%s: in_dtype %d", fn, f.in_dtype);
    if (f.out_dtype != f.in_dtype) return fail(MI_ERR_INVALID_ARG, "%s: out_dtype %d is not in_dtype %d", fn, f.out_dtype, f.in_dtype);
    if (f.batch == 0) return fail(MI_ERR_INVALID_ARG, "%s: batch 0", fn);
    if (!mi_fused_attn_supported(f.C, f.heads))
        return fail(MI_ERR_UNSUPPORTED, "%s: unsupported C=%u heads=%u (need heads | C and C/heads <= 64)", fn, f.C, f.heads);
    if (f.batch > 65535 || f.heads > 65535) return fail(MI_ERR_UNSUPPORTED, "%s: batch/heads > 65535", fn);
    if (f.Tq && (!f.q || !f.out || !x.dout || !x.dq)) return fail(MI_ERR_INVALID_ARG, "%s: null q, out, dout or dq", fn);
    if (f.Tk && (!f.k || !f.v || !x.dk || !x.dv)) return fail(MI_ERR_INVALID_ARG, "%s: null k, v, dk or dv", fn);
    const float hd = static_cast<float>(f.C / f.heads);
    const float scale = f.scale != 0.0f ? f.scale : 1.0f / sqrtf(hd);
    if (!(fabsf(scale) < INFINITY)) return fail(MI_ERR_INVALID_ARG, "%s: scale is not finite", fn);

    BwdArgs a{};
    const uint64_t e = f.in_dtype == MI_F16 ? 2 : 4;
    const struct {
        const void* p;
        uint64_t ld, s;
        uint32_t T;
        Tensor* t;
        const char* name;
    } in[8] = {{f.q, f.ldq, f.sq, f.Tq, &a.q, "q"},         {f.k, f.ldk, f.sk, f.Tk, &a.k, "k"},
               {f.v, f.ldv, f.sv, f.Tk, &a.v, "v"},         {f.out, f.ldo, f.so, f.Tq, &a.o, "out"},
               {x.dout, x.lddout, x.sdout, f.Tq, &a.g, "dout"}, {x.dq, x.lddq, x.sdq, f.Tq, &a.dq, "dq"},
               {x.dk, x.lddk, x.sdk, f.Tk, &a.dk, "dk"},    {x.dv, x.lddv, x.sdv, f.Tk, &a.dv, "dv"}};
    Span span[8];
    const bool vec = wide(x), vout = wide_out(x);
    for (int i = 0; i < 8; ++i) {
        const uint64_t ld = in[i].ld ? in[i].ld : f.C, s = in[i].s ? in[i].s : in[i].T * ld;
        if (ld < f.C) return fail(MI_ERR_INVALID_ARG, "%s: token stride of %s < C", fn, in[i].name);
        // 64 rows of a tile stay below 2^30 bytes (32-bit buffer offsets)
        if (ld >= (1ull << 22)) return fail(MI_ERR_UNSUPPORTED, "%s: token stride of %s too large", fn, in[i].name);
        if (i >= 5 && f.batch > 1 && in[i].T && s < (in[i].T - 1) * ld + f.C)
            return fail(MI_ERR_INVALID_ARG, "%s: batch rows of %s overlap", fn, in[i].name);
        if (!aligned(in[i].p, e)) return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
        *in[i].t = Tensor{in[i].p, ld, s, f.C / f.heads};
        span[i] = Span{in[i].p, in[i].T ? ((f.batch - 1) * s + (in[i].T - 1) * ld + f.C) * e : 0};
    }
    for (int o = 5; o < 8; ++o)
        for (int i = 0; i < o; ++i)
            if (overlaps(span[o].p, span[o].bytes, span[i].p, span[i].bytes) &&
                !(i >= 5 && interleaved(*in[o].t, *in[i].t, in[o].T, in[i].T, f.batch, f.C, e)))
                return fail(MI_ERR_ALIASING, "%s: %s overlaps %s", fn, in[o].name, in[i].name);
    a.batch = f.batch;
    a.Tq = f.Tq;
    a.Tk = f.Tk;
    a.heads = f.heads;
    a.hd = f.C / f.heads;
    a.causal = f.causal ? 1 : 0;
    a.kv_len = f.kv_len;
    a.scale = scale;
    a.sgn = scale < 0.0f ? -1.0f : 1.0f;
    a.c = fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f);  // a masked score stays -inf
    a.ohd = a.hd;
    if (f.Tq == 0) {
        if (f.Tk == 0) return MI_OK;
        const uint64_t n = static_cast<uint64_t>(f.batch) * f.Tk * f.C;
        const dim3 grid(static_cast<unsigned>(std::min<uint64_t>(ceil_div(n, 256), 1024)), 2);
        if (e == 2) attn_bwd_zero_kernel<_Float16><<<grid, 256, 0, stream>>>(a);
        else attn_bwd_zero_kernel<float><<<grid, 256, 0, stream>>>(a);
        return check_launch(fn);
    }
    a.qblocks = ceil_div(f.Tq, kB);
    const int st = plan(f, a.qd, a.kd, fn);
    if (st) return st;
    const bool packed = e == 4 || !vec;
    const Layout l = layout(f.batch, f.heads, f.Tq, f.Tk, packed, e == 4, vout);
    const uint64_t bhs = static_cast<uint64_t>(f.batch) * f.heads;
    if (!ws || ws_bytes < l.total)
        return fail(MI_ERR_INVALID_ARG, "%s: workspace %llu bytes < %llu needed", fn,
                    static_cast<unsigned long long>(ws ? ws_bytes : 0), static_cast<unsigned long long>(l.total));
    if (!aligned(ws, 16)) return fail(MI_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
    for (int i = 0; i < 8; ++i)
        if (overlaps(ws, l.total, span[i].p, span[i].bytes)) return fail(MI_ERR_ALIASING, "%s: workspace overlaps %s", fn, in[i].name);
    char* w = static_cast<char*>(ws);
    a.lse = reinterpret_cast<float*>(w);
    a.delta = reinterpret_cast<float*>(w + l.delta);
    a.rexp = packed ? reinterpret_cast<int*>(w + l.rexp) : nullptr;
    a.maxes = reinterpret_cast<float*>(w + l.maxes);
    a.part = reinterpret_cast<float*>(w + l.part);
    a.vin = vec ? 1u : 0u;
    if (!vout) {
        char* p = w + l.outs;
        Tensor* t[3] = {&a.dq, &a.dk, &a.dv};
        for (int i = 0; i < 3; ++i) {
            const uint64_t T = i ? f.Tk : f.Tq;
            a.user[i] = *t[i];
            *t[i] = Tensor{p, 64, f.heads * T * 64, T * 64};
            p += bhs * T * 64 * e;
        }
        a.ohd = 64;
    }
    if (packed) {
        _Float16* p = reinterpret_cast<_Float16*>(w + l.planes);
        const uint64_t np = e == 4 ? 2 : 1;
        auto take = [&](uint32_t T, uint64_t plane) {
            const Operand x{p, 64, static_cast<uint64_t>(f.heads) * T * 64, static_cast<uint64_t>(T) * 64, plane};
            p += np * plane;
            return x;
        };
        a.xq = take(f.Tq, l.qplane);
        a.xg = take(f.Tq, l.qplane);
        a.xk = take(f.Tk, l.kplane);
        a.xv = take(f.Tk, l.kplane);
        if (e == 4) launch<float, true>(a, stream);
        else launch<_Float16, true>(a, stream);
    } else {
        auto direct = [&](const Tensor& t) { return Operand{static_cast<const _Float16*>(t.p), t.ld, t.s, a.hd, 0}; };
        a.xq = direct(a.q);
        a.xg = direct(a.g);
        a.xk = direct(a.k);
        a.xv = direct(a.v);
        launch<_Float16, false>(a, stream);
    }
    return check_launch(fn);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" uint64_t mi_fused_attention_bwd_ws_bytes(const mi_attn_bwd_args* args) {
    if (!args) return 0;
    const mi_attn_args& f = args->fwd;
    if (!f.batch || !f.Tq || !mi_fused_attn_supported(f.C, f.heads) || (f.in_dtype != MI_F32 && f.in_dtype != MI_F16)) return 0;
    Deal qd, kd;
    if (plan(f, qd, kd, "mi_fused_attention_bwd_ws_bytes") != MI_OK) return 0;
    const bool f32 = f.in_dtype == MI_F32;
    return layout(f.batch, f.heads, f.Tq, f.Tk, f32 || !wide(*args), f32, wide_out(*args)).total;
}

extern "C" int mi_fused_attention_bwd(const mi_attn_bwd_args* args, void* workspace, uint64_t workspace_bytes, void* stream) {
    if (!args) return fail(MI_ERR_INVALID_ARG, "mi_fused_attention_bwd: null args");
    return run(*args, workspace, workspace_bytes, static_cast<hipStream_t>(stream), "mi_fused_attention_bwd");
}

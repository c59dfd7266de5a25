// attention_bwd.hip -- gradients of the fused attention (attention.hip) for gfx950.
//
// With S = scale Q K^T (+ mask), P = softmax(S) per query i and O = P V:
//   delta_i = sum_d dO_id O_id          (= sum_j P_ij dP_ij)
//   dP = dO V^T,   dS = P (dP - delta)
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO
// P is never stored: two kernels recompute it, one for queries, one for keys.
//
// attn_bwd_q_kernel: a workgroup owns 128 queries of one (batch, head), 4 waves x 32, and walks over 64-key tiles of K
// and V in LDS. S^T = K Q^T and dP^T = V dO^T leave a lane with one query and 32 keys, so the softmax is the forward
// pass's online one: with the running maximum m, dQ accumulates exp2(s - m) (dP - delta) K and is rescaled with the row
// sum l when m rises (lazily: kLazy); dQ = scale / l times that. Nothing but Q, K, V, O and dO is needed from the
// forward pass; m + log2 l and delta of each row go to the workspace for the other kernel.
// attn_bwd_k_kernel: a workgroup owns 128 keys, 4 waves x 32, and walks over 64-query tiles of Q and dO.
// S = Q K^T and dP = dO V^T leave a lane with one key and 32 queries; P = exp2(s - (m + log2 l)). dV^T = dO^T P and
// dK^T = Q^T dS take P and dS from the registers they are in (the MFMA's output order of the contracted index is the
// order in which the other operand is read).
// Every MFMA is v_mfma_f32_32x32x16_f16: seven products of Tq x Tk x 64 instead of five, for no atomic additions and
// no dQ partials in memory (results repeat bit for bit).
//
// Each tile is staged row-major (64 rows x 64 columns fp16); 16-byte chunk c of row r lies at slot c ^ f(r), f the bit
// reversal of (r / 2) % 8. That makes both uses free of bank conflicts: the 16-byte row fragments (16 rows of one chunk:
// every slot of either half once) and the transposing reads of ds_read_b64_tr_b16 (four rows of four chunks: the
// reversal puts rows r and r + 2 into different halves of a row).
//
// fp32 tensors are carried as fp16 pairs x = hi + lo and three MFMAs per product (hi hi + hi lo + lo hi), as in the
// forward pass; P and dS too. fp16's range is kept by powers of two, which are exact:
//   * dS of a query row, in the first kernel, by the row's largest |dO| (kRowExp);
//   * P, in the second kernel, by 2^14 (weights of 2^-28 are normal numbers then); dS by what keeps
//     2^14 (64 max|dO| max|V| + max|delta|) under 2^15, max|dO| and max|delta| over the (batch, head), max|V| over the
//     wave's keys: dS cannot overflow, and a weight of 2^-20 still has all its bits;
//   * dO, fp32 only, by its largest element (of the row, or of the (batch, head)), taken to 2^8.
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace mi {
namespace {

constexpr int kB = 128;                  // queries (keys) per workgroup
constexpr int kTile = 64;                // keys (queries) per staged tile
// The running max rises when a score passes it by this (exp2 domain), and the power of two that a row's largest |dO| is
// taken to in dS: exp2(s - m) (dP - delta) stays in fp16's range for |V| up to 32 even where 64 products agree in sign. A
// pair's low part is a subnormal number where dS is small, so fp32 takes it larger and rescales more often.
template <int NP>
constexpr float kLazy = NP == 2 ? 2.0f : 8.0f;
template <int NP>
constexpr int kRowExp = NP == 2 ? 2 : -4;
constexpr int kPairExp = 8;              // fp32: the power of two that the largest |dO| is taken to in its pairs
constexpr int kPExp = 14;                // P's power of two in the key kernel
constexpr uint32_t kOob = 0x80000000u;   // a buffer offset past every record: the load returns zeros

struct Tensor {
    const void* p;
    uint64_t ld, s;  // token and batch strides, elements
};
struct BwdArgs {
    Tensor q, k, v, o, g;     // g: dO
    Tensor dq, dk, dv;
    uint32_t batch, Tq, Tk, heads, hd;
    int causal;
    const int32_t* kv_len;
    float c;                  // |scale| log2(e)
    float sgn, scale;         // the scale's sign, and itself
    // workspace: per (batch, head) rows of qpad = 128 ceil(Tq / 128): m + log2 l (+inf: no key), delta; then per
    // 128 queries max|dO| and max|delta|; then the query parts' dK and dV
    float *lse, *delta, *maxes, *part;
    uint32_t qblocks, kblocks, splits;
    uint32_t vout;            // dq, dk and dv take 4-element stores
};

__device__ __forceinline__ uint32_t keys_of(const BwdArgs& a, uint32_t b) {
    if (!a.kv_len) return a.Tk;
    const int32_t l = a.kv_len[b];
    return l < 0 ? 0u : min(static_cast<uint32_t>(l), a.Tk);
}
template <typename T>
__device__ __forceinline__ const T* head_of(const Tensor& t, uint32_t b, uint32_t h, uint32_t hd) {
    return static_cast<const T*>(t.p) + b * t.s + static_cast<uint64_t>(h) * hd;
}
// bit reversal of (r / 2) % 8
__device__ __forceinline__ int swz(int r) { return ((r >> 3) & 1) | ((r >> 1) & 2) | ((r << 1) & 4); }

// Eight consecutive elements of a row, those at or past `valid` zero, as fp16 and, for fp32, fp16 residuals, times sc.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int valid, float sc, half8& hi, half8& lo) {
    T x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<T>(0.0f);
    if constexpr (VEC) {
        typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
        if (valid > 0) {
#pragma unroll
            for (int i = 0; i < 8 * static_cast<int>(sizeof(T)) / 16; ++i) {
                const V v = reinterpret_cast<const V*>(p)[i];
#pragma unroll
                for (int e = 0; e < static_cast<int>(16 / sizeof(T)); ++e) x[i * (16 / sizeof(T)) + e] = v[e];
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < valid) x[e] = p[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (sizeof(T) == 4) {
            const float v = x[e] * sc;
            hi[e] = static_cast<_Float16>(v);
            lo[e] = static_cast<_Float16>(v - static_cast<float>(hi[e]));
        } else {
            hi[e] = sc < 0.0f ? -x[e] : x[e];  // fp16: the sign alone
        }
    }
}
__device__ __forceinline__ half8 zero8() { return half8{0, 0, 0, 0, 0, 0, 0, 0}; }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
// The exponent e of a positive x in [2^e, 2^(e+1)); zero and subnormals -127.
__device__ __forceinline__ int exponent(float x) { return static_cast<int>(__float_as_uint(x) >> 23) - 127; }

// One staged operand: 64 rows of up to 64 columns of a [rows, ld] tensor, two LDS stages of NP planes.
// fp16 rows of whole 16-byte chunks travel straight into LDS; others through registers (converted on the way).
template <typename T, bool VEC>
struct Stage {
    static constexpr bool kDma = VEC && sizeof(T) == 2;
    static constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    static constexpr int kPlane = kTile * 64, kHalves = 2 * NP * kPlane;
    _Float16* lds;
    const T* base;
    uint64_t ld;
    uint32_t rows;  // rows of the tensor that are read; others are zeros
    int hd, tid;
    float sc;       // fp32: the elements' power of two
    half8 r[kDma ? 1 : 2][NP];

    __device__ __forceinline__ Stage(_Float16* l, const T* b, uint64_t ld_, uint32_t rows_, uint32_t hd_, int tid_, float sc_ = 1.0f)
        : lds(l), base(b), ld(ld_), rows(rows_), hd(static_cast<int>(hd_)), tid(tid_), sc(sc_) {}
    // chunk tid + 256 i of the tile: row c / 8, slot c % 8
    __device__ __forceinline__ void load(uint32_t row0, int st) {
        if constexpr (kDma) {
            const uint32_t n = row0 < rows ? min(rows - row0, static_cast<uint32_t>(kTile)) : 0u;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<T*>(base + static_cast<uint64_t>(n ? row0 : 0u) * ld), 0,
                n ? static_cast<int>(((n - 1) * ld + hd) * 2) : 0, 0x00020000);
            const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int piece = wave * 2 + i, row = 8 * piece + (lane >> 3), c = (lane & 7) ^ swz(row);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void*)(lds + st * NP * kPlane + piece * 512), 16,
                    c * 8 < hd ? (row * static_cast<uint32_t>(ld) + c * 8) * 2u : kOob, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int ch = tid + 256 * i, row = ch >> 3, c = (ch & 7) ^ swz(row);
                const bool in = row0 + row < rows;
                half8 lo = zero8();
                load8<T, VEC>(base + static_cast<uint64_t>(in ? row0 + row : 0u) * ld + (c * 8 < hd ? c * 8 : 0), in ? hd - c * 8 : 0, sc,
                              r[i][0], lo);
                if constexpr (NP == 2) r[i][1] = lo;
            }
        }
    }
    __device__ __forceinline__ void store(int st) {
        if constexpr (!kDma) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    *reinterpret_cast<half8*>(lds + (st * NP + p) * kPlane + (tid + 256 * i) * 8) = r[i][p];
        }
    }
    // this thread's loads of a tile are in LDS (before the barrier that hands it over)
    __device__ __forceinline__ void settle() {
        if constexpr (kDma) __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    // rows 32 t + l32, columns 16 s + 8 g .. + 7
    __device__ __forceinline__ half8 row_frag(int st, int p, int t, int s, int l32, int g) const {
        return *reinterpret_cast<const half8*>(lds + (st * NP + p) * kPlane + (32 * t + l32) * 64 + (((2 * s + g) ^ swz(l32)) * 8));
    }
    // column 32 u + l32, rows 32 t + 16 sp + 4 g + {0..3, 8..11}
    __device__ __forceinline__ half8 col_frag(int st, int p, int t, int sp, int u, int lane) const {
        const int g = lane >> 5, rk = (lane >> 2) & 3, d = 32 * u + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        half4 x[2];
#pragma unroll
        for (int rd = 0; rd < 2; ++rd) {
            const int row = 32 * t + 16 * sp + 8 * rd + 4 * g + rk;
            x[rd] = lds_read_tr16(lds + (st * NP + p) * kPlane + row * 64 + (((d >> 3) ^ swz(row)) * 8) + (d & 7));
        }
        return half8{x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
    }
};

// acc += a b of one 16-deep slice: one MFMA, or three of the pairs' planes (those with a residual first).
template <int NP>
__device__ __forceinline__ floatx16 mma(const half8 (&x)[NP], const half8 (&y)[NP], floatx16 acc) {
    if constexpr (NP == 2) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[1], y[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[0], y[1], acc, 0, 0, 0);
    }
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x[0], y[0], acc, 0, 0, 0);
}
// Elements 8 sp .. 8 sp + 7 of x as an MFMA operand. The empty register constraint holds the fp32 value: the rounding to hi
// must not fuse into the multiplication that made it (a mixed-precision fma rounds the exact product), or lo, the rest of
// the fp32 value, would belong to another hi now and then (a row in a hundred off by 1e-4).
template <int NP>
__device__ __forceinline__ void operand(const float (&x)[16], int sp, half8 (&f)[NP]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v = x[8 * sp + i];
        if constexpr (NP == 2) asm volatile("" : "+v"(v));
        f[0][i] = static_cast<_Float16>(v);
        if constexpr (NP == 2) f[NP - 1][i] = static_cast<_Float16>(v - static_cast<float>(f[0][i]));
    }
}

// Columns 32 u + 8 (r / 4) + 4 g + r % 4 of one row of T from two accumulator tiles, times f.
template <typename T>
__device__ __forceinline__ void store_row(T* row, const floatx16 (&acc)[2], float f, int hd, int g, bool vec) {
    typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * u + 8 * q + 4 * g;
            if (d >= hd) continue;
            const T4 v = {static_cast<T>(acc[u][4 * q] * f), static_cast<T>(acc[u][4 * q + 1] * f),
                          static_cast<T>(acc[u][4 * q + 2] * f), static_cast<T>(acc[u][4 * q + 3] * f)};
            if (vec) {
                *reinterpret_cast<T4*>(row + d) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < hd) row[d + e] = v[e];
            }
        }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256, 2) void attn_bwd_q_kernel(BwdArgs a) {
    typedef Stage<T, VEC> St;
    constexpr int NP = St::NP;
    __shared__ __attribute__((aligned(16))) _Float16 smem[2 * St::kHalves];
    __shared__ float wmax[2][4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, g = lane >> 5;
    const uint32_t blk = xcd_swizzle(blockIdx.x, gridDim.x);
    const uint32_t qb = blk % a.qblocks, bh = blk / a.qblocks;
    const uint32_t h = bh % a.heads, b = bh / a.heads;
    const uint32_t q0 = qb * kB, qi = q0 + wave * 32 + l32;
    const int hd = static_cast<int>(a.hd);
    const uint32_t L = keys_of(a, b);
    const uint32_t kend = a.causal ? min(L, q0 + kB) : L;
    // tiles that end at or before kfull need no mask for any query of this wave
    uint32_t kfull = L / kTile * kTile;
    if (a.causal) kfull = min(kfull, (q0 + wave * 32 + 1) / kTile * kTile);

    St K(smem, head_of<T>(a.k, b, h, a.hd), a.k.ld, kend, a.hd, tid);
    St V(smem + St::kHalves, head_of<T>(a.v, b, h, a.hd), a.v.ld, kend, a.hd, tid);
    const uint32_t ntiles = (kend + kTile - 1) / kTile;
    if (ntiles) {
        K.load(0, 0);
        V.load(0, 0);
    }

    // this lane's query: fragments of Q (with the scale's sign) and dO, delta, max|dO|
    const bool in = qi < a.Tq;
    const T* qp = head_of<T>(a.q, b, h, a.hd) + static_cast<uint64_t>(in ? qi : 0u) * a.q.ld;
    const T* op = head_of<T>(a.o, b, h, a.hd) + static_cast<uint64_t>(in ? qi : 0u) * a.o.ld;
    const T* gp = head_of<T>(a.g, b, h, a.hd) + static_cast<uint64_t>(in ? qi : 0u) * a.g.ld;
    half8 qf[4][NP], gf[4][NP];
    float delta = 0.0f, gmax = 0.0f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int d = 16 * s + 8 * g, n = in ? hd - d : 0;
        half8 lo = zero8();
        load8<T, VEC>(qp + (d < hd ? d : 0), n, a.sgn, qf[s][0], lo);
        if constexpr (NP == 2) qf[s][NP - 1] = lo;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) {
                const float x = static_cast<float>(gp[d + e]);
                delta = __builtin_fmaf(x, static_cast<float>(op[d + e]), delta);
                gmax = fmaxf(gmax, fabsf(x));
            }
    }
    delta += __shfl_xor(delta, 32);
    gmax = fmaxf(gmax, __shfl_xor(gmax, 32));
    // the row's power of two: max|dO| to 2^kRowExp in dS, to 2^kPairExp in the pairs
    const int ge = max(-100, min(100, kRowExp<NP> - exponent(gmax)));
    const float gsc = ldexpf(1.0f, ge);
    constexpr float kPairUp = NP == 2 ? 64.0f : 1.0f;
    static_assert(NP == 1 || kPairExp - kRowExp<2> == 6, "2^6 between the pairs of dO and dS");
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int d = 16 * s + 8 * g;
        half8 lo = zero8();
        load8<T, VEC>(gp + (d < hd ? d : 0), in ? hd - d : 0, NP == 2 ? gsc * kPairUp : 1.0f, gf[s][0], lo);
        if constexpr (NP == 2) gf[s][NP - 1] = lo;
    }
    const float dscale = NP == 2 ? 1.0f / kPairUp : gsc;
    const float ds0 = delta * gsc;
    const float bmax = wave_max(gmax), dmax = wave_max(fabsf(delta));
    if (lane == 0) {
        wmax[0][wave] = bmax;
        wmax[1][wave] = dmax;
    }

    floatx16 acc[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][r] = acc[1][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    if (ntiles) {
        K.store(0);
        V.store(0);
        K.settle();
    }
    __syncthreads();
    for (uint32_t it = 0; it < ntiles; ++it) {
        const int st = it & 1;
        const bool more = it + 1 < ntiles;
        if (more) {
            K.load((it + 1) * kTile, st ^ 1);
            V.load((it + 1) * kTile, st ^ 1);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            floatx16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                half8 kf[NP], vf[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    kf[p] = K.row_frag(st, p, t, i, l32, g);
                    vf[p] = V.row_frag(st, p, t, i, l32, g);
                }
                s = mma(kf, qf[i], s);
                dp = mma(vf, gf[i], dp);
            }
            const uint32_t k0 = it * kTile + 32 * t;
            if (it * kTile >= kfull) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t key = k0 + 8 * (r >> 2) + 4 * g + (r & 3);
                    if (key >= L || (a.causal && key > qi)) s[r] = -INFINITY;
                }
            }
            float mx = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
            mx = fmaxf(mx, __shfl_xor(mx, 32)) * a.c;
            if (__any(mx > m + kLazy<NP>)) {
                const float mn = fmaxf(m, mx);
                const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    acc[0][r] *= alpha;
                    acc[1][r] *= alpha;
                }
            }
            const float mu = m == -INFINITY ? 0.0f : m;
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -mu));
                l += p;
                ds[r] = p * __builtin_fmaf(dp[r], dscale, -ds0);
            }
#pragma unroll
            for (int sp = 0; sp < 2; ++sp) {
                half8 df[NP];
                operand<NP>(ds, sp, df);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    half8 kt[NP];
#pragma unroll
                    for (int p = 0; p < NP; ++p) kt[p] = K.col_frag(st, p, t, sp, u, lane);
                    acc[u] = mma(kt, df, acc[u]);
                }
            }
        }
        if (more) {
            K.store(st ^ 1);
            V.store(st ^ 1);
            K.settle();
        }
        __syncthreads();
    }
    l += __shfl_xor(l, 32);
    const uint64_t row = static_cast<uint64_t>(bh) * a.qblocks * kB + q0 + wave * 32 + l32;
    if (g == 0) {
        // a row without keys, or past Tq: its P is 0 in the key kernel whatever its scores
        a.lse[row] = in && l > 0.0f ? m + __builtin_log2f(l) : INFINITY;
        a.delta[row] = in ? delta : 0.0f;
    }
    if (tid < 2) {
        float x = wmax[tid][0];
#pragma unroll
        for (int w = 1; w < 4; ++w) x = fmaxf(x, wmax[tid][w]);
        a.maxes[(static_cast<uint64_t>(bh) * a.qblocks + qb) * 2 + tid] = x;
    }
    if (!in) return;
    const float f = l > 0.0f ? ldexpf(a.scale / l, -ge) : 0.0f;
    T* out = const_cast<T*>(head_of<T>(a.dq, b, h, a.hd)) + static_cast<uint64_t>(qi) * a.dq.ld;
    store_row(out, acc, f, hd, g, a.vout);
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256, 2) void attn_bwd_k_kernel(BwdArgs a) {
    typedef Stage<T, VEC> St;
    constexpr int NP = St::NP;
    __shared__ __attribute__((aligned(16))) _Float16 smem[2 * St::kHalves];
    __shared__ __attribute__((aligned(16))) float rowv[2][2][kTile];  // [stage][m + log2 l - kPExp, delta][query]
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, g = lane >> 5;
    const uint32_t blk = xcd_swizzle(blockIdx.x, gridDim.x);
    // parts of one key block are neighbours: they share its XCD with the head's other key blocks
    const uint32_t part = blk % a.splits, kb = blk / a.splits % a.kblocks, bh = blk / a.splits / a.kblocks;
    const uint32_t h = bh % a.heads, b = bh / a.heads;
    const uint32_t k0 = kb * kB, kj = k0 + wave * 32 + l32;
    const int hd = static_cast<int>(a.hd);
    const uint32_t L = keys_of(a, b);

    // max|dO| and max|delta| of the (batch, head)
    float gm = 0.0f, dm = 0.0f;
    for (uint32_t i = lane; i < a.qblocks; i += 64) {
        const float* x = a.maxes + (static_cast<uint64_t>(bh) * a.qblocks + i) * 2;
        gm = fmaxf(gm, x[0]);
        dm = fmaxf(dm, x[1]);
    }
    gm = wave_max(gm);
    dm = wave_max(dm);
    const int ge = NP == 2 ? max(-100, min(100, kPairExp - exponent(gm))) : 0;  // fp32: dO times 2^ge

    // this lane's key: fragments of K (with the scale's sign) and V
    const bool in = kj < L;
    const T* kp = head_of<T>(a.k, b, h, a.hd) + static_cast<uint64_t>(in ? kj : 0u) * a.k.ld;
    const T* vp = head_of<T>(a.v, b, h, a.hd) + static_cast<uint64_t>(in ? kj : 0u) * a.v.ld;
    half8 kf[4][NP], vf[4][NP];
    float vm = 0.0f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int d = 16 * s + 8 * g, n = in ? hd - d : 0;
        half8 lo = zero8();
        load8<T, VEC>(kp + (d < hd ? d : 0), n, a.sgn, kf[s][0], lo);
        if constexpr (NP == 2) kf[s][NP - 1] = lo;
        load8<T, VEC>(vp + (d < hd ? d : 0), n, 1.0f, vf[s][0], lo);
        if constexpr (NP == 2) vf[s][NP - 1] = lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) vm = fmaxf(vm, fabsf(static_cast<float>(vf[s][0][e])));
    }
    vm = wave_max(vm);
    // dS times 2^(kPExp + se) stays under 2^15; dP already carries 2^ge
    const int se = max(-100, min(100, 15 - kPExp - 1 - exponent(64.0f * gm * vm + dm)));
    const float psc = ldexpf(1.0f, se - ge), dsc = ldexpf(1.0f, se);

    // query tiles of this part; causal: from the first one with a query at or past the block's first key
    const uint32_t tiles = (a.Tq + kTile - 1) / kTile;
    const uint32_t first = a.causal ? min(k0 / kTile, tiles) : 0u;
    const uint32_t t0 = first + static_cast<uint32_t>(static_cast<uint64_t>(tiles - first) * part / a.splits);
    const uint32_t t1 = k0 < L ? first + static_cast<uint32_t>(static_cast<uint64_t>(tiles - first) * (part + 1) / a.splits) : t0;

    St Q(smem, head_of<T>(a.q, b, h, a.hd), a.q.ld, a.Tq, a.hd, tid);
    St G(smem + St::kHalves, head_of<T>(a.g, b, h, a.hd), a.g.ld, a.Tq, a.hd, tid, ldexpf(1.0f, ge));
    const float* lse = a.lse + static_cast<uint64_t>(bh) * a.qblocks * kB;
    const float* del = a.delta + static_cast<uint64_t>(bh) * a.qblocks * kB;
    float rv = 0.0f;  // threads 0..127: the next tile's row values
    auto load_rows = [&](uint32_t q0) {
        if (tid < kTile) rv = lse[q0 + tid] - static_cast<float>(kPExp);
        else if (tid < 2 * kTile) rv = del[q0 + tid - kTile];
    };
    auto store_rows = [&](int st) {
        if (tid < 2 * kTile) rowv[st][tid >> 6][tid & 63] = rv;
    };

    floatx16 dk[2], dv[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[0][r] = dk[1][r] = dv[0][r] = dv[1][r] = 0.0f;
    if (t0 < t1) {
        Q.load(t0 * kTile, 0);
        G.load(t0 * kTile, 0);
        load_rows(t0 * kTile);
        Q.store(0);
        G.store(0);
        store_rows(0);
        Q.settle();
    }
    __syncthreads();
    for (uint32_t it = t0; it < t1; ++it) {
        const int st = (it - t0) & 1;
        const bool more = it + 1 < t1;
        if (more) {
            Q.load((it + 1) * kTile, st ^ 1);
            G.load((it + 1) * kTile, st ^ 1);
            load_rows((it + 1) * kTile);
        }
        // causal: tiles that start at or past the wave's last key need no mask
        const bool mask = a.causal && it * kTile < k0 + wave * 32 + 31;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            floatx16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                half8 qf[NP], gf[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    qf[p] = Q.row_frag(st, p, t, i, l32, g);
                    gf[p] = G.row_frag(st, p, t, i, l32, g);
                }
                s = mma(qf, kf[i], s);
                dp = mma(gf, vf[i], dp);
            }
            float p[16], ds[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const floatx4 lq = *reinterpret_cast<const floatx4*>(&rowv[st][0][32 * t + 8 * q + 4 * g]);
                const floatx4 dq = *reinterpret_cast<const floatx4*>(&rowv[st][1][32 * t + 8 * q + 4 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * q + e;
                    p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -lq[e]));
                    if (mask && it * kTile + 32 * t + 8 * q + 4 * g + e < kj) p[r] = 0.0f;
                    ds[r] = p[r] * __builtin_fmaf(dp[r], psc, -dq[e] * dsc);
                }
            }
#pragma unroll
            for (int sp = 0; sp < 2; ++sp) {
                half8 pf[NP], df[NP];
                operand<NP>(p, sp, pf);
                operand<NP>(ds, sp, df);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    half8 gt[NP], qt[NP];
#pragma unroll
                    for (int pl = 0; pl < NP; ++pl) {
                        gt[pl] = G.col_frag(st, pl, t, sp, u, lane);
                        qt[pl] = Q.col_frag(st, pl, t, sp, u, lane);
                    }
                    dv[u] = mma(gt, pf, dv[u]);
                    dk[u] = mma(qt, df, dk[u]);
                }
            }
        }
        if (more) {
            Q.store(st ^ 1);
            G.store(st ^ 1);
            store_rows(st ^ 1);
            Q.settle();
        }
        __syncthreads();
    }
    if (kj >= a.Tk) return;
    // keys past their row's length get zeros
    const float fv = in ? ldexpf(1.0f, -kPExp - ge) : 0.0f;
    const float fk = in ? ldexpf(a.scale, -kPExp - se) : 0.0f;
    if (!in)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[0][r] = dk[1][r] = dv[0][r] = dv[1][r] = 0.0f;
    if (a.splits > 1) {
        // [part][dk, dv][batch, head][Tk][64]
        const uint64_t plane = static_cast<uint64_t>(a.batch) * a.heads * a.Tk * 64;
        float* P = a.part + part * 2 * plane + (static_cast<uint64_t>(bh) * a.Tk + kj) * 64;
        store_row(P, dk, fk, 64, g, true);
        store_row(P + plane, dv, fv, 64, g, true);
        return;
    }
    store_row(const_cast<T*>(head_of<T>(a.dk, b, h, a.hd)) + static_cast<uint64_t>(kj) * a.dk.ld, dk, fk, hd, g, a.vout);
    store_row(const_cast<T*>(head_of<T>(a.dv, b, h, a.hd)) + static_cast<uint64_t>(kj) * a.dv.ld, dv, fv, hd, g, a.vout);
}

// The query parts' dK (blockIdx.y = 0) and dV (1), added in order: 16 threads a row of 64 columns.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_sum_kernel(BwdArgs a) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const uint64_t rows = static_cast<uint64_t>(a.batch) * a.heads * a.Tk, plane = rows * 64;
    const uint64_t row = blockIdx.x * 16ull + (threadIdx.x >> 4);
    const int d = (threadIdx.x & 15) * 4, hd = static_cast<int>(a.hd);
    if (row >= rows || d >= hd) return;
    const float* p = a.part + blockIdx.y * plane + row * 64 + d;
    floatx4 v = *reinterpret_cast<const floatx4*>(p);
    for (uint32_t s = 1; s < a.splits; ++s) v += *reinterpret_cast<const floatx4*>(p + s * 2 * plane);
    const uint32_t bh = static_cast<uint32_t>(row / a.Tk), kj = static_cast<uint32_t>(row % a.Tk);
    const Tensor& t = blockIdx.y ? a.dv : a.dk;
    T* out = const_cast<T*>(head_of<T>(t, bh / a.heads, bh % a.heads, a.hd)) + static_cast<uint64_t>(kj) * t.ld + d;
    if (a.vout) {
        *reinterpret_cast<T4*>(out) = T4{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < hd) out[e] = static_cast<T>(v[e]);
    }
}

// Parts of the queries for the key kernel: as many as bring its grid to the GPU's CUs, each of two tiles at least.
uint32_t query_parts(uint64_t blocks, uint32_t Tq) {
    const uint64_t tiles = ceil_div(Tq, kTile);
    return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(256 / std::max<uint64_t>(blocks, 1), tiles / 2)));
}

struct Layout {
    uint64_t rows, maxes, part, total;  // bytes of one row array, offsets of the others
};
Layout layout(uint32_t batch, uint32_t heads, uint32_t Tq, uint32_t Tk, uint32_t splits) {
    Layout l;
    const uint64_t bh = static_cast<uint64_t>(batch) * heads, qb = ceil_div(Tq, kB);
    l.rows = bh * qb * kB * 4;
    l.maxes = 2 * l.rows;
    l.part = (l.maxes + bh * qb * 8 + 255) / 256 * 256;
    l.total = l.part + (splits > 1 ? static_cast<uint64_t>(splits) * 2 * bh * Tk * 64 * 4 : 0);
    return l;
}

template <typename T, bool VEC>
void launch(const BwdArgs& a, hipStream_t s) {
    const unsigned bh = a.batch * a.heads;
    attn_bwd_q_kernel<T, VEC><<<a.qblocks * bh, 256, 0, s>>>(a);
    if (a.Tk == 0) return;
    attn_bwd_k_kernel<T, VEC><<<a.kblocks * bh * a.splits, 256, 0, s>>>(a);
    if (a.splits > 1) attn_bwd_sum_kernel<T><<<dim3(ceil_div(static_cast<uint64_t>(bh) * a.Tk, 16), 2), 256, 0, s>>>(a);
}

// Zeros, for a call without queries.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_zero_kernel(BwdArgs a) {
    const uint64_t C = static_cast<uint64_t>(a.heads) * a.hd, n = static_cast<uint64_t>(a.batch) * a.Tk * C;
    const Tensor& t = blockIdx.y ? a.dv : a.dk;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += static_cast<uint64_t>(gridDim.x) * 256) {
        const uint64_t r = i / C;
        static_cast<T*>(const_cast<void*>(t.p))[r / a.Tk * t.s + r % a.Tk * t.ld + i % C] = static_cast<T>(0.0f);
    }
}

struct Span {
    const void* p;
    uint64_t bytes;
};

// Two outputs whose byte spans overlap without sharing an element: column blocks of one matrix (the joint Q / K / V
// gradient [rows, 3C]), the same strides and C columns apart at least.
bool interleaved(const Tensor& x, const Tensor& y, uint64_t C, uint64_t e) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(x.p), q = reinterpret_cast<uintptr_t>(y.p);
    const uint64_t apart = (p > q ? p - q : q - p);
    return x.ld == y.ld && x.s == y.s && apart >= C * e && apart + C * e <= x.ld * e;
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
    bool vec = f.C / f.heads % 8 == 0, vout = f.C / f.heads % 4 == 0;
    for (int i = 0; i < 8; ++i) {
        const uint64_t ld = in[i].ld ? in[i].ld : f.C, s = in[i].s ? in[i].s : in[i].T * ld;
        if (ld < f.C) return fail(MI_ERR_INVALID_ARG, "%s: token stride of %s < C", fn, in[i].name);
        // 64 rows of a tile stay below 2^30 bytes (32-bit buffer offsets)
        if (ld >= (1ull << 22)) return fail(MI_ERR_UNSUPPORTED, "%s: token stride of %s too large", fn, in[i].name);
        if (i >= 5 && f.batch > 1 && in[i].T && s < (in[i].T - 1) * ld + f.C)
            return fail(MI_ERR_INVALID_ARG, "%s: batch rows of %s overlap", fn, in[i].name);
        if (!aligned(in[i].p, e)) return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
        *in[i].t = Tensor{in[i].p, ld, s};
        span[i] = Span{in[i].p, in[i].T ? ((f.batch - 1) * s + (in[i].T - 1) * ld + f.C) * e : 0};
        if (i < 5) vec = vec && aligned(in[i].p, 16) && ld * e % 16 == 0 && (f.batch == 1 || s * e % 16 == 0);
        else vout = vout && aligned(in[i].p, 4 * e) && ld % 4 == 0 && (f.batch == 1 || s % 4 == 0);
    }
    for (int o = 5; o < 8; ++o)
        for (int i = 0; i < o; ++i)
            if (overlaps(span[o].p, span[o].bytes, span[i].p, span[i].bytes) &&
                !(i >= 5 && interleaved(*in[o].t, *in[i].t, f.C, e)))
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
    a.vout = vout ? 1u : 0u;
    const uint64_t bh = static_cast<uint64_t>(f.batch) * f.heads;
    if (f.Tq == 0) {
        if (f.Tk == 0) return MI_OK;
        const uint64_t n = static_cast<uint64_t>(f.batch) * f.Tk * f.C;
        const dim3 grid(static_cast<unsigned>(std::min<uint64_t>(ceil_div(n, 256), 1024)), 2);
        if (e == 2) attn_bwd_zero_kernel<_Float16><<<grid, 256, 0, stream>>>(a);
        else attn_bwd_zero_kernel<float><<<grid, 256, 0, stream>>>(a);
        return check_launch(fn);
    }
    a.qblocks = ceil_div(f.Tq, kB);
    a.kblocks = ceil_div(f.Tk, kB);
    a.splits = query_parts(bh * a.kblocks, f.Tq);
    if (bh * a.qblocks >= (1u << 23) || bh * a.kblocks * a.splits >= (1u << 23))
        return fail(MI_ERR_UNSUPPORTED, "%s: batch * heads * tokens too large", fn);
    const Layout l = layout(f.batch, f.heads, f.Tq, f.Tk, a.splits);
    if (!ws || ws_bytes < l.total)
        return fail(MI_ERR_INVALID_ARG, "%s: workspace %llu bytes < %llu needed", fn,
                    static_cast<unsigned long long>(ws ? ws_bytes : 0), static_cast<unsigned long long>(l.total));
    if (!aligned(ws, 16)) return fail(MI_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
    for (int i = 0; i < 8; ++i)
        if (overlaps(ws, l.total, span[i].p, span[i].bytes)) return fail(MI_ERR_ALIASING, "%s: workspace overlaps %s", fn, in[i].name);
    char* w = static_cast<char*>(ws);
    a.lse = reinterpret_cast<float*>(w);
    a.delta = reinterpret_cast<float*>(w + l.rows);
    a.maxes = reinterpret_cast<float*>(w + l.maxes);
    a.part = reinterpret_cast<float*>(w + l.part);
    if (e == 2 && vec) launch<_Float16, true>(a, stream);
    else if (e == 2) launch<_Float16, false>(a, stream);
    else if (vec) launch<float, true>(a, stream);
    else launch<float, false>(a, stream);
    return check_launch(fn);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" uint64_t mi_fused_attention_bwd_ws_bytes(const mi_attn_bwd_args* args) {
    if (!args) return 0;
    const mi_attn_args& f = args->fwd;
    if (!f.batch || !f.Tq || !mi_fused_attn_supported(f.C, f.heads)) return 0;
    const uint64_t bh = static_cast<uint64_t>(f.batch) * f.heads;
    return layout(f.batch, f.heads, f.Tq, f.Tk, query_parts(bh * ceil_div(f.Tk, kB), f.Tq)).total;
}

extern "C" int mi_fused_attention_bwd(const mi_attn_bwd_args* args, void* workspace, uint64_t workspace_bytes, void* stream) {
    if (!args) return fail(MI_ERR_INVALID_ARG, "mi_fused_attention_bwd: null args");
    return run(*args, workspace, workspace_bytes, static_cast<hipStream_t>(stream), "mi_fused_attention_bwd");
}

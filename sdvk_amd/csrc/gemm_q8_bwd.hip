// gemm_q8_bwd.hip -- the input gradient of a frozen Q8_0 linear for gfx950:
//   dA[M,K] (=|+=) dC[M,N] . deq(W[N,K])
// for the forward product C = A . deq(W)^T of gemm_q8.hip (the weights are frozen, so there is no dW).
//
// A workgroup computes a BM x BN tile of dA (BN columns k, whole 32-wide blocks) in steps of NS rows n of W:
//   * dC's rows are staged row-major in LDS, 128 bytes of a row per step;
//   * a step's BN / 32 blocks of each of NS weight rows are dequantised once per workgroup and staged row-major
//     [n][k]; the sum runs over n, so a weight fragment has to be k-major: ds_read_b64_tr_b16 transposes on the way
//     out of LDS (row stride BN + 32 halves, so that the four rows of a 32-lane read cover all banks);
//   * v_mfma_f32_32x32x16_f16 of the transposed product (a lane holds one row of dA and runs of four columns).
//
// fp16: dC as it is, w = fp16(d * q), fp32 sums, dA rounded once. The forward product rounds the weights alike: this is the
//   gradient of what ran (3e-4 of unrounded weights' in the mean, with the result's own rounding, which alone is 2e-4;
//   weights as pairs would take two products).
// fp32: both operands as fp16 pairs x = hi + lo and three products (hi hi + hi lo + lo hi): what is dropped is
//   2^-22 of a product, the accuracy of an fp32 product summed in fp32. fp16's range is kept by powers of two, which
//   are exact: the weights times 2^6 (|w| < 1023; the pair's absolute error 2^-31 is then 2^-25 of a weight of 0.02);
//   each row of dC by its own exponent, which follows the row's largest element seen so far (gradients of 1e-8 and
//   of 1e4 keep all their bits). A row's exponent falls by a step only when an element would pass 2^14 (its first
//   elements are taken to 2^9 .. 2^10), and the row's sums are then brought down with it.
//
// Measured (MI355X, us a call): fp16 2048x1280x5120 (M x N x K) 45 (600 TFLOP/s: 640 tiles of 128x128 on 512 places, MFMAs
// busy 29% of cycles, LDS 48%, and a barrier per step), 1976x10240x1280 71; fp32 1152x1280x1280 29 (five parts,
// 23 and 6 for their sum), 2048x1280x5120 105; 2x1280x1280 6.1 (gemm_q8_bwd_few_kernel).
//
// Grids too small to fill the GPU split N when the caller gives a workspace: each part stores its sums, fp32, and a
// second kernel adds them in order (results repeat bit for bit).
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace mi {
namespace {

constexpr uint32_t kPast = 0x80000000u;  // a buffer offset past every record: the load returns zeros
constexpr int kWExp = 6;                 // fp32: the weights' power of two
constexpr float kRowMax = 16384.0f;      // fp32: a row's exponent falls when an element passes this
constexpr int kRowExp = 9;               // ... and takes the row's largest element to [2^9, 2^10)

struct BwdArgs {
    const void* dC;
    const uint8_t* W;
    void* dA;
    float* part;         // N parts: [splits][M][K] fp32, else NULL
    uint32_t M, N, K, ldc, lda, mode;
    uint32_t rowbytes;   // of a weight row
    uint32_t tiles_m, tiles_k, group_m;
    uint32_t steps, steps_per_split;
    uint32_t vec;        // dA's rows (or the parts') take 4-element stores
};

// dA from one 32 x 32 accumulator tile at a time, through a wave-private LDS region (row stride 36 floats): eight
// lanes store a row's 32 columns. e: the lane's row exponents (fp32).
constexpr int kStageLd = 36;
constexpr int kStageFloats = 32 * kStageLd;

template <typename T, int FM, int FN>
__device__ __forceinline__ void store_tiles(const BwdArgs& a, float* stage, uint32_t mw, uint32_t kw, const floatx16 (&acc)[FM][FN],
                                            const int (&e)[FM], int lane, float* part) {
    const int l32 = lane & 31, g = lane >> 5;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T* const out = static_cast<T*>(a.dA);
    for (int b = 0; b < FM * FN; ++b) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                if (b == i * FN + j) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        floatx4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                        if constexpr (sizeof(T) == 4) {
#pragma unroll
                            for (int x = 0; x < 4; ++x) v[x] = ldexpf(v[x], -(e[i] + kWExp));
                        }
                        *reinterpret_cast<floatx4*>(&stage[l32 * kStageLd + 8 * q + 4 * g]) = v;
                    }
                }
        __builtin_amdgcn_wave_barrier();
        const uint32_t mb = mw + 32 * (b / FN), k = kw + 32 * (b % FN) + (lane & 7) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (lane >> 3) + 8 * i;
            const uint32_t m = mb + row;
            floatx4 v = *reinterpret_cast<const floatx4*>(&stage[row * kStageLd + (lane & 7) * 4]);
            if (m >= a.M || k >= a.K) continue;  // K is a multiple of 32: a tile is inside or past it
            if (part) {
                *reinterpret_cast<floatx4*>(part + static_cast<uint64_t>(m) * a.K + k) = v;
                continue;
            }
            T* p = out + static_cast<uint64_t>(m) * a.lda + k;
            if (a.vec) {
                if (a.mode) {
                    const T4 old = *reinterpret_cast<const T4*>(p);
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] += static_cast<float>(old[x]);
                }
                *reinterpret_cast<T4*>(p) = T4{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
            } else {
#pragma unroll
                for (int x = 0; x < 4; ++x) p[x] = static_cast<T>(a.mode ? static_cast<float>(p[x]) + v[x] : v[x]);
            }
        }
        __builtin_amdgcn_wave_barrier();  // every read of this tile precedes the next tile's writes
    }
}

template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false)));
}

// ANY: dC's rows or its N do not allow 16-byte loads (element-wise ones instead).
template <typename T, int BM, int BN, int WM, int WN, bool ANY>
__global__ __launch_bounds__(WM * WN * 64) void gemm_q8_bwd_kernel(BwdArgs a) {
    constexpr bool kPair = sizeof(T) == 4;
    constexpr int NP = kPair ? 2 : 1;
    constexpr int NT = WM * WN * 64;
    constexpr int NS = 128 / static_cast<int>(sizeof(T));    // n per step: 128 bytes of a dC row
    constexpr int AV = 16 / static_cast<int>(sizeof(T));     // dC elements per 16-byte unit
    constexpr int LDA = NS + 8, LDW = BN + 32;               // LDS row strides in halves
    constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
    constexpr int A_IT = BM * 8 / NT;
    constexpr int KB = BN / 32, W_BLOCKS = NS * KB;          // blocks of a step
    constexpr int PARTS = W_BLOCKS >= NT ? 1 : NT / W_BLOCKS >= 4 ? 4 : NT / W_BLOCKS;  // threads per block
    constexpr int QD = 8 / PARTS;                            // q dwords per thread
    constexpr int W_IT = (W_BLOCKS * PARTS + NT - 1) / NT;
    static_assert(BM * 8 % NT == 0 && W_BLOCKS * PARTS % NT == 0, "staging must divide evenly");
    constexpr int kAPlane = BM * LDA, kWPlane = NS * LDW;
    constexpr int kStage = NP * (kAPlane + kWPlane);
    constexpr int kHalves = 2 * kStage > 2 * NT / 64 * kStageFloats ? 2 * kStage : 2 * NT / 64 * kStageFloats;
    __shared__ __attribute__((aligned(16))) _Float16 smem[kHalves];
    __shared__ int rowexp[kPair ? 2 * BM : 1];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, g = lane >> 5;
    const int wm = wave % WM, wn = wave / WM;

    // tile order: groups of group_m row panels, column-major inside a group, one contiguous chunk per XCD
    const unsigned lin = xcd_swizzle(blockIdx.x, gridDim.x);
    const uint32_t gsz = a.group_m * a.tiles_k;
    const uint32_t grp = lin / gsz, rem = lin % gsz;
    const uint32_t rows_in = min(a.group_m, a.tiles_m - grp * a.group_m);
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((grp * a.group_m + rem % rows_in) * BM);
    const uint32_t k0 = __builtin_amdgcn_readfirstlane((rem / rows_in) * BN);
    const uint32_t s_begin = blockIdx.y * a.steps_per_split;
    const uint32_t s_end = min(a.steps, s_begin + a.steps_per_split);

    const T* const panel = static_cast<const T*>(a.dC) + static_cast<uint64_t>(m0) * a.ldc;
    const uint32_t rows = min(a.M - m0, static_cast<uint32_t>(BM));
    const __amdgpu_buffer_rsrc_t rA = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(panel), 0, static_cast<int>(((rows - 1) * a.ldc + a.N) * sizeof(T)), 0x00020000);
    const __amdgpu_buffer_rsrc_t rW = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(a.W), 0, static_cast<int>((a.N * a.rowbytes + 15u) & ~15u), 0x00020000);

    // dC: unit f of the step is row f / 8, elements AV (f % 8) .. of the step's NS
    uint32_t a_off[A_IT];
#pragma unroll
    for (int i = 0; i < A_IT; ++i) {
        const uint32_t row = (tid + i * NT) >> 3;
        a_off[i] = row < rows ? row * a.ldc * sizeof(T) : kPast;
    }
    // W: thread u handles part u % PARTS of block u / PARTS: row n = block / KB, column block % KB (a wave writes runs of
    // whole rows to LDS; parts a wave apart, four lanes met in a bank: 2048x1280x5120 fp16 51.0 us, now 45.8). 64 (32) rows
    // of 34 * K / 32 bytes are a multiple of 4 bytes, so a thread's place in its dwords is the same every step.
    uint32_t w_off[W_IT], w_n[W_IT], w_sel[W_IT], w_d[W_IT];
#pragma unroll
    for (int i = 0; i < W_IT; ++i) {
        const uint32_t u = tid + i * NT, blk = u / PARTS, pt = u % PARTS;
        w_n[i] = blk / KB;
        const uint32_t byte = w_n[i] * a.rowbytes + min(k0 / 32 + blk % KB, a.K / 32 - 1) * 34;
        const uint32_t q = byte + 2 + pt * (QD * 4);
        w_d[i] = byte;
        w_off[i] = q & ~3u;
        w_sel[i] = (q & 2u) ? 0x05040302u : 0x03020100u;  // bytes 2..5 or 0..3 of (x[j+1]:x[j])
    }

    typedef T Unit __attribute__((ext_vector_type(AV)));
    Unit areg[2][A_IT];
    uint32_t wq[2][W_IT][QD + 1], wd[2][W_IT];
    auto past = [](bool in) {
        // (opaque: a select of the offset becomes a branch around the loads, and a load under a branch makes every later
        // wait retire the loads in flight)
        uint32_t top = in ? 0u : kPast;
        asm volatile("" : "+v"(top));
        return top;
    };
    auto load_step = [&](uint32_t step, auto RS) {
        constexpr int rs = decltype(RS)::value;
        const uint32_t n0 = __builtin_amdgcn_readfirstlane(step * NS);
#pragma unroll
        for (int i = 0; i < A_IT; ++i) {
            const uint32_t n = n0 + ((tid + i * NT) & 7) * AV;
            if constexpr (ANY) {
                const uint32_t row = (tid + i * NT) >> 3;
#pragma unroll
                for (int e = 0; e < AV; ++e)
                    areg[rs][i][e] = row < rows && n + e < a.N ? panel[static_cast<uint64_t>(row) * a.ldc + n + e] : static_cast<T>(0.0f);
            } else {
                // units past N read as zeros: offsets with the top bit set are out of range
                const uint32_t off = (a_off[i] + ((tid + i * NT) & 7) * 16u) | past(n < a.N);
                areg[rs][i] = __builtin_bit_cast(Unit, __builtin_amdgcn_raw_buffer_load_b128(rA, off, n0 * sizeof(T), 0));
            }
        }
        const uint32_t soff = n0 * a.rowbytes;
#pragma unroll
        for (int i = 0; i < W_IT; ++i) {
            const uint32_t out = past(n0 + w_n[i] < a.N);  // rows past N read as zeros
            const uint32_t o = w_off[i] | out;
            if constexpr (QD == 8) {
                const auto x0 = __builtin_amdgcn_raw_buffer_load_b128(rW, o, soff, 0);
                const auto x1 = __builtin_amdgcn_raw_buffer_load_b128(rW, o + 16, soff, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    wq[rs][i][e] = x0[e];
                    wq[rs][i][QD / 2 + e] = x1[e];
                }
            } else if constexpr (QD == 4) {
                const auto x0 = __builtin_amdgcn_raw_buffer_load_b128(rW, o, soff, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e) wq[rs][i][e] = x0[e];
            } else {
                const auto x0 = __builtin_amdgcn_raw_buffer_load_b64(rW, o, soff, 0);
                wq[rs][i][0] = x0[0];
                wq[rs][i][1] = x0[1];
            }
            // (the last block's window may end past W: the whole offset is in voffset, where the range check counts it)
            wq[rs][i][QD] = __builtin_amdgcn_raw_buffer_load_b32(rW, (w_off[i] + soff + 4 * QD) | out, 0, 0);
            wd[rs][i] = __builtin_amdgcn_raw_buffer_load_b16(rW, w_d[i] | out, soff, 0);
        }
    };

    float neg1 = -1.0f;  // (residual2)
    asm volatile("" : "+v"(neg1));
    int re[A_IT];  // fp32: the exponents of this thread's rows (the same in the eight threads of a row)
#pragma unroll
    for (int i = 0; i < A_IT; ++i) re[i] = 127;
    auto store_step = [&](auto RS, auto ST) {
        constexpr int rs = decltype(RS)::value, st = decltype(ST)::value;
        _Float16* const As = smem + st * kStage;
        _Float16* const Ws = As + NP * kAPlane;
#pragma unroll
        for (int i = 0; i < A_IT; ++i) {
            const int f = tid + i * NT;
            _Float16* dst = As + (f >> 3) * LDA + (f & 7) * AV;
            if constexpr (kPair) {
                const floatx4 x = areg[rs][i];
                float mx = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
                mx = dpp_max<0xb1>(mx);   // quad_perm [1, 0, 3, 2]
                mx = dpp_max<0x4e>(mx);   // quad_perm [2, 3, 0, 1]
                mx = dpp_max<0x141>(mx);  // row_half_mirror: the row's eight lanes
                const int low = min(re[i], kRowExp + 127 - static_cast<int>(__float_as_uint(mx) >> 23));
                re[i] = ldexpf(mx, re[i]) > kRowMax ? low : re[i];
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = ldexpf(x[e], re[i]);
                const half2 h0 = pack2(v[0], v[1]), h1 = pack2(v[2], v[3]);
                const half2 l0 = residual2(h0, v[0], v[1], neg1), l1 = residual2(h1, v[2], v[3], neg1);
                *reinterpret_cast<half4*>(dst) = half4{h0[0], h0[1], h1[0], h1[1]};
                *reinterpret_cast<half4*>(dst + kAPlane) = half4{l0[0], l0[1], l1[0], l1[1]};
                if ((f & 7) == 0) rowexp[st * BM + (f >> 3)] = re[i];
            } else {
                *reinterpret_cast<half8*>(dst) = __builtin_bit_cast(half8, areg[rs][i]);
            }
        }
#pragma unroll
        for (int i = 0; i < W_IT; ++i) {
            const int u = tid + i * NT, blk = u / PARTS, pt = u % PARTS;
            _Float16* dst = Ws + (blk / KB) * LDW + (blk % KB) * 32 + pt * (QD * 4);
            const _Float16 d = __builtin_bit_cast(_Float16, static_cast<uint16_t>(wd[rs][i]));
            uint32_t q[QD];
#pragma unroll
            for (int j = 0; j < QD; ++j) q[j] = __builtin_amdgcn_perm(wq[rs][i][j + 1], wq[rs][i][j], w_sel[i]);
#pragma unroll
            for (int j = 0; j < QD; j += 2) {
                if constexpr (kPair) {
                    // 64 d q is exact in fp32 (19 bits), and so is each step to it
                    const float s = static_cast<float>(d) * (1 << kWExp), s128 = -128.0f * s;
                    half8 hi, lo;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        float w[2];
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t byte = ((q[j + e / 4] ^ 0x80808080u) >> (8 * (e % 4 + x))) & 0xffu;
                            w[x] = __builtin_fmaf(static_cast<float>(byte), s, s128);
                        }
                        const half2 h = pack2(w[0], w[1]), l = residual2(h, w[0], w[1], neg1);
                        hi[e] = h[0];
                        hi[e + 1] = h[1];
                        lo[e] = l[0];
                        lo[e + 1] = l[1];
                    }
                    *reinterpret_cast<half8*>(dst + 4 * j) = hi;
                    *reinterpret_cast<half8*>(dst + 4 * j + kWPlane) = lo;
                } else {
                    *reinterpret_cast<half8*>(dst + 4 * j) = dequant8_f16(q[j], q[j + 1], d);
                }
            }
        }
    };

    floatx16 acc[FM][FN];
    int ce[FM];  // fp32: the exponents that the sums of this lane's rows carry
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        ce[i] = 127;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    }
    // W^T fragment: lane (k = l32, g) takes n = 16 s + 8 g + 0..7 as two transposing reads of four rows; lane i of a
    // 16-lane group supplies row i / 4, columns 4 (i % 4) .. + 3 of the group's 16
    const int w_rd = (8 * g + ((lane >> 2) & 3)) * LDW + wn * TN + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int a_rd = (wm * TM + l32) * LDA + 8 * g;
    auto compute = [&](auto ST) {
        constexpr int st = decltype(ST)::value;
        const _Float16* const As = smem + st * kStage;
        const _Float16* const Ws = As + NP * kAPlane;
        if constexpr (kPair) {
            int ne[FM];
            bool moved = false;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                ne[i] = rowexp[st * BM + wm * TM + 32 * i + l32];
                moved |= ne[i] != ce[i];
            }
            if (__any(moved)) {
#pragma unroll
                for (int i = 0; i < FM; ++i) {
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[i][j][r] = ldexpf(acc[i][j][r], ne[i] - ce[i]);
                    ce[i] = ne[i];
                }
            }
        }
#pragma unroll
        for (int s = 0; s < NS / 16; ++s) {
            half8 af[NP][FM], wf[NP][FN];
#pragma unroll
            for (int pl = 0; pl < NP; ++pl) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    af[pl][i] = *reinterpret_cast<const half8*>(&As[pl * kAPlane + a_rd + 32 * i * LDA + 16 * s]);
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    const _Float16* p = &Ws[pl * kWPlane + w_rd + 16 * s * LDW + 32 * j];
                    const half4 x = lds_read_tr16(p), y = lds_read_tr16(p + 4 * LDW);
                    wf[pl][j] = half8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
                }
            }
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    if constexpr (kPair) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[NP - 1][j], af[0][i], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[0][j], af[NP - 1][i], acc[i][j], 0, 0, 0);
                    }
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[0][j], af[0][i], acc[i][j], 0, 0, 0);
                }
        }
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;

    // The step's MFMAs with the next fragment reads and a share of the conversions and LDS writes between them. Only the
    // 256-row tiles have the CU to themselves; of the others two or three workgroups fill each other's gaps. us with and
    // without the order, fp16: 256x128 1976x10240x1280 76.6 / 79.7, 8192x1920x640 37.9 / 41.2, 988x1280x5120 26.7 / 28.9;
    // 128x128 2048x1280x5120 54.8 / 51.8; 64x64 576x1280x1280 11.7 / 10.8. fp32: 256x128 1976x10240x1280 212 / 214.
    constexpr bool kMix = !ANY && BM == 256;
    constexpr int kMfma = FM * FN * (NS / 16) * (kPair ? 3 : 1);
    constexpr int kRead0 = NP * (FM + 2 * FN), kReads = kRead0 * (NS / 16);
    constexpr int kWrites = NP * (A_IT + W_IT * QD / 2);
    constexpr int kValu = kPair ? A_IT * 30 + W_IT * QD * 17 : W_IT * QD * 8;
    // Step j computes from LDS stage j & 1 while the loads of step j + 2 are in flight; those of step j + 1 are then
    // stored into the other stage. Loads past the last step re-read it and are not used.
    const uint32_t n_steps = s_end - s_begin, last = s_end - 1;
    load_step(s_begin, S0{});
    store_step(S0{}, S0{});
    load_step(min(s_begin + 1, last), S1{});
    __syncthreads();
    uint32_t j = 0;
    for (; j + 2 <= n_steps; j += 2) {
        load_step(min(s_begin + j + 2, last), S0{});
        __builtin_amdgcn_sched_barrier(0);
        compute(S0{});
        store_step(S1{}, S1{});
        if constexpr (kMix) interleave_step<kMfma, kRead0, kReads - kRead0, kValu, kWrites>();
        __syncthreads();
        load_step(min(s_begin + j + 3, last), S1{});
        __builtin_amdgcn_sched_barrier(0);
        compute(S1{});
        // an odd last step is the one just stored; an even one needs nothing more, and storing the last step again
        // would not change the sums, but would count its rows' exponents twice: the same exponents
        store_step(S0{}, S0{});
        if constexpr (kMix) interleave_step<kMfma, kRead0, kReads - kRead0, kValu, kWrites>();
        __syncthreads();
    }
    if (j < n_steps) compute(S0{});
    __syncthreads();  // every wave is done with the operand tiles before LDS is reused
    store_tiles<T, FM, FN>(a, reinterpret_cast<float*>(smem) + wave * kStageFloats, m0 + wm * TM, k0 + wn * TN, acc, ce, lane,
                           a.part ? a.part + static_cast<uint64_t>(blockIdx.y) * a.M * a.K : nullptr);
}

// The N parts' sums in order: dA = P0 + P1 + ... (+ dA).
template <typename T>
__global__ __launch_bounds__(256) void gemm_q8_bwd_sum_kernel(const float* P, uint32_t splits, T* dA, uint32_t M, uint32_t K,
                                                              uint32_t lda, uint32_t mode, uint32_t vec) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const uint64_t plane = static_cast<uint64_t>(M) * K, total = plane / 4;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < total; i += static_cast<uint64_t>(gridDim.x) * 256) {
        const float* p = P + 4 * i;
        floatx4 v = *reinterpret_cast<const floatx4*>(p);
        uint32_t s = 1;
        for (; s + 3 < splits; s += 4) {
            const floatx4 x0 = *reinterpret_cast<const floatx4*>(p + s * plane), x1 = *reinterpret_cast<const floatx4*>(p + (s + 1) * plane),
                          x2 = *reinterpret_cast<const floatx4*>(p + (s + 2) * plane), x3 = *reinterpret_cast<const floatx4*>(p + (s + 3) * plane);
            v += x0;
            v += x1;
            v += x2;
            v += x3;
        }
        for (; s < splits; ++s) v += *reinterpret_cast<const floatx4*>(p + s * plane);
        const uint32_t m = static_cast<uint32_t>(4 * i / K), k = static_cast<uint32_t>(4 * i % K);
        T* o = dA + static_cast<uint64_t>(m) * lda + k;
        T4 old = {0, 0, 0, 0};
        if (mode) {
            if (vec) old = *reinterpret_cast<const T4*>(o);
            else
#pragma unroll
                for (int x = 0; x < 4; ++x) old[x] = o[x];
        }
        T4 r;
#pragma unroll
        for (int x = 0; x < 4; ++x) r[x] = static_cast<T>(mode ? v[x] + static_cast<float>(old[x]) : v[x]);
        if (vec) *reinterpret_cast<T4*>(o) = r;
        else
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] = r[x];
    }
}

// N == 0: a sum over nothing.
template <typename T>
__global__ __launch_bounds__(256) void gemm_q8_bwd_zero_kernel(T* dA, uint32_t M, uint32_t K, uint32_t lda) {
    const uint64_t total = static_cast<uint64_t>(M) * K;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < total; i += static_cast<uint64_t>(gridDim.x) * 256)
        dA[i / K * lda + i % K] = static_cast<T>(0.0f);
}

constexpr uint32_t kCUs = 256;

enum BuildId { k256x128 = 0, k128x128 = 1, k64x64 = 2, k256x256 = 3, kFew = 4 };
static_assert(k256x256 + 1 == kGemmBwdBuilds, "mi_tuning_set bounds gemm_bwd_cfg by kGemmBwdBuilds");

struct Plan {
    int build;
    uint32_t splits;
};

uint32_t n_step(bool f32) { return f32 ? 32 : 64; }

// The parts that whole steps make of N when `splits` are asked for: none empty.
uint32_t launched_splits(uint32_t N, bool f32, uint32_t splits) {
    const uint32_t steps = ceil_div(N, n_step(f32));
    return ceil_div(steps, ceil_div(steps, splits));
}

// Few rows: dA = dC . deq(W) for up to MR rows in one launch, in fp32 for either type (w = d * q exact). What bounds it is
// the latency of a launch and of its loads: a workgroup takes one 32-wide block of columns and all of N, a wave's lanes 8
// rows n by the 8 dwords of a block, the 16 waves 128 rows at a time, kDeep times that in flight. The lanes of a column are
// added by shuffles, the waves through LDS, always in the same order. 2x1280x1280 fp32: 6.3 us, of which a launch is 3.9
// (64x64 tiles in 12 parts and their sum: 8.3).
constexpr uint32_t kFewRows = 4;
constexpr int kFewWaves = 16;
constexpr uint32_t kFewMaxK = 1u << 27;  // K / 32 workgroups of 1024 threads: a launch counts them in 32 bits

template <typename T, int MR>
__global__ __launch_bounds__(kFewWaves * 64) void gemm_q8_bwd_few_kernel(BwdArgs a) {
    constexpr int kDeep = MR <= 2 ? 8 : 4;
    constexpr uint32_t kRows = kFewWaves * 8;
    __shared__ float sums[kFewWaves][MR][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 7;
    const uint8_t* const col = a.W + static_cast<uint64_t>(blockIdx.x) * 34;
    const T* const dC = static_cast<const T*>(a.dC);
    float acc[MR][4];
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][e] = 0.0f;
    for (uint32_t n0 = 0; n0 < a.N; n0 += kRows * kDeep) {
        uint32_t q[kDeep];
        _Float16 d[kDeep];
        T x[kDeep][MR];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const uint32_t n = n0 + u * kRows + wave * 8 + (lane >> 3), at = min(n, a.N - 1);
            const uint8_t* p = col + static_cast<uint64_t>(at) * a.rowbytes;
            d[u] = *reinterpret_cast<const _Float16*>(p);
            __builtin_memcpy(&q[u], p + 2 + 4 * c, 4);  // (2-byte aligned)
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const T v = dC[static_cast<uint64_t>(min(static_cast<uint32_t>(m), a.M - 1)) * a.ldc + at];
                x[u][m] = n < a.N ? v : static_cast<T>(0.0f);
            }
        }
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const float s = static_cast<float>(d[u]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = s * static_cast<float>(static_cast<int8_t>(q[u] >> (8 * e)));
#pragma unroll
                for (int m = 0; m < MR; ++m) acc[m][e] = __builtin_fmaf(static_cast<float>(x[u][m]), w, acc[m][e]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int o = 8; o < 64; o <<= 1) acc[m][e] += __shfl_xor(acc[m][e], o);
        if (lane < 8) *reinterpret_cast<floatx4*>(&sums[wave][m][4 * c]) = floatx4{acc[m][0], acc[m][1], acc[m][2], acc[m][3]};
    }
    __syncthreads();
    const uint32_t m = tid / 32, k = tid % 32;
    if (m >= a.M) return;  // (MR of the 32 rows that the threads cover have sums)
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) v += sums[w][m][k];
    T* out = static_cast<T*>(a.dA) + static_cast<uint64_t>(m) * a.lda + blockIdx.x * 32 + k;
    *out = static_cast<T>(a.mode ? static_cast<float>(*out) + v : v);
}

// What a build costs, us: `base` (launch, first loads, last stores) and a step of its workgroups with 1, 2 or 3 of them on
// a CU (LDS allows no more of the larger tiles). Fitted to a sweep of every build and number of parts over the layers of
// 512- to 1024-pixel images (MI355X, operands of full entropy, calls back to back); examples in us, build:parts measured
// (256x128, 128x128, 64x64, 256x256): fp16 2048x1280x5120 48.0 / 45.9 / 72.7 / 46.5, 8192x1920x640 33.1 / 40.0 / 51.3 /
// 46.0, 576x1280x1280 16.9 / 14.4 / 9.7, 1976x10240x1280 in 3 parts 71.8 / 83.1, in 5 parts 256x256 78.6; fp32
// 1152x1280x1280 29.0 in 5 parts / 30.3 in 2 / 34.9 / 32.9 in 8, 2048x1280x5120 142 / 130 / - / 105, 1976x10240x1280 203 in
// 3 parts / 236 / - / 184 in 5. fp32's three products per pair of fragments gain from 256x256 tiles, fp16's one does not: it
// has no such build.
struct Cost {
    uint32_t bm, bk, per_cu;
    double base, step[3];
};
constexpr Cost kCost[2][kGemmBwdBuilds] = {
    {{256, 128, 1, 6.0, {1.00}}, {128, 128, 2, 4.5, {0.68, 1.25}}, {64, 64, 3, 2.8, {0.35, 0.62, 0.90}}, {}},
    {{256, 128, 1, 7.0, {1.60}}, {128, 128, 1, 5.0, {1.08}}, {64, 64, 3, 3.0, {0.62, 0.87, 1.18}}, {256, 256, 1, 9.0, {2.41}}}};

double cost_us(const Cost& c, uint32_t M, uint32_t K, uint32_t steps, uint32_t splits) {
    const uint64_t wgs = static_cast<uint64_t>(ceil_div(M, c.bm)) * ceil_div(K, c.bk) * splits;
    const uint64_t rounds = wgs / (kCUs * c.per_cu);
    const uint32_t last = static_cast<uint32_t>(wgs % (kCUs * c.per_cu));
    double us = static_cast<double>(rounds) * c.step[c.per_cu - 1];
    if (last) us += c.step[ceil_div(last, kCUs) - 1];
    us = c.base + us * ceil_div(steps, splits);
    // the parts' planes are written and read back, by a launch of its own
    if (splits > 1) us += 3.0 + static_cast<double>(splits) * M * K * 8 / 5.5e6;
    return us;
}

Plan choose(uint32_t M, uint32_t N, uint32_t K, bool f32, bool allow_split) {
    const int forced = tuning().gemm_bwd_cfg.load(std::memory_order_relaxed);
    if (forced >= 0) {
        const uint32_t s = static_cast<uint32_t>(tuning().gemm_bwd_splits.load(std::memory_order_relaxed));
        return Plan{forced, allow_split ? launched_splits(N, f32, s) : 1u};
    }
    Plan best{k64x64, 1};
    double best_us = 1e300;
    // The kernel for few rows: one launch and no parts, but all of N in one workgroup, at a quarter of the loads in flight
    // that the parts have. us against the best build and parts, fp32 / fp16: 1x1280x1280 5.7 : 8.3 / 5.6 : 7.6, 2x640x1280
    // 4.7 : 7.8 / 4.7 : 6.0, 4x1280x1280 6.9 : 8.3 / 7.0 : 7.6, 2x5120x640 12.7 : 11.1 / 12.8 : 8.0; with eight rows
    // 8x1280x1280 9.8 : 8.6 / 10.2 : 7.5.
    if (M <= kFewRows && K < kFewMaxK) {
        best = Plan{kFew, 1};
        best_us = 4.0 + N * (0.0013 + 0.00025 * M);
    }
    for (int b = 0; b < (f32 ? kGemmBwdBuilds : kGemmBwdBuilds - 1); ++b)
        for (uint32_t splits : {1u, 2u, 3u, 4u, 5u, 8u, 12u, 16u}) {
            if (splits > 1 && (!allow_split || launched_splits(N, f32, splits) != splits)) continue;
            const double us = cost_us(kCost[f32][b], M, K, ceil_div(N, n_step(f32)), splits);
            if (us < best_us) {
                best_us = us;
                best = Plan{b, splits};
            }
        }
    return best;
}

uint64_t part_bytes(uint32_t M, uint32_t K, uint32_t splits) { return splits > 1 ? static_cast<uint64_t>(splits) * M * K * 4 : 0; }

template <typename T, int BM, int BN, int WM, int WN, bool ANY>
void launch_build(BwdArgs a, uint32_t splits, hipStream_t s) {
    a.tiles_m = ceil_div(a.M, BM);
    a.tiles_k = ceil_div(a.K, BN);
    a.group_m = std::min(a.tiles_m, 4u);
    a.steps = ceil_div(a.N, 128 / sizeof(T));
    a.steps_per_split = ceil_div(a.steps, splits);
    gemm_q8_bwd_kernel<T, BM, BN, WM, WN, ANY><<<dim3(a.tiles_m * a.tiles_k, splits), WM * WN * 64, 0, s>>>(a);
}

template <typename T>
void launch_few(const BwdArgs& a, hipStream_t s) {
    const unsigned grid = a.K / 32, block = kFewWaves * 64;
    if (a.M == 1) gemm_q8_bwd_few_kernel<T, 1><<<grid, block, 0, s>>>(a);
    else if (a.M == 2) gemm_q8_bwd_few_kernel<T, 2><<<grid, block, 0, s>>>(a);
    else gemm_q8_bwd_few_kernel<T, kFewRows><<<grid, block, 0, s>>>(a);
}

template <typename T>
void launch(const BwdArgs& a, const Plan& p, bool any, hipStream_t s) {
    if (p.build == kFew) launch_few<T>(a, s);
    else if (any) launch_build<T, 64, 64, 2, 2, true>(a, p.splits, s);
    else if (sizeof(T) == 4 && p.build == k256x256) launch_build<float, 256, 256, 4, 2, false>(a, p.splits, s);
    else if (p.build == k256x128 || p.build == k256x256) launch_build<T, 256, 128, 4, 2, false>(a, p.splits, s);
    else if (p.build == k128x128) launch_build<T, 128, 128, 4, 2, false>(a, p.splits, s);
    else launch_build<T, 64, 64, 2, 2, false>(a, p.splits, s);
    if (!a.part) return;
    const uint64_t units = static_cast<uint64_t>(a.M) * a.K / 4;
    gemm_q8_bwd_sum_kernel<T><<<static_cast<unsigned>(std::min<uint64_t>(ceil_div(units, 256), 2048)), 256, 0, s>>>(
        a.part, p.splits, static_cast<T*>(a.dA), a.M, a.K, a.lda, a.mode, a.vec);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" uint64_t mi_gemm_nt_q8_0_bwd_ws_bytes(uint32_t M, uint32_t N, uint32_t K, int dtype) {
    if (M == 0 || N == 0 || K == 0 || K % 32 || (dtype != MI_F32 && dtype != MI_F16)) return 0;
    return part_bytes(M, K, choose(M, N, K, dtype == MI_F32, true).splits);
}

extern "C" int mi_gemm_nt_q8_0_bwd(const void* dC, const void* W, void* dA, int dtype, uint32_t M, uint32_t N, uint32_t K,
                                   uint32_t mode, uint32_t ldc, uint32_t lda, void* workspace, uint64_t workspace_bytes,
                                   void* stream) {
    const char* fn = "mi_gemm_nt_q8_0_bwd";
    if (M == 0 || K == 0) return MI_OK;
    if (dtype != MI_F32 && dtype != MI_F16) return fail(MI_ERR_INVALID_ARG, "%s: dtype %d", fn, dtype);
    if (!dA || (N && (!dC || !W))) return fail(MI_ERR_INVALID_ARG, "%s: null pointer", fn);
    if (mode > 1) return fail(MI_ERR_INVALID_ARG, "%s: mode %u (0 = store, 1 = accumulate)", fn, mode);
    if (K % 32) return fail(MI_ERR_UNSUPPORTED, "%s: K=%u is not a multiple of 32 (Q8_0 block)", fn, K);
    if (ldc == 0) ldc = N;
    if (lda == 0) lda = K;
    if (ldc < N || lda < K) return fail(MI_ERR_INVALID_ARG, "%s: ldc %u < N %u or lda %u < K %u", fn, ldc, N, lda, K);
    const uint64_t e = dtype == MI_F16 ? 2 : 4;
    if (!aligned(W, 16)) return fail(MI_ERR_ALIGNMENT, "%s: W must be 16-byte aligned", fn);
    if (!aligned(dC, e) || !aligned(dA, e)) return fail(MI_ERR_ALIGNMENT, "%s: dC and dA must be aligned to their element size", fn);
    const uint64_t wbytes = static_cast<uint64_t>(N) * (K / 32) * 34;
    // 32-bit buffer offsets, the upper half of which reads as zeros
    if (wbytes + 16 >= kPast) return fail(MI_ERR_UNSUPPORTED, "%s: weight >= 2 GiB", fn);
    if (static_cast<uint64_t>(ldc) * e * 256 >= kPast) return fail(MI_ERR_UNSUPPORTED, "%s: ldc=%u too large", fn, ldc);
    if (static_cast<uint64_t>(ceil_div(M, 64)) * ceil_div(K, 64) >= (1u << 23)) return fail(MI_ERR_UNSUPPORTED, "%s: M=%u K=%u too large", fn, M, K);
    const uint64_t cbytes = N ? (static_cast<uint64_t>(M - 1) * ldc + N) * e : 0, abytes = (static_cast<uint64_t>(M - 1) * lda + K) * e;
    if (overlaps(dA, abytes, dC, cbytes) || overlaps(dA, abytes, W, wbytes))
        return fail(MI_ERR_ALIASING, "%s: dA overlaps an input", fn);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (N == 0) {
        if (mode == 1) return MI_OK;
        const unsigned grid = static_cast<unsigned>(std::min<uint64_t>(ceil_div(static_cast<uint64_t>(M) * K, 256), 2048));
        if (dtype == MI_F16) gemm_q8_bwd_zero_kernel<_Float16><<<grid, 256, 0, s>>>(static_cast<_Float16*>(dA), M, K, lda);
        else gemm_q8_bwd_zero_kernel<float><<<grid, 256, 0, s>>>(static_cast<float*>(dA), M, K, lda);
        return check_launch(fn);
    }
    Plan p = choose(M, N, K, dtype == MI_F32, workspace != nullptr);
    if (part_bytes(M, K, p.splits) > workspace_bytes) p = choose(M, N, K, dtype == MI_F32, false);
    const uint64_t need = part_bytes(M, K, p.splits);
    if (need) {
        if (!aligned(workspace, 16)) return fail(MI_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
        if (overlaps(workspace, need, dC, cbytes) || overlaps(workspace, need, W, wbytes) || overlaps(workspace, need, dA, abytes))
            return fail(MI_ERR_ALIASING, "%s: workspace overlaps an operand", fn);
    }
    BwdArgs a{};
    a.dC = dC;
    a.W = static_cast<const uint8_t*>(W);
    a.dA = dA;
    a.part = need ? static_cast<float*>(workspace) : nullptr;
    a.M = M;
    a.N = N;
    a.K = K;
    a.ldc = ldc;
    a.lda = lda;
    a.mode = mode;
    a.rowbytes = (K / 32) * 34;
    a.vec = aligned(dA, 4 * e) && lda % 4 == 0 ? 1u : 0u;
    const bool any = !aligned(dC, 16) || (ldc * e) % 16 || (N * e) % 16;
    if (dtype == MI_F16) launch<_Float16>(a, p, any, s);
    else launch<float>(a, p, any, s);
    return check_launch(fn);
}

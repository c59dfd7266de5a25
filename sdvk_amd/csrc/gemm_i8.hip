// gemm_i8.hip -- linears in 8-bit integers for gfx950: the token quantiser and the product
//   C[m,n] (=|+=) sa[m] sw[n] sum_k A[m,k] W[n,k] (+ bias[n])
// of codes with a scale for each row of A (a token) and of W (a channel).
//
// The sum is exact in 32-bit integers (K <= 131071: |code| <= 128), so every plan gives the same bits; the epilogue is one
// conversion, one product and one fma in fp32: fma(float(sum) * sa, sw, bias).
#include "common.hpp"
#include "quant.hpp"

#include <algorithm>
#include <type_traits>

namespace mi {
namespace {

constexpr uint32_t kMaxGrid = 1u << 20;  // workgroups of a launch that strides over its units
constexpr uint32_t kMaxFastCols = 8192;  // columns of a row that stays in registers
constexpr uint32_t kMaxSize = 1u << 31;  // rows and columns of a product, rows of the quantiser ...
constexpr uint32_t kMaxCols = 1u << 30;  // ... and its columns: counted in 32 bits with a tile or a wave past the end
constexpr uint32_t kMaxK = 131071;       // 2^31 / 2^14
constexpr uint64_t kMaxLd = 1u << 22;    // row strides that a tile's 320 rows address in 31 bits

struct I8Args {
    const int8_t *A, *W;
    const float *sa, *sw, *bias;
    void* C;
    uint32_t M, N, K, mode;
    uint64_t lda, ldw, ldc;
    uint32_t tiles_m, tiles_n, group_m;
    uint32_t wide;  // C's rows take 16-byte stores
};

constexpr uint32_t kPast = 0x80000000u;  // a buffer offset past every record: the load returns zeros
constexpr int kAll = 0x7fffffff;         // bytes of a resource that kPast alone is past

// C from a sum: mode 0 stores, mode 1 adds, mode 2 adds with the bias (NULL for mode 1). An fp32 number also where fp16 is stored: as one
// instruction with that rounding, which the compiler would make of some results and not of others, one in 10^5 had other bits.
template <typename TC>
__device__ __forceinline__ float result(int acc, float sa, float sw, float bias) {
    float r = __builtin_fmaf(static_cast<float>(acc) * sa, sw, bias);
    if constexpr (sizeof(TC) == 2) asm volatile("" : "+v"(r));
    return r;
}
template <typename TC>
__device__ __forceinline__ void store_one(const I8Args& a, uint32_t m, uint32_t n, int acc, float sa) {
    float v = result<TC>(acc, sa, a.sw[n], a.bias ? a.bias[n] : 0.0f);
    TC* p = static_cast<TC*>(a.C) + m * a.ldc + n;
    if (a.mode) v += static_cast<float>(*p);
    *p = static_cast<TC>(v);
}

// The scales and biases of V columns.
template <int V>
struct Columns {
    float sw[V], bias[V];
};
// V neighbouring results of row m: whole runs (16-byte aligned, in range), or element by element.
template <typename TC, int V>
__device__ __forceinline__ void store_run(const I8Args& a, uint32_t m, uint32_t n, const int (&acc)[V], float sa, const Columns<V>& c, bool whole) {
    typedef TC Run __attribute__((ext_vector_type(V)));
    TC* p = static_cast<TC*>(a.C) + m * a.ldc + n;
    if (whole) {
        Run r;
        if (a.mode) {
            const Run old = *reinterpret_cast<const Run*>(p);
#pragma unroll
            for (int e = 0; e < V; ++e) r[e] = static_cast<TC>(result<TC>(acc[e], sa, c.sw[e], c.bias[e]) + static_cast<float>(old[e]));
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) r[e] = static_cast<TC>(result<TC>(acc[e], sa, c.sw[e], c.bias[e]));
        }
        *reinterpret_cast<Run*>(p) = r;
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (n + e < a.N) {
            float v = result<TC>(acc[e], sa, c.sw[e], c.bias[e]);
            if (a.mode) v += static_cast<float>(p[e]);
            p[e] = static_cast<TC>(v);
        }
}

// Any K, any alignment: a 64 x 64 tile in steps of 32 codes, 4 x 4 outputs a thread, four products an instruction; bound by its
// byte loads: 2048x10240x1280 489 us, tiles 32; 154x1280x2048 154, waves that split K 5.
template <typename TC>
__global__ __launch_bounds__(256) void gemm_i8_any_kernel(I8Args a) {
    __shared__ __attribute__((aligned(4))) int8_t at[64][36], wt[64][36];
    const uint32_t tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const uint32_t tiles_n = (a.N + 63) / 64;
    const uint64_t tiles = static_cast<uint64_t>((a.M + 63) / 64) * tiles_n;  // (M, N <= 2^31)
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t m0 = static_cast<uint32_t>(t / tiles_n) * 64, n0 = static_cast<uint32_t>(t % tiles_n) * 64;
        int acc[4][4] = {};
        for (uint32_t k0 = 0; k0 < a.K; k0 += 32) {
            for (uint32_t i = tid; i < 64 * 32; i += 256) {
                const uint32_t r = i >> 5, k = i & 31;
                const bool in = k0 + k < a.K;
                at[r][k] = in && m0 + r < a.M ? a.A[(m0 + r) * a.lda + k0 + k] : static_cast<int8_t>(0);
                wt[r][k] = in && n0 + r < a.N ? a.W[(n0 + r) * a.ldw + k0 + k] : static_cast<int8_t>(0);
            }
            __syncthreads();
            for (int k = 0; k < 32; k += 4) {
                int x[4], w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = *reinterpret_cast<const int*>(&at[ty + 16 * i][k]);
                    w[i] = *reinterpret_cast<const int*>(&wt[tx + 16 * i][k]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_sdot4(x[i], w[j], acc[i][j], false);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = m0 + ty + 16 * i;
            if (m >= a.M) continue;
            const float sa = a.sa[m];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t n = n0 + tx + 16 * j;
                if (n < a.N) store_one<TC>(a, m, n, acc[i][j], sa);
            }
        }
    }
}

// ---- tiles ---------------------------------------------------------------------------
//
// A workgroup computes a BM x BN tile of C in steps of 128 codes. A step's rows go from memory straight into LDS
// (buffer loads with an LDS destination: 8 rows of 128 bytes an instruction), a ring of NS stages deep. An LDS row is 128 bytes, its
// eight 16-byte slots in the order slot ^ (row / 2) % 8, so that the 16 rows that a fragment read takes at a time lie in
// different banks; the loads' lanes permute their addresses accordingly (the 128 bytes of a row stay one segment).
// The product is transposed (W is the MFMA's A operand): a lane holds one row m of C and runs of four columns.
// Codes past K and rows past M or N are zeros: their lanes' offsets are out of the resources' range.
// What bounds it: a CU is fed about 75 bytes a ns (128 x 128 and four stages 0.42 us a step), so tiles as large as the registers allow where
// there are enough of them: 256 x 320 reads 72 KB for 10.5 M products, 128 x 128 32 KB for 2.1 M. 2048x10240x1280 fp16 (256 x 320, a tile a
// CU, 1670 TOP/s over the call) takes 15.2 us with K = 128, 31.7 with 1280, 51.2 with 2560: a step is 1.95 us in a long run (its MFMAs at
// 80% of their rate at the 1.67 GHz that the card then holds), and 11 to 12 us are the launch, the first loads and 42 MB of C that all CUs
// store at once, with no product beside them.
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ uint32_t swz(uint32_t row) { return (row >> 1) & 7u; }
__device__ __forceinline__ void wait_lds() {  // lgkmcnt(0)
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);  // no access that follows moves before the wait
}
// Waits until at most N of the wave's loads are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "vmcnt has six bits");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
// A barrier that waits for nothing else: __syncthreads() would wait for every load on its way. A wave has the fragments of the step
// before when it gets here (its products have taken them).
__device__ __forceinline__ void barrier() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_sched_barrier(0);
    wait_lds();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// 16 bytes a lane from base + off + at (zeros for off = kPast) to LDS: lane l's to dst + 16 l. The range check subtracts `at` from the
// resource's bytes in 32 bits: those are more than any `at`, so that the difference cannot wrap.
__device__ __forceinline__ void load_lds(const int8_t* base, int8_t* dst, uint32_t off, int at) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base), 0, kAll, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(dst), 16, off, at, 0, 0);
}

// Rows of one operand: IT load instructions a wave brings into LDS (rows 8 (IT wave + i) .. + 7).
template <int IT>
struct Rows {
    const int8_t* base;
    uint32_t off[IT], col[2], K;  // col: the lane's place in 128 codes, by the parity of its eight rows
    int at;                       // bytes into a stage
    // rows r0 .. r0 + count - 1 of X at stride ld; further ones are zeros
    __device__ __forceinline__ Rows(const int8_t* X, uint64_t ld, uint32_t r0, uint32_t count, uint32_t K_, int wave, int lane) : K(K_) {
        base = X + r0 * ld;
        at = wave * IT * 1024;
#pragma unroll
        for (int i = 0; i < 2; ++i) col[i] = ((lane & 7) ^ swz(8 * (wave * IT + i) + (lane >> 3))) * 16;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const uint32_t r = 8 * (wave * IT + i) + (lane >> 3);
            off[i] = r < count ? r * static_cast<uint32_t>(ld) + col[i & 1] : kPast;
        }
    }
    // (steps in turn: a lane whose codes are past K once stays there)
    __device__ __forceinline__ void load(int8_t* stage, uint32_t k0) {
        if (k0 + 128 > K) {
#pragma unroll
            for (int i = 0; i < IT; ++i) off[i] = k0 + col[i & 1] < K ? off[i] : kPast;
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) load_lds(base, stage + at + i * 1024, off[i], static_cast<int>(k0));
    }
};

// Rows and columns of the tile that workgroup `b` of tiles_m x tiles_n computes: neighbouring workgroups of an XCD share
// group_m rows of tiles.
__device__ __forceinline__ void tile_of(const I8Args& a, uint32_t b, uint32_t& tm, uint32_t& tn) {
    const uint32_t t = xcd_swizzle(b, a.tiles_m * a.tiles_n);
    const uint32_t per = a.group_m * a.tiles_n, g = t / per, i = t % per;
    const uint32_t rows = min(a.group_m, a.tiles_m - g * a.group_m);
    tm = g * a.group_m + i % rows;
    tn = i / rows;
}

// A wave's sums of R rows and TN columns at a time leave through LDS (a region of its own), so that whole runs of a row are stored.
template <typename TC, int TN, int R_>
struct Out {
    static constexpr int R = R_, kLd = TN + 4, kInts = R * kLd;
    static constexpr int V = 16 / static_cast<int>(sizeof(TC)), LPR = TN / V, RPI = 64 / LPR;  // columns a lane, lanes a row, rows at a time
};

template <typename TC, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(WM * WN * 64) void gemm_i8_tile_kernel(I8Args a) {
    constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
    constexpr int A_IT = BM / 8 / NW, W_IT = BN / 8 / NW, T = NW * 64;
    // the epilogue's regions: P waves' in each of the two larger stage arrays, Q in each of the others, 32 rows each where they fit
    constexpr int kBig = 128 * (BM > BN ? BM : BN), kSmall = 128 * (BM > BN ? BN : BM), kRow = (TN + 4) * 4;
    constexpr int R = 2 * (kBig / (32 * kRow) + kSmall / (32 * kRow)) >= NW ? 32 : 16;
    typedef Out<TC, TN, R> O;
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "loads divide evenly");
    constexpr int P = kBig / (O::kInts * 4), Q = kSmall / (O::kInts * 4);
    static_assert(2 * (P + Q) >= NW, "the epilogue's regions fit the stages");
    // arrays of their own: the compiler then knows that reads of one stage do not wait for the loads into the other
    __shared__ __attribute__((aligned(16))) int8_t as0[BM * 128], as1[BM * 128], ws0[BN * 128], ws1[BN * 128];
    __shared__ __attribute__((aligned(16))) int8_t as2[NS > 2 ? BM * 128 : 16], ws2[NS > 2 ? BN * 128 : 16];
    __shared__ __attribute__((aligned(16))) int8_t as3[NS > 3 ? BM * 128 : 16], ws3[NS > 3 ? BN * 128 : 16];
    static_assert(NS >= 2 && NS <= 4, "two to four stages");
    // the tile's scales and biases, read while the first codes are on their way: from memory in the epilogue each would cost a
    // round trip
    __shared__ __attribute__((aligned(16))) float sas[BM], sws[BN], biases[BN];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, g = lane >> 5, wm = wave % WM, wn = wave / WM;
    uint32_t tm, tn;
    tile_of(a, blockIdx.x, tm, tn);
    const uint32_t m0 = tm * BM, n0 = tn * BN;
    Rows<A_IT> ra(a.A, a.lda, m0, min(static_cast<uint32_t>(BM), a.M - m0), a.K, wave, lane);
    Rows<W_IT> rw(a.W, a.ldw, n0, min(static_cast<uint32_t>(BN), a.N - n0), a.K, wave, lane);
    int at[4];  // the lane's piece of a 32-row block, for each 32 codes of a step
#pragma unroll
    for (int s = 0; s < 4; ++s) at[s] = l32 * 128 + (((2 * s + g) ^ swz(l32)) * 16);
    intx16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    // the fragments of the next 32 codes are read ahead of the products of these
    auto compute = [&](const int8_t* as, const int8_t* ws) {
        const int8_t* ap = as + wm * TM * 128;
        const int8_t* wp = ws + wn * TN * 128;
        intx4 x[2][FM], w[2][FN];
        auto read = [&](auto S) {
            constexpr int s = decltype(S)::value;
#pragma unroll
            for (int i = 0; i < FM; ++i) x[s & 1][i] = *reinterpret_cast<const intx4*>(ap + i * 4096 + at[s]);
#pragma unroll
            for (int j = 0; j < FN; ++j) w[s & 1][j] = *reinterpret_cast<const intx4*>(wp + j * 4096 + at[s]);
        };
        auto multiply = [&](auto S) {
            constexpr int s = decltype(S)::value;
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[s & 1][j], x[s & 1][i], acc[i][j], 0, 0, 0);
        };
        read(std::integral_constant<int, 0>{});
        __builtin_amdgcn_sched_barrier(0);
        read(std::integral_constant<int, 1>{});
        multiply(std::integral_constant<int, 0>{});
        __builtin_amdgcn_sched_barrier(0);
        read(std::integral_constant<int, 2>{});
        multiply(std::integral_constant<int, 1>{});
        __builtin_amdgcn_sched_barrier(0);
        read(std::integral_constant<int, 3>{});
        multiply(std::integral_constant<int, 2>{});
        __builtin_amdgcn_sched_barrier(0);
        multiply(std::integral_constant<int, 3>{});
    };
    auto load = [&](int8_t* as, int8_t* ws, uint32_t k) {  // past K: zeros
        ra.load(as, k);
        rw.load(ws, k);
    };
    const uint32_t steps = (a.K + 127) / 128;
    uint32_t k = 0;  // of the next step to compute
    // (their loads first: what waits for them then waits for no codes)
    float sa_[(BM + T - 1) / T], sw_[(BN + T - 1) / T], bias_[(BN + T - 1) / T];
#pragma unroll
    for (int i = 0; i < (BM + T - 1) / T; ++i) sa_[i] = a.sa[min(m0 + min(tid + i * T, BM - 1), a.M - 1)];
#pragma unroll
    for (int i = 0; i < (BN + T - 1) / T; ++i) {
        const uint32_t c = min(n0 + min(tid + i * T, BN - 1), a.N - 1);
        sw_[i] = a.sw[c];
        bias_[i] = a.bias ? a.bias[c] : 0.0f;
    }
    __builtin_amdgcn_sched_barrier(0);
    load(as0, ws0, k);
    if constexpr (NS > 2) load(as1, ws1, k + 128);
    if constexpr (NS > 3) load(as2, ws2, k + 256);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < (BM + T - 1) / T; ++i)
        if (tid + i * T < BM) sas[tid + i * T] = sa_[i];
#pragma unroll
    for (int i = 0; i < (BN + T - 1) / T; ++i)
        if (tid + i * T < BN) {
            sws[tid + i * T] = sw_[i];
            biases[tid + i * T] = bias_[i];
        }
    // One step: its loads have landed (a wave's own, then with the barrier everybody's, and everybody has read the step before), the
    // loads of the step NS - 1 ahead go where that one was, and its products run.
    auto step = [&](auto S) {
        constexpr int s = decltype(S)::value, f = (s + NS - 1) % NS;
        wait_loads<(NS - 2) * (A_IT + W_IT)>();
        barrier();
        load(f == 0 ? as0 : f == 1 ? as1 : f == 2 ? as2 : as3, f == 0 ? ws0 : f == 1 ? ws1 : f == 2 ? ws2 : ws3, k + (NS - 1) * 128);
        compute(s == 0 ? as0 : s == 1 ? as1 : s == 2 ? as2 : as3, s == 0 ? ws0 : s == 1 ? ws1 : s == 2 ? ws2 : ws3);
        k += 128;
    };
    // NS steps a trip, the last ones behind them (leaving the loop in its middle would copy every sum)
    for (uint32_t p = steps / NS; p > 0; --p) {
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        if constexpr (NS > 2) step(std::integral_constant<int, 2>{});
        if constexpr (NS > 3) step(std::integral_constant<int, 3>{});
    }
    const uint32_t rest = steps % NS;
    if (rest > 0) {
        step(std::integral_constant<int, 0>{});
        if constexpr (NS > 2) {
            if (rest > 1) {
                step(std::integral_constant<int, 1>{});
                if constexpr (NS > 3) {
                    if (rest > 2) step(std::integral_constant<int, 2>{});
                }
            }
        }
    }
    wait_loads<0>();
    __syncthreads();
    // (every wave has read its last step, no load is on its way: the stages are free)
    int8_t* const big = (BM > BN ? wave < P ? as0 : as1 : wave < P ? ws0 : ws1) + wave % P * O::kInts * 4;
    int8_t* const small = (BM > BN ? wave - 2 * P < Q ? ws0 : ws1 : wave - 2 * P < Q ? as0 : as1) + (wave < 2 * P ? 0 : (wave - 2 * P) % (Q ? Q : 1)) * O::kInts * 4;
    int* const stage = reinterpret_cast<int*>(wave < 2 * P ? big : small);
    const int lrow = lane / O::LPR, lcol = lane % O::LPR * O::V;
    const bool busy = lane < O::LPR * O::RPI;
    const uint32_t n = n0 + wn * TN + lcol;
    Columns<O::V> cols;
#pragma unroll
    for (int e = 0; e < O::V; ++e) {
        cols.sw[e] = sws[wn * TN + lcol + e];
        cols.bias[e] = biases[wn * TN + lcol + e];
    }
    auto rows = [&](int i, auto WHOLE) {
#pragma unroll
        for (int h = 0; h < 32; h += O::R) {
            const int r0 = wm * TM + 32 * i + h;
            if (O::R == 32 || (l32 & 16) == h) {
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<intx4*>(&stage[(l32 % O::R) * O::kLd + 32 * j + 8 * q + 4 * g]) =
                            intx4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int t = 0; t < O::R; t += O::RPI) {
                const int row = t + lrow;
                if (busy && row < O::R) {
                    const uint32_t m = m0 + r0 + row;
                    int v[O::V];
#pragma unroll
                    for (int e = 0; e < O::V; e += 4) {
                        const intx4 x = *reinterpret_cast<const intx4*>(&stage[row * O::kLd + lcol + e]);
#pragma unroll
                        for (int y = 0; y < 4; ++y) v[e + y] = x[y];
                    }
                    if constexpr (decltype(WHOLE)::value) store_run<TC, O::V>(a, m, n, v, sas[r0 + row], cols, true);
                    else if (m < a.M && n < a.N) store_run<TC, O::V>(a, m, n, v, sas[r0 + row], cols, a.wide && n + O::V <= a.N);
                }
            }
            __builtin_amdgcn_wave_barrier();  // every read of these rows precedes the next rows' writes
        }
    };
    if (a.wide && m0 + BM <= a.M && n0 + BN <= a.N) {
#pragma unroll
        for (int i = 0; i < FM; ++i) rows(i, std::true_type{});
    } else {
#pragma unroll
        for (int i = 0; i < FM; ++i) rows(i, std::false_type{});
    }
}

// ---- small grids: a workgroup's waves split K ---------------------------------------------
//
// Eight waves compute the same 32 x 32 tile, each from the 128-code steps wave, wave + 8, ... through LDS stages of its own
// (no barrier: a wave waits for its own loads alone), and add their sums through LDS. One launch, no workspace. Bound by the launch and two
// round trips of loads: 154x1280x2048 4.7 us, tiles of 64 x 64 6.4.
template <typename TC>
__global__ __launch_bounds__(512) void gemm_i8_split_kernel(I8Args a) {
    constexpr int kWave = 64 * 128;  // bytes of a wave's stage: 32 rows of A, 32 of W
    constexpr int kLd = 36;
    __shared__ __attribute__((aligned(16))) int8_t st0[8 * kWave], st1[8 * kWave];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, g = lane >> 5;
    uint32_t tm, tn;
    tile_of(a, blockIdx.x, tm, tn);
    const uint32_t m0 = tm * 32, n0 = tn * 32;
    Rows<4> ra(a.A, a.lda, m0, min(32u, a.M - m0), a.K, 0, lane), rw(a.W, a.ldw, n0, min(32u, a.N - n0), a.K, 0, lane);
    int8_t* const s0 = st0 + wave * kWave;
    int8_t* const s1 = st1 + wave * kWave;
    intx16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0;
    auto load = [&](int8_t* st, uint32_t k) {
        wait_lds();  // reads of what the loads replace
        ra.load(st, k);
        rw.load(st + 4096, k);
    };
    auto compute = [&](const int8_t* st) {
        __builtin_amdgcn_wave_barrier();  // (a wave's wait is for the loads of all its lanes)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int at = l32 * 128 + (((2 * s + g) ^ swz(l32)) * 16);
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*reinterpret_cast<const intx4*>(st + 4096 + at),
                                                        *reinterpret_cast<const intx4*>(st + at), acc, 0, 0, 0);
        }
    };
    uint32_t k = wave * 128;
    if (k < a.K) load(s0, k);
    while (k < a.K) {
        if (k + 1024 < a.K) {
            load(s1, k + 1024);
            wait_loads<8>();  // (the other stage's)
        } else {
            wait_loads<0>();
        }
        compute(s0);
        k += 1024;
        if (k >= a.K) break;
        if (k + 1024 < a.K) {
            load(s0, k + 1024);
            wait_loads<8>();
        } else {
            wait_loads<0>();
        }
        compute(s1);
        k += 1024;
    }
    __syncthreads();
    int* const red = reinterpret_cast<int*>(st0);
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<intx4*>(&red[(wave * 32 + l32) * kLd + 8 * q + 4 * g]) = intx4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    __syncthreads();
    if (tid >= 256) return;
    const uint32_t row = tid >> 3, c = (tid & 7) * 4, m = m0 + row, n = n0 + c;
    if (m >= a.M || n >= a.N) return;
    Columns<4> cols;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        cols.sw[e] = a.sw[min(n + e, a.N - 1)];
        cols.bias[e] = a.bias ? a.bias[min(n + e, a.N - 1)] : 0.0f;
    }
    const float sa = a.sa[m];
    int v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        const intx4 x = *reinterpret_cast<const intx4*>(&red[(w * 32 + row) * kLd + c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += x[e];
    }
    store_run<TC, 4>(a, m, n, v, sa, cols, a.wide && n + 4 <= a.N);
}

// ---- few rows ------------------------------------------------------------------------------
//
// Up to 16 rows (single tokens): a workgroup takes 16 columns and its eight waves the 256-code pieces of K in turn, the
// weights straight from memory into MFMA operands (16 rows x 64 bytes an instruction); the sums are added through LDS. 2x1280x1280 3.0 us
// (an empty launch 2.0 by the same clock); K below 2048 leaves waves idle (1280 three of the eight).
constexpr uint32_t kFewRows = 16;

template <typename TC>
__global__ __launch_bounds__(512) void gemm_i8_few_kernel(I8Args a) {
    constexpr int kLd = 20;
    __shared__ __attribute__((aligned(16))) int red[8][16 * kLd];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t l16 = lane & 15, c = lane >> 4, n0 = blockIdx.x * 16;
    const uint32_t rows = min(16u, a.N - n0);
    const __amdgpu_buffer_rsrc_t rA = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.A), 0, static_cast<int>((a.M - 1) * a.lda + a.K), 0x00020000);
    const __amdgpu_buffer_rsrc_t rW = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.W + n0 * a.ldw), 0,
                                                                        static_cast<int>((rows - 1) * a.ldw + a.K), 0x00020000);
    const uint32_t oa = l16 < a.M ? l16 * static_cast<uint32_t>(a.lda) : kPast, ow = l16 < rows ? l16 * static_cast<uint32_t>(a.ldw) : kPast;
    intx4 acc = {0, 0, 0, 0};
    for (uint32_t k0 = wave * 256; k0 < a.K; k0 += 2048) {
        intx4 x[4], w[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint32_t k = k0 + 64 * s + 16 * c;
            w[s] = __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(rW, k < a.K && l16 < rows ? ow + k : kPast, 0, 0));
            x[s] = __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(rA, k < a.K && l16 < a.M ? oa + k : kPast, 0, 0));
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[s], x[s], acc, 0, 0, 0);
    }
    *reinterpret_cast<intx4*>(&red[wave][l16 * kLd + 4 * c]) = acc;  // row m = l16, columns 4c .. 4c + 3
    __syncthreads();
    if (tid >= 256) return;
    const uint32_t m = tid >> 4, col = tid & 15, n = n0 + col;
    if (m >= a.M || n >= a.N) return;
    int v = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += red[w][m * kLd + col];
    store_one<TC>(a, m, n, v, a.sa[m]);
}

// A wave takes a row at a time: its largest magnitude, then its codes.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_any_kernel(const T* x, int8_t* q, float* scale, uint64_t rows, uint32_t cols,
                                                                uint64_t ldx, uint64_t ldq) {
    const uint32_t lane = threadIdx.x & 63;
    for (uint64_t r = blockIdx.x * 4ull + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4ull) {
        const T* xr = x + r * ldx;
        uint32_t top = 0;
        for (uint32_t c = lane; c < cols; c += 64) top = max(top, magnitude_bits(static_cast<float>(xr[c])));
        const RowScale s = row_scale(wave_max(top));
        for (uint32_t c = lane; c < cols; c += 64) q[r * ldq + c] = static_cast<int8_t>(quant_code(static_cast<float>(xr[c]), s));
        if (lane == 0) scale[r] = s.scale;
    }
}

// Rows of whole 16-byte vectors, cols <= 8192 (E values a lane, NV vectors): a wave takes a row, or the W = 4 waves of a workgroup do, and it
// stays in their registers from its largest magnitude to its codes, so it is read once. Lanes past the row repeat its last vector and
// store nothing. Bound by memory and, for few rows, by the launch: 2048 x 5120 fp16 (31 MB) 8.3 us with four waves a row, 10.2 with one,
// whose registers leave two waves a SIMD; 4096 x 8192 fp16 17.9 / 35, 64 x 4096 fp16 4.2 / 5.8; but 8192 x 640 fp16 8.8 / 5.2: up to three
// vectors a lane are one wave's.
template <typename T, int NV, int W>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* x, int8_t* q, float* scale, uint32_t rows, uint32_t cols, uint64_t ldx,
                                                            uint64_t ldq) {
    constexpr int E = 16 / static_cast<int>(sizeof(T));
    typedef T VT __attribute__((ext_vector_type(E)));
    __shared__ uint32_t tops[2][4];  // (a row's, and the next one's: one barrier a row)
    const uint32_t wave = threadIdx.x >> 6, at = threadIdx.x % (64 * W), vecs = cols / E;
    uint32_t turn = 0;
    for (uint64_t r = blockIdx.x * (4ull / W) + wave / W; r < rows; r += gridDim.x * (4ull / W), turn ^= 1) {
        const T* xr = x + r * ldx;
        VT v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = *reinterpret_cast<const VT*>(xr + min(at + 64 * W * i, vecs - 1) * E);
        uint32_t top = 0;
        if constexpr (E == 8) {
            // fp16 magnitudes order as 16-bit integers, two at a time
            typedef uint16_t U8 __attribute__((ext_vector_type(8)));
            U8 m = __builtin_bit_cast(U8, v[0]) & static_cast<uint16_t>(0x7fff);
#pragma unroll
            for (int i = 1; i < NV; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(U8, v[i]) & static_cast<uint16_t>(0x7fff));
            uint16_t t = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) t = t > m[e] ? t : m[e];
            top = magnitude_bits(static_cast<float>(__builtin_bit_cast(_Float16, t)));
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) top = max(top, magnitude_bits(static_cast<float>(v[i][e])));
        }
        top = wave_max(top);
        if constexpr (W > 1) {  // (every wave of the workgroup has this row)
            if ((threadIdx.x & 63) == 0) tops[turn][wave] = top;
            __syncthreads();
            top = max(max(tops[turn][0], tops[turn][1]), max(tops[turn][2], tops[turn][3]));
        }
        const RowScale s = row_scale(top);
        int8_t* qr = q + r * ldq;
        uint32_t w[NV * E / 4];
        quant_codes<NV * E>([&](int i) { return static_cast<float>(v[i / E][i % E]); }, s, w);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at + 64 * W * i < vecs) {
                uint32_t* p = reinterpret_cast<uint32_t*>(qr + (at + 64 * W * i) * E);
                if constexpr (E == 8) {
                    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
                    *reinterpret_cast<u2*>(p) = u2{w[2 * i], w[2 * i + 1]};
                } else {
                    *p = w[i];
                }
            }
        if (at == 0) scale[r] = s.scale;
    }
}

unsigned grid_of(uint64_t units) { return static_cast<unsigned>(std::min<uint64_t>(units, kMaxGrid)); }

uint64_t span(uint64_t rows, uint64_t ld, uint64_t cols) { return rows ? (rows - 1) * ld + cols : 0; }

// Builds: 0 any shape, 1 few rows, 2 waves split K (32 x 32), the others tiles: 8 is 3 with three stages, 5 is 4 with four (and eight
// waves: one workgroup a CU, whose loads alone have to hide their latency).
//
// The cost of a tile build, n tiles on the fullest of 256 CUs: 3 + n (tile + steps step). It is there to rank builds: what a call's C
// costs beyond its tiles' share is the same for all and is not in it, nor is C's type, nor the lower clock of long runs of products.
// us (MI355X, fp16 C) of builds 3, 8, 4, 5, 6, 7, and by the cost where a rule does not keep the build out:
//   576x1280x1280     5.3  5.3  8.7  7.9 15.0 24.4   (5.5  4.7   -   9.2 15.8 24.5)
//   2048x1280x1280    8.3  9.2  9.4  8.7 15.6 24.9   (9.1   -    -   9.2 15.8 24.5)
//   2048x1280x5120   24.9 25.7 30.1 21.5 45.5 67.0  (25.6   -    -  21.9 44.0 65.9)
//   8192x640x2560    25.3 23.7 20.8 24.4 27.0 40.2  (27.0   -  22.2 23.9 25.2 38.3)
//   8192x640x640      9.4  9.9  9.3 12.0 11.6 18.8   (9.8   -   9.6 11.3 11.1 17.6)
//   2048x10240x1280  48.3 49.9 35.2 40.3 35.2 32.3  (53.0   -  30.0 34.2 28.6 24.5)
// The fastest is chosen in each, and so it is with fp32 C (2048x1280x5120 21.7, 8192x640x2560 22.2, 2048x10240x1280 35.7: 4 us more for C).
// (128 x 128 with two groups of waves that take the steps in turn: 24.8 for 2048x1280x5120; 128 x 80 in 256 workgroups of four waves of 64 x 80,
// half of each step's codes each, with the next step's fragments read ahead: 21.8; 256 x 256, 256 x 128, 128 x 64, 128 x 192 and
// 64 x 128 tiles were between their neighbours.)
struct Build {
    uint32_t bm, bn;
    float tile_us, step_us;
};
constexpr Build kBuilds[kGemmI8Builds] = {{64, 64, 0, 0},          {16, 16, 0, 0},           {32, 32, 0, 0},           {64, 64, 0.2f, 0.23f},  {128, 128, 1.2f, 0.42f},
                                          {128, 128, 2.05f, 0.42f}, {192, 256, 3.4f, 0.94f}, {256, 320, 7.7f, 1.38f}, {64, 64, 0.2f, 0.15f}};
enum { kAny = 0, kFew = 1, kSplitK = 2, k64 = 3, k128 = 4, k128x4 = 5, k192 = 6, k256 = 7, k64x3 = 8 };

int choose(const I8Args& a) {
    const bool vec = a.K % 16 == 0 && a.lda % 16 == 0 && a.ldw % 16 == 0 && aligned(a.A, 16) && aligned(a.W, 16) &&
                     a.lda <= kMaxLd && a.ldw <= kMaxLd;
    if (!vec) return kAny;
    // (a launch has fewer than 2^32 threads)
    auto tiles = [&](int b) { return static_cast<uint64_t>(ceil_div(a.M, kBuilds[b].bm)) * ceil_div(a.N, kBuilds[b].bn); };
    auto fits = [&](int b) { return tiles(b) < (1u << 23) && (b != kFew || a.M <= kFewRows); };
    const int cfg = tuning().gemm_i8_cfg.load();
    if (cfg >= 0 && fits(cfg)) return cfg;
    if (fits(kFew)) return kFew;
    if (static_cast<uint64_t>(ceil_div(a.M, 64)) * ceil_div(a.N, 64) <= 128) return kSplitK;
    int best = kAny;
    float least = 0.0f;
    for (int b = k64; b <= k64x3; ++b) {
        if (!fits(b)) continue;
        const uint64_t n = (tiles(b) + 255) / 256;
        if (b == k64x3 && n > 2) continue;  // three workgroups a CU; with more tiles four are faster
        if (b == k128 && n < 2) continue;   // two workgroups a CU hide each other's latency; one needs four stages
        // (three of its four places on a CU taken: 0.19 us a tile and step with 40 steps, 0.16 with 10, where two take 0.23 and 0.14, four 0.20
        // and 0.18, six 0.21 and 0.20; 2048x1280x1280 has three)
        const float step = b == k64 && n == 3 ? 0.183f : kBuilds[b].step_us;
        const float us = static_cast<float>(n) * (kBuilds[b].tile_us + ceil_div(a.K, 128) * step);
        if (best == kAny || us < least) {
            best = b;
            least = us;
        }
    }
    return best;
}

template <typename TC>
void launch_product(I8Args a, hipStream_t s) {
    const int build = choose(a);
    if (build == kAny) {
        gemm_i8_any_kernel<TC><<<grid_of(static_cast<uint64_t>(ceil_div(a.M, 64)) * ceil_div(a.N, 64)), 256, 0, s>>>(a);
        return;
    }
    a.wide = a.ldc % (16 / sizeof(TC)) == 0 && aligned(a.C, 16);
    a.tiles_m = ceil_div(a.M, kBuilds[build].bm);
    a.tiles_n = ceil_div(a.N, kBuilds[build].bn);
    a.group_m = std::min(a.tiles_m, 8u);
    const unsigned grid = a.tiles_m * a.tiles_n;
    switch (build) {
        case kFew: gemm_i8_few_kernel<TC><<<grid, 512, 0, s>>>(a); break;
        case kSplitK: gemm_i8_split_kernel<TC><<<grid, 512, 0, s>>>(a); break;
        case k64: gemm_i8_tile_kernel<TC, 64, 64, 2, 2, 2><<<grid, 256, 0, s>>>(a); break;
        case k128: gemm_i8_tile_kernel<TC, 128, 128, 2, 2, 2><<<grid, 256, 0, s>>>(a); break;
        case k128x4: gemm_i8_tile_kernel<TC, 128, 128, 4, 2, 4><<<grid, 512, 0, s>>>(a); break;
        case k192: gemm_i8_tile_kernel<TC, 192, 256, 2, 4, 2><<<grid, 512, 0, s>>>(a); break;
        case k256: gemm_i8_tile_kernel<TC, 256, 320, 4, 2, 2><<<grid, 512, 0, s>>>(a); break;
        default: gemm_i8_tile_kernel<TC, 64, 64, 2, 2, 3><<<grid, 256, 0, s>>>(a); break;
    }
}

template <typename T>
void launch_quantize(const T* x, int8_t* q, float* scale, uint32_t rows, uint32_t cols, uint64_t ldx, uint64_t ldq, hipStream_t s) {
    constexpr uint32_t E = 16 / sizeof(T);
    const uint32_t nv = ceil_div(cols, 64 * E);
    const unsigned grid = grid_of((static_cast<uint64_t>(rows) + 3) / 4), wide = grid_of(rows);
    if (cols % E != 0 || ldx % E != 0 || ldq % E != 0 || !aligned(x, 16) || !aligned(q, E) || cols > kMaxFastCols)
        quantize_rows_any_kernel<T><<<grid, 256, 0, s>>>(x, q, scale, rows, cols, ldx, ldq);
    else if (nv <= 2) quantize_rows_kernel<T, 2, 1><<<grid, 256, 0, s>>>(x, q, scale, rows, cols, ldx, ldq);
    else if (nv <= 3) quantize_rows_kernel<T, 3, 1><<<grid, 256, 0, s>>>(x, q, scale, rows, cols, ldx, ldq);
    else if (nv <= 8) quantize_rows_kernel<T, 2, 4><<<wide, 256, 0, s>>>(x, q, scale, rows, cols, ldx, ldq);
    else if (nv <= 12) quantize_rows_kernel<T, 3, 4><<<wide, 256, 0, s>>>(x, q, scale, rows, cols, ldx, ldq);
    else if (sizeof(T) == 2 || nv <= 16) quantize_rows_kernel<T, 4, 4><<<wide, 256, 0, s>>>(x, q, scale, rows, cols, ldx, ldq);
    else if constexpr (sizeof(T) == 4) quantize_rows_kernel<T, 8, 4><<<wide, 256, 0, s>>>(x, q, scale, rows, cols, ldx, ldq);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_quantize_rows_i8(const void* x, int dtype, int8_t* q, float* scale, uint32_t rows, uint32_t cols, uint32_t ldx,
                                   uint32_t ldq, void* stream) {
    const char* fn = "mi_quantize_rows_i8";
    if (dtype != MI_F32 && dtype != MI_F16) return fail(MI_ERR_INVALID_ARG, "%s: dtype %d", fn, dtype);
    if (rows == 0 || cols == 0) return MI_OK;
    if (rows > kMaxSize || cols > kMaxCols) return fail(MI_ERR_UNSUPPORTED, "%s: rows %u > 2^31 or columns %u > 2^30", fn, rows, cols);
    if (!x || !q || !scale) return fail(MI_ERR_INVALID_ARG, "%s: null pointer", fn);
    const uint64_t lx = ldx ? ldx : cols, lq = ldq ? ldq : cols, e = dtype == MI_F16 ? 2 : 4;
    if (lx < cols || lq < cols) return fail(MI_ERR_INVALID_ARG, "%s: a row stride below %u columns", fn, cols);
    if (!aligned(x, e) || !aligned(scale, 4)) return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
    const uint64_t nx = span(rows, lx, cols) * e, nq = span(rows, lq, cols), ns = static_cast<uint64_t>(rows) * 4;
    if (overlaps(q, nq, x, nx) || overlaps(scale, ns, x, nx)) return fail(MI_ERR_ALIASING, "%s: an output overlaps x", fn);
    if (overlaps(q, nq, scale, ns)) return fail(MI_ERR_ALIASING, "%s: q and scale overlap", fn);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == MI_F16) launch_quantize(static_cast<const _Float16*>(x), q, scale, rows, cols, lx, lq, s);
    else launch_quantize(static_cast<const float*>(x), q, scale, rows, cols, lx, lq, s);
    return check_launch(fn);
}

extern "C" int mi_gemm_nt_i8(const int8_t* A, const float* a_scale, const int8_t* W, const float* w_scale, const float* bias, void* C,
                             int c_dtype, uint32_t M, uint32_t N, uint32_t K, uint32_t mode, uint32_t lda, uint32_t ldw, uint32_t ldc,
                             void* stream) {
    const char* fn = "mi_gemm_nt_i8";
    if (c_dtype != MI_F32 && c_dtype != MI_F16) return fail(MI_ERR_INVALID_ARG, "%s: c_dtype %d", fn, c_dtype);
    if (mode > 2) return fail(MI_ERR_INVALID_ARG, "%s: mode %u", fn, mode);
    if (M == 0 || N == 0) return MI_OK;
    if (M > kMaxSize || N > kMaxSize) return fail(MI_ERR_UNSUPPORTED, "%s: M %u or N %u > 2^31", fn, M, N);
    if (K == 0 || K > kMaxK) return fail(MI_ERR_UNSUPPORTED, "%s: K %u (1 .. %u: the sum is held in 32 bits)", fn, K, kMaxK);
    if (!A || !a_scale || !W || !w_scale || !C) return fail(MI_ERR_INVALID_ARG, "%s: null pointer", fn);
    I8Args a{A, W, a_scale, w_scale, mode == 1 ? nullptr : bias, C, M, N, K, mode, lda ? lda : K, ldw ? ldw : K, ldc ? ldc : N, 0, 0, 0, 0};
    if (a.lda < K || a.ldw < K || a.ldc < N) return fail(MI_ERR_INVALID_ARG, "%s: a row stride below its row", fn);
    const uint64_t e = c_dtype == MI_F16 ? 2 : 4;
    if (!aligned(a_scale, 4) || !aligned(w_scale, 4) || !aligned(bias, 4) || !aligned(C, e))
        return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
    const uint64_t nc = span(M, a.ldc, N) * e;
    const struct {
        const void* p;
        uint64_t bytes;
    } in[5] = {{A, span(M, a.lda, K)}, {W, span(N, a.ldw, K)}, {a_scale, M * 4ull}, {w_scale, N * 4ull}, {a.bias, N * 4ull}};
    for (const auto& i : in)
        if (overlaps(C, nc, i.p, i.bytes)) return fail(MI_ERR_ALIASING, "%s: C overlaps an input", fn);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (c_dtype == MI_F16) launch_product<_Float16>(a, s);
    else launch_product<float>(a, s);
    return check_launch(fn);
}

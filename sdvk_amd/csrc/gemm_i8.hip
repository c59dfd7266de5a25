// gemm_i8.hip -- linears in 8-bit integers for gfx950: the token quantiser and the product
//   C[m,n] (=|+=) sa[m] sw[n] sum_k A[m,k] W[n,k] (+ bias[n])
// of codes with a scale for each row of A (a token) and of W (a channel).
//
// The sum is exact in 32-bit integers (K <= 131071: |code| <= 128), so every plan gives the same bits; the epilogue is one
// conversion, one product and one fma in fp32: fma(float(sum) * sa, sw, bias).
#include "common.hpp"
#include "quant.hpp"

#include <algorithm>

namespace mi {
namespace {

constexpr uint32_t kMaxGrid = 1u << 20;  // workgroups of a launch that strides over its units
constexpr uint32_t kMaxK = 131071;       // 2^31 / 2^14

struct I8Args {
    const int8_t *A, *W;
    const float *sa, *sw, *bias;
    void* C;
    uint32_t M, N, K, mode;
    uint64_t lda, ldw, ldc;
};

// mode 0 stores, mode 1 adds, mode 2 adds with the bias (NULL for mode 1).
template <typename TC>
__device__ __forceinline__ void store_one(const I8Args& a, uint32_t m, uint32_t n, int acc, float sa) {
    const float b = a.bias ? a.bias[n] : 0.0f;
    float v = __builtin_fmaf(static_cast<float>(acc) * sa, a.sw[n], b);
    TC* p = static_cast<TC*>(a.C) + m * a.ldc + n;
    if (a.mode) v += static_cast<float>(*p);
    *p = static_cast<TC>(v);
}

// Any K, any alignment: a 64 x 64 tile in steps of 32 codes, 4 x 4 outputs a thread.
template <typename TC>
__global__ __launch_bounds__(256) void gemm_i8_any_kernel(I8Args a) {
    __shared__ int8_t at[64][36], wt[64][36];
    const uint32_t tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const uint32_t tiles_n = (a.N + 63) / 64;
    const uint64_t tiles = static_cast<uint64_t>((a.M + 63) / 64) * tiles_n;
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
            for (int k = 0; k < 32; ++k) {
                int x[4], w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = at[ty + 16 * i][k];
                    w[i] = wt[tx + 16 * i][k];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] += x[i] * w[j];
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

unsigned grid_of(uint64_t units) { return static_cast<unsigned>(std::min<uint64_t>(units, kMaxGrid)); }

uint64_t span(uint64_t rows, uint64_t ld, uint64_t cols) { return rows ? (rows - 1) * ld + cols : 0; }

template <typename TC>
void launch_product(const I8Args& a, hipStream_t s) {
    gemm_i8_any_kernel<TC><<<grid_of(static_cast<uint64_t>(ceil_div(a.M, 64)) * ceil_div(a.N, 64)), 256, 0, s>>>(a);
}

template <typename T>
void launch_quantize(const T* x, int8_t* q, float* scale, uint32_t rows, uint32_t cols, uint64_t ldx, uint64_t ldq, hipStream_t s) {
    quantize_rows_any_kernel<T><<<grid_of((static_cast<uint64_t>(rows) + 3) / 4), 256, 0, s>>>(x, q, scale, rows, cols, ldx, ldq);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_quantize_rows_i8(const void* x, int dtype, int8_t* q, float* scale, uint32_t rows, uint32_t cols, uint32_t ldx,
                                   uint32_t ldq, void* stream) {
    const char* fn = "mi_quantize_rows_i8";
    if (dtype != MI_F32 && dtype != MI_F16) return fail(MI_ERR_INVALID_ARG, "%s: dtype %d", fn, dtype);
    if (rows == 0 || cols == 0) return MI_OK;
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
    if (K == 0 || K > kMaxK) return fail(MI_ERR_UNSUPPORTED, "%s: K %u (1 .. %u: the sum is held in 32 bits)", fn, K, kMaxK);
    if (!A || !a_scale || !W || !w_scale || !C) return fail(MI_ERR_INVALID_ARG, "%s: null pointer", fn);
    I8Args a{A, W, a_scale, w_scale, mode == 1 ? nullptr : bias, C, M, N, K, mode, lda ? lda : K, ldw ? ldw : K, ldc ? ldc : N};
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

// glue_bwd.hip -- backward passes of the block glue (glue.hip) for gfx950: LayerNorm and GEGLU.
//
// LayerNorm, y = xh * gamma + beta, xh = (x - mean) * inv, inv = 1 / sqrt(var + eps) per row of d:
//   w      = dy * gamma
//   dx     = inv * (w - mean(w) - xh * mean(w * xh)) (+ res, the residual stream's gradient)
//   dgamma = sum over rows of dy * xh,   dbeta = sum over rows of dy
// mean and inv are recomputed from x (two passes over the row in registers, as in the forward kernel), so
// nothing has to be kept from the forward pass but x.
//
// GEGLU, y = v * gelu(g) for h = [v | g]: geglu_grad (common.hpp).
//
// Both are HBM-bound: every element is read and written once. LayerNorm's column sums stay in a lane's
// registers over the rows of its wave, are added over the workgroup's waves in LDS and go to the workspace
// as one partial row per workgroup, which a second kernel adds in a fixed order (results repeat bit for bit).
//
// Measured (MI355X): LayerNorm 8192 x 640 fp32 with res 16.3 us (84 MB: 5.2 TB/s, what a copy of that size reaches in the
// last-level cache) and 3.8 us for the sum of the partial rows; 77 x 768 with an fp16 dy 4.8 and 2.9 us (latency). GEGLU
// 2048 x 5120 fp32 30.9 us with its tensors in cache, 39.6 us with others in turn (210 MB: 5.3 TB/s), fp16 22.0 us (147 MB).
#include "common.hpp"

#include <algorithm>

namespace mi {
namespace {

constexpr uint32_t kMaxParts = 512;  // partial rows of dgamma / dbeta: two workgroups per CU
constexpr int kColRows = 64;         // rows per workgroup of the general column sums, at least
constexpr uint32_t kMaxRows = 1u << 31;
constexpr uint32_t kMaxCols = 1u << 30;  // 2 d columns of sums and a stride of 64 are counted in 32 bits
constexpr uint32_t kMaxGrid = 1u << 20;  // workgroups of a launch that strides over rows or columns (2^32 threads are refused)

// The wave's sum in every lane, the same bits in each (glue.hip's order: quads, half rows, rows, halves).
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = dpp_add<0xb1>(v);   // quad_perm [1, 0, 3, 2]
    v = dpp_add<0x4e>(v);   // quad_perm [2, 3, 0, 1]
    v = dpp_add<0x141>(v);  // row_half_mirror
    v = dpp_add<0x140>(v);  // row_mirror
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
}

// Four consecutive elements of a row of T from a buffer resource, as fp32; j: their index / 4.
template <typename T>
__device__ __forceinline__ floatx4 load4(__amdgpu_buffer_rsrc_t r, uint32_t j) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, j * 16, 0, 0));
    } else {
        const half4 h = __builtin_bit_cast(half4, __builtin_amdgcn_raw_buffer_load_b64(r, j * 8, 0, 0));
        return floatx4{static_cast<float>(h[0]), static_cast<float>(h[1]), static_cast<float>(h[2]), static_cast<float>(h[3])};
    }
}

// Vector rows: d % 4 == 0, d <= 256 NC, 16-byte aligned fp32 tensors, 8-byte aligned fp16 dy. A wave takes rows
// blockIdx.x * 4 + wave, + 4 gridDim.x, ...; the lane's columns are 4 (lane + 64 i) + e, chunks past d read as
// zeros (out of the resource's range) and are never stored. part: [gridDim.x][2][d], or NULL (no weight gradients).
// us a call, this kernel against the general one: 8192x640 fp32 18.7 : 35, 4096x2560 fp32 43.6 : 93, fp16 dy 67 : 89,
// 4096x4096 fp32 61 : 150, fp16 dy 79 : 126, 77x4096 fp16 dy 20 : 47 (NC 16 with an fp16 dy spills 137 registers).
template <typename TD, int NC>
__global__ __launch_bounds__(256) void layernorm_bwd_vec_kernel(const float* x, const float* gamma, const TD* dy,
                                                                const float* res, float* dx, float* part, uint32_t rows,
                                                                uint32_t d, float eps) {
    __shared__ __attribute__((aligned(16))) float sums[3][64 * 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t n4 = d / 4;
    const int nbytes = static_cast<int>(d * 4);
    floatx4 gm[NC], sg[NC], sb[NC];
    if (gamma) {
        const __amdgpu_buffer_rsrc_t rg = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(gamma), 0, nbytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < NC; ++i) gm[i] = load4<float>(rg, lane + 64 * i);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) sg[i] = sb[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + wave); row < rows; row += gridDim.x * 4) {
        const uint64_t at = static_cast<uint64_t>(row) * d;
        const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(x + at), 0, nbytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t ry = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<TD*>(dy + at), 0, static_cast<int>(d * sizeof(TD)), 0x00020000);
        const __amdgpu_buffer_rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<float*>(res ? res + at : x), 0, res ? nbytes : 0, 0x00020000);
        floatx4 c[NC], w[NC], r[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) c[i] = load4<float>(rx, lane + 64 * i);
#pragma unroll
        for (int i = 0; i < NC; ++i) w[i] = load4<TD>(ry, lane + 64 * i);
#pragma unroll
        for (int i = 0; i < NC; ++i) r[i] = load4<float>(rr, lane + 64 * i);  // zeros without res
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i) s += (c[i][0] + c[i][1]) + (c[i][2] + c[i][3]);
        const float mean = wave_sum(s) / static_cast<float>(d);
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const bool in = lane + 64u * i < n4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[i][e] = in ? c[i][e] - mean : 0.0f;
                ss += c[i][e] * c[i][e];
            }
        }
        const float inv = 1.0f / sqrtf(wave_sum(ss) / static_cast<float>(d) + eps);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[i][e] *= inv;  // xh
                sg[i][e] += w[i][e] * c[i][e];
                sb[i][e] += w[i][e];
                if (gamma) w[i][e] *= gm[i][e];
                s1 += w[i][e];
                s2 += w[i][e] * c[i][e];
            }
        s1 = wave_sum(s1) / static_cast<float>(d);
        s2 = wave_sum(s2) / static_cast<float>(d);
        float* out = dx + at;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const uint32_t j = lane + 64 * i;
            if (j < n4) {
                floatx4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = inv * (w[i][e] - s1 - c[i][e] * s2) + r[i][e];
                *reinterpret_cast<floatx4*>(out + 4 * j) = v;
            }
        }
    }
    if (!part) return;
    // the four waves' sums of one 256-column chunk at a time, waves in order
    float* P = part + static_cast<uint64_t>(blockIdx.x) * 2 * d;
#pragma unroll
    for (int k = 0; k < 2 * NC; ++k) {
        const int i = k >> 1;
        floatx4 v = (k & 1) ? sb[i] : sg[i];
        if (wave > 0) *reinterpret_cast<floatx4*>(&sums[wave - 1][lane * 4]) = v;
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int u = 0; u < 3; ++u) v += *reinterpret_cast<const floatx4*>(&sums[u][lane * 4]);
            const uint32_t j = lane + 64 * i;
            if (j < n4) *reinterpret_cast<floatx4*>(P + (k & 1) * d + 4 * j) = v;
        }
        __syncthreads();
    }
}

// Any d, any alignment: a wave takes a row at a time (as above), each pass over memory. stats: [rows][2] of mean and inv for the column
// sums, or NULL.
template <typename TD>
__global__ __launch_bounds__(256) void layernorm_bwd_kernel(const float* x, const float* gamma, const TD* dy,
                                                            const float* res, float* dx, float* stats, uint32_t rows,
                                                            uint32_t d, float eps) {
    const int lane = threadIdx.x & 63;
    for (uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += gridDim.x * 4) {
        const uint64_t at = static_cast<uint64_t>(row) * d;
        const float* xr = x + at;
        const TD* yr = dy + at;
        float s = 0.0f;
        for (uint32_t j = lane; j < d; j += 64) s += xr[j];
        const float mean = wave_sum(s) / static_cast<float>(d);
        float ss = 0.0f;
        for (uint32_t j = lane; j < d; j += 64) {
            const float v = xr[j] - mean;
            ss += v * v;
        }
        const float inv = 1.0f / sqrtf(wave_sum(ss) / static_cast<float>(d) + eps);
        float s1 = 0.0f, s2 = 0.0f;
        for (uint32_t j = lane; j < d; j += 64) {
            const float w = static_cast<float>(yr[j]) * (gamma ? gamma[j] : 1.0f);
            s1 += w;
            s2 += w * ((xr[j] - mean) * inv);
        }
        s1 = wave_sum(s1) / static_cast<float>(d);
        s2 = wave_sum(s2) / static_cast<float>(d);
        for (uint32_t j = lane; j < d; j += 64) {
            const float w = static_cast<float>(yr[j]) * (gamma ? gamma[j] : 1.0f);
            const float v = inv * (w - s1 - (xr[j] - mean) * inv * s2);
            dx[at + j] = res ? v + res[at + j] : v;
        }
        if (stats && lane == 0) {
            stats[2 * static_cast<uint64_t>(row)] = mean;
            stats[2 * static_cast<uint64_t>(row) + 1] = inv;
        }
    }
}

// Column sums of rows [y * per, (y + 1) * per) at 64 columns at a time: four row groups of a workgroup, added in order.
template <typename TD>
__global__ __launch_bounds__(256) void layernorm_cols_kernel(const float* x, const TD* dy, const float* stats, float* part,
                                                             uint32_t rows, uint32_t d, uint32_t per) {
    __shared__ float sums[2][4][64];
    const uint32_t lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
    const uint32_t r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
    for (uint32_t j0 = blockIdx.x * 64; j0 < d; j0 += gridDim.x * 64) {
        const uint32_t j = j0 + lane;
        float sg = 0.0f, sb = 0.0f;
        if (j < d)
            for (uint32_t r = r0 + grp; r < r1; r += 4) {
                const uint64_t at = static_cast<uint64_t>(r) * d + j;
                const float w = static_cast<float>(dy[at]);
                sg += w * ((x[at] - stats[2 * static_cast<uint64_t>(r)]) * stats[2 * static_cast<uint64_t>(r) + 1]);
                sb += w;
            }
        sums[0][grp][lane] = sg;
        sums[1][grp][lane] = sb;
        __syncthreads();
        if (grp < 2 && j < d)
            part[(static_cast<uint64_t>(blockIdx.y) * 2 + grp) * d + j] =
                ((sums[grp][0][lane] + sums[grp][1][lane]) + sums[grp][2][lane]) + sums[grp][3][lane];
        __syncthreads();  // the sums are free for the next columns
    }
}

// dgamma and dbeta from `parts` partial rows of [2][d]: 32 columns at a time, 32 groups of rows (g, g + 32, ...)
// whose sums are added in a fixed tree.
__global__ __launch_bounds__(1024) void layernorm_parts_kernel(const float* part, float* dgamma, float* dbeta,
                                                               uint32_t parts, uint32_t d) {
    __shared__ float sums[32][33];
    const uint32_t lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const uint64_t width = 2ull * d;
    for (uint64_t j0 = blockIdx.x * 32ull; j0 < width; j0 += gridDim.x * 32ull) {
        const uint64_t j = j0 + lane;
        float s = 0.0f;
        if (j < width) {
            uint32_t p = grp;
            for (; p + 96 < parts; p += 128) {
                const float* q = part + static_cast<uint64_t>(p) * width + j;
                const float a = q[0], b = q[32 * width], c = q[64 * width], e = q[96 * width];
                s += (a + b) + (c + e);
            }
            for (; p < parts; p += 32) s += part[static_cast<uint64_t>(p) * width + j];
        }
        sums[grp][lane] = s;
        __syncthreads();
        for (uint32_t o = 16; o > 0; o >>= 1) {
            if (grp < o) sums[grp][lane] += sums[grp + o][lane];
            __syncthreads();
        }
        if (grp == 0 && j < width) {  // (a lane reads what it alone writes for the next columns)
            if (j < d) dgamma[j] = sums[0][lane];
            else dbeta[j - d] = sums[0][lane];
        }
    }
}

uint32_t vec_parts(uint32_t rows) { return std::min(ceil_div(rows, 4), kMaxParts); }
uint32_t col_parts(uint32_t rows) { return std::min(ceil_div(rows, kColRows), kMaxParts); }
uint64_t stats_bytes(uint32_t rows) { return (static_cast<uint64_t>(rows) * 8 + 255) / 256 * 256; }

uint64_t norm_ws_bytes(uint32_t rows, uint32_t d) {
    return rows && d ? stats_bytes(rows) + static_cast<uint64_t>(vec_parts(rows)) * 2 * d * 4 : 0;
}

template <typename TD>
void launch_norm_vec(const float* x, const float* gamma, const TD* dy, const float* res, float* dx, float* part,
                     uint32_t rows, uint32_t d, float eps, hipStream_t s) {
    // with weight gradients the rows are strided over the partial rows' workgroups, else each wave takes one
    const unsigned grid = part ? vec_parts(rows) : std::min(ceil_div(rows, 4), kMaxGrid);
    const uint32_t nc = ceil_div(d / 4, 64u);
    if (nc <= 2) layernorm_bwd_vec_kernel<TD, 2><<<grid, 256, 0, s>>>(x, gamma, dy, res, dx, part, rows, d, eps);
    else if (nc <= 3) layernorm_bwd_vec_kernel<TD, 3><<<grid, 256, 0, s>>>(x, gamma, dy, res, dx, part, rows, d, eps);
    else if (nc <= 5) layernorm_bwd_vec_kernel<TD, 5><<<grid, 256, 0, s>>>(x, gamma, dy, res, dx, part, rows, d, eps);
    else if (nc <= 8) layernorm_bwd_vec_kernel<TD, 8><<<grid, 256, 0, s>>>(x, gamma, dy, res, dx, part, rows, d, eps);
    else layernorm_bwd_vec_kernel<TD, 16><<<grid, 256, 0, s>>>(x, gamma, dy, res, dx, part, rows, d, eps);
}

template <typename TD>
void launch_norm(const float* x, const float* gamma, const TD* dy, const float* res, float* dx, float* dgamma,
                 float* dbeta, void* ws, uint32_t rows, uint32_t d, float eps, bool vec, hipStream_t s) {
    float* stats = dgamma ? static_cast<float*>(ws) : nullptr;
    float* part = dgamma ? reinterpret_cast<float*>(static_cast<char*>(ws) + stats_bytes(rows)) : nullptr;
    uint32_t parts;
    if (vec) {
        launch_norm_vec(x, gamma, dy, res, dx, part, rows, d, eps, s);
        parts = vec_parts(rows);
    } else {
        layernorm_bwd_kernel<TD><<<std::min(ceil_div(rows, 4), kMaxGrid), 256, 0, s>>>(x, gamma, dy, res, dx, stats, rows, d, eps);
        if (!dgamma) return;
        const uint32_t per = ceil_div(rows, col_parts(rows));
        parts = ceil_div(rows, per);
        layernorm_cols_kernel<TD><<<dim3(std::min(ceil_div(d, 64), kMaxGrid), parts), 256, 0, s>>>(x, dy, stats, part, rows, d, per);
    }
    if (dgamma) layernorm_parts_kernel<<<std::min(ceil_div(2ull * d, 32), kMaxGrid), 1024, 0, s>>>(part, dgamma, dbeta, parts, d);
}

// Thread (x, y) of the grid takes columns 4 (blockIdx.x * 256 + tid) .. + 3 of rows blockIdx.y, + gridDim.y, ...
// F % 4 == 0, rows 16-byte aligned (8-byte for fp16 dy and dh). dh may be h itself (each thread reads its value and gate
// elements before it writes them).
template <typename T>
__global__ __launch_bounds__(256) void geglu_bwd_vec_kernel(const float* h, const T* dy, T* dh, uint32_t rows, uint32_t F) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const uint32_t f4 = F / 4;
    const uint32_t j = blockIdx.x * 256 + threadIdx.x;
    if (j >= f4) return;
    for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const floatx4* hr = reinterpret_cast<const floatx4*>(h + static_cast<uint64_t>(r) * 2 * F);
        const floatx4 v = hr[j], g = hr[f4 + j];
        const T4 y = reinterpret_cast<const T4*>(dy + static_cast<uint64_t>(r) * F)[j];
        T4 dv, dg;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a, b;
            geglu_grad(v[e], g[e], static_cast<float>(y[e]), a, b);
            dv[e] = static_cast<T>(a);
            dg[e] = static_cast<T>(b);
        }
        T4* out = reinterpret_cast<T4*>(dh + static_cast<uint64_t>(r) * 2 * F);
        out[j] = dv;
        out[f4 + j] = dg;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void geglu_bwd_kernel(const float* h, const T* dy, T* dh, uint32_t rows, uint32_t F) {
    const uint64_t total = static_cast<uint64_t>(rows) * F;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < total; i += static_cast<uint64_t>(gridDim.x) * 256) {
        const uint64_t r = i / F, at = r * 2 * F + i % F;
        float a, b;
        geglu_grad(h[at], h[at + F], static_cast<float>(dy[i]), a, b);
        dh[at] = static_cast<T>(a);
        dh[at + F] = static_cast<T>(b);
    }
}

template <typename T>
void launch_geglu(const float* h, const T* dy, T* dh, uint32_t rows, uint32_t F, hipStream_t s) {
    if (F % 4 == 0 && aligned(h, 16) && aligned(dy, 4 * sizeof(T)) && aligned(dh, 4 * sizeof(T))) {
        const unsigned gx = ceil_div(F / 4, 256);
        const unsigned gy = static_cast<unsigned>(std::min<uint64_t>(rows, std::max<uint64_t>(1, 2048 / gx)));
        geglu_bwd_vec_kernel<T><<<dim3(gx, gy), 256, 0, s>>>(h, dy, dh, rows, F);
    } else {
        const uint64_t wgs = (static_cast<uint64_t>(rows) * F + 255) / 256;
        geglu_bwd_kernel<T><<<static_cast<unsigned>(std::min<uint64_t>(wgs, 2048)), 256, 0, s>>>(h, dy, dh, rows, F);
    }
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" uint64_t mi_layernorm_bwd_ws_bytes(uint32_t rows, uint32_t d) { return norm_ws_bytes(rows, d); }

extern "C" int mi_layernorm_bwd(const float* x, const float* gamma, const void* dy, int dy_dtype, const float* res, float* dx,
                                float* dgamma, float* dbeta, uint32_t rows, uint32_t d, float eps, void* workspace,
                                uint64_t workspace_bytes, void* stream) {
    const char* fn = "mi_layernorm_bwd";
    if (!x || !dy || !dx) return fail(MI_ERR_INVALID_ARG, "%s: null pointer", fn);
    if (dy_dtype != MI_F32 && dy_dtype != MI_F16) return fail(MI_ERR_INVALID_ARG, "%s: dy_dtype %d", fn, dy_dtype);
    if ((dgamma == nullptr) != (dbeta == nullptr)) return fail(MI_ERR_INVALID_ARG, "%s: dgamma and dbeta go together", fn);
    if (d == 0) return fail(MI_ERR_INVALID_ARG, "%s: d == 0", fn);
    if (rows > kMaxRows || d > kMaxCols) return fail(MI_ERR_UNSUPPORTED, "%s: rows %u > 2^31 or d %u > 2^30", fn, rows, d);
    const uint64_t ey = dy_dtype == MI_F16 ? 2 : 4;
    if (!aligned(x, 4) || !aligned(gamma, 4) || !aligned(dy, ey) || !aligned(res, 4) || !aligned(dx, 4) ||
        !aligned(dgamma, 4) || !aligned(dbeta, 4))
        return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
    const uint64_t n = static_cast<uint64_t>(rows) * d, cols = static_cast<uint64_t>(d) * 4;
    const struct {
        const void* p;
        uint64_t bytes;
    } in[4] = {{x, n * 4}, {gamma, cols}, {dy, n * ey}, {res, n * 4}}, out[3] = {{dx, n * 4}, {dgamma, cols}, {dbeta, cols}};
    const uint64_t need = dgamma ? norm_ws_bytes(rows, d) : 0;
    for (int o = 0; o < 3; ++o) {
        for (int i = 0; i < 4; ++i)
            if (overlaps(out[o].p, out[o].bytes, in[i].p, in[i].bytes) && !(o == 0 && i == 3 && res == dx))
                return fail(MI_ERR_ALIASING, "%s: an output overlaps an input (only dx may be res itself)", fn);
        for (int q = 0; q < o; ++q)
            if (overlaps(out[o].p, out[o].bytes, out[q].p, out[q].bytes))
                return fail(MI_ERR_ALIASING, "%s: outputs overlap each other", fn);
    }
    if (need) {
        if (!workspace || workspace_bytes < need)
            return fail(MI_ERR_INVALID_ARG, "%s: workspace %llu bytes < %llu needed for dgamma and dbeta", fn,
                        static_cast<unsigned long long>(workspace ? workspace_bytes : 0), static_cast<unsigned long long>(need));
        if (!aligned(workspace, 16)) return fail(MI_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
        for (int i = 0; i < 4; ++i)
            if (overlaps(workspace, need, in[i].p, in[i].bytes) || (i < 3 && overlaps(workspace, need, out[i].p, out[i].bytes)))
                return fail(MI_ERR_ALIASING, "%s: workspace overlaps a tensor", fn);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows == 0) {
        // sums over no rows
        if (dgamma) layernorm_parts_kernel<<<std::min(ceil_div(2ull * d, 32), kMaxGrid), 1024, 0, s>>>(nullptr, dgamma, dbeta, 0, d);
        return check_launch(fn);
    }
    const bool vec = d % 4 == 0 && d <= kLayerNormVecMax && aligned(x, 16) && aligned(dx, 16) && aligned(dy, 4 * ey) &&
                     (!gamma || aligned(gamma, 16)) && (!res || aligned(res, 16));
    if (dy_dtype == MI_F16)
        launch_norm(x, gamma, static_cast<const _Float16*>(dy), res, dx, dgamma, dbeta, workspace, rows, d, eps, vec, s);
    else
        launch_norm(x, gamma, static_cast<const float*>(dy), res, dx, dgamma, dbeta, workspace, rows, d, eps, vec, s);
    return check_launch(fn);
}

extern "C" int mi_geglu_bwd(const float* h, const void* dy, void* dh, int dtype, uint32_t rows, uint32_t F, void* stream) {
    const char* fn = "mi_geglu_bwd";
    if (!h || !dy || !dh) return fail(MI_ERR_INVALID_ARG, "%s: null pointer", fn);
    if (dtype != MI_F32 && dtype != MI_F16) return fail(MI_ERR_INVALID_ARG, "%s: dtype %d", fn, dtype);
    if (rows == 0 || F == 0) return MI_OK;
    if (rows > kMaxRows) return fail(MI_ERR_UNSUPPORTED, "%s: rows %u > 2^31", fn, rows);
    const uint64_t e = dtype == MI_F16 ? 2 : 4, n = static_cast<uint64_t>(rows) * F;
    if (!aligned(h, 4) || !aligned(dy, e) || !aligned(dh, e))
        return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
    if (overlaps(dh, n * 2 * e, dy, n * e) || (overlaps(dh, n * 2 * e, h, n * 8) && !(dtype == MI_F32 && dh == h)))
        return fail(MI_ERR_ALIASING, "%s: dh overlaps an input (an fp32 dh may be h itself)", fn);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == MI_F16) launch_geglu(h, static_cast<const _Float16*>(dy), static_cast<_Float16*>(dh), rows, F, s);
    else launch_geglu(h, static_cast<const float*>(dy), static_cast<float*>(dh), rows, F, s);
    return check_launch(fn);
}

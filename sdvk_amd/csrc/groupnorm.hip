// groupnorm.hip -- GroupNorm with an optional SiLU on channels-last tensors for gfx950, forward and backward.
//
// x [batch][pixels][C]; group g of an image is channels g cg .. g cg + cg - 1 (cg = C / groups) of all its pixels, n = pixels cg
// values with mean m and variance v:
//   xh = (x - m) inv, inv = 1 / sqrt(v + eps);  z = xh gamma + beta;  y = z or z sigma(z)
//   w  = dy act'(z);  dgamma = sum over batch and pixels of w xh,  dbeta = sum of w
//   dx = inv (w gamma - mean_g(w gamma) - xh mean_g(w gamma xh)) (+ res)
// y may leave as 8-bit rows (one pixel's channels) with a scale each: quant.hpp.
//
// Statistics: an image's rows are cut into chunks. A chunk's sums are taken about a shift, the mean of some of its own values,
// so that neither a large common mean nor an outlier cancels the variance (the shift lies within sqrt(n / m) standard
// deviations of the chunk's mean, m the values that made it); the chunks' means and variances are then joined in 64 bits.
// A mean is held as two floats, a chunk's and a group's: with the first alone x - m would be off by 2^-24 m, which a large mean over
// a small spread shows.
#include "common.hpp"
#include "quant.hpp"

#include <algorithm>

namespace mi {
namespace {

constexpr uint32_t kMaxGrid = 1u << 20;   // workgroups of a launch that strides over its units
constexpr uint32_t kChunkValues = 16384;  // values of a chunk, at least (but for the last), and ...
constexpr uint32_t kChunkMax = 2048;      // ... rows at most: the longest chain of fp32 additions
constexpr uint32_t kChunks = 256;         // chunks of all images, about: a workgroup per CU (images of 4 M values and more; kChunkValues
                                          // binds the others: 576 x 1280 has 45 chunks)
// Parts (of 16 bytes) that all workgroups together read where each joins an image's statistics by itself; more are joined by a launch of
// its own. us of a call by themselves / by a launch: 576 x 1280 in 8 bits (2^16.9 parts) 13.2 / 14.6, 2304 x 640 in 8 bits (2^18.95) 12.9 /
// 14.8, 2 x 1024 x 1280 in 8 bits (2^19.5) 19.6 / 19.0, 1024 x 2560 fp16 (2^20.2) 14.2 / 14.9, 4096 x 640 fp32 (2^20.6) 16.9 / 15.6,
// 2 x 16384 x 320 fp16 (2^21) 23.3 / 22.5, 16384 x 320 fp16 (2^22) 21.3 / 17.8: equal somewhere from 2^19.5 to 2^20.5.
constexpr uint64_t kJoinParts = 1u << 19;

struct Stat {  // of one group of one image, 16 bytes: what `stats` holds
    float mean, low, inv, zero;
};
struct Part {  // of one group of one chunk: its mean as two floats, var = mean of (x - mean)^2 (their sum could pass fp32's range)
    float mean, low, var, zero;
};
__device__ __forceinline__ Part part_of(double mean, double var) {
    const float hi = static_cast<float>(mean);
    return Part{hi, static_cast<float>(mean - static_cast<double>(hi)), static_cast<float>(var), 0.0f};
}

// Squares are summed in fp32, of differences times a power of two: fp32 values below 1e18 differ by 2e18 at most, and the longest sums
// are 2048 of a column and 4096 of a wave's lanes, 4096 (2e18 / 16)^2 = 6.4e37 in all. (fp16 values stay below 2^17.)
template <typename TX>
constexpr float kDown = sizeof(TX) == 4 ? 0.0625f : 1.0f;
template <typename TX>
constexpr double kUp = 1.0 / kDown<TX>;
// (x - shift) kDown of a shift that is held times kDown: exactly that multiple of the rounded difference
template <typename TX>
__device__ __forceinline__ float down(float x, float shift) {
    if constexpr (sizeof(TX) == 4) return __builtin_fmaf(x, kDown<TX>, -shift);
    return x - shift;
}

struct GnArgs {
    const void* x;
    const float *gamma, *beta;
    void* y;
    float* y_scale;
    Stat* stats;
    Part* part;
    uint32_t batch, pixels, C, groups, cg;
    uint32_t chunk, nchunk;  // rows of a chunk, chunks of an image
    uint32_t cut, ncut;      // rows of a workgroup that stores y or dx, of such workgroups an image
    uint32_t joined;         // stats hold the statistics; 0: they are joined from part
    float eps;
    uint64_t ldx, ldy, sx, sy;
};

struct GnBwdArgs {
    GnArgs f;
    const void *dy, *res;
    void* dx;
    float *dgamma, *dbeta;
    float* cpart;  // [batch][nchunk][2][C]: sums of w and of w xh
    float* gsum;   // [batch][groups][2]: mean(w gamma), mean(w gamma xh)
    float* gpart;  // [batch][nchunk][groups][2]: a chunk's sums of w gamma and w gamma xh
    uint64_t lddy, ldres, lddx, sdy, sres, sdx;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

__device__ __forceinline__ double not_below_zero(double v) { return v < 0.0 ? 0.0 : v; }  // (a NaN stays)

// z = xh gamma + beta as one fma of x - mean: s.low inv gamma is far below beta's rounding unless the mean is large.
struct Coef {
    float mean, a, b;
};
__device__ __forceinline__ Coef coef(const Stat& s, float gamma, float beta) {
    const float a = s.inv * gamma;
    return Coef{s.mean, a, __builtin_fmaf(-s.low, a, beta)};
}
__device__ __forceinline__ float apply(float x, const Coef& k) { return __builtin_fmaf(x - k.mean, k.a, k.b); }

constexpr float kLog2e = 1.44269504088896340736f;
// z sigma(z). The exponential and the reciprocal are the hardware's (1 ulp each); the exponent's argument is off by 2^-24 of
// itself, which is |z| 2^-24 of the result: no more than z's own rounding does to it. Where the exponential overflows (z < -88) or
// its reciprocal is no normal number the result is zero for one below 1e-36.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == MI_ACT_NONE) return z;
    return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
}
// act'(z) = sigma(z) (1 + z sigma(-z)), sigma(-z) = e sigma(z); e is held at 2^126, so that e sigma stays 1
template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == MI_ACT_NONE) return 1.0f;
    const float e = __builtin_amdgcn_exp2f(fminf(-kLog2e * z, 126.0f));
    const float s = __builtin_amdgcn_rcpf(1.0f + e);
    return s * __builtin_fmaf(z, e * s, 1.0f);
}

// ---- any shape and alignment -------------------------------------------------------
//
// Element by element, four or five launches; bound by the loads' latency (2 x 4096 x 640 fp16 backward with the statistics 110 us, by
// vectors 33).

// One group of one chunk per workgroup; two passes over its values, sums in 64 bits.
template <typename TX>
__global__ __launch_bounds__(256) void gn_part_any_kernel(GnArgs a) {
    __shared__ double red[3][4];
    const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const uint64_t units = static_cast<uint64_t>(a.batch) * a.nchunk * a.groups;
    const uint32_t step_r = 256 / a.cg, step_c = 256 % a.cg;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t g = static_cast<uint32_t>(u % a.groups);
        const uint64_t bc = u / a.groups;
        const uint32_t c = static_cast<uint32_t>(bc % a.nchunk), b = static_cast<uint32_t>(bc / a.nchunk);
        const uint32_t r0 = c * a.chunk, rows = min(a.chunk, a.pixels - r0);
        const TX* x = static_cast<const TX*>(a.x) + b * a.sx + r0 * a.ldx + static_cast<uint64_t>(g) * a.cg;
        const uint64_t n = static_cast<uint64_t>(rows) * a.cg;
        const uint32_t first_r = tid / a.cg, first_c = tid % a.cg;
        double s = wave_sum(first_r < rows ? static_cast<double>(x[first_r * a.ldx + first_c]) : 0.0);
        if (lane == 0) red[0][wave] = s;
        __syncthreads();
        const float shift = static_cast<float>(((red[0][0] + red[0][1]) + (red[0][2] + red[0][3])) /
                                               static_cast<double>(min(n, static_cast<uint64_t>(256))));
        double d1 = 0.0, d2 = 0.0;
        for (uint32_t r = first_r, ch = first_c; r < rows;) {
            const double d = static_cast<double>(static_cast<float>(x[r * a.ldx + ch])) - static_cast<double>(shift);
            d1 += d;
            d2 += d * d;
            r += step_r;
            ch += step_c;
            if (ch >= a.cg) {
                ch -= a.cg;
                ++r;
            }
        }
        d1 = wave_sum(d1);
        d2 = wave_sum(d2);
        if (lane == 0) {
            red[1][wave] = d1;
            red[2][wave] = d2;
        }
        __syncthreads();
        if (tid == 0) {
            d1 = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
            d2 = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
            const double rest = d1 / static_cast<double>(n);
            a.part[bc * a.groups + g] = part_of(static_cast<double>(shift) + rest, not_below_zero(d2 - d1 * rest) / static_cast<double>(n));
        }
        __syncthreads();  // the sums are free for the next unit
    }
}

// Sums of the chunks' means and deviations about `ref`, in 64 bits, over the chunks first, first + n, ... of a group whose parts begin at
// p: (sum of values - ref, sum of squares about ref). Eight chunks' loads are in flight: one after another they would cost a
// round trip each.
__device__ __forceinline__ void join(const GnArgs& a, const Part* p, uint32_t first, uint32_t n, double ref, double& s1, double& s2) {
    s1 = s2 = 0.0;
    for (uint32_t c0 = first; c0 < a.nchunk; c0 += 8 * n) {
        Part q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = p[static_cast<uint64_t>(min(c0 + i * n, a.nchunk - 1)) * a.groups];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t c = c0 + i * n;
            if (c < a.nchunk) {
                const double k = static_cast<double>(min(a.chunk, a.pixels - c * a.chunk)) * a.cg;
                const double d = (static_cast<double>(q[i].mean) - ref) + static_cast<double>(q[i].low);
                s1 += k * d;
                s2 += k * (static_cast<double>(q[i].var) + d * d);
            }
        }
    }
}
__device__ __forceinline__ Stat stat_of(const GnArgs& a, double ref, double s1, double s2) {
    const double total = static_cast<double>(a.pixels) * a.cg, off = s1 / total, mean = ref + off;
    const double var = not_below_zero(s2 - s1 * off) / total;
    const float hi = static_cast<float>(mean);
    return Stat{hi, static_cast<float>(mean - static_cast<double>(hi)), static_cast<float>(1.0 / sqrt(var + static_cast<double>(a.eps))), 0.0f};
}

// Joins the chunks of a group, a wave each.
__global__ __launch_bounds__(256) void gn_join_kernel(GnArgs a) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t units = static_cast<uint64_t>(a.batch) * a.groups;
    for (uint64_t u = blockIdx.x * 4ull + (threadIdx.x >> 6); u < units; u += gridDim.x * 4ull) {
        const Part* p = a.part + u / a.groups * a.nchunk * a.groups + u % a.groups;
        const Part first = p[0];
        const double ref = static_cast<double>(first.mean) + static_cast<double>(first.low);
        double s1, s2;
        join(a, p, lane, 64, ref, s1, s2);
        s1 = wave_sum(s1);
        s2 = wave_sum(s2);
        if (lane == 0) a.stats[u] = stat_of(a, ref, s1, s2);
    }
}

// A wave takes a row at a time.
template <typename TX, typename TY, int ACT>
__global__ __launch_bounds__(256) void gn_apply_any_kernel(GnArgs a) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t rows = static_cast<uint64_t>(a.batch) * a.pixels;
    for (uint64_t row = blockIdx.x * 4ull + (threadIdx.x >> 6); row < rows; row += gridDim.x * 4ull) {
        const uint64_t b = row / a.pixels, r = row % a.pixels;
        const TX* x = static_cast<const TX*>(a.x) + b * a.sx + r * a.ldx;
        TY* y = static_cast<TY*>(a.y) + b * a.sy + r * a.ldy;
        const Stat* st = a.stats + b * a.groups;
        auto value = [&](uint32_t c) {
            const Coef k = coef(st[c / a.cg], a.gamma ? a.gamma[c] : 1.0f, a.beta ? a.beta[c] : 0.0f);
            return activate<ACT>(apply(static_cast<float>(x[c]), k));
        };
        if constexpr (sizeof(TY) == 1) {
            uint32_t top = 0;
            for (uint32_t c = lane; c < a.C; c += 64) top = max(top, magnitude_bits(value(c)));
            const RowScale s = row_scale(wave_max(top));
            for (uint32_t c = lane; c < a.C; c += 64) y[c] = static_cast<int8_t>(quant_code(value(c), s));
            if (lane == 0) a.y_scale[row] = s.scale;
        } else {
            for (uint32_t c = lane; c < a.C; c += 64) y[c] = static_cast<TY>(value(c));
        }
    }
}

// Sums of w and w xh over a chunk's rows, 64 channels at a time: four row groups of a workgroup, added in order.
template <typename TX, typename TD, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_cols_any_kernel(GnBwdArgs a) {
    __shared__ float sums[2][4][64];
    const GnArgs& f = a.f;
    const uint32_t lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
    const uint32_t blocks = (f.C + 63) / 64;
    const uint64_t units = static_cast<uint64_t>(f.batch) * f.nchunk * blocks;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t c = static_cast<uint32_t>(u % blocks) * 64 + lane;
        const uint64_t bc = u / blocks, b = bc / f.nchunk;
        const uint64_t r0 = (bc % f.nchunk) * f.chunk;
        const uint32_t rows = min(f.chunk, static_cast<uint32_t>(f.pixels - r0));
        float s1 = 0.0f, s2 = 0.0f;
        if (c < f.C) {
            const Stat st = f.stats[b * f.groups + c / f.cg];
            const Coef one = coef(st, 1.0f, 0.0f);
            const float gamma = f.gamma ? f.gamma[c] : 1.0f, beta = f.beta ? f.beta[c] : 0.0f;
            const TX* x = static_cast<const TX*>(f.x) + b * f.sx + r0 * f.ldx + c;
            const TD* dy = static_cast<const TD*>(a.dy) + b * a.sdy + r0 * a.lddy + c;
            for (uint32_t r = grp; r < rows; r += 4) {
                const float xh = apply(static_cast<float>(x[r * f.ldx]), one);
                const float w = static_cast<float>(dy[r * a.lddy]) * slope<ACT>(__builtin_fmaf(xh, gamma, beta));
                s1 += w;
                s2 += w * xh;
            }
        }
        sums[0][grp][lane] = s1;
        sums[1][grp][lane] = s2;
        __syncthreads();
        if (grp < 2 && c < f.C)
            a.cpart[(bc * 2 + grp) * f.C + c] = ((sums[grp][0][lane] + sums[grp][1][lane]) + sums[grp][2][lane]) + sums[grp][3][lane];
        __syncthreads();  // the sums are free for the next unit
    }
}

// A group's sums over the chunks' columns (a wave each), in 64 bits.
__global__ __launch_bounds__(256) void gn_bwd_groups_kernel(GnBwdArgs a) {
    const GnArgs& f = a.f;
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t units = static_cast<uint64_t>(f.batch) * f.groups;
    for (uint64_t u = blockIdx.x * 4ull + (threadIdx.x >> 6); u < units; u += gridDim.x * 4ull) {
        const uint64_t b = u / f.groups;
        const uint32_t c0 = static_cast<uint32_t>(u % f.groups) * f.cg;
        const float* p = a.cpart + b * f.nchunk * 2 * f.C;
        double s1 = 0.0, s2 = 0.0;
        for (uint32_t k = 0; k < f.nchunk; ++k, p += 2ull * f.C)
            for (uint32_t c = lane; c < f.cg; c += 64) {
                const double gamma = f.gamma ? static_cast<double>(f.gamma[c0 + c]) : 1.0;
                s1 += gamma * static_cast<double>(p[c0 + c]);
                s2 += gamma * static_cast<double>(p[f.C + c0 + c]);
            }
        const double n = static_cast<double>(f.pixels) * f.cg;
        s1 = wave_sum(s1) / n;
        s2 = wave_sum(s2) / n;
        if (lane == 0) {
            a.gsum[2 * u] = static_cast<float>(s1);
            a.gsum[2 * u + 1] = static_cast<float>(s2);
        }
    }
}

// dgamma and dbeta: 64 channels at a time, four groups of partial rows, in 64 bits. parts == 0: sums over nothing.
__global__ __launch_bounds__(256) void gn_bwd_params_kernel(const float* cpart, float* dgamma, float* dbeta, uint64_t parts, uint32_t C) {
    __shared__ double sums[2][4][64];
    const uint32_t lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
    for (uint32_t c0 = blockIdx.x * 64; c0 < C; c0 += gridDim.x * 64) {
        const uint32_t c = c0 + lane;
        double s1 = 0.0, s2 = 0.0;
        if (c < C)
            for (uint64_t p = grp; p < parts; p += 4) {
                s1 += static_cast<double>(cpart[p * 2 * C + c]);
                s2 += static_cast<double>(cpart[(p * 2 + 1) * C + c]);
            }
        sums[0][grp][lane] = s1;
        sums[1][grp][lane] = s2;
        __syncthreads();
        if (grp < 2 && c < C) {
            const double s = (sums[grp][0][lane] + sums[grp][1][lane]) + (sums[grp][2][lane] + sums[grp][3][lane]);
            (grp ? dgamma : dbeta)[c] = static_cast<float>(s);
        }
        __syncthreads();
    }
}

template <typename TX, typename TD, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_apply_any_kernel(GnBwdArgs a) {
    const GnArgs& f = a.f;
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t rows = static_cast<uint64_t>(f.batch) * f.pixels;
    for (uint64_t row = blockIdx.x * 4ull + (threadIdx.x >> 6); row < rows; row += gridDim.x * 4ull) {
        const uint64_t b = row / f.pixels, r = row % f.pixels;
        const TX* x = static_cast<const TX*>(f.x) + b * f.sx + r * f.ldx;
        const TD* dy = static_cast<const TD*>(a.dy) + b * a.sdy + r * a.lddy;
        const TX* res = a.res ? static_cast<const TX*>(a.res) + b * a.sres + r * a.ldres : nullptr;
        TX* dx = static_cast<TX*>(a.dx) + b * a.sdx + r * a.lddx;
        for (uint32_t c = lane; c < f.C; c += 64) {
            const uint64_t g = b * f.groups + c / f.cg;
            const Stat st = f.stats[g];
            const float gamma = f.gamma ? f.gamma[c] : 1.0f, beta = f.beta ? f.beta[c] : 0.0f;
            const float xh = apply(static_cast<float>(x[c]), coef(st, 1.0f, 0.0f));
            const float w = static_cast<float>(dy[c]) * slope<ACT>(__builtin_fmaf(xh, gamma, beta));
            const float t = __builtin_fmaf(w, gamma, -a.gsum[2 * g]);
            const float d = st.inv * __builtin_fmaf(-xh, a.gsum[2 * g + 1], t);
            dx[c] = static_cast<TX>(res ? d + static_cast<float>(res[c]) : d);
        }
    }
}

// ---- rows of 16-byte vectors ---------------------------------------------------------
//
// C and the strides multiples of a vector (16 bytes of x: E values), 16-byte aligned tensors, C <= 4096, groups <= 256. A workgroup of T
// threads takes a chunk: thread t holds the columns E (t % V) .. + E - 1 (V = C / E vectors a row) of the rows t / V, + T / V, ...,
// with what it needs of its columns in registers.
//
// Statistics: a thread sums x - x0 and its square for each of its columns, x0 the column's first value of its own, and after 17, 65,
// 257 and 1025 rows the mean of those (about the first value alone, an outlier there that makes the variance multiplies the sums' rounding
// by the rows of a thread: of 2048 the variance was 8% off); the threads' sums are joined in 64 bits.
// All of it is bound by memory: every pass reads x once (and dy), and one stores y or dx. One 2^20 x 128 image, fp16 (268 MB): sums 75 us (3.6
// TB/s), join 5, store 85 (6.3 TB/s, part of x from the last-level cache). 2 x 16384 x 320 fp16 (21 MB): 9.5, 3.3 and 9.0 us, of which 2 are
// the launch. Backward 2 x 4096 x 640 fp16 (10 MB a tensor): sums 10.0 us, dx and the weights' gradients 13.0.
constexpr uint32_t kFastChannels = 4096, kFastGroups = 256;
constexpr int kRows = 4;  // rows a thread has in flight

typedef float float2v __attribute__((ext_vector_type(2)));
template <typename T>
struct Vec {
    static constexpr int E = 16 / static_cast<int>(sizeof(T));
    typedef T type __attribute__((ext_vector_type(E)));
};
// E neighbouring values of T, 16-byte aligned at most (eight floats are two vectors).
template <typename T, int E>
struct Run {
    typedef T type __attribute__((ext_vector_type(E), aligned(E * sizeof(T) > 16 ? 16 : E * sizeof(T))));
};

// A group's lanes: the largest power of two (at most 64) of threads that T threads have for each of G groups at once.
__device__ __forceinline__ uint32_t lanes_of(uint32_t T, uint32_t G) {
    uint32_t n = 1;
    while (n < 64 && 2 * n * G <= T) n *= 2;
    return n;
}
template <typename F>
__device__ __forceinline__ F lanes_sum(F v, uint32_t n) {  // over n neighbouring lanes
    for (uint32_t o = 1; o < n; o <<= 1) v += __shfl_xor(v, static_cast<int>(o));
    return v;
}

// The statistics of image b's groups into st[G], by all threads: loaded, or joined from the chunks as gn_join_kernel does.
__device__ __forceinline__ void image_stats(const GnArgs& a, uint64_t b, Stat* st) {
    const uint32_t T = blockDim.x, tid = threadIdx.x;
    if (a.joined) {
        for (uint32_t g = tid; g < a.groups; g += T) st[g] = a.stats[b * a.groups + g];
        __syncthreads();
        return;
    }
    const uint32_t n = lanes_of(T, a.groups), lane = tid % n, per = T / n;
    for (uint32_t g0 = 0; g0 < a.groups; g0 += per) {
        const uint32_t g = min(g0 + tid / n, a.groups - 1);
        const Part* p = a.part + b * a.nchunk * a.groups + g;
        const Part first = p[0];
        const double ref = static_cast<double>(first.mean) + static_cast<double>(first.low);
        double s1, s2;
        join(a, p, lane, n, ref, s1, s2);
        s1 = lanes_sum(s1, n);
        s2 = lanes_sum(s2, n);
        if (lane == 0 && g0 + tid / n < a.groups) st[g] = stat_of(a, ref, s1, s2);
    }
    __syncthreads();
}

// The E values of gamma or beta from column c0 on (`other` without them).
template <int E>
__device__ __forceinline__ void column_values(const float* p, uint32_t c0, float other, float (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = p ? p[c0 + e] : other;
}
// The groups of columns c0 .. c0 + E - 1, by one division.
template <int E>
__device__ __forceinline__ void column_groups(uint32_t c0, uint32_t cg, uint32_t (&g)[E]) {
    uint32_t q = c0 / cg, r = c0 - q * cg;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        g[e] = q;
        if (++r == cg) {
            r = 0;
            ++q;
        }
    }
}

// What a thread needs of E columns from c0 on.
template <int E>
struct Cols {
    float mean[E], a[E], b[E];
    // before the statistics are there: gamma and beta
    __device__ __forceinline__ void load(const GnArgs& f, uint32_t c0) {
        column_values(f.gamma, c0, 1.0f, a);
        column_values(f.beta, c0, 0.0f, b);
    }
    __device__ __forceinline__ void set(const GnArgs& f, const Stat* st, uint32_t c0) {
        uint32_t g[E];
        column_groups(c0, f.cg, g);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const Coef k = coef(st[g[e]], a[e], b[e]);
            mean[e] = k.mean;
            a[e] = k.a;
            b[e] = k.b;
        }
    }
};

// Grid: batch * nchunk. LDS: 3 floats a thread's column. LONG: a thread may take more than kShort rows (the code for them costs 2 x 16384 x
// 320 fp16, eleven rows a thread, 0.1 us of 21.8, 1024 x 1280 fp32 backward 0.2 of 21.7).
constexpr uint32_t kShort = 1 + 4 * kRows;
template <typename TX, bool LONG>
__global__ __launch_bounds__(4096 / Vec<TX>::E) void gn_part_kernel(GnArgs a) {
    constexpr int E = Vec<TX>::E;
    typedef typename Vec<TX>::type VT;
    extern __shared__ __attribute__((aligned(16))) float red[];  // [3][T / V][C]: x0, sums of x - x0, of its square, of values times kDown
    const uint32_t T = blockDim.x, tid = threadIdx.x, V = a.C / E, rows_at = T / V;
    const uint32_t ty = tid / V, tx = tid % V;
    const uint64_t b = blockIdx.x / a.nchunk;
    const uint32_t chunk = blockIdx.x % a.nchunk, r0 = chunk * a.chunk, rows = min(a.chunk, a.pixels - r0);
    const TX* x = static_cast<const TX*>(a.x) + b * a.sx + static_cast<uint64_t>(r0) * a.ldx + tx * E;
    float x0[E], s1[E], s2[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x0[e] = s1[e] = s2[e] = 0.0f;
    const bool in = ty < rows_at;
    if (in && ty < rows) {
        const VT v = *reinterpret_cast<const VT*>(x + ty * a.ldx);
#pragma unroll
        for (int e = 0; e < E; ++e) x0[e] = static_cast<float>(v[e]) * kDown<TX>;
        // (a batch's rows past the chunk repeat its last row and add nothing: one by one they would cost a round trip each)
        uint32_t batch = 0, next = 4;
        for (uint32_t r = ty + rows_at; r < rows; r += kRows * rows_at) {
            VT w[kRows];
#pragma unroll
            for (int i = 0; i < kRows; ++i) w[i] = *reinterpret_cast<const VT*>(x + min(r + i * rows_at, rows - 1) * a.ldx);
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const bool whole = r + i * rows_at < rows;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = whole ? down<TX>(static_cast<float>(w[i][e]), x0[e]) : 0.0f;
                    s1[e] += d;
                    s2[e] = __builtin_fmaf(d, d, s2[e]);
                }
            }
            // the sums so far, about their mean
            if (LONG && ++batch == next && r + kRows * rows_at < rows) {
                next *= 4;
                const float k = static_cast<float>(1 + kRows * batch);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float mean = x0[e] + s1[e] / k;
                    const double t = static_cast<double>(mean) - static_cast<double>(x0[e]), u = static_cast<double>(s1[e]);
                    s2[e] = static_cast<float>(static_cast<double>(s2[e]) + t * (k * t - 2.0 * u));
                    s1[e] = static_cast<float>(u - k * t);
                    x0[e] = mean;
                }
            }
        }
    }
    const uint32_t plane = rows_at * a.C;
    if (in) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t i = ty * a.C + tx * E + e;
            red[i] = x0[e];
            red[plane + i] = s1[e];
            red[2 * plane + i] = s2[e];
        }
    }
    __syncthreads();
    // a group's sums about its first thread's first value, in 64 bits
    const uint32_t n = lanes_of(T, a.groups), lane = tid % n, per = T / n;
    const uint32_t used = min(rows_at, rows);
    for (uint32_t g0 = 0; g0 < a.groups; g0 += per) {
        const uint32_t g = min(g0 + tid / n, a.groups - 1);
        const float ref = red[g * a.cg];
        double t1 = 0.0, t2 = 0.0;
        for (uint32_t y = 0; y < used; ++y) {
            const double k = static_cast<double>((rows - y + rows_at - 1) / rows_at);  // rows of this thread
            for (uint32_t c = lane; c < a.cg; c += n) {
                const uint32_t i = y * a.C + g * a.cg + c;
                const double d = static_cast<double>(red[i]) - static_cast<double>(ref), u = static_cast<double>(red[plane + i]);
                t1 += u + k * d;
                t2 += static_cast<double>(red[2 * plane + i]) + d * (2.0 * u + k * d);
            }
        }
        t1 = lanes_sum(t1, n);
        t2 = lanes_sum(t2, n);
        if (lane == 0 && g0 + tid / n < a.groups) {
            const double each = 1.0 / (static_cast<double>(rows) * a.cg), rest = t1 * each;
            a.part[static_cast<uint64_t>(blockIdx.x) * a.groups + g] =
                part_of((static_cast<double>(ref) + rest) * kUp<TX>, not_below_zero(t2 - t1 * rest) * each * (kUp<TX> * kUp<TX>));
        }
    }
}

// Grid: batch * ncut, an image's workgroups from its last rows to its first: those that the statistics have read last are still
// in the last-level cache. LDS: the statistics.
template <typename TX, typename TY, int ACT>
__global__ __launch_bounds__(4096 / Vec<TX>::E) void gn_apply_kernel(GnArgs a) {
    constexpr int E = Vec<TX>::E;
    typedef typename Vec<TX>::type VT;
    typedef typename Run<TY, E>::type YT;
    extern __shared__ __attribute__((aligned(16))) Stat st[];
    const uint32_t T = blockDim.x, tid = threadIdx.x, V = a.C / E, rows_at = T / V;
    const uint32_t ty = tid / V, tx = tid % V;
    const uint32_t wg = gridDim.x - 1 - blockIdx.x;
    const uint64_t b = wg / a.ncut;
    const uint32_t r0 = wg % a.ncut * a.cut, rows = min(a.cut, a.pixels - r0);
    const TX* x = static_cast<const TX*>(a.x) + b * a.sx + static_cast<uint64_t>(r0) * a.ldx + tx * E;
    // the first rows are on their way while the statistics are joined
    VT w[kRows];
    auto load = [&](uint32_t r) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) w[i] = *reinterpret_cast<const VT*>(x + min(r + i * rows_at, rows - 1) * a.ldx);
    };
    load(ty);
    Cols<E> k;
    k.load(a, tx * E);
    image_stats(a, b, st);
    if (!a.joined && r0 == 0 && a.stats)
        for (uint32_t g = tid; g < a.groups; g += T) a.stats[b * a.groups + g] = st[g];
    if (ty >= rows_at) return;
    k.set(a, st, tx * E);
    TY* y = static_cast<TY*>(a.y) + b * a.sy + static_cast<uint64_t>(r0) * a.ldy + tx * E;
    auto store = [&](uint32_t r, const VT& v) {
        YT o;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = static_cast<TY>(activate<ACT>(__builtin_fmaf(static_cast<float>(v[e]) - k.mean[e], k.a[e], k.b[e])));
        *reinterpret_cast<YT*>(y + r * a.ldy) = o;
    };
    for (uint32_t r = ty; r < rows; r += kRows * rows_at) {
        if (r != ty) load(r);
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (r + i * rows_at < rows) store(r + i * rows_at, w[i]);
    }
}

// 8-bit rows: a wave takes two rows at a time, four columns (lane + 64 i) each, so that a row's largest value is the wave's. Grid: batch *
// ncut, T threads. 2 x 4096 x 640 fp16 7.1 us (16 MB), bound by the instructions of the quantiser and of the statistics' use.
template <typename TX, int ACT, int NV, int T>
__global__ __launch_bounds__(T) void gn_apply_i8_kernel(GnArgs a) {
    typedef TX VT __attribute__((ext_vector_type(4)));
    extern __shared__ __attribute__((aligned(16))) Stat st[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, v4 = a.C / 4;
    const uint32_t wg = gridDim.x - 1 - blockIdx.x;
    const uint64_t b = wg / a.ncut;
    const uint32_t r0 = wg % a.ncut * a.cut, rows = min(a.cut, a.pixels - r0);
    const TX* x = static_cast<const TX*>(a.x) + b * a.sx + static_cast<uint64_t>(r0) * a.ldx;
    int8_t* y = static_cast<int8_t*>(a.y) + b * a.sy + static_cast<uint64_t>(r0) * a.ldy;
    constexpr int kPair = NV > 10 ? 1 : 2;  // (16 vectors leave registers for one row)
    constexpr uint32_t kWaves = T / 64;
    VT v[kPair][NV];
    auto load = [&](uint32_t r) {
#pragma unroll
        for (int u = 0; u < kPair; ++u)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                v[u][i] = *reinterpret_cast<const VT*>(x + min(r + u * kWaves, rows - 1) * a.ldx + min(lane + 64 * i, v4 - 1) * 4);
    };
    load(tid >> 6);  // on their way while the statistics are joined
    Cols<4> k[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) k[i].load(a, min(lane + 64 * i, v4 - 1) * 4);
    image_stats(a, b, st);
    if (!a.joined && r0 == 0 && a.stats)
        for (uint32_t g = tid; g < a.groups; g += T) a.stats[b * a.groups + g] = st[g];
#pragma unroll
    for (int i = 0; i < NV; ++i) k[i].set(a, st, min(lane + 64 * i, v4 - 1) * 4);
    for (uint32_t r = tid >> 6; r < rows; r += kPair * kWaves) {
        if (r != tid >> 6) load(r);
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
            const uint32_t row = r + u * kWaves;
            if (row >= rows) break;  // (the wave's: every lane agrees)
            float z[NV][4];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z[i][e] = activate<ACT>(__builtin_fmaf(static_cast<float>(v[u][i][e]) - k[i].mean[e], k[i].a[e], k[i].b[e]));
                    top = max(top, magnitude_bits(z[i][e]));  // (lanes past the row repeat its last columns)
                }
            const RowScale s = row_scale(wave_max(top));
            uint32_t w[NV];
            quant_codes<NV * 4>([&](int i) { return z[i / 4][i % 4]; }, s, w);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (lane + 64 * i < v4) *reinterpret_cast<uint32_t*>(y + row * a.ldy + (lane + 64 * i) * 4) = w[i];
            if (lane == 0) a.y_scale[b * a.pixels + r0 + row] = s.scale;
        }
    }
}

// Sums of a chunk's w and w xh for each column, and of w gamma and w gamma xh for each group. Grid: batch * nchunk. LDS: the
// statistics, then 2 floats a thread's column.
template <typename TX, typename TD, int ACT>
__global__ __launch_bounds__(4096 / Vec<TX>::E) void gn_bwd_cols_kernel(GnBwdArgs a) {
    constexpr int E = Vec<TX>::E;
    typedef typename Vec<TX>::type VT;
    typedef typename Run<TD, E>::type DT;
    extern __shared__ __attribute__((aligned(16))) Stat st[];
    const GnArgs& f = a.f;
    float* const red = reinterpret_cast<float*>(st + f.groups);
    const uint32_t T = blockDim.x, tid = threadIdx.x, V = f.C / E, rows_at = T / V;
    const uint32_t ty = tid / V, tx = tid % V;
    const uint64_t b = blockIdx.x / f.nchunk;
    const uint32_t chunk = blockIdx.x % f.nchunk, r0 = chunk * f.chunk, rows = min(f.chunk, f.pixels - r0);
    const TX* x = static_cast<const TX*>(f.x) + b * f.sx + static_cast<uint64_t>(r0) * f.ldx + tx * E;
    const TD* dy = static_cast<const TD*>(a.dy) + b * a.sdy + static_cast<uint64_t>(r0) * a.lddy + tx * E;
    VT v[2];
    DT d[2];
    auto load = [&](uint32_t r) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t q = min(r + i * rows_at, rows - 1);
            v[i] = *reinterpret_cast<const VT*>(x + q * f.ldx);
            d[i] = *reinterpret_cast<const DT*>(dy + q * a.lddy);
        }
    };
    load(ty);  // on their way while the statistics are joined
    float mean[E], inv[E], low[E], gamma[E], beta[E], s1[E], s2[E];
    column_values(f.gamma, tx * E, 1.0f, gamma);
    column_values(f.beta, tx * E, 0.0f, beta);
    image_stats(f, b, st);
    if (!f.joined && chunk == 0)
        for (uint32_t g = tid; g < f.groups; g += T) f.stats[b * f.groups + g] = st[g];
    const uint32_t plane = rows_at * f.C;
    if (ty < rows_at) {
        uint32_t g[E];
        column_groups(tx * E, f.cg, g);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const Coef one = coef(st[g[e]], 1.0f, 0.0f);
            mean[e] = one.mean;
            inv[e] = one.a;
            low[e] = one.b;
            s1[e] = s2[e] = 0.0f;
        }
        auto add = [&](const VT& vr, const DT& dr, bool whole) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float xh = __builtin_fmaf(static_cast<float>(vr[e]) - mean[e], inv[e], low[e]);
                const float w = static_cast<float>(dr[e]) * slope<ACT>(__builtin_fmaf(xh, gamma[e], beta[e]));
                s1[e] += whole ? w : 0.0f;
                s2[e] = whole ? __builtin_fmaf(w, xh, s2[e]) : s2[e];
            }
        };
        for (uint32_t r = ty; r < rows; r += 2 * rows_at) {
            if (r != ty) load(r);
#pragma unroll
            for (int i = 0; i < 2; ++i) add(v[i], d[i], r + i * rows_at < rows);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t i = ty * f.C + tx * E + e;
            red[i] = s1[e];
            red[plane + i] = s2[e];
        }
    }
    __syncthreads();
    // each column over the threads that share it; the sums stay in the first row's places for the groups
    float* const out = a.cpart + static_cast<uint64_t>(blockIdx.x) * 2 * f.C;
    for (uint32_t c = tid; c < f.C; c += T) {
        float u1 = red[c], u2 = red[plane + c];
        for (uint32_t y = 1; y < rows_at; ++y) {
            u1 += red[y * f.C + c];
            u2 += red[plane + y * f.C + c];
        }
        out[c] = u1;
        out[f.C + c] = u2;
        const float gamma = f.gamma ? f.gamma[c] : 1.0f;
        red[c] = u1 * gamma;
        red[plane + c] = u2 * gamma;
    }
    __syncthreads();
    const uint32_t n = lanes_of(T, f.groups), lane = tid % n, per = T / n;
    for (uint32_t g0 = 0; g0 < f.groups; g0 += per) {
        const uint32_t g = min(g0 + tid / n, f.groups - 1);
        double t1 = 0.0, t2 = 0.0;
        for (uint32_t c = lane; c < f.cg; c += n) {
            t1 += static_cast<double>(red[g * f.cg + c]);
            t2 += static_cast<double>(red[plane + g * f.cg + c]);
        }
        t1 = lanes_sum(t1, n);
        t2 = lanes_sum(t2, n);
        if (lane == 0 && g0 + tid / n < f.groups) {
            float* const o = a.gpart + (static_cast<uint64_t>(blockIdx.x) * f.groups + g) * 2;
            o[0] = static_cast<float>(t1);
            o[1] = static_cast<float>(t2);
        }
    }
}

// dx. Grid: batch * ncut, then (with dgamma) the workgroups of the weights' gradients, 32 columns each. LDS: the statistics, the groups'
// means (two floats each), or 32 doubles for each 32 threads.
template <typename TX, typename TD, int ACT>
__global__ __launch_bounds__(4096 / Vec<TX>::E) void gn_bwd_apply_kernel(GnBwdArgs a) {
    constexpr int E = Vec<TX>::E;
    typedef typename Vec<TX>::type VT;
    typedef typename Run<TD, E>::type DT;
    extern __shared__ __attribute__((aligned(16))) Stat st[];
    const GnArgs& f = a.f;
    const uint32_t T = blockDim.x, tid = threadIdx.x;
    const uint32_t images = f.batch * f.ncut;
    if (blockIdx.x >= images) {
        double* const sums = reinterpret_cast<double*>(st);
        const uint32_t lane = tid & 31, grp = tid >> 5, groups = T >> 5, parts = f.batch * f.nchunk;
        const uint32_t j = (blockIdx.x - images) * 32 + lane;
        double s = 0.0;
        if (j < 2 * f.C) {
            const float* q = a.cpart + j;
            const uint64_t w = 2ull * f.C;
            uint32_t p = grp;
            for (; p + 3 * groups < parts; p += 4 * groups) {
                const float v0 = q[p * w], v1 = q[(p + groups) * w], v2 = q[(p + 2 * groups) * w], v3 = q[(p + 3 * groups) * w];
                s += (static_cast<double>(v0) + static_cast<double>(v1)) + (static_cast<double>(v2) + static_cast<double>(v3));
            }
            for (; p < parts; p += groups) s += static_cast<double>(q[p * w]);
        }
        sums[tid] = s;
        __syncthreads();
        if (grp == 0 && j < 2 * f.C) {
            for (uint32_t i = 1; i < groups; ++i) s += sums[i * 32 + lane];
            if (j < f.C) a.dbeta[j] = static_cast<float>(s);
            else a.dgamma[j - f.C] = static_cast<float>(s);
        }
        return;
    }
    float* const gs = reinterpret_cast<float*>(st + f.groups);
    const uint32_t V = f.C / E, rows_at = T / V, ty = tid / V, tx = tid % V;
    const uint32_t wg = images - 1 - blockIdx.x;
    const uint64_t b = wg / f.ncut;
    const uint32_t r0 = wg % f.ncut * f.cut, rows = min(f.cut, f.pixels - r0);
    const TX* x = static_cast<const TX*>(f.x) + b * f.sx + static_cast<uint64_t>(r0) * f.ldx + tx * E;
    const TD* dy = static_cast<const TD*>(a.dy) + b * a.sdy + static_cast<uint64_t>(r0) * a.lddy + tx * E;
    const TX* res = a.res ? static_cast<const TX*>(a.res) + b * a.sres + static_cast<uint64_t>(r0) * a.ldres + tx * E : nullptr;
    TX* dx = static_cast<TX*>(a.dx) + b * a.sdx + static_cast<uint64_t>(r0) * a.lddx + tx * E;
    VT v[2], s[2];
    DT d[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) s[i][e] = static_cast<TX>(0.0f);
    auto load = [&](uint32_t r) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t q = min(r + i * rows_at, rows - 1);
            v[i] = *reinterpret_cast<const VT*>(x + q * f.ldx);
            d[i] = *reinterpret_cast<const DT*>(dy + q * a.lddy);
            // (a thread's own rows alone: dx may be res, and another thread stores them)
            if (res && r + i * rows_at < rows && ty < rows_at) s[i] = *reinterpret_cast<const VT*>(res + q * a.ldres);
        }
    };
    load(ty);  // on their way while the sums are joined
    float mean[E], inv[E], low[E], gamma[E], beta[E], m1[E], m2[E];
    column_values(f.gamma, tx * E, 1.0f, gamma);
    column_values(f.beta, tx * E, 0.0f, beta);
    for (uint32_t g = tid; g < f.groups; g += T) st[g] = f.stats[b * f.groups + g];
    {
        const uint32_t n = lanes_of(T, f.groups), lane = tid % n, per = T / n;
        const double total = static_cast<double>(f.pixels) * f.cg;
        for (uint32_t g0 = 0; g0 < f.groups; g0 += per) {
            const uint32_t g = min(g0 + tid / n, f.groups - 1);
            const float2v* p = reinterpret_cast<const float2v*>(a.gpart) + b * f.nchunk * f.groups + g;
            double t1 = 0.0, t2 = 0.0;
            for (uint32_t c0 = lane; c0 < f.nchunk; c0 += 8 * n) {
                float2v q[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = p[static_cast<uint64_t>(min(c0 + i * n, f.nchunk - 1)) * f.groups];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c0 + i * n < f.nchunk) {
                        t1 += static_cast<double>(q[i][0]);
                        t2 += static_cast<double>(q[i][1]);
                    }
            }
            t1 = lanes_sum(t1, n);
            t2 = lanes_sum(t2, n);
            if (lane == 0 && g0 + tid / n < f.groups) {
                gs[2 * g] = static_cast<float>(t1 / total);
                gs[2 * g + 1] = static_cast<float>(t2 / total);
            }
        }
    }
    __syncthreads();
    if (ty >= rows_at) return;
    // dx = inv (w gamma - m1 - xh m2)
    uint32_t g[E];
    column_groups(tx * E, f.cg, g);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const Coef one = coef(st[g[e]], 1.0f, 0.0f);
        mean[e] = one.mean;
        inv[e] = one.a;
        low[e] = one.b;
        m1[e] = gs[2 * g[e]];
        m2[e] = gs[2 * g[e] + 1];
    }
    auto store = [&](uint32_t r, const VT& vr, const DT& dr, const VT& sr) {
        VT o;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float xh = __builtin_fmaf(static_cast<float>(vr[e]) - mean[e], inv[e], low[e]);
            const float w = static_cast<float>(dr[e]) * slope<ACT>(__builtin_fmaf(xh, gamma[e], beta[e]));
            const float q = inv[e] * __builtin_fmaf(-xh, m2[e], __builtin_fmaf(w, gamma[e], -m1[e]));
            o[e] = static_cast<TX>(res ? q + static_cast<float>(sr[e]) : q);
        }
        *reinterpret_cast<VT*>(dx + r * a.lddx) = o;
    };
    for (uint32_t r = ty; r < rows; r += 2 * rows_at) {
        if (r != ty) load(r);
        store(r, v[0], d[0], s[0]);
        if (r + rows_at < rows) store(r + rows_at, v[1], d[1], s[1]);
    }
}

// ---- a group in a workgroup's registers --------------------------------------------------
//
// Images of few pixels: a workgroup holds one group of one image, loads it once and stores y: one launch instead of two or three, which
// wait for each other. A thread's unit is VE neighbouring values, NU units at most. The sums are taken about the mean
// that a first sum gives. us this way / in launches: 256 x 1280 fp32 6.2 / 9.7, 2 x 1024 x 1280 fp16 13.2 / 14.8, but 1024 x 1920 fp32 15.5 / 13.6:
// a CU takes 256 bytes of x a thread at most. Backward 256 x 1280 fp32 8.8 / 12.4, 2 x 576 x 1280 fp16 20.4 / 17.0: eight units.
constexpr uint32_t kSlabThreads = 512, kSlabChannels = 1024, kSlabGroups = 1u << 20, kSlabBytes = 256;
constexpr int kBwdSlabUnits = 8;

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_sum32(float v) {
    v = dpp_add<0xb1>(v);   // quad_perm [1, 0, 3, 2]
    v = dpp_add<0x4e>(v);   // quad_perm [2, 3, 0, 1]
    v = dpp_add<0x141>(v);  // row_half_mirror
    v = dpp_add<0x140>(v);  // row_mirror
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
}

template <typename TX, typename TY, int ACT, int VE, int NU>
__global__ __launch_bounds__(512) void gn_slab_kernel(GnArgs a) {
    constexpr uint32_t T = kSlabThreads;
    typedef TX VT __attribute__((ext_vector_type(VE)));
    typedef TY YT __attribute__((ext_vector_type(VE)));
    __shared__ float sums[3][T / 64];
    __shared__ float ca[kSlabChannels], cb[kSlabChannels];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t b = blockIdx.x / a.groups, g = blockIdx.x % a.groups;
    const uint32_t upr = a.cg / VE, units = a.pixels * upr, step_r = T / upr, step_c = T % upr;
    const uint32_t row0 = tid / upr, col0 = tid % upr;
    const TX* x = static_cast<const TX*>(a.x) + b * a.sx + static_cast<uint64_t>(g) * a.cg;
    TY* y = static_cast<TY*>(a.y) + b * a.sy + static_cast<uint64_t>(g) * a.cg;
    for (uint32_t c = tid; c < a.cg; c += T) {
        ca[c] = a.gamma ? a.gamma[g * a.cg + c] : 1.0f;
        cb[c] = a.beta ? a.beta[g * a.cg + c] : 0.0f;
    }
    VT v[NU];
    uint32_t row = row0, col = col0;
    auto next = [&]() {
        row += step_r;
        col += step_c;
        if (col >= upr) {
            col -= upr;
            ++row;
        }
    };
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        const bool in = tid + i * T < units;
        v[i] = *reinterpret_cast<const VT*>(x + (in ? row : 0u) * a.ldx + (in ? col : 0u) * VE);
        next();
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) s += tid + i * T < units ? static_cast<float>(v[i][e]) : 0.0f;
    s = wave_sum32(s);
    if (lane == 0) sums[0][wave] = s;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < T / 64; ++w) t += static_cast<double>(sums[0][w]);
    const float ref = static_cast<float>(t / (static_cast<double>(a.pixels) * a.cg)) * kDown<TX>;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float d = tid + i * T < units ? down<TX>(static_cast<float>(v[i][e]), ref) : 0.0f;
            s1 += d;
            s2 = __builtin_fmaf(d, d, s2);
        }
    s1 = wave_sum32(s1);
    s2 = wave_sum32(s2);
    if (lane == 0) {
        sums[1][wave] = s1;
        sums[2][wave] = s2;
    }
    __syncthreads();
    double d1 = 0.0, d2 = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < T / 64; ++w) {
        d1 += static_cast<double>(sums[1][w]);
        d2 += static_cast<double>(sums[2][w]);
    }
    const Stat st = stat_of(a, ref * kUp<TX>, d1 * kUp<TX>, d2 * (kUp<TX> * kUp<TX>));
    for (uint32_t c = tid; c < a.cg; c += T) {
        const Coef k = coef(st, ca[c], cb[c]);
        ca[c] = k.a;
        cb[c] = k.b;
    }
    if (tid == 0) a.stats[blockIdx.x] = st;
    __syncthreads();
    row = row0;
    col = col0;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        if (tid + i * T < units) {
            YT o;
#pragma unroll
            for (int e = 0; e < VE; ++e)
                o[e] = static_cast<TY>(activate<ACT>(__builtin_fmaf(static_cast<float>(v[i][e]) - st.mean, ca[col * VE + e], cb[col * VE + e])));
            *reinterpret_cast<YT*>(y + row * a.ldy + col * VE) = o;
        }
        next();
    }
}

// The gradients of one group of one image: x and dy are loaded once. The threads in use are a multiple of a row's units, so that a thread's
// columns are the same in all of its rows and their sums stay in registers. part: [batch][2][C] of the weights' gradients, to
// be summed over the images, or NULL; with one image they are stored as they are.
template <typename TX, typename TD, int ACT, int VE, int NU>
__global__ __launch_bounds__(512) void gn_bwd_slab_kernel(GnBwdArgs a, uint32_t recompute) {
    constexpr uint32_t T = kSlabThreads;
    typedef TX VT __attribute__((ext_vector_type(VE)));
    typedef TD DT __attribute__((ext_vector_type(VE)));
    __shared__ float sums[4][T / 64];
    __shared__ float red[2][T * VE];
    const GnArgs& f = a.f;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t b = blockIdx.x / f.groups, g = blockIdx.x % f.groups;
    const uint32_t upr = f.cg / VE, rows_at = T / upr, row0 = tid / upr, col = tid % upr * VE, c0 = g * f.cg + col;
    const bool use = row0 < rows_at;
    const TX* x = static_cast<const TX*>(f.x) + b * f.sx + c0;
    const TD* dy = static_cast<const TD*>(a.dy) + b * a.sdy + c0;
    auto in = [&](int i) { return use && row0 + i * rows_at < f.pixels; };
    VT v[NU];
    DT d[NU];
#pragma unroll
    for (int i = 0; i < NU; ++i) v[i] = *reinterpret_cast<const VT*>(x + (in(i) ? row0 + i * rows_at : 0u) * f.ldx);
#pragma unroll
    for (int i = 0; i < NU; ++i) d[i] = *reinterpret_cast<const DT*>(dy + (in(i) ? row0 + i * rows_at : 0u) * a.lddy);
    float gamma[VE], beta[VE];
    column_values(f.gamma, c0, 1.0f, gamma);
    column_values(f.beta, c0, 0.0f, beta);
    auto total = [&](int k, float s) {  // over the workgroup, in 64 bits over the waves
        s = wave_sum32(s);
        if (lane == 0) sums[k][wave] = s;
    };
    auto read = [&](int k) {
        double t = 0.0;
#pragma unroll
        for (uint32_t w = 0; w < T / 64; ++w) t += static_cast<double>(sums[k][w]);
        return t;
    };
    const double n = static_cast<double>(f.pixels) * f.cg;
    Stat st;
    if (recompute) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) s += in(i) ? static_cast<float>(v[i][e]) : 0.0f;
        total(0, s);
        __syncthreads();
        const float ref = static_cast<float>(read(0) / n) * kDown<TX>;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float q = in(i) ? down<TX>(static_cast<float>(v[i][e]), ref) : 0.0f;
                s1 += q;
                s2 = __builtin_fmaf(q, q, s2);
            }
        total(1, s1);
        total(2, s2);
        __syncthreads();
        st = stat_of(f, ref * kUp<TX>, read(1) * kUp<TX>, read(2) * (kUp<TX> * kUp<TX>));
        __syncthreads();  // the sums are free
    } else {
        st = f.stats[blockIdx.x];
    }
#pragma unroll
    for (int i = 0; i < NU; ++i) asm volatile("" : "+v"(v[i]));
    const Coef one = coef(st, 1.0f, 0.0f);
    float u1[VE], u2[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) u1[e] = u2[e] = 0.0f;
    auto xhat = [&](int i, int e) { return __builtin_fmaf(static_cast<float>(v[i][e]) - one.mean, one.a, one.b); };
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float xh = xhat(i, e), w = static_cast<float>(d[i][e]) * slope<ACT>(__builtin_fmaf(xh, gamma[e], beta[e]));
            u1[e] += in(i) ? w : 0.0f;
            u2[e] = in(i) ? __builtin_fmaf(w, xh, u2[e]) : u2[e];
        }
    float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        t1 += u1[e] * gamma[e];
        t2 += u2[e] * gamma[e];
        red[0][tid * VE + e] = u1[e];
        red[1][tid * VE + e] = u2[e];
    }
    total(0, t1);
    total(3, t2);
    __syncthreads();
    const float m1 = static_cast<float>(read(0) / n), m2 = static_cast<float>(read(3) / n);
    if (a.dgamma) {
        // a column's sums: eight threads, rows r, r + 8, ... each (a row of threads is cg values)
        for (uint32_t j0 = 0; j0 < 2 * f.cg; j0 += T / 8) {
            const uint32_t j = min(j0 + tid / 8, 2 * f.cg - 1), c = j % f.cg;
            const float* q = red[j / f.cg] + c;
            float s = 0.0f;
            for (uint32_t r = tid % 8; r < rows_at; r += 8) s += q[r * f.cg];
            s = lanes_sum(s, 8);
            if (tid % 8 == 0 && j0 + tid / 8 < 2 * f.cg) {
                if (f.batch > 1) a.cpart[(static_cast<uint64_t>(b) * 2 + j / f.cg) * f.C + g * f.cg + c] = s;
                else (j < f.cg ? a.dbeta : a.dgamma)[g * f.cg + c] = s;
            }
        }
    }
    if (!use) return;
    // what the sums took of x and dy is computed again: kept, it would not fit the registers
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        asm volatile("" : "+v"(v[i]));
        asm volatile("" : "+v"(d[i]));
    }
    TX* dx = static_cast<TX*>(a.dx) + b * a.sdx + c0;
    const TX* res = a.res ? static_cast<const TX*>(a.res) + b * a.sres + c0 : nullptr;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
        if (!in(i)) continue;
        const uint64_t r = row0 + i * rows_at;
        VT o, q;
#pragma unroll
        for (int e = 0; e < VE; ++e) q[e] = static_cast<TX>(0.0f);
        if (res) q = *reinterpret_cast<const VT*>(res + r * a.ldres);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float xh = xhat(i, e), w = static_cast<float>(d[i][e]) * slope<ACT>(__builtin_fmaf(xh, gamma[e], beta[e]));
            const float t = st.inv * __builtin_fmaf(-xh, m2, __builtin_fmaf(w, gamma[e], -m1));
            o[e] = static_cast<TX>(res ? t + static_cast<float>(q[e]) : t);
        }
        *reinterpret_cast<VT*>(dx + r * a.lddx) = o;
    }
}

// ---- host ------------------------------------------------------------------------------

constexpr uint32_t kMaxBatch = 1u << 20, kMaxChannels = 1u << 20;
constexpr uint64_t kMaxRows = 1ull << 31;

void set_chunks(GnArgs& a) {
    const uint64_t pixels = std::max(a.pixels, 1u);
    const uint64_t most = std::max<uint64_t>(pixels * a.C / kChunkValues, 1);
    const uint64_t least = (pixels + kChunkMax - 1) / kChunkMax;
    const uint64_t want = std::min(pixels, std::max<uint64_t>(std::min<uint64_t>(most, kChunks / std::max(a.batch, 1u)), least));
    a.chunk = ceil_div(pixels, want);
    a.nchunk = ceil_div(pixels, a.chunk);
    // two workgroups store what one has summed
    a.cut = ceil_div(a.chunk, 2);
    a.ncut = ceil_div(pixels, a.cut);
}

// Threads of a workgroup whose threads take `vectors` columns: the smallest count from 512 on that leaves a tenth idle at most, or the
// one that leaves fewest.
uint32_t threads_for(uint32_t vectors, uint32_t most) {
    uint32_t best = 512;
    float use = 0.0f;
    for (uint32_t t = 512; t <= most; t += 64) {
        const float u = static_cast<float>(t / vectors * vectors) / static_cast<float>(t);
        if (u > use + 0.001f) {
            use = u;
            best = t;
        }
        if (use >= 0.9f) break;
    }
    return best;
}

bool sizes_ok(uint32_t batch, uint32_t pixels, uint32_t channels, uint32_t groups) {
    return channels != 0 && groups != 0 && channels % groups == 0 && batch <= kMaxBatch && channels <= kMaxChannels &&
           static_cast<uint64_t>(batch) * pixels <= kMaxRows;
}

uint64_t up(uint64_t n) { return (n + 255) / 256 * 256; }
uint64_t stat_bytes(const GnArgs& a) { return up(static_cast<uint64_t>(a.batch) * a.groups * sizeof(Stat)); }
uint64_t part_bytes(const GnArgs& a) { return up(static_cast<uint64_t>(a.batch) * a.nchunk * a.groups * sizeof(Part)); }
uint64_t cpart_bytes(const GnArgs& a) { return up(static_cast<uint64_t>(a.batch) * a.nchunk * 2 * a.C * 4); }
uint64_t gpart_bytes(const GnArgs& a) { return up(static_cast<uint64_t>(a.batch) * a.nchunk * a.groups * 8); }
uint64_t gsum_bytes(const GnArgs& a) { return up(static_cast<uint64_t>(a.batch) * a.groups * 8); }

GnArgs sized(uint32_t batch, uint32_t pixels, uint32_t channels, uint32_t groups) {
    GnArgs a{};
    a.batch = batch;
    a.pixels = pixels;
    a.C = channels;
    a.groups = groups;
    a.cg = channels / groups;
    set_chunks(a);
    return a;
}

unsigned grid_of(uint64_t units) { return static_cast<unsigned>(std::min<uint64_t>(units, kMaxGrid)); }

struct Span {
    const void* p;
    uint64_t bytes;
};
// The bytes from a strided tensor's first element to behind its last; false where that passes 2^62.
bool span(const void* p, uint32_t batch, uint32_t pixels, uint32_t C, uint64_t ld, uint64_t s, uint64_t esz, Span& out) {
    const __uint128_t last = static_cast<__uint128_t>(batch - 1) * s + static_cast<__uint128_t>(pixels - 1) * ld + C;
    if (last > (static_cast<__uint128_t>(1) << 60)) return false;
    out = Span{p, static_cast<uint64_t>(last) * esz};
    return true;
}
// Whether no two rows of an output overlap: image after image, or the images' rows in turn.
bool rows_apart(uint32_t batch, uint32_t pixels, uint32_t C, uint64_t ld, uint64_t s) {
    if (batch <= 1) return true;
    const __uint128_t image = static_cast<__uint128_t>(pixels - 1) * ld + C;
    if (pixels <= 1) return s >= C;
    return s >= image || (s >= C && ld >= static_cast<__uint128_t>(batch - 1) * s + C);
}

uint64_t esize(int dtype) { return dtype == MI_F32 ? 4 : dtype == MI_F16 ? 2 : 1; }

// What both directions check of the forward call's arguments, strides filled in. need_y: the forward call itself.
int check_args(const char* fn, const mi_groupnorm_args* g, GnArgs& a, bool need_y, Span& x, Span& y) {
    if (!g) return fail(MI_ERR_INVALID_ARG, "%s: null arguments", fn);
    if (g->x_dtype != MI_F32 && g->x_dtype != MI_F16) return fail(MI_ERR_INVALID_ARG, "%s: x_dtype %d", fn, g->x_dtype);
    if (g->y_dtype != MI_F32 && g->y_dtype != MI_F16 && !(need_y && g->y_dtype == MI_I8))
        return fail(MI_ERR_INVALID_ARG, "%s: y_dtype %d", fn, g->y_dtype);
    if (g->act != MI_ACT_NONE && g->act != MI_ACT_SILU) return fail(MI_ERR_INVALID_ARG, "%s: act %d", fn, g->act);
    if (!(g->eps >= 0.0f) || g->eps > 3.4e38f) return fail(MI_ERR_INVALID_ARG, "%s: eps %g", fn, static_cast<double>(g->eps));
    if (g->channels == 0 || g->groups == 0 || g->channels % g->groups != 0)
        return fail(MI_ERR_INVALID_ARG, "%s: %u channels in %u groups", fn, g->channels, g->groups);
    if (!sizes_ok(g->batch, g->pixels, g->channels, g->groups))
        return fail(MI_ERR_UNSUPPORTED, "%s: batch %u > 2^20, batch * pixels > 2^31 or channels %u > 2^20", fn, g->batch, g->channels);
    a = sized(g->batch, g->pixels, g->channels, g->groups);
    a.x = g->x;
    a.gamma = g->gamma;
    a.beta = g->beta;
    a.y = g->y;
    a.y_scale = g->y_scale;
    a.eps = g->eps;
    a.ldx = g->ldx ? g->ldx : g->channels;
    a.ldy = g->ldy ? g->ldy : g->channels;
    a.sx = g->sx ? g->sx : a.ldx * g->pixels;
    a.sy = g->sy ? g->sy : a.ldy * g->pixels;
    if (g->batch == 0 || g->pixels == 0) return MI_OK;
    if (!g->x || (need_y && !g->y)) return fail(MI_ERR_INVALID_ARG, "%s: null pointer", fn);
    if (need_y && (g->y_dtype == MI_I8) != (g->y_scale != nullptr))
        return fail(MI_ERR_INVALID_ARG, "%s: y_scale belongs to MI_I8 rows", fn);
    if (a.ldx < g->channels || (need_y && a.ldy < g->channels))
        return fail(MI_ERR_INVALID_ARG, "%s: a row stride below %u channels", fn, g->channels);
    if (!span(a.x, a.batch, a.pixels, a.C, a.ldx, a.sx, esize(g->x_dtype), x) ||
        (need_y && !span(a.y, a.batch, a.pixels, a.C, a.ldy, a.sy, esize(g->y_dtype), y)))
        return fail(MI_ERR_UNSUPPORTED, "%s: a tensor spans 2^60 elements or more", fn);
    if (need_y && !rows_apart(a.batch, a.pixels, a.C, a.ldy, a.sy))
        return fail(MI_ERR_INVALID_ARG, "%s: rows of y overlap each other", fn);
    if (!aligned(a.x, esize(g->x_dtype)) || (need_y && !aligned(a.y, esize(g->y_dtype))) || !aligned(a.gamma, 4) || !aligned(a.beta, 4) ||
        !aligned(a.y_scale, 4))
        return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
    if (!aligned(g->stats, 16)) return fail(MI_ERR_ALIGNMENT, "%s: stats must be 16-byte aligned", fn);
    return MI_OK;
}

// No output overlaps an input or another output; same[o] (or -1) names the input that output o may be itself.
int check_overlaps(const char* fn, const Span* out, int nout, const Span* in, int nin, int may_o, int may_i) {
    for (int o = 0; o < nout; ++o) {
        for (int i = 0; i < nin; ++i)
            if (overlaps(out[o].p, out[o].bytes, in[i].p, in[i].bytes) && !(o == may_o && i == may_i && out[o].p == in[i].p))
                return fail(MI_ERR_ALIASING, "%s: an output or the workspace overlaps an input", fn);
        for (int q = 0; q < o; ++q)
            if (overlaps(out[o].p, out[o].bytes, out[q].p, out[q].bytes))
                return fail(MI_ERR_ALIASING, "%s: outputs or the workspace overlap each other", fn);
    }
    return MI_OK;
}

int check_ws(const char* fn, const void* ws, uint64_t have, uint64_t need) {
    if (!ws || have < need)
        return fail(MI_ERR_INVALID_ARG, "%s: workspace %llu bytes < %llu needed", fn, static_cast<unsigned long long>(ws ? have : 0),
                    static_cast<unsigned long long>(need));
    if (!aligned(ws, 16)) return fail(MI_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", fn);
    return MI_OK;
}

// Whether x's rows are whole 16-byte vectors, and so are the same columns of the other tensors (`e` values of `esz` bytes).
template <typename TX>
bool fast_x(const GnArgs& a) {
    constexpr uint32_t E = Vec<TX>::E;
    return a.C % E == 0 && a.C <= kFastChannels && a.groups <= kFastGroups && a.ldx % E == 0 && a.sx % E == 0 && aligned(a.x, 16);
}
bool fast_rows(const void* p, uint64_t ld, uint64_t s, uint32_t e, uint64_t esz) {  // (esz e is a power of two)
    return !p || (ld % e == 0 && s % e == 0 && aligned(p, std::min<uint64_t>(16, e * esz)));
}

// The sums of the chunks. Returns whether they are joined into a.stats (else every workgroup that needs them joins them).
template <typename TX>
bool launch_stats(const GnArgs& a, bool fast, hipStream_t s) {
    if (fast) {
        constexpr uint32_t E = Vec<TX>::E;
        const uint32_t T = threads_for(a.C / E, 4096 / E), rows_at = T / (a.C / E);
        const uint32_t lds = 3 * rows_at * a.C * sizeof(float);
        if (a.chunk > kShort * rows_at) gn_part_kernel<TX, true><<<a.batch * a.nchunk, T, lds, s>>>(a);
        else gn_part_kernel<TX, false><<<a.batch * a.nchunk, T, lds, s>>>(a);
        if (static_cast<uint64_t>(a.nchunk) * a.groups * a.batch * a.ncut <= kJoinParts) return false;
    } else {
        gn_part_any_kernel<TX><<<grid_of(static_cast<uint64_t>(a.batch) * a.nchunk * a.groups), 256, 0, s>>>(a);
    }
    gn_join_kernel<<<grid_of((static_cast<uint64_t>(a.batch) * a.groups + 3) / 4), 256, 0, s>>>(a);
    return true;
}

template <typename TX, typename TY, int ACT>
void launch_apply(const GnArgs& a, hipStream_t s) {
    const uint32_t T = threads_for(a.C / Vec<TX>::E, 4096 / Vec<TX>::E);
    gn_apply_kernel<TX, TY, ACT><<<a.batch * a.ncut, T, a.groups * sizeof(Stat), s>>>(a);
}

template <typename TX, int ACT>
void launch_apply_i8(const GnArgs& a, hipStream_t s) {
    const unsigned grid = a.batch * a.ncut, lds = a.groups * sizeof(Stat);
    const uint32_t nv = ceil_div(a.C / 4, 64u);
    if (nv <= 1) gn_apply_i8_kernel<TX, ACT, 1, 512><<<grid, 512, lds, s>>>(a);
    else if (nv <= 3) gn_apply_i8_kernel<TX, ACT, 3, 512><<<grid, 512, lds, s>>>(a);
    else if (nv <= 5) gn_apply_i8_kernel<TX, ACT, 5, 512><<<grid, 512, lds, s>>>(a);
    else if (nv <= 10) gn_apply_i8_kernel<TX, ACT, 10, 256><<<grid, 256, lds, s>>>(a);
    else gn_apply_i8_kernel<TX, ACT, 16, 256><<<grid, 256, lds, s>>>(a);
}

// Launches gn_slab_kernel for units of VE values where a group fits and its rows allow them.
template <typename TX, typename TY, int ACT, int VE>
bool launch_slab(const GnArgs& a, hipStream_t s) {
    const uint64_t units = static_cast<uint64_t>(a.pixels) * a.cg / VE;
    if (a.cg % VE != 0 || a.cg > kSlabChannels || units > 32 * kSlabThreads || units * VE * sizeof(TX) > kSlabBytes * kSlabThreads || !fast_rows(a.x, a.ldx, a.sx, VE, sizeof(TX)) ||
        !fast_rows(a.y, a.ldy, a.sy, VE, sizeof(TY)))
        return false;
    const unsigned grid = a.batch * a.groups;
    constexpr int kMost = kSlabBytes / (VE * sizeof(TX));
    if (units <= 8 * kSlabThreads) gn_slab_kernel<TX, TY, ACT, VE, 8><<<grid, kSlabThreads, 0, s>>>(a);
    else if (units <= 16 * kSlabThreads) gn_slab_kernel<TX, TY, ACT, VE, 16><<<grid, kSlabThreads, 0, s>>>(a);
    else if constexpr (kMost > 16) gn_slab_kernel<TX, TY, ACT, VE, 32><<<grid, kSlabThreads, 0, s>>>(a);
    return true;
}

template <typename TX, typename TY, int ACT>
void launch_forward(GnArgs a, hipStream_t s) {
    if constexpr (sizeof(TY) != 1) {
        // (a row's scale needs all groups)
        if (static_cast<uint64_t>(a.batch) * a.groups <= kSlabGroups && (launch_slab<TX, TY, ACT, 4>(a, s) || launch_slab<TX, TY, ACT, 2>(a, s))) return;
    }
    const bool fx = fast_x<TX>(a);
    const bool fast = fx && fast_rows(a.y, a.ldy, a.sy, sizeof(TY) == 1 ? 4 : Vec<TX>::E, sizeof(TY));
    a.joined = launch_stats<TX>(a, fx, s);
    if (fast) {
        if constexpr (sizeof(TY) == 1) launch_apply_i8<TX, ACT>(a, s);
        else launch_apply<TX, TY, ACT>(a, s);
        return;
    }
    if (!a.joined) gn_join_kernel<<<grid_of((static_cast<uint64_t>(a.batch) * a.groups + 3) / 4), 256, 0, s>>>(a);
    gn_apply_any_kernel<TX, TY, ACT><<<grid_of((static_cast<uint64_t>(a.batch) * a.pixels + 3) / 4), 256, 0, s>>>(a);
}

template <typename TX, typename TY>
void launch_forward(const GnArgs& a, int act, hipStream_t s) {
    if (act == MI_ACT_SILU) launch_forward<TX, TY, MI_ACT_SILU>(a, s);
    else launch_forward<TX, TY, MI_ACT_NONE>(a, s);
}

template <typename TX>
void launch_forward(const GnArgs& a, int y_dtype, int act, hipStream_t s) {
    if (y_dtype == MI_F32) launch_forward<TX, float>(a, act, s);
    else if (y_dtype == MI_F16) launch_forward<TX, _Float16>(a, act, s);
    else launch_forward<TX, int8_t>(a, act, s);
}

// Launches gn_bwd_slab_kernel for units of VE values where a group fits and its rows allow them.
template <typename TX, typename TD, int ACT, int VE>
bool launch_bwd_slab(const GnBwdArgs& a, bool stats, hipStream_t s) {
    const GnArgs& f = a.f;
    if (f.cg % VE != 0 || f.cg / VE > kSlabThreads) return false;
    const uint32_t rows_at = kSlabThreads / (f.cg / VE);
    const uint64_t units = (static_cast<uint64_t>(f.pixels) + rows_at - 1) / rows_at;  // a thread's
    if (units > kBwdSlabUnits || !fast_rows(f.x, f.ldx, f.sx, VE, sizeof(TX)) || !fast_rows(a.dy, a.lddy, a.sdy, VE, sizeof(TD)) ||
        !fast_rows(a.dx, a.lddx, a.sdx, VE, sizeof(TX)) || !fast_rows(a.res, a.ldres, a.sres, VE, sizeof(TX)))
        return false;
    const unsigned grid = f.batch * f.groups;
    gn_bwd_slab_kernel<TX, TD, ACT, VE, kBwdSlabUnits><<<grid, kSlabThreads, 0, s>>>(a, stats);
    if (a.dgamma && f.batch > 1) gn_bwd_params_kernel<<<grid_of(ceil_div(f.C, 64)), 256, 0, s>>>(a.cpart, a.dgamma, a.dbeta, f.batch, f.C);
    return true;
}

template <typename TX, typename TD, int ACT>
void launch_backward(GnBwdArgs a, bool stats, hipStream_t s) {
    GnArgs& f = a.f;
    constexpr uint32_t E = Vec<TX>::E;
    if (static_cast<uint64_t>(f.batch) * f.groups <= kSlabGroups &&
        (launch_bwd_slab<TX, TD, ACT, 4>(a, stats, s) || launch_bwd_slab<TX, TD, ACT, 2>(a, stats, s)))
        return;
    const bool fx = fast_x<TX>(f);
    const bool fast = fx && fast_rows(a.dy, a.lddy, a.sdy, E, sizeof(TD)) && fast_rows(a.dx, a.lddx, a.sdx, E, sizeof(TX)) &&
                      fast_rows(a.res, a.ldres, a.sres, E, sizeof(TX));
    f.joined = stats ? launch_stats<TX>(f, fx, s) : 1;
    if (fast) {
        const uint32_t T = threads_for(f.C / E, 4096 / E), rows_at = T / (f.C / E);
        const uint32_t lds = f.groups * sizeof(Stat);
        gn_bwd_cols_kernel<TX, TD, ACT><<<f.batch * f.nchunk, T, lds + 2 * rows_at * f.C * sizeof(float), s>>>(a);
        const uint32_t apply = f.batch * f.ncut + (a.dgamma ? ceil_div(2ull * f.C, 32) : 0);
        gn_bwd_apply_kernel<TX, TD, ACT><<<apply, T, std::max<uint32_t>(lds + f.groups * 8, T * 8), s>>>(a);
        return;
    }
    if (!f.joined) gn_join_kernel<<<grid_of((static_cast<uint64_t>(f.batch) * f.groups + 3) / 4), 256, 0, s>>>(f);
    gn_bwd_cols_any_kernel<TX, TD, ACT><<<grid_of(static_cast<uint64_t>(f.batch) * f.nchunk * ceil_div(f.C, 64)), 256, 0, s>>>(a);
    gn_bwd_groups_kernel<<<grid_of((static_cast<uint64_t>(f.batch) * f.groups + 3) / 4), 256, 0, s>>>(a);
    if (a.dgamma)
        gn_bwd_params_kernel<<<grid_of(ceil_div(f.C, 64)), 256, 0, s>>>(a.cpart, a.dgamma, a.dbeta, static_cast<uint64_t>(f.batch) * f.nchunk, f.C);
    gn_bwd_apply_any_kernel<TX, TD, ACT><<<grid_of((static_cast<uint64_t>(f.batch) * f.pixels + 3) / 4), 256, 0, s>>>(a);
}

template <typename TX, typename TD>
void launch_backward(const GnBwdArgs& a, int act, bool stats, hipStream_t s) {
    if (act == MI_ACT_SILU) launch_backward<TX, TD, MI_ACT_SILU>(a, stats, s);
    else launch_backward<TX, TD, MI_ACT_NONE>(a, stats, s);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" uint64_t mi_groupnorm_ws_bytes(uint32_t batch, uint32_t pixels, uint32_t channels, uint32_t groups) {
    if (!sizes_ok(batch, pixels, channels, groups) || batch == 0 || pixels == 0) return 0;
    const GnArgs a = sized(batch, pixels, channels, groups);
    return stat_bytes(a) + part_bytes(a);
}

extern "C" int mi_groupnorm(const mi_groupnorm_args* args, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* fn = "mi_groupnorm";
    GnArgs a;
    Span x{}, y{};
    if (int st = check_args(fn, args, a, true, x, y)) return st;
    if (a.batch == 0 || a.pixels == 0) return MI_OK;
    const uint64_t need = mi_groupnorm_ws_bytes(a.batch, a.pixels, a.C, a.groups), cols = static_cast<uint64_t>(a.C) * 4;
    if (int st = check_ws(fn, workspace, workspace_bytes, need)) return st;
    const Span in[3] = {x, {a.gamma, cols}, {a.beta, cols}};
    const Span out[4] = {y, {a.y_scale, static_cast<uint64_t>(a.batch) * a.pixels * 4},
                         {args->stats, static_cast<uint64_t>(a.batch) * a.groups * sizeof(Stat)}, {workspace, need}};
    if (int st = check_overlaps(fn, out, 4, in, 3, -1, -1)) return st;
    a.stats = args->stats ? reinterpret_cast<Stat*>(args->stats) : static_cast<Stat*>(workspace);
    a.part = reinterpret_cast<Part*>(static_cast<char*>(workspace) + stat_bytes(a));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (args->x_dtype == MI_F32) launch_forward<float>(a, args->y_dtype, args->act, s);
    else launch_forward<_Float16>(a, args->y_dtype, args->act, s);
    return check_launch(fn);
}

extern "C" uint64_t mi_groupnorm_bwd_ws_bytes(uint32_t batch, uint32_t pixels, uint32_t channels, uint32_t groups) {
    if (!sizes_ok(batch, pixels, channels, groups) || batch == 0 || pixels == 0) return 0;
    const GnArgs a = sized(batch, pixels, channels, groups);
    return stat_bytes(a) + part_bytes(a) + gsum_bytes(a) + gpart_bytes(a) + cpart_bytes(a);
}

extern "C" int mi_groupnorm_bwd(const mi_groupnorm_bwd_args* args, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* fn = "mi_groupnorm_bwd";
    if (!args) return fail(MI_ERR_INVALID_ARG, "%s: null arguments", fn);
    GnBwdArgs a{};
    Span x{}, none{}, dy{}, res{}, dx{};
    if (int st = check_args(fn, &args->fwd, a.f, false, x, none)) return st;
    const GnArgs& f = a.f;
    const mi_groupnorm_args& g = args->fwd;
    if ((args->dgamma == nullptr) != (args->dbeta == nullptr)) return fail(MI_ERR_INVALID_ARG, "%s: dgamma and dbeta go together", fn);
    if (!aligned(args->dgamma, 4) || !aligned(args->dbeta, 4))
        return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
    a.dgamma = args->dgamma;
    a.dbeta = args->dbeta;
    const uint64_t cols = static_cast<uint64_t>(f.C) * 4;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (f.batch == 0 || f.pixels == 0) {
        if (!a.dgamma) return MI_OK;
        if (overlaps(a.dgamma, cols, a.dbeta, cols)) return fail(MI_ERR_ALIASING, "%s: outputs overlap each other", fn);
        gn_bwd_params_kernel<<<grid_of(ceil_div(f.C, 64)), 256, 0, s>>>(nullptr, a.dgamma, a.dbeta, 0, f.C);
        return check_launch(fn);
    }
    if (!args->dy || !args->dx) return fail(MI_ERR_INVALID_ARG, "%s: null pointer", fn);
    a.dy = args->dy;
    a.res = args->res;
    a.dx = args->dx;
    a.lddy = args->lddy ? args->lddy : f.C;
    a.ldres = args->ldres ? args->ldres : f.C;
    a.lddx = args->lddx ? args->lddx : f.C;
    a.sdy = args->sdy ? args->sdy : a.lddy * f.pixels;
    a.sres = args->sres ? args->sres : a.ldres * f.pixels;
    a.sdx = args->sdx ? args->sdx : a.lddx * f.pixels;
    if (a.lddy < f.C || a.lddx < f.C || (a.res && a.ldres < f.C))
        return fail(MI_ERR_INVALID_ARG, "%s: a row stride below %u channels", fn, f.C);
    const uint64_t ex = esize(g.x_dtype), ed = esize(g.y_dtype);
    if (!span(a.dy, f.batch, f.pixels, f.C, a.lddy, a.sdy, ed, dy) || !span(a.dx, f.batch, f.pixels, f.C, a.lddx, a.sdx, ex, dx) ||
        (a.res && !span(a.res, f.batch, f.pixels, f.C, a.ldres, a.sres, ex, res)))
        return fail(MI_ERR_UNSUPPORTED, "%s: a tensor spans 2^60 elements or more", fn);
    if (!rows_apart(f.batch, f.pixels, f.C, a.lddx, a.sdx)) return fail(MI_ERR_INVALID_ARG, "%s: rows of dx overlap each other", fn);
    if (!aligned(a.dy, ed) || !aligned(a.dx, ex) || !aligned(a.res, ex))
        return fail(MI_ERR_ALIGNMENT, "%s: tensors must be aligned to their element size", fn);
    const uint64_t need = mi_groupnorm_bwd_ws_bytes(f.batch, f.pixels, f.C, f.groups);
    if (int st = check_ws(fn, workspace, workspace_bytes, need)) return st;
    const Span in[6] = {x, {f.gamma, cols}, {f.beta, cols}, dy, {g.stats, static_cast<uint64_t>(f.batch) * f.groups * sizeof(Stat)}, res};
    const Span out[4] = {dx, {a.dgamma, cols}, {a.dbeta, cols}, {workspace, need}};
    // dx may be res itself: a value is read before it is written, by the same lane
    const bool same = a.res == a.dx && a.ldres == a.lddx && a.sres == a.sdx;
    if (int st = check_overlaps(fn, out, 4, in, 6, same ? 0 : -1, 5)) return st;
    char* ws = static_cast<char*>(workspace);
    a.f.stats = g.stats ? reinterpret_cast<Stat*>(g.stats) : reinterpret_cast<Stat*>(ws);
    a.f.part = reinterpret_cast<Part*>(ws + stat_bytes(f));
    a.gsum = reinterpret_cast<float*>(ws + stat_bytes(f) + part_bytes(f));
    a.gpart = reinterpret_cast<float*>(ws + stat_bytes(f) + part_bytes(f) + gsum_bytes(f));
    a.cpart = reinterpret_cast<float*>(ws + stat_bytes(f) + part_bytes(f) + gsum_bytes(f) + gpart_bytes(f));
    const bool stats = !g.stats;
    if (g.x_dtype == MI_F32) {
        if (g.y_dtype == MI_F32) launch_backward<float, float>(a, g.act, stats, s);
        else launch_backward<float, _Float16>(a, g.act, stats, s);
    } else {
        if (g.y_dtype == MI_F32) launch_backward<_Float16, float>(a, g.act, stats, s);
        else launch_backward<_Float16, _Float16>(a, g.act, stats, s);
    }
    return check_launch(fn);
}

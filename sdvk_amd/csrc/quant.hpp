// quant.hpp -- rows of 8-bit codes with a scale each: what gemm_i8.hip's quantiser and groupnorm.hip's 8-bit output share.
//
//   scale = max(max|x|, 127 * 2^-126) / 127 in fp32,  code = x / scale rounded to the nearest integer, ties to even
//
// The quotient is exact: which of two integers is nearest is decided by x - code * scale, which fp32 holds without rounding (a
// multiple of the smaller operand's last place, no larger than the scale); twice it is held against the scale (half a scale below
// 2^-125 is no fp32 number if its last place is odd). The floor keeps 1 / scale finite: rows smaller
// than it (zeros among them) get codes in steps of 2^-126. A row that holds an infinity or a NaN gets the scale NaN
// and codes 0, so that everything computed from it is NaN.
#pragma once

#include "common.hpp"

namespace mi {

struct RowScale {
    float scale, inv;
};

// |v| as an unsigned integer that orders like it, infinities and NaN above every number.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = max(v, __shfl_xor(v, o));
    return v;
}

// top: the row's largest magnitude_bits. inv == 0 marks a row without numbers.
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
    if (top >= 0x7f800000u) return RowScale{__uint_as_float(0x7fc00000u), 0.0f};
    const float s = fmaxf(__uint_as_float(top), 127.0f * 1.17549435082228750797e-38f) / 127.0f;
    return RowScale{s, 1.0f / s};
}

constexpr float kQuantMagic = 12582912.0f;  // 1.5 * 2^23: a sum of it and a code holds the code in its low bits

// v / scale rounded, as kQuantMagic + code: the fma's rounding is that of v * inv, which is off by 2^-17 at most, so where
// the exact rest is under half a step the code is the nearest integer. rest: the largest of those seen.
__device__ __forceinline__ float quant_fast(float v, const RowScale& s, float& rest) {
    const float t = __builtin_fmaf(v, s.inv, kQuantMagic);
    rest = fmaxf(rest, fabsf(__builtin_fmaf(kQuantMagic - t, s.scale, v)));
    return t;
}
// ... put right where it is a tie or went one too far (t's last place is one code).
__device__ __forceinline__ float quant_right(float v, float t, const RowScale& s) {
    if (s.inv == 0.0f) return kQuantMagic;
    const float r = __builtin_fmaf(kQuantMagic - t, s.scale, v);
    const uint32_t bits = __float_as_uint(t);
    // over half a step, or half a step and an odd code: magnitudes order as integers
    const bool wrong = magnitude_bits(r + r) + (bits & 1u) > __float_as_uint(s.scale);
    return wrong ? __uint_as_float(r > 0.0f ? bits + 1 : bits - 1) : t;
}
__device__ __forceinline__ int quant_code(float v, const RowScale& s) {
    float rest = 0.0f;
    const float t = quant_right(v, quant_fast(v, s, rest), s);
    return static_cast<int8_t>(__float_as_uint(t) & 0xffu);
}

// N codes of value(0) .. value(N - 1), four a dword. One value in 2^18 or a tie sends its lane through quant_right (code of its own for
// every value, or branches among them, made the kernels wait for instructions: 2048 x 5120 fp16 14 us).
template <int N, typename F>
__device__ __forceinline__ void quant_codes(const F& value, const RowScale& s, uint32_t (&out)[N / 4]) {
    float t[N], rest = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = quant_fast(value(i), s, rest);
    if (!(rest + rest < s.scale)) {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = quant_right(value(i), t[i], s);
    }
#pragma unroll
    for (int i = 0; i < N; i += 4)
        out[i / 4] = __builtin_amdgcn_perm(__float_as_uint(t[i + 1]), __float_as_uint(t[i]), 0x0c0c0400u) |
                     __builtin_amdgcn_perm(__float_as_uint(t[i + 3]), __float_as_uint(t[i + 2]), 0x04000c0cu);
}

}  // namespace mi

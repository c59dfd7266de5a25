// quant.hpp -- rows of 8-bit codes with a scale each: what gemm_i8.hip's quantiser and groupnorm.hip's 8-bit output share.
//
//   scale = max(max|x|, 127 * 2^-126) / 127 in fp32,  code = x / scale rounded to the nearest integer, ties to even
//
// The quotient is exact: which of two integers is nearest is decided by x - code * scale, which fp32 holds without rounding (a
// multiple of the smaller operand's last place, no larger than the scale). The floor keeps 1 / scale finite: rows smaller
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

__device__ __forceinline__ int quant_code(float v, const RowScale& s) {
    if (s.inv == 0.0f) return 0;
    // within 2^-15 of the quotient: off by one at most, near a tie
    float q = rintf(v * s.inv);
    const float rest = __builtin_fmaf(-q, s.scale, v), half = 0.5f * s.scale;  // exact
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (rest > half || (rest == half && odd)) q += 1.0f;
    else if (rest < -half || (rest == -half && odd)) q -= 1.0f;
    return static_cast<int>(q);
}

// Four codes as bytes. Adding 1.5 * 2^23 rounds the product v / scale to an integer in the sum's low bits, whose low byte is the code;
// where what is left of every value is less than half a step the codes are the nearest integers, and a lane that holds a tie
// or a quotient that rounded over one (one value in 2^16) takes quant_code.
__device__ __forceinline__ uint32_t quant_codes4(const float (&v)[4], const RowScale& s) {
    constexpr float kMagic = 12582912.0f;
    float t[4], rest = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        t[e] = __builtin_fmaf(v[e], s.inv, kMagic);
        rest = fmaxf(rest, fabsf(__builtin_fmaf(kMagic - t[e], s.scale, v[e])));
    }
    if (!(rest < 0.5f * s.scale)) {
        uint32_t r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) r |= (static_cast<uint32_t>(quant_code(v[e], s)) & 0xffu) << (8 * e);
        return r;
    }
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[1]), __float_as_uint(t[0]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t[3]), __float_as_uint(t[2]), 0x04000c0cu);
    return lo | hi;
}

}  // namespace mi

// Four bits a number, for weights and for cached keys and values.
//
// A group of neighbouring numbers x (32 of a cached head; 32, 64 or 128 of a weight's row) is held as a scale s with four
// significant bits, a zero z and a code c for each number, z and c in 0..15; the number then stands for s · (c − z):
//     lo = min(0, min x), hi = max(0, max x)
//     s = (hi − lo) / 15 rounded UP to four significant bits, z = round(−lo / s), c = clamp(round(x / s) + z, 0, 15)
// with the exact quotients rounded to nearest, ties to even. A group with hi − lo < 2^-100 stands for zeros (s = z = c = 0),
// one with an entry that is not finite or beyond 2^100 for NaN (s NaN, z = c = 0).
//
// Why so: |c − z| has four bits, so s · (c − z) has eight and IS a bfloat16, and every kernel, whichever way it takes the
// numbers apart, multiplies the same ones; and s and z fit one 16-bit word, the bfloat16 of s with z in the four low bits
// of its mantissa, which are free. What it costs: a step up to an eighth wider than the range needs (a sixteenth on average).
//
// Codes lie eight to a word such that (word >> 4 j) & 0x000f000f is the pair of numbers 2 j and 2 j + 1, as the
// halves of a tensor-core operand's register: nibble j holds number 2 j, nibble j + 4 number 2 j + 1. With 0x4300 in
// front a code is the bfloat16 128 + c, and 128 + c minus 128 + z is exact.
#pragma once
#include "common.cuh"

namespace {

__device__ __forceinline__ uint32_t q4_pair(uint32_t word, int j) { return ((word >> (4 * j)) & 0x000f000fu) | 0x43004300u; }
__device__ __forceinline__ float q4_scale_of(uint32_t meta) { return __uint_as_float((meta & 0xfff0u) << 16); }
__device__ __forceinline__ float q4_value(int code, uint32_t meta) { return q4_scale_of(meta) * (float)(code - (int)(meta & 15u)); }

__device__ __forceinline__ uint32_t bf2_sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
    return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmul2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
    return *(const uint32_t*)&r;
}

struct Q4Scale { float s, inv; int z; };

// s and z of a group from its bounds (lo <= 0 <= hi), in 64 bits: hi − lo and the quotients are compared with values that
// they may equal (a multiple of s halfway between two codes, a power of two's boundary).
__device__ __forceinline__ Q4Scale q4_group(float lo, float hi, bool bad) {
    Q4Scale g{0.0f, 0.0f, 0};
    const double r = (double)hi - (double)lo;
    if (bad) { g.s = __int_as_float(0x7fc00000); return g; }
    if (r < 7.888609052210118e-31) return g;                         // 2^-100
    long long bits = __double_as_longlong(r / 15.0);
    constexpr long long LOW = (1ll << 49) - 1;                       // all but four significant bits
    bits = (bits + LOW) & ~LOW;
    const double s = __longlong_as_double(bits);
    g.s = (float)s;
    g.inv = 1.0f / g.s;
    g.z = __double2int_rn(-(double)lo / s);
    return g;
}

// The code of x: a quotient by the reciprocal, at most one off, and the remainder x − s·t, which is exact (s·t has eight
// bits and x's last place is below s's), decides.
__device__ __forceinline__ int q4_code(float x, const Q4Scale& g) {
    if (!(g.s > 0.0f)) return 0;                                     // zeros, NaN
    float t = rintf(x * g.inv);
    const float d = fmaf(-g.s, t, x), over = 2.0f * fabsf(d) - g.s;  // exact: both are multiples of x's last place
    if (over > 0.0f || (over == 0.0f && ((int)t & 1))) t += copysignf(1.0f, d);
    return min(15, max(0, (int)t + g.z));
}

__device__ __forceinline__ uint32_t q4_meta(const Q4Scale& g) { return ((__float_as_uint(g.s) >> 16) & 0xfff0u) | (uint32_t)g.z; }

__device__ __forceinline__ bool q4_bad(float x) { return !(fabsf(x) <= 1.2676506002282294e30f); }      // 2^100; NaN too

}  // namespace

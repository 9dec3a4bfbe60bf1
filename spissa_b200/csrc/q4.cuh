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
#include <cuda_fp16.h>

namespace {

__device__ __forceinline__ uint32_t q4_pair(uint32_t word, int j) { return ((word >> (4 * j)) & 0x000f000fu) | 0x43004300u; }
__device__ __forceinline__ float q4_scale_of(uint32_t meta) { return __uint_as_float((meta & 0xfff0u) << 16); }
__device__ __forceinline__ float q4_value(int code, uint32_t meta) { return q4_scale_of(meta) * (float)(code - (int)(meta & 15u)); }

// (c − z) 2^-9 as two float16 numbers, exactly. The bits in their places (w & 0x000f000f, or w & 0x00f000f0) ARE the float16 numbers
// c · 2^-24 (16 c · 2^-24), and so are z's; 2^15 makes ordinary numbers of them: tensor cores align a subnormal operand by the exponent it
// is written with, and its product loses up to ten of the 24 bits (float32 products 3.5e-6 off where these are 2.4e-7).
__device__ __forceinline__ uint32_t q4_zero(uint32_t z) {
    const __half2 r = __hmul2(*(const __half2*)&z, __float2half2_rn(-32768.0f));
    return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t q4_minus(uint32_t c, uint32_t zero) {
    const __half2 r = __hfma2(*(const __half2*)&c, __float2half2_rn(32768.0f), *(const __half2*)&zero);
    return *(const uint32_t*)&r;
}

__device__ __forceinline__ uint32_t bf2_sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
    return *(const uint32_t*)&r;
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmul2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
    return *(const uint32_t*)&r;
}

struct Q4Scale { float s, inv; int z; };

// round(x / s), ties to even, |x / s| < 2^20: a quotient by the reciprocal, rounded in the place of ones of 1.5 · 2^23 and at most
// one off; the remainder x − s·t, which is exact (s·t has eight bits and x's last place is below s's), decides.
__device__ __forceinline__ int q4_round(float x, float s, float inv) {
    const float y = fmaf(x, inv, 12582912.0f), d = fmaf(-s, y - 12582912.0f, x), over = 2.0f * fabsf(d) - s;
    int t = __float_as_int(y) - 0x4b400000;
    if (over >= 0.0f && (over > 0.0f || (t & 1))) t += d > 0.0f ? 1 : -1;      // (over is exact: both are multiples of x's last place)
    return t;
}

// (hi − lo) / 15 rounded up to four significant bits, or 0 below 2^-100, in 64 bits: a range may be a multiple of 15 exactly
static __device__ __noinline__ float q4_step(float lo, float hi) {
    const double r = (double)hi - (double)lo;
    if (r < 7.888609052210118e-31) return 0.0f;
    constexpr long long LOW = (1ll << 49) - 1;                       // all but four significant bits
    return (float)__longlong_as_double((__double_as_longlong(r / 15.0) + LOW) & ~LOW);
}

// s and z of a group from its bounds (lo <= 0 <= hi). The quotient in 32 bits is off by at most four of its last places, so
// rounding it up gives the same unless it lies within 16 of a number of four bits.
__device__ __forceinline__ Q4Scale q4_group(float lo, float hi, bool bad) {
    Q4Scale g{0.0f, 0.0f, 0};
    if (bad) { g.s = __int_as_float(0x7fc00000); return g; }
    const float r = hi - lo;
    const uint32_t q = __float_as_uint(r * (1.0f / 15.0f)), low = q & 0xfffffu;
    g.s = __uint_as_float((q & ~0xfffffu) + 0x100000u);
    if (low - 16u > 0xfffffu - 32u || r < 1.6e-30f) g.s = q4_step(lo, hi);
    if (g.s > 0.0f) {
        asm("rcp.approx.f32 %0, %1;" : "=f"(g.inv) : "f"(g.s));
        g.z = q4_round(-lo, g.s, g.inv);
    }
    return g;
}

__device__ __forceinline__ int q4_code(float x, const Q4Scale& g) {
    if (!(g.s > 0.0f)) return 0;                                     // zeros, NaN
    return min(15, max(0, q4_round(x, g.s, g.inv) + g.z));
}

__device__ __forceinline__ uint32_t q4_meta(const Q4Scale& g) { return ((__float_as_uint(g.s) >> 16) & 0xfff0u) | (uint32_t)g.z; }

__device__ __forceinline__ bool q4_bad(float x) { return !(fabsf(x) <= 1.2676506002282294e30f); }      // 2^100; NaN too

}  // namespace

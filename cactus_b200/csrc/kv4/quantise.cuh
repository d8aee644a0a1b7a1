// The 4-bit KV cache's quantisation of a group: its step and its codes, of the exact differences. Shared by
// the kernels that write rows into pages.
#pragma once
#include "../common.cuh"

namespace cb {
namespace kv4 {

// What the rounding of d = a - b took away: a - b - d, exactly (Knuth's two-sum).
__device__ __forceinline__ float rest_of_difference(float a, float b, float d) {
    const float c = __fsub_rn(d, a);
    return __fsub_rn(__fsub_rn(a, __fsub_rn(d, c)), __fadd_rn(b, c));
}

// (hi - lo) / 15 rounded towards zero to fp16: the product with 1/15 is a unit in the last place off at
// most, and fifteen times an fp16 number is exact in fp32. The difference is not where hi and lo are of
// very different sizes, but its rounding keeps the order: only where it equals what it is compared with
// does the rest decide.
__device__ __forceinline__ __half step_of(float hi, float lo) {
    const float range = __fsub_rn(hi, lo);
    const unsigned short s = __half_as_ushort(__float2half_rz(__fmul_rn(range, 1.0f / 15.0f)));
    const float at = __fmul_rn(__half2float(__ushort_as_half(s)), 15.0f);
    const float above = __fmul_rn(__half2float(__ushort_as_half((unsigned short)(s + 1))), 15.0f);
    const bool less = rest_of_difference(hi, lo, range) < 0.0f;
    const bool up = above < range || (above == range && !less), down = at > range || (at == range && less);
    return __ushort_as_half((unsigned short)(s + (up ? 1 : 0) - (down ? 1 : 0)));
}

// The codes of 8 elements of a group as a word: each quotient (x - lo) / step rounded half to even, at most
// 15. The product with the reciprocal is within 4e-6 of a quotient below 16 (2^-23 for the reciprocal, 2^-24
// for the product and for the difference), so where every product is further than that from a half its
// rounding is the quotient's; else (rare) the differences are compared with the half steps about them
// (exact in fp32), and their rests decide where they are equal; so they are where the step is so small (a
// few of fp16's smallest units) that a quotient can pass 15.5. Adding 1.5 * 2^23 rounds to an integer and leaves it in the low bits.
__device__ __forceinline__ uint32_t quant_codes(const __half2* h, float lo, float step) {
    const float magic = 12582912.0f;
    float inv, far = 0.0f, x[8];
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 p = __half22float2(h[j]);
        x[2 * j] = __fsub_rn(p.x, lo);
        x[2 * j + 1] = __fsub_rn(p.y, lo);
    }
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t = fmaf(x[j], inv, magic);
        far = fmaxf(far, fabsf(fmaf(x[j], inv, -__fsub_rn(t, magic))));
        w += __float_as_uint(t) << (4 * j);  // 0x4B400000 + code: the sum of the constants is taken off below
    }
    w -= 0x4B400000u * 0x11111111u;
    if (far > 0.499992f || step < 0x1p-18f) {
        w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 p = __half22float2(h[j / 2]);
            const float n = floorf(__fmul_rn(x[j], inv));  // the quotient is in n - 4e-6 .. n + 1 + 4e-6
            const float half = __fmul_rn(n + 0.5f, step), rest = rest_of_difference(j & 1 ? p.y : p.x, lo, x[j]);
            const bool up = x[j] > half || (x[j] == half && (rest > 0.0f || (rest == 0.0f && ((int)n & 1))));
            w |= (uint32_t)min((int)n + up, 15) << (4 * j);
        }
    }
    return w;
}

}  // namespace kv4
}  // namespace cb

// Quantisation of a block of fp32 values to e4m3 with one scale, shared by the kernels that produce 8-bit rows.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace b200moe {
namespace fp8_block {

constexpr float kMax = 448.f;            // largest finite e4m3
constexpr float kFloor = 0x1p-100f;      // a block's largest magnitude counts as at least this much

// code = e4m3_rne(x * 448 / a), and where x and a are bf16 values the codes are those of the exact quotient: x * 448 and a are then
// integers of at most 11 and 8 bits times powers of two, so a quotient that is no tie of e4m3 is at least 2^-13 (relative) away
// from one, and one that is a tie has at most five bits and comes out of the correction step as it is: the first guess
// is good to about 2^-21, its remainder is exact (11 bits), and what the step leaves is of the second order.
// x * 448 / a = x' / a' with x' = x * 7 * 2^-4 and a' = a * 2^-10: neither product overflows, and neither is rounded where it matters.
__device__ __forceinline__ float reciprocal(float a) {  // good to 2^-23, a normal
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}
// The largest magnitude of three; a NaN stays one.
__device__ __forceinline__ float max_magnitude(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
struct Quantizer {
    float scale;
    float a, inv;  // a', 1 / a' (0 for a block that is not finite: zeros have code 0 there)
    // `top`: the largest magnitude of the block, or infinity / NaN where the block holds one
    __device__ __forceinline__ explicit Quantizer(float top) {
        const bool finite = top < INFINITY;  // (not NaN either)
        const float m = fmaxf(top, kFloor);
        a = finite ? m * 0x1p-10f : 0.f;
        inv = finite ? reciprocal(a) : 0.f;
        // m / 448 by the same correction step (for bf16 m the quotient rounded to nearest, which the tests check for all of them)
        constexpr float kInv = 1.f / kMax;
        const float q = m * kInv;
        scale = finite ? fmaf(fmaf(-q, kMax, m), kInv, q) : __uint_as_float(0x7FC00000u);
    }
    // what codes2() needs, for a thread that did not see the block's magnitude
    __device__ __forceinline__ float2 packed() const { return make_float2(a, inv); }
    __device__ __forceinline__ explicit Quantizer(const float2& p) : scale(0.f), a(p.x), inv(p.y) {}
    // two codes, the first value's in the low byte
    __device__ __forceinline__ uint32_t codes2(f32x2 x) const {
        const f32x2 inv2 = pack_f32x2(inv, inv), a2 = pack_f32x2(-a, -a);
        x = mul_f32x2(x, pack_f32x2(0.4375f, 0.4375f));
        const f32x2 q = mul_f32x2(x, inv2);
        const f32x2 y = fma_f32x2(fma_f32x2(q, a2, x), inv2, q);
        uint16_t o;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(o) : "f"(f32x2_hi(y)), "f"(f32x2_lo(y)));
        return o;
    }
    __device__ __forceinline__ bool finite() const { return inv != 0.f; }
};

}  // namespace fp8_block
}  // namespace b200moe

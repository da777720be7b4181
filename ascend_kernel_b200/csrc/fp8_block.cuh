// Quantisation of a block of fp32 values to e4m3 with one scale, shared by the kernels that produce 8-bit rows.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace b200moe {
namespace fp8_block {

constexpr int kBlock = 128;
constexpr float kMax = 448.f;            // largest finite e4m3
constexpr float kFloor = 0x1p-100f;      // a block's largest magnitude counts as at least this much

// code = e4m3_rne(x * 448 / a), and where x and a are bf16 values the codes are those of the exact quotient: x * 448 and a are then
// integers of at most 11 and 8 bits times powers of two, so a quotient that is no tie of e4m3 is at least 2^-13 (relative) away
// from one, and one that is a tie has at most five bits and comes out of the correction step as it is (r, the remainder, is
// exact, and what the step leaves is of the second order in a first guess good to 2^-22).
struct Quantizer {
    float scale;
    float inv_, a_, step_;  // 448 / a, a * 2^-10, 2^10 / a
    bool finite_;
    // `top`: the largest magnitude of the block, or infinity / NaN where the block holds one
    __device__ __forceinline__ explicit Quantizer(float top) {
        finite_ = top < INFINITY;
        const float a = fmaxf(top, kFloor);
        scale = finite_ ? a / kMax : __uint_as_float(0x7FC00000u);
        inv_ = finite_ ? kMax / a : 0.f;
        a_ = a * 0x1p-10f;
        step_ = inv_ * (1024.f / kMax);
    }
    // what four() needs, for a thread that did not see the block's magnitude
    __device__ __forceinline__ float4 packed() const { return make_float4(inv_, a_, step_, finite_ ? 1.f : 0.f); }
    __device__ __forceinline__ explicit Quantizer(const float4& p) : scale(0.f), inv_(p.x), a_(p.y), step_(p.z), finite_(p.w != 0.f) {}
    __device__ __forceinline__ float ratio(float x) const {
        // x * 448 / a = (x * 7 * 2^-4) / (a * 2^-10): neither product overflows, and neither is rounded where it matters
        const float q = x * inv_;
        const float r = fmaf(-q, a_, x * 0.4375f);
        return fmaf(r, step_, q);
    }
    __device__ __forceinline__ uint32_t four(float x0, float x1, float x2, float x3) const {
        if (!finite_) return 0u;
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(ratio(x0), ratio(x1)), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(ratio(x2), ratio(x3)), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    }
};

}  // namespace fp8_block
}  // namespace b200moe

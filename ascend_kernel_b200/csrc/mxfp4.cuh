// Quantisation of a block of 32 fp32 values to e2m1 with one power-of-two scale, shared by the kernels that produce 4-bit rows.
#pragma once

#include "common.cuh"

namespace b200moe {
namespace mxfp4 {

constexpr uint32_t kLowest = 127 - 100;  // smallest scale byte of a block that is finite
constexpr uint32_t kNaN = 255;

// Bytes of a row of scales: whole words of four.
__host__ __device__ constexpr int64_t scale_width(int64_t K) { return (K + 127) / 128 * 4; }

// The scale byte for a block's largest magnitude (its bits): the smallest power of two 2^e with magnitude <= 7 * 2^e, so that the nearest
// code is 6 at most and no value is further than half a step of its binade from its code.  The exponent of the magnitude less two, one
// more where the significand is over 1.75; an infinity or a NaN makes the scale NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    const int e = (int)((top + 0x1FFFFFu) >> 23) - 2;
    return top >= 0x7F800000u ? kNaN : (uint32_t)max(e, (int)kLowest);
}
// 2^-e; 0 where the block is not finite
__device__ __forceinline__ float inverse(uint32_t byte) { return byte == kNaN ? 0.f : __uint_as_float((254u - byte) << 23); }
// Eight codes, element i in nibble i: nearest, ties to even, at most 6.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        "mov.b32 %0, {b0, b1, b2, b3};\n"
        "}\n"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

}  // namespace mxfp4
}  // namespace b200moe

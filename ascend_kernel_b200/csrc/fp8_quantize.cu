// Rows of bf16 quantised to e4m3 with one fp32 scale per 128 elements, optionally gathered by an index on the way (token rows
// into expert order).
//
//   a = max(2^-100, largest magnitude of the block);  scale = a / 448;  code = e4m3_rne(x * 448 / a)
//
// The floor keeps the quotient finite for a block of zeros.  A block that holds an infinity or a NaN gets the scale NaN (and
// codes 0): everything that it stands for is NaN, as every sum over the row would be.
#include <cuda_fp8.h>

#include "common.cuh"
#include "fp8_block.cuh"

namespace b200moe {

// A half-warp takes a block: 16 lanes x 8 elements.  A warp takes kBlocks blocks of a row at a time.
constexpr int kQuantPairs = 4;  // pairs of blocks a warp has in flight

__global__ void __launch_bounds__(256) fp8_quantize_rows_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ index,
                                                                uint2* __restrict__ codes, float* __restrict__ scale, int n_src,
                                                                long long n_units, int units_per_row, int K8, int KB) {
    const int lane = threadIdx.x & 31, half = lane >> 4, l16 = lane & 15;
    const long long unit = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (unit >= n_units) return;
    const long long row = unit / units_per_row;
    const int b0 = (int)(unit % units_per_row) * (2 * kQuantPairs) + half;
    const long long from = index ? (long long)__ldg(index + row) : row;
    const bool inside = (unsigned long long)from < (unsigned long long)n_src;
    const uint4* src = x + (inside ? from : 0) * K8;
    uint4 v[kQuantPairs];
#pragma unroll
    for (int i = 0; i < kQuantPairs; ++i) {
        const int c = (b0 + 2 * i) * 16 + l16;
        v[i] = inside && c < K8 ? __ldg(src + c) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < kQuantPairs; ++i) {
        const int b = b0 + 2 * i, c = b * 16 + l16;
        uint32_t m = __vmaxu2(__vmaxu2(v[i].x & 0x7FFF7FFFu, v[i].y & 0x7FFF7FFFu), __vmaxu2(v[i].z & 0x7FFF7FFFu, v[i].w & 0x7FFF7FFFu));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
        // magnitudes of bf16 order as their bits do, and infinities and NaN come last
        const uint32_t top = max(m & 0xFFFFu, m >> 16);
        const fp8_block::Quantizer q(__uint_as_float(top << 16));
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t o[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            o[j] = q.four(__uint_as_float(w[2 * j] << 16), __uint_as_float(w[2 * j] & 0xFFFF0000u),
                          __uint_as_float(w[2 * j + 1] << 16), __uint_as_float(w[2 * j + 1] & 0xFFFF0000u));
        if (c < K8) codes[row * K8 + c] = make_uint2(o[0], o[1]);
        if (l16 == 0 && b < KB) scale[row * KB + b] = q.scale;
    }
}

}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_fp8_quantize_rows(const void* x, const int32_t* index, void* codes, float* scale, int64_t n_src,
                                         int64_t n_rows, int64_t K, void* stream) {
    if (n_src < 0 || n_rows < 0 || K <= 0 || (K % 16) != 0 || n_src > 0x7FFFFFFFLL || n_rows > 0x7FFFFFFFLL || K > 0x7FFFFFF0LL ||
        (!index && n_rows > n_src))
        return B200MOE_ERR_SHAPE;
    if (n_rows == 0) return B200MOE_OK;
    if ((!x && n_src > 0) || !codes || !scale) return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(x) || !aligned16(codes)) return B200MOE_ERR_ALIGNMENT;
    const int KB = (int)((K + 127) / 128), upr = (KB + 2 * kQuantPairs - 1) / (2 * kQuantPairs);
    const long long units = n_rows * upr, blocks = (units + 7) / 8;
    if (blocks > 0x7FFFFFFFLL) return B200MOE_ERR_SHAPE;
    fp8_quantize_rows_kernel<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint4*>(x), index, static_cast<uint2*>(codes), scale, (int)n_src, units, upr, (int)(K / 8), KB);
    B200MOE_CUDA_TRY(cudaGetLastError());
    return B200MOE_OK;
}

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

// Eight lanes take a block, 16 elements (32 bytes in, 16 out) each, a warp four blocks at a time and kSteps times as many in flight.
// (16 lanes of 8 elements: twice the shuffles and twice the work per block; 4096 tokens x 8, 7168: 139 us, see below.)
constexpr int kSteps = 2;
constexpr int kWarpBlocks = 4 * kSteps;

__global__ void __launch_bounds__(256) fp8_quantize_rows_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ index,
                                                                uint4* __restrict__ codes, float* __restrict__ scale, int n_src, int K16,
                                                                int KB) {
    const int lane = threadIdx.x & 31, l8 = lane & 7;
    const long long row = blockIdx.x;
    const int b0 = ((int)blockIdx.y * (int)(blockDim.x >> 5) + (int)(threadIdx.x >> 5)) * kWarpBlocks + (lane >> 3);
    const long long from = index ? (long long)__ldg(index + row) : row;
    const bool inside = (unsigned long long)from < (unsigned long long)n_src;
    const uint4* src = x + (inside ? from : 0) * K16 * 2;
    uint4 v[kSteps][2];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int c = (b0 + 4 * i) * 8 + l8;
        const bool some = inside && c < K16;
        v[i][0] = some ? __ldg(src + 2 * c) : make_uint4(0u, 0u, 0u, 0u);
        v[i][1] = some ? __ldg(src + 2 * c + 1) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int b = b0 + 4 * i, c = b * 8 + l8;
        const uint32_t w[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
        // magnitudes of bf16 order as their bits do, and infinities and NaN come last
        const fp8_block::Quantizer q(__uint_as_float(max(m & 0xFFFFu, m >> 16) << 16));
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = q.codes2(pack_u32x2(w[2 * j] << 16, w[2 * j] & 0xFFFF0000u));
            const uint32_t hi = q.codes2(pack_u32x2(w[2 * j + 1] << 16, w[2 * j + 1] & 0xFFFF0000u));
            o[j] = q.finite() ? lo | (hi << 16) : 0u;
        }
        if (c < K16) codes[row * K16 + c] = make_uint4(o[0], o[1], o[2], o[3]);
        if (l8 == 0 && b < KB) scale[row * KB + b] = q.scale;
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
    // a CTA for a row and up to eight warps' blocks of it
    const int KB = (int)((K + 127) / 128), units = (KB + kWarpBlocks - 1) / kWarpBlocks, warps = units < 8 ? units : 8;
    const int groups = (units + warps - 1) / warps;
    if (groups > 65535) return B200MOE_ERR_SHAPE;
    fp8_quantize_rows_kernel<<<dim3((unsigned)n_rows, (unsigned)groups), 32 * warps, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint4*>(x), index, static_cast<uint4*>(codes), scale, (int)n_src, (int)(K / 16), KB);
    B200MOE_CUDA_TRY(cudaGetLastError());
    return B200MOE_OK;
}

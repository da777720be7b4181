// Rows of bf16 quantised to e2m1 with one power-of-two scale per 32 elements, optionally gathered by an index on the way
// (token rows into expert order).
//
//   2^e = the smallest power of two with (largest magnitude of the block) <= 7 * 2^e, e at least -100;  code = e2m1_rne(x / 2^e)
//
// Division by a power of two is exact, so the codes are those of the definition.  A block that holds an infinity or a NaN gets the scale
// NaN (and codes 0): everything that it stands for is NaN, as every sum over the row would be.
#include <algorithm>

#include "common.cuh"
#include "mxfp4.cuh"

namespace b200moe {
namespace mq {

// Two lanes take a block, 16 elements (32 bytes in, 8 out) each, a warp kSteps times 16 blocks; a CTA takes a row or up to eight warps'
// blocks of it.  Bound by memory where the rows are read once (4096 of 7168: 12.1 us, 6.2 TB/s), by its launch where they are few (2.6 us).
constexpr int kSteps = 2;
constexpr int kWarpChunks = 32 * kSteps;  // of 16 elements

__global__ void __launch_bounds__(256) quantize_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ index,
                                                       uint2* __restrict__ codes, uint8_t* __restrict__ scale, int n_src, int K16,
                                                       int width) {
    const int lane = threadIdx.x & 31;
    const long long row = blockIdx.x;
    const int c0 = ((int)blockIdx.y * (int)(blockDim.x >> 5) + (int)(threadIdx.x >> 5)) * kWarpChunks + lane;
    const long long from = index ? (long long)__ldg(index + row) : row;
    const bool inside = (unsigned long long)from < (unsigned long long)n_src;
    const uint4* src = x + (inside ? from : 0) * K16 * 2;
    uint4 v[kSteps][2];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int c = c0 + 32 * i;
        const bool some = inside && c < K16;
        v[i][0] = some ? __ldg(src + 2 * c) : make_uint4(0u, 0u, 0u, 0u);
        v[i][1] = some ? __ldg(src + 2 * c + 1) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int c = c0 + 32 * i, b = c >> 1;
        const uint32_t w[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
        // magnitudes order as their bits do, infinities and NaN last: both halves of a word at once
        uint32_t m2 = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m2 = __vmaxu2(m2, w[j] & 0x7FFF7FFFu);
        m2 = __vmaxu2(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
        const uint32_t byte = mxfp4::scale_byte(max(m2 << 16, m2 & 0xFFFF0000u));
        const float inv = mxfp4::inverse(byte);
        float lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lo[2 * j] = __uint_as_float(w[j] << 16) * inv;
            lo[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u) * inv;
            hi[2 * j] = __uint_as_float(w[4 + j] << 16) * inv;
            hi[2 * j + 1] = __uint_as_float(w[4 + j] & 0xFFFF0000u) * inv;
        }
        const bool finite = byte != mxfp4::kNaN;
        if (c < K16) codes[row * K16 + c] = finite ? make_uint2(mxfp4::codes8(lo), mxfp4::codes8(hi)) : make_uint2(0u, 0u);
        if ((lane & 1) == 0 && b < width) scale[row * width + b] = c < K16 ? (uint8_t)byte : (uint8_t)0;
    }
    grid_dep_launch();
}

// Row index[i] of quantised rows -> row i: a warp per row, eight 16-byte loads in flight, the next row's index fetched meanwhile.
constexpr int kUnroll = 8;
__global__ void __launch_bounds__(256) gather_kernel(const uint4* __restrict__ src_codes, const uint32_t* __restrict__ src_scale,
                                                     const int32_t* __restrict__ index, uint4* __restrict__ codes,
                                                     uint32_t* __restrict__ scale, int n_src, int n_rows, int K32, int words) {
    const int lane = threadIdx.x & 31, n_warps = gridDim.x * (blockDim.x >> 5);
    int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    int from = row < n_rows ? __ldg(index + row) : 0;
    grid_dep_wait();
    for (; row < n_rows; row += n_warps) {
        const bool inside = (unsigned)from < (unsigned)n_src;
        const uint4* s = src_codes + (long long)(inside ? from : 0) * K32;
        const uint32_t* ss = src_scale + (long long)(inside ? from : 0) * words;
        uint4* d = codes + (long long)row * K32;
        uint32_t* ds = scale + (long long)row * words;
        if (row + n_warps < n_rows) from = __ldg(index + row + n_warps);
        for (int c = lane; c < words; c += 32) {
            uint32_t v = mxfp4::kLowest * 0x01010101u;  // (of a row of zeros)
            if (K32 - 4 * c < 4) v &= (1u << (8 * (K32 - 4 * c))) - 1;
            ds[c] = inside ? __ldcg(ss + c) : v;
        }
        for (int c = lane; c < K32; c += 32 * kUnroll) {
            uint4 v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                v[u] = inside && c + 32 * u < K32 ? __ldcg(s + c + 32 * u) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (c + 32 * u < K32) d[c + 32 * u] = v[u];
        }
    }
}

static bool sizes_ok(int64_t n_src, int64_t n_rows, int64_t K) {
    return n_src >= 0 && n_src <= 0x3FFFFFFFLL && n_rows >= 0 && n_rows <= 0x3FFFFFFFLL && K > 0 && K <= 0x3FFFFFFLL;
}

// Whether the rows of x are quantised once, into scratch, and their bytes gathered: where an index names every row of x four times or
// more and the second launch does not matter.  Every row of the result quantised | two passes, us (rows of x, times each is named, K): 4096 x 8,
// 7168: 66.0 | 40.5; 1024 x 8, 7168: 18.5 | 12.3; 512 x 8, 7168: 11.1 | 8.2; 256 x 8, 7168: 7.5 | 6.2; 128 x 8, 7168: 6.2 | 6.2; 4096 x 8, 2048:
// 36.9 | 16.4; 4096 x 4, 7168: 35.5 | 28.7; 4096 x 2, 7168: 20.5 | 21.3.
static bool two_passes(int64_t n_src, int64_t n_rows, int64_t K) { return n_rows >= 4 * n_src && n_rows * K >= (12ll << 20); }

static int launch_quantize(const void* x, const int32_t* index, void* codes, uint8_t* scale, int64_t n_src, int64_t n_rows, int64_t K,
                           cudaStream_t st) {
    const int width = (int)mxfp4::scale_width(K), units = (2 * width + kWarpChunks - 1) / kWarpChunks, warps = std::min(units, 8);
    const int groups = (units + warps - 1) / warps;
    quantize_kernel<<<dim3((unsigned)n_rows, (unsigned)groups), 32 * warps, 0, st>>>(static_cast<const uint4*>(x), index,
                                                                                    static_cast<uint2*>(codes), scale, (int)n_src,
                                                                                    (int)(K / 16), width);
    B200MOE_CUDA_TRY(cudaGetLastError());
    return B200MOE_OK;
}

}  // namespace mq
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_mxfp4_quantize_rows_scratch_bytes(int64_t n_src, int64_t n_rows, int64_t K, int has_index) {
    if (!mq::sizes_ok(n_src, n_rows, K) || (K % 32) != 0 || n_src == 0 || !has_index || !mq::two_passes(n_src, n_rows, K)) return 0;
    return (size_t)n_src * ((size_t)K / 2 + (size_t)mxfp4::scale_width(K));
}

extern "C" int b200moe_mxfp4_quantize_rows(const void* x, const int32_t* index, void* codes, uint8_t* scale, int64_t n_src,
                                           int64_t n_rows, int64_t K, void* scratch, size_t scratch_bytes, void* stream) {
    if (!mq::sizes_ok(n_src, n_rows, K) || (K % 32) != 0 || (!index && n_rows > n_src)) return B200MOE_ERR_SHAPE;
    if (n_rows == 0) return B200MOE_OK;
    if ((!x && n_src > 0) || !codes || !scale) return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(x) || !aligned16(codes) || (reinterpret_cast<uintptr_t>(scale) & 3u) != 0 || !aligned16(scratch)) return B200MOE_ERR_ALIGNMENT;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t need = b200moe_mxfp4_quantize_rows_scratch_bytes(n_src, n_rows, K, index != nullptr);
    if (need == 0 || !scratch || scratch_bytes < need) return mq::launch_quantize(x, index, codes, scale, n_src, n_rows, K, st);
    uint8_t* once = static_cast<uint8_t*>(scratch);
    uint8_t* once_scale = once + (size_t)n_src * (size_t)(K / 2);
    const int rc = mq::launch_quantize(x, nullptr, once, once_scale, n_src, n_src, K, st);
    if (rc != B200MOE_OK) return rc;
    const int64_t want = (n_rows + 7) / 8, most = 8LL * sm_count();
    B200MOE_CUDA_TRY(launch_dependent(mq::gather_kernel, (unsigned)(want < most ? want : most), 256, 0, st,
                                      reinterpret_cast<const uint4*>(once), reinterpret_cast<const uint32_t*>(once_scale), index,
                                      static_cast<uint4*>(codes), reinterpret_cast<uint32_t*>(scale), (int)n_src, (int)n_rows,
                                      (int)(K / 32), (int)(mxfp4::scale_width(K) / 4)));
    return B200MOE_OK;
}

// Rows of bf16 quantised to e4m3 with one fp32 scale per 128 elements, optionally gathered by an index on the way (token rows
// into expert order).
//
//   a = max(2^-100, largest magnitude of the block);  scale = a / 448;  code = e4m3_rne(x * 448 / a)
//
// The floor keeps the quotient finite for a block of zeros.  A block that holds an infinity or a NaN gets the scale NaN (and
// codes 0): everything that it stands for is NaN, as every sum over the row would be.
#include "common.cuh"
#include "fp8_block.cuh"

namespace b200moe {
namespace fq {

// Eight lanes take a block, 16 elements (32 bytes in, 16 out) each, a warp kSteps times four blocks; a CTA takes a row or up to eight
// warps' blocks of it.  Bound by memory where the rows are read once (32768 rows of 7168: 104 us, 6.8 TB/s; of 2048:
// 37 us; 4096 of 7168: 15.6 us, 5.7 TB/s), by its launch where they are few (8 rows: 1.8 us).  Tried and not kept: one step (104 us where two take
// 84: 4096 rows of 7168, each named eight times), four (88), warps that walk over rows with the next one's loads under way (88 - 92).
constexpr int kSteps = 2;
constexpr int kWarpBlocks = 4 * kSteps;

__global__ void __launch_bounds__(256) quantize_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ index,
                                                       uint4* __restrict__ codes, float* __restrict__ scale, int n_src, int K16, int KB) {
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
        float f[16], m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            f[2 * j] = __uint_as_float(w[j] << 16);
            f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            m = fp8_block::max_magnitude(m, f[2 * j], f[2 * j + 1]);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = fp8_block::max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        const fp8_block::Quantizer q(m);
        if (!q.finite()) {
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] = 0.f;
        }
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            o[j] = q.codes2(pack_f32x2(f[4 * j], f[4 * j + 1])) | (q.codes2(pack_f32x2(f[4 * j + 2], f[4 * j + 3])) << 16);
        if (c < K16) codes[row * K16 + c] = make_uint4(o[0], o[1], o[2], o[3]);
        if (l8 == 0 && b < KB) scale[row * KB + b] = q.scale;
    }
    grid_dep_launch();
}

// Row index[i] of quantised rows -> row i: a warp per row, eight 16-byte loads in flight, the next row's index fetched meanwhile.
constexpr int kUnroll = 8;
__global__ void __launch_bounds__(256) gather_kernel(const uint4* __restrict__ src_codes, const float* __restrict__ src_scale,
                                                     const int32_t* __restrict__ index, uint4* __restrict__ codes,
                                                     float* __restrict__ scale, int n_src, int n_rows, int K16, int KB) {
    const int lane = threadIdx.x & 31, n_warps = gridDim.x * (blockDim.x >> 5);
    int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    int from = row < n_rows ? __ldg(index + row) : 0;
    grid_dep_wait();
    for (; row < n_rows; row += n_warps) {
        const bool inside = (unsigned)from < (unsigned)n_src;
        const uint4* s = src_codes + (long long)(inside ? from : 0) * K16;
        const float* ss = src_scale + (long long)(inside ? from : 0) * KB;
        uint4* d = codes + (long long)row * K16;
        float* ds = scale + (long long)row * KB;
        if (row + n_warps < n_rows) from = __ldg(index + row + n_warps);
        for (int c = lane; c < KB; c += 32) ds[c] = inside ? __ldcg(ss + c) : fp8_block::kFloor / fp8_block::kMax;
        for (int c = lane; c < K16; c += 32 * kUnroll) {
            uint4 v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                v[u] = inside && c + 32 * u < K16 ? __ldcg(s + c + 32 * u) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (c + 32 * u < K16) d[c + 32 * u] = v[u];
        }
    }
}

static bool sizes_ok(int64_t n_src, int64_t n_rows, int64_t K) {
    return n_src >= 0 && n_src <= 0x3FFFFFFFLL && n_rows >= 0 && n_rows <= 0x3FFFFFFFLL && K > 0 && K <= 0x3FFFFFFLL;
}

// Whether the rows of x are quantised once, into scratch, and their bytes gathered: where an index names every row of x four times or
// more and the second launch does not matter.  Every row of the result quantised | two passes, us (rows of x, times each is named,
// K): 4096 x 8, 7168: 84.0 | 69.6 (cudaMemset takes 62 for as many bytes); 1024 x 8, 7168: 22.6 | 18.5; 512 x 8, 7168: 12.3 | 12.2;
// 256 x 8, 7168: 10.6 | 15.8; 4096 x 8, 2048: 37.9 | 22.5; 4096 x 2, 7168: 24.6 | 29.1.
static bool two_passes(int64_t n_src, int64_t n_rows, int64_t K) { return n_rows >= 4 * n_src && n_rows * K >= (32ll << 20); }

static int launch_quantize(const void* x, const int32_t* index, void* codes, float* scale, int64_t n_src, int64_t n_rows, int64_t K,
                           cudaStream_t st) {
    const int KB = (int)((K + 127) / 128), units = (KB + kWarpBlocks - 1) / kWarpBlocks, warps = units < 8 ? units : 8;
    const int groups = (units + warps - 1) / warps;
    quantize_kernel<<<dim3((unsigned)n_rows, (unsigned)groups), 32 * warps, 0, st>>>(static_cast<const uint4*>(x), index,
                                                                                    static_cast<uint4*>(codes), scale, (int)n_src,
                                                                                    (int)(K / 16), KB);
    B200MOE_CUDA_TRY(cudaGetLastError());
    return B200MOE_OK;
}

}  // namespace fq
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_fp8_quantize_rows_scratch_bytes(int64_t n_src, int64_t n_rows, int64_t K, int has_index) {
    if (!fq::sizes_ok(n_src, n_rows, K) || n_src == 0 || !has_index || !fq::two_passes(n_src, n_rows, K)) return 0;
    return (size_t)n_src * ((size_t)K + 4u * (size_t)((K + 127) / 128));
}

extern "C" int b200moe_fp8_quantize_rows(const void* x, const int32_t* index, void* codes, float* scale, int64_t n_src,
                                         int64_t n_rows, int64_t K, void* scratch, size_t scratch_bytes, void* stream) {
    if (!fq::sizes_ok(n_src, n_rows, K) || (K % 16) != 0 || (!index && n_rows > n_src)) return B200MOE_ERR_SHAPE;
    if (n_rows == 0) return B200MOE_OK;
    if ((!x && n_src > 0) || !codes || !scale) return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(x) || !aligned16(codes) || !aligned16(scratch)) return B200MOE_ERR_ALIGNMENT;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t need = b200moe_fp8_quantize_rows_scratch_bytes(n_src, n_rows, K, index != nullptr);
    if (need == 0 || !scratch || scratch_bytes < need) return fq::launch_quantize(x, index, codes, scale, n_src, n_rows, K, st);
    uint8_t* once = static_cast<uint8_t*>(scratch);
    float* once_scale = reinterpret_cast<float*>(once + (size_t)n_src * (size_t)K);
    const int rc = fq::launch_quantize(x, nullptr, once, once_scale, n_src, n_src, K, st);
    if (rc != B200MOE_OK) return rc;
    const int64_t want = (n_rows + 7) / 8, most = 8LL * sm_count();
    B200MOE_CUDA_TRY(launch_dependent(fq::gather_kernel, (unsigned)(want < most ? want : most), 256, 0, st,
                                      reinterpret_cast<const uint4*>(once), static_cast<const float*>(once_scale), index,
                                      static_cast<uint4*>(codes), scale, (int)n_src, (int)n_rows, (int)(K / 16), (int)((K + 127) / 128)));
    return B200MOE_OK;
}

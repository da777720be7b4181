// Grouped GEMM whose two operands are 8-bit floats with one scale per block of 128:
//
//   y[m, n] = sum over blocks kb of 128 k:  x_scale[m, kb] * weight_scale[g, kb, n / 128] * sum_{k in kb} x[m, k] * w[g, k, n]
//
// x e4m3 [M, K] with fp32 scales per row and 128 k, weights e4m3 [G, K, N] with fp32 scales per 128 x 128.
#include <cuda_fp8.h>

#include "common.cuh"
#include "fp8_block.cuh"

namespace b200moe {
namespace fb {

struct Args {
    const uint8_t* x;
    const float* x_scale;
    const uint8_t* weight;
    const float* w_scale;
    const int64_t* group_list;
    void* out;
    float* out_scale;
    int M, K, N, G, gl_type, KB, NB;
    int* status;
    int* findings;
};

__device__ __forceinline__ float e4m3_to_float(uint32_t code) {
    __nv_fp8_e4m3 v;
    v.__x = (__nv_fp8_storage_t)code;
    return (float)v;
}

constexpr int kRows = 16;
template <bool GATE_UP>
__global__ void __launch_bounds__(GATE_UP ? 256 : 128) simple_kernel(const Args a) {
    __shared__ int row_start[kMaxExperts + 1];
    __shared__ float xs[kRows][128];
    __shared__ alignas(16) float h[kRows][128];
    load_row_starts(a.group_list, a.G, a.M, a.gl_type, row_start, a.status);
    int tile = blockIdx.y, g = 0, r0 = 0, rows = 0;
    for (;; ++g) {
        if (g == a.G) return;
        const int n = row_start[g + 1] - row_start[g], tiles = (n + kRows - 1) / kRows;
        if (tile < tiles) {
            r0 = row_start[g] + tile * kRows;
            rows = min(kRows, n - tile * kRows);
            break;
        }
        tile -= tiles;
    }
    const int half = threadIdx.x >> 7, c = threadIdx.x & 127;
    const int col = blockIdx.x * 128 + c + (GATE_UP ? half * (a.N >> 1) : 0);
    float acc[kRows] = {};
    for (int kb = 0; kb < a.KB; ++kb) {
        const int k0 = kb * 128, kn = min(128, a.K - k0);
        __syncthreads();
        for (int i = threadIdx.x; i < kRows * 128; i += blockDim.x) {
            const int r = i >> 7, k = i & 127;
            xs[r][k] = r < rows && k < kn ? e4m3_to_float(a.x[(size_t)(r0 + r) * a.K + k0 + k]) : 0.f;
        }
        __syncthreads();
        float part[kRows] = {};
        if (col < a.N) {
            for (int k = 0; k < kn; ++k) {
                const float w = e4m3_to_float(a.weight[((size_t)g * a.K + k0 + k) * a.N + col]);
#pragma unroll
                for (int r = 0; r < kRows; ++r) part[r] = fmaf(xs[r][k], w, part[r]);
            }
            const float ws = a.w_scale[((size_t)g * a.KB + kb) * a.NB + (col >> 7)];
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                if (r < rows) acc[r] = fmaf(part[r], ws * a.x_scale[(size_t)(r0 + r) * a.KB + kb], acc[r]);
        }
    }
    if constexpr (!GATE_UP) {
        if (col < a.N)
            for (int r = 0; r < rows; ++r) static_cast<__nv_bfloat16*>(a.out)[(size_t)(r0 + r) * a.N + col] = __float2bfloat16_rn(acc[r]);
    } else {
        __syncthreads();
        if (half == 1)
            for (int r = 0; r < kRows; ++r) xs[r][c] = acc[r];
        __syncthreads();
        if (half == 0)
            for (int r = 0; r < kRows; ++r) h[r][c] = acc[r] / (1.f + expf(-acc[r])) * xs[r][c];
        __syncthreads();
        const int inter = a.N >> 1;
        for (int r = threadIdx.x >> 5; r < rows; r += 8) {
            const int lane = threadIdx.x & 31;
            const float4 v = reinterpret_cast<const float4*>(h[r])[lane];
            uint32_t top = 0;  // magnitudes order as their bits do, infinities and NaN last
            top = max(max(__float_as_uint(v.x) & 0x7FFFFFFFu, __float_as_uint(v.y) & 0x7FFFFFFFu),
                      max(__float_as_uint(v.z) & 0x7FFFFFFFu, __float_as_uint(v.w) & 0x7FFFFFFFu));
            top = __reduce_max_sync(0xffffffffu, top);
            const fp8_block::Quantizer q(__uint_as_float(top));
            reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + (size_t)(r0 + r) * inter + blockIdx.x * 128)[lane] = q.four(v.x, v.y, v.z, v.w);
            if (lane == 0) a.out_scale[(size_t)(r0 + r) * (inter >> 7) + blockIdx.x] = q.scale;
        }
    }
}

__global__ void keep_finding_kernel(const int* status, int* findings) {
    if (status[0] != 0 && atomicCAS(findings, 0, status[0]) == 0) findings[1] = status[1];
}

}  // namespace fb
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_grouped_gemm_fp8_block_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t G, int gate_up_silu) {
    return B200MOE_STATUS_BYTES;
}

extern "C" int b200moe_grouped_gemm_fp8_block(const void* x, const float* x_scale, const void* weight, const float* weight_scale,
                                              const int64_t* group_list, void* out, float* out_scale, int64_t M, int64_t K, int64_t N,
                                              int64_t G, int group_list_type, int gate_up_silu, void* workspace,
                                              size_t workspace_bytes, int32_t* findings, void* stream) {
    if (M < 0 || K <= 0 || N <= 0 || G <= 0 || G > kMaxExperts || (K % 16) != 0 || (N % 16) != 0 || M > 0x3FFFFFFFLL ||
        K > 0x3FFFFFFFLL || N > 0x3FFFFFFFLL || (gate_up_silu && (N % 256) != 0))
        return B200MOE_ERR_SHAPE;
    if (group_list_type != B200MOE_GROUP_LIST_CUMSUM && group_list_type != B200MOE_GROUP_LIST_COUNTS) return B200MOE_ERR_ARGUMENT;
    if (gate_up_silu != 0 && gate_up_silu != 1) return B200MOE_ERR_ARGUMENT;
    if (M == 0) return B200MOE_OK;
    if (!x || !x_scale || !weight || !weight_scale || !group_list || !out || (gate_up_silu && !out_scale))
        return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(x) || !aligned16(weight) || !aligned16(out)) return B200MOE_ERR_ALIGNMENT;
    if (!workspace || workspace_bytes < b200moe_grouped_gemm_fp8_block_workspace_bytes(M, K, N, G, gate_up_silu))
        return B200MOE_ERR_WORKSPACE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    fb::Args a;
    a.x = static_cast<const uint8_t*>(x);
    a.x_scale = x_scale;
    a.weight = static_cast<const uint8_t*>(weight);
    a.w_scale = weight_scale;
    a.group_list = group_list;
    a.out = out;
    a.out_scale = out_scale;
    a.M = (int)M; a.K = (int)K; a.N = (int)N; a.G = (int)G;
    a.gl_type = group_list_type;
    a.KB = (int)((K + 127) / 128);
    a.NB = (int)((N + 127) / 128);
    a.status = static_cast<int*>(workspace);
    a.findings = findings;
    B200MOE_CUDA_TRY(cudaMemsetAsync(workspace, 0, B200MOE_STATUS_BYTES, st));
    const long long tiles = (M + fb::kRows - 1) / fb::kRows + G;
    if (tiles > 65535) return B200MOE_ERR_SHAPE;
    const dim3 grid((unsigned)(gate_up_silu ? N / 256 : a.NB), (unsigned)tiles);
    if (gate_up_silu) fb::simple_kernel<true><<<grid, 256, 0, st>>>(a);
    else fb::simple_kernel<false><<<grid, 128, 0, st>>>(a);
    B200MOE_CUDA_TRY(cudaGetLastError());
    if (findings) {
        fb::keep_finding_kernel<<<1, 1, 0, st>>>(a.status, findings);
        B200MOE_CUDA_TRY(cudaGetLastError());
    }
    return B200MOE_OK;
}

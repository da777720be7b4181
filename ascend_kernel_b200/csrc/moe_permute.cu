// Tokens on their way to the experts and back, with gradients: the stable sort of the (token, j) pairs by expert, the rows
// of the sorted pairs, and the weighted sum of a token's rows.
//
//   sort      slot[p] = number of kept pairs of smaller experts + number of earlier pairs of the same expert; token_of[slot[p]] = p / k
//   dispatch  rows[slot[t, j]] = x[t];                      grad_x[t] = sum_j grad_rows[slot[t, j]]
//   combine   out[t] = sum_j w[t, j] y[slot[t, j]];         grad_y[slot[t, j]] = w[t, j] g[t],  grad_w[t, j] = <g[t], y[slot[t, j]]>
//
// A pair whose expert is outside 0 .. E - 1 is dropped: slot -1, no row, no part in a sum.  Rows behind the kept pairs (token_of -1)
// are zero, and so are their gradients.  No floating-point atomics and a fixed order of every sum: the same bits each time.
#include <algorithm>

#include "common.cuh"
#include "ptx.cuh"

namespace b200moe {
namespace mp {

constexpr int kMaxTopK = 32;

// ---- the sort ---------------------------------------------------------------------------------------------------------
//
// A CTA takes a range of pairs, each of its warps a part of that.  Two passes over the ids: count per warp and expert
// in shared memory, then, with every warp's first position of every expert in the counts' place, hand the positions out.  In a
// warp, lanes of the same expert find one another by a vote on each bit of its number, and take positions in the order of their lanes.  Short calls
// are one CTA's; where there are more, a first kernel leaves each CTA's counts in scratch memory, and every CTA of the second adds up those before it,
// its own counting done beside the first kernel.
//
// Measured, one call after the other, us (256 experts): 37 x 8 pairs 4.2, 512 x 8 10, 65536 x 8 16.4 (of its 6.3 MB the memory takes 1): launches and the chains
// of shared-memory latencies in between.  Tried and not kept: the match instruction (22.6), clusters that add up their counts in
// distributed shared memory (18 in clusters of 4, 31 of 8, which do not all fit at once), stores put in order in shared memory first (16.4).

constexpr int kWarps = 32, kFewWarps = 8;
constexpr int kRoom = 32;          // sums of the warps, in static shared memory
// Pairs of a call that is one CTA's.  One CTA | two kernels, us (256 experts; 1024): 2048 pairs 8.2 | 14.3; 11.3 | 22.5, 4096 pairs 10.3 | 14.3; 12.3 | 22.5, 6144
// pairs 16.4 | 13.8; 20.5 | 22.5, 8192 pairs 18.4 | 13.8; 22.5 | 22.5.
constexpr int kOnePairs = 4096;
constexpr int kMostCtas = 128;
constexpr int kBatch = 4;          // ids a lane has at a time

struct SortArgs {
    const int32_t* idx;
    long long* counts;
    int32_t* token_of;
    int32_t* slot;
    int32_t* totals;   // [E][kMostCtas]
    int P, E, k, cta_pairs, warp_pairs;
    int bits;          // of an expert's number
    unsigned long long per_k;  // ceil(2^35 / k)
};

// p / k: with p < 2^30 and k <= 32 the rounding of per_k adds less than 31 * 2^30 < 2^35
__device__ __forceinline__ int token_of_pair(const SortArgs& a, int p) {
    return a.k == 1 ? p : (int)(((unsigned long long)(unsigned)p * a.per_k) >> 35);
}

// The lanes whose expert is the same; for a lane without one (-1) it means nothing.  (A vote for each bit: the match instruction takes as many
// steps as there are different numbers.)
__device__ __forceinline__ unsigned same_expert(int e, int bits) {
    unsigned same = __ballot_sync(0xffffffffu, e >= 0);
#pragma unroll
    for (int b = 0; b < 10; ++b) {
        if (b >= bits) break;
        const bool mine = (e >> b) & 1;
        const unsigned set = __ballot_sync(0xffffffffu, mine);
        same &= mine ? set : ~set;
    }
    return same;
}

// A warp's pairs, 32 * kBatch at a time: [first, end) and the ids of a batch (-1: none).
struct WarpRange {
    long long first;
    int end;
};
__device__ __forceinline__ WarpRange warp_range(const SortArgs& a) {
    const long long cta_end = min((long long)a.P, ((long long)blockIdx.x + 1) * a.cta_pairs);
    const long long first = (long long)blockIdx.x * a.cta_pairs + (long long)(threadIdx.x >> 5) * a.warp_pairs;
    return {first, (int)min(cta_end, first + a.warp_pairs)};
}
__device__ __forceinline__ void load_batch(const SortArgs& a, long long p0, int end, int (&e)[kBatch]) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const long long p = p0 + 32 * i + (threadIdx.x & 31);
        e[i] = p < end ? __ldg(a.idx + p) : -1;
        if ((unsigned)e[i] >= (unsigned)a.E) e[i] = -1;
    }
}
// Counts a batch on top of `mine`, the warp's counts by expert, in the order of the pairs; rank[i]: the pairs of the same expert before.
__device__ __forceinline__ void count_batch(const SortArgs& a, const int (&e)[kBatch], int* mine, int (&rank)[kBatch]) {
    unsigned peers[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) peers[i] = same_expert(e[i], a.bits);
    const unsigned lower = (1u << (threadIdx.x & 31)) - 1;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const int below = __popc(peers[i] & lower);
        int before = 0;
        if (e[i] >= 0) before = mine[e[i]];
        __syncwarp();
        if (e[i] >= 0 && below == 0) mine[e[i]] = before + __popc(peers[i]);
        __syncwarp();
        rank[i] = before + below;
    }
}

// The first pass: hist[warp][e] = the warp's pairs of expert e; e and rank are those of its last batch.
template <int WARPS>
__device__ __forceinline__ void count_pairs(const SortArgs& a, int* hist, int (&e)[kBatch], int (&rank)[kBatch]) {
    const WarpRange w = warp_range(a);
    load_batch(a, w.first, w.end, e);
    for (int i = threadIdx.x; i < WARPS * a.E; i += WARPS * 32) hist[i] = 0;
    __syncthreads();
    int* mine = hist + (threadIdx.x >> 5) * a.E;
    for (long long p0 = w.first; p0 < w.end; p0 += 32 * kBatch) {
        if (p0 != w.first) load_batch(a, p0, w.end, e);
        count_batch(a, e, mine, rank);
    }
    __syncthreads();
}

// hist -> the sums over the warps before each; returns expert threadIdx.x's pairs in the CTA.
template <int WARPS>
__device__ __forceinline__ int scan_warps(const SortArgs& a, int* hist) {
    int total = 0;
    if ((int)threadIdx.x < a.E) {
        int c[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) c[w] = hist[w * a.E + threadIdx.x];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            hist[w * a.E + threadIdx.x] = total;
            total += c[w];
        }
    }
    return total;
}

// Sum over the threads below and, in `all`, over all of the CTA.
template <int WARPS>
__device__ __forceinline__ int cta_exclusive_sum(int v, int& all, int* room) {
    int sum;
    const int below = warp_exclusive_sum(v, sum);
    if ((threadIdx.x & 31) == 31) room[threadIdx.x >> 5] = sum;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const int before = warp_exclusive_sum(lane < WARPS ? room[lane] : 0, all);
    return below + __shfl_sync(0xffffffffu, before, threadIdx.x >> 5);
}

// The second pass: base[e] is where the CTA's pairs of expert e begin.  A warp with one batch still has its ranks.
__device__ __forceinline__ void place_pairs(const SortArgs& a, int* hist, const int* base, int kept, int (&e)[kBatch], int (&rank)[kBatch]) {
    const WarpRange w = warp_range(a);
    int* mine = hist + (threadIdx.x >> 5) * a.E;
    const bool once = a.warp_pairs <= 32 * kBatch;
    for (long long p0 = w.first; p0 < w.end; p0 += 32 * kBatch) {
        if (!once) {
            load_batch(a, p0, w.end, e);
            count_batch(a, e, mine, rank);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int p = (int)p0 + 32 * i + (int)(threadIdx.x & 31);
            const int at = e[i] < 0 ? -1 : base[e[i]] + rank[i] + (once ? mine[e[i]] : 0);
            if (p < w.end) a.slot[p] = at;
            if (at >= 0) a.token_of[at] = token_of_pair(a, p);
        }
    }
    for (long long r = (long long)kept + blockIdx.x * blockDim.x + threadIdx.x; r < a.P; r += (long long)gridDim.x * blockDim.x) a.token_of[r] = -1;
}

// A call that is one CTA's; E <= 32 WARPS.
template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) sort_one_kernel(const SortArgs a) {
    extern __shared__ int smem[];  // [WARPS][E], [E]
    __shared__ int s_room[kRoom];
    int *hist = smem, *base = hist + WARPS * a.E;
    int id[kBatch], rank[kBatch], kept;
    count_pairs<WARPS>(a, hist, id, rank);
    const int total = scan_warps<WARPS>(a, hist);
    const int start = cta_exclusive_sum<WARPS>(total, kept, s_room);
    if ((int)threadIdx.x < a.E) {
        base[threadIdx.x] = start;
        a.counts[threadIdx.x] = total;
    }
    __syncthreads();
    place_pairs(a, hist, base, kept, id, rank);
}

__global__ void __launch_bounds__(kWarps * 32, 1) sort_count_kernel(const SortArgs a) {
    extern __shared__ int smem[];  // [kWarps][E]
    int id[kBatch], rank[kBatch];
    count_pairs<kWarps>(a, smem, id, rank);
    if ((int)threadIdx.x < a.E) {
        int total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) total += smem[w * a.E + threadIdx.x];
        a.totals[threadIdx.x * kMostCtas + blockIdx.x] = total;
    }
    grid_dep_launch();
}

__global__ void __launch_bounds__(kWarps * 32, 1) sort_place_kernel(const SortArgs a) {
    extern __shared__ int smem[];  // [kWarps][E], twice [E]
    __shared__ int s_room[kRoom];
    int *hist = smem, *base = hist + kWarps * a.E, *alls = base + a.E;
    const int e = threadIdx.x;
    int id[kBatch], rank[kBatch], kept;
    count_pairs<kWarps>(a, hist, id, rank);
    scan_warps<kWarps>(a, hist);
    // every expert's pairs in the CTAs before this one and in all: a warp an expert, a lane four CTAs
    const int lane = threadIdx.x & 31;
    grid_dep_wait();
#pragma unroll 4
    for (int x = threadIdx.x >> 5; x < a.E; x += kWarps) {
        static_assert(kMostCtas == 4 * 32, "CTAs of a lane");
        const int4 v = __ldcg(reinterpret_cast<const int4*>(a.totals + x * kMostCtas) + lane);
        const int c[4] = {v.x, v.y, v.z, v.w};
        int before = 0, all = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (4 * lane + i < (int)gridDim.x) all += c[i];
            if (4 * lane + i < (int)blockIdx.x) before += c[i];
        }
        before = __reduce_add_sync(0xffffffffu, before);
        all = __reduce_add_sync(0xffffffffu, all);
        if (lane == 0) {
            base[x] = before;
            alls[x] = all;
        }
    }
    __syncthreads();
    const int all = e < a.E ? alls[e] : 0;
    const int start = cta_exclusive_sum<kWarps>(all, kept, s_room);
    if (e < a.E) {
        base[e] += start;
        if (blockIdx.x == 0) a.counts[e] = all;
    }
    __syncthreads();
    place_pairs(a, hist, base, kept, id, rank);
}

static bool sort_sizes_ok(int64_t T, int64_t E, int64_t k) {
    return T >= 0 && E > 0 && E <= kMaxExperts && k > 0 && k <= kMaxTopK && T <= 0x3FFFFFFF / k;
}
// The number of CTAs and the pairs of each.
static int ctas_of(int64_t P) {
    if (P <= kOnePairs) return 1;
    return (int)std::min<int64_t>(kMostCtas, (P + 1023) / 1024);
}
static int cta_pairs_of(int64_t P) {
    const int64_t n = (P + ctas_of(P) - 1) / ctas_of(P);
    return (int)((n + 1023) / 1024 * 1024);
}

// ---- rows ---------------------------------------------------------------------------------------------------------------
//
// A CTA of 256 threads takes a token, 16 bytes a thread at a time, and where tokens are few several CTAs share its columns (not those that add up the
// products for a weight's gradient).  Memory bounds all of them.  4096 tokens x 8 rows of 7168 bf16, us: dispatch 92 (529 MB, 5.7 TB/s: nine
// tenths of it written), its gradient 82 (6.5 TB/s), combine 83, its gradients 160 (6.2 TB/s; of the rows alone 93); 509 x 2 rows of 2048 fp32: 4.2, 4.1, 4.1, 6.2.  Tried and not kept: streaming loads and stores, with which 8 x 4096 rows of
// 2048 bf16 gain (dispatch 28.7 -> 23.9, its gradient 27.0 -> 22.5, combine 28.7 -> 23.9) and the joint gradients of rows of 7168 lose (160 -> 171): of
// calls right behind one another, where a part of that is what the call before has left in L2.

// 16 bytes of a row as fp32 and back.
template <class T>
struct Piece;
template <>
struct Piece<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
};
template <>
struct Piece<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
        v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};

constexpr int kRowThreads = 256;

// The token's slots, -1 where one is no row of the P there are; in shared memory for all of the CTA.
__device__ __forceinline__ void load_slots(const int32_t* slot, long long t, int k, long long P, int* s_slot) {
    if ((int)threadIdx.x < k) {
        const int s = __ldg(slot + t * k + threadIdx.x);
        s_slot[threadIdx.x] = (unsigned)s < (unsigned)P ? s : -1;
    }
}

// Rows t k .. t k + k - 1 that no pair has: zeros.
__device__ __forceinline__ void clear_rows(const int32_t* token_of, long long t, int k, uint4* rows, int width16) {
    for (int j = 0; j < k; ++j)
        if (__ldg(token_of + t * k + j) < 0) {
            uint4* d = rows + (t * k + j) * width16;
            for (int c = blockIdx.y * kRowThreads + threadIdx.x; c < width16; c += gridDim.y * kRowThreads) d[c] = make_uint4(0u, 0u, 0u, 0u);
        }
}

// A CTA per token: its row is read once and stored to every slot.
__global__ void __launch_bounds__(kRowThreads) dispatch_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ token_of,
                                                               const int32_t* __restrict__ slot, uint4* __restrict__ rows, int k,
                                                               int width16) {
    __shared__ int s_slot[kMaxTopK];
    const long long t = blockIdx.x;
    load_slots(slot, t, k, (long long)gridDim.x * k, s_slot);
    __syncthreads();
    for (int c = blockIdx.y * kRowThreads + threadIdx.x; c < width16; c += gridDim.y * kRowThreads) {
        const uint4 v = __ldg(x + t * width16 + c);
        for (int j = 0; j < k; ++j)
            if (s_slot[j] >= 0) rows[(long long)s_slot[j] * width16 + c] = v;
    }
    clear_rows(token_of, t, k, rows, width16);
}

// out[t] = sum_j w[t, j] y[slot[t, j]], w 1 where there is none; fp32 sums in the order of j.
template <class T, bool WEIGHTED>
__global__ void __launch_bounds__(kRowThreads) sum_kernel(const uint4* __restrict__ y, const float* __restrict__ weight,
                                                          const int32_t* __restrict__ slot, uint4* __restrict__ out, int k, int width16) {
    constexpr int N = Piece<T>::N;
    __shared__ int s_slot[kMaxTopK];
    __shared__ float s_w[kMaxTopK];
    const long long t = blockIdx.x;
    load_slots(slot, t, k, (long long)gridDim.x * k, s_slot);
    if (WEIGHTED && (int)threadIdx.x < k) s_w[threadIdx.x] = __ldg(weight + t * k + threadIdx.x);
    __syncthreads();
    for (int c = blockIdx.y * kRowThreads + threadIdx.x; c < width16; c += gridDim.y * kRowThreads) {
        float acc[N] = {};
        for (int j0 = 0; j0 < k; j0 += 8) {
            uint4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < k && s_slot[j0 + j] >= 0) v[j] = __ldg(y + (long long)s_slot[j0 + j] * width16 + c);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < k && s_slot[j0 + j] >= 0) {
                    const float w = WEIGHTED ? s_w[j0 + j] : 1.f;
                    float f[N];
                    Piece<T>::unpack(v[j], f);
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[i] = WEIGHTED ? fmaf(w, f[i], acc[i]) : acc[i] + f[i];
                }
        }
        out[t * width16 + c] = Piece<T>::pack(acc);
    }
}

// Gradient of the weighted sum, a CTA per token: its row of g stays in L1 for the token's slots, eight of which are taken at a time.
template <class T, bool GRAD_Y, bool GRAD_W>
__global__ void __launch_bounds__(kRowThreads) combine_grad_kernel(const uint4* __restrict__ y, const float* __restrict__ weight,
                                                                   const int32_t* __restrict__ token_of, const int32_t* __restrict__ slot,
                                                                   const uint4* __restrict__ grad, uint4* __restrict__ grad_y,
                                                                   float* __restrict__ grad_w, int k, int width16) {
    constexpr int N = Piece<T>::N, kRowWarps = kRowThreads / 32;
    __shared__ int s_slot[kMaxTopK];
    __shared__ float s_w[kMaxTopK];
    __shared__ float s_dot[kRowWarps][8];
    const long long t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    load_slots(slot, t, k, (long long)gridDim.x * k, s_slot);
    if ((int)threadIdx.x < k) s_w[threadIdx.x] = __ldg(weight + t * k + threadIdx.x);
    __syncthreads();
    for (int j0 = 0; j0 < k; j0 += 8) {
        float dot[8] = {};
        for (int c = threadIdx.x; c < width16; c += kRowThreads) {
            uint4 v[8];
            const uint4 q = __ldg(grad + t * width16 + c);
            if constexpr (GRAD_W) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j0 + j < k && s_slot[j0 + j] >= 0) v[j] = __ldg(y + (long long)s_slot[j0 + j] * width16 + c);
            }
            float g[N];
            Piece<T>::unpack(q, g);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < k && s_slot[j0 + j] >= 0) {
                    if constexpr (GRAD_W) {
                        float f[N];
                        Piece<T>::unpack(v[j], f);
#pragma unroll
                        for (int i = 0; i < N; ++i) dot[j] = fmaf(g[i], f[i], dot[j]);
                    }
                    if constexpr (GRAD_Y) {
                        float o[N];
#pragma unroll
                        for (int i = 0; i < N; ++i) o[i] = s_w[j0 + j] * g[i];
                        grad_y[(long long)s_slot[j0 + j] * width16 + c] = Piece<T>::pack(o);
                    }
                }
        }
        if constexpr (GRAD_W) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
            if (lane == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) s_dot[warp][j] = dot[j];
            }
            __syncthreads();
            if (threadIdx.x < 8 && j0 + (int)threadIdx.x < k) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kRowWarps; ++w) sum += s_dot[w][threadIdx.x];
                grad_w[t * k + j0 + threadIdx.x] = sum;
            }
            __syncthreads();
        }
    }
    if constexpr (GRAD_Y) clear_rows(token_of, t, k, grad_y, width16);
}

static bool row_sizes_ok(int64_t T, int64_t k, int64_t width) {
    return T >= 0 && k > 0 && k <= kMaxTopK && T <= 0x3FFFFFFF / k && width > 0 && width % 8 == 0 && width <= 0x3FFFFFF;
}
static int width16_of(int64_t width, int fp32) { return (int)(width / (fp32 ? 4 : 8)); }
// CTAs that share a token's row where tokens are few.
static unsigned row_parts(int64_t T, int width16) {
    const int64_t want = 4 * sm_count() / std::max<int64_t>(T, 1), most = (width16 + kRowThreads - 1) / kRowThreads;
    return (unsigned)std::max<int64_t>(1, std::min(want, most));
}

}  // namespace mp
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_moe_sort_scratch_bytes(int64_t n_tokens, int64_t n_experts, int64_t top_k) {
    if (!mp::sort_sizes_ok(n_tokens, n_experts, top_k)) return 0;
    const int ctas = mp::ctas_of(n_tokens * top_k);
    return ctas == 1 ? 0 : (size_t)mp::kMostCtas * (size_t)n_experts * 4;
}

extern "C" int b200moe_moe_sort(const int32_t* idx, int64_t n_tokens, int64_t n_experts, int64_t top_k, int64_t* counts,
                                int32_t* token_of, int32_t* slot, void* scratch, size_t scratch_bytes, void* stream) {
    if (!mp::sort_sizes_ok(n_tokens, n_experts, top_k)) return B200MOE_ERR_SHAPE;
    if (!counts || (n_tokens > 0 && (!idx || !token_of || !slot))) return B200MOE_ERR_NULL_POINTER;
    const size_t need = b200moe_moe_sort_scratch_bytes(n_tokens, n_experts, top_k);
    if (need > 0 && (!scratch || scratch_bytes < need)) return B200MOE_ERR_WORKSPACE;
    if (need > 0 && !aligned16(scratch)) return B200MOE_ERR_ALIGNMENT;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    mp::SortArgs a = {};
    a.idx = idx;
    a.counts = reinterpret_cast<long long*>(counts);
    a.token_of = token_of;
    a.slot = slot;
    a.totals = static_cast<int32_t*>(scratch);
    a.P = (int)(n_tokens * top_k); a.E = (int)n_experts; a.k = (int)top_k;
    while ((1 << a.bits) < a.E) ++a.bits;
    a.per_k = ((1ull << 35) + (unsigned)a.k - 1) / (unsigned)a.k;
    const int ctas = mp::ctas_of(a.P);
    // Eight warps where the call has pairs for no more: less to clear and to add up.
    const bool few = ctas == 1 && a.E <= mp::kFewWarps * 32 && a.P <= 32 * mp::kBatch * mp::kFewWarps;
    const int warps = few ? mp::kFewWarps : mp::kWarps;
    a.cta_pairs = mp::cta_pairs_of(a.P);
    a.warp_pairs = std::max(1, ((std::min(a.P, a.cta_pairs) + warps - 1) / warps + 31) / 32) * 32;
    const size_t smem = (size_t)(warps + 2) * (size_t)a.E * 4;
    // (what a launch has without asking for more holds the static part too)
    const auto opt_in = [&](void (*kernel)(mp::SortArgs)) {
        if (smem + mp::kRoom * sizeof(int) <= 48 * 1024) return cudaSuccess;
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (mp::kWarps + 2) * kMaxExperts * 4);
    };
    if (need == 0) {
        const auto kernel = few ? mp::sort_one_kernel<mp::kFewWarps> : mp::sort_one_kernel<mp::kWarps>;
        B200MOE_CUDA_TRY(opt_in(kernel));
        kernel<<<1, warps * 32, smem, st>>>(a);
        B200MOE_CUDA_TRY(cudaGetLastError());
        return B200MOE_OK;
    }
    B200MOE_CUDA_TRY(opt_in(mp::sort_count_kernel));
    B200MOE_CUDA_TRY(opt_in(mp::sort_place_kernel));
    mp::sort_count_kernel<<<(unsigned)ctas, warps * 32, smem, st>>>(a);
    B200MOE_CUDA_TRY(cudaGetLastError());
    B200MOE_CUDA_TRY(launch_dependent(mp::sort_place_kernel, (unsigned)ctas, (unsigned)(warps * 32), smem, st, a));
    return B200MOE_OK;
}

extern "C" int b200moe_moe_dispatch(const void* x, int fp32, const int32_t* token_of, const int32_t* slot, void* rows, int64_t n_tokens,
                                    int64_t top_k, int64_t width, void* stream) {
    if (!mp::row_sizes_ok(n_tokens, top_k, width)) return B200MOE_ERR_SHAPE;
    if (fp32 != 0 && fp32 != 1) return B200MOE_ERR_ARGUMENT;
    if (n_tokens == 0) return B200MOE_OK;
    if (!x || !token_of || !slot || !rows) return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(x) || !aligned16(rows)) return B200MOE_ERR_ALIGNMENT;
    const int w16 = mp::width16_of(width, fp32);
    mp::dispatch_kernel<<<dim3((unsigned)n_tokens, mp::row_parts(n_tokens, w16)), mp::kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint4*>(x), token_of, slot, static_cast<uint4*>(rows), (int)top_k, w16);
    B200MOE_CUDA_TRY(cudaGetLastError());
    return B200MOE_OK;
}

namespace b200moe {
namespace mp {
static int launch_sum(const void* y, int fp32, const float* weight, const int32_t* slot, void* out, int64_t T, int64_t k, int64_t width,
                      void* stream) {
    const int w16 = width16_of(width, fp32);
    void (*kernel)(const uint4*, const float*, const int32_t*, uint4*, int, int);
    if (fp32) kernel = weight ? sum_kernel<float, true> : sum_kernel<float, false>;
    else kernel = weight ? sum_kernel<__nv_bfloat16, true> : sum_kernel<__nv_bfloat16, false>;
    kernel<<<dim3((unsigned)T, row_parts(T, w16)), kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint4*>(y), weight, slot, static_cast<uint4*>(out), (int)k, w16);
    B200MOE_CUDA_TRY(cudaGetLastError());
    return B200MOE_OK;
}
}  // namespace mp
}  // namespace b200moe

extern "C" int b200moe_moe_dispatch_grad(const void* grad_rows, int fp32, const int32_t* slot, void* grad_x, int64_t n_tokens,
                                         int64_t top_k, int64_t width, void* stream) {
    if (!mp::row_sizes_ok(n_tokens, top_k, width)) return B200MOE_ERR_SHAPE;
    if (fp32 != 0 && fp32 != 1) return B200MOE_ERR_ARGUMENT;
    if (n_tokens == 0) return B200MOE_OK;
    if (!grad_rows || !slot || !grad_x) return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(grad_rows) || !aligned16(grad_x)) return B200MOE_ERR_ALIGNMENT;
    return mp::launch_sum(grad_rows, fp32, nullptr, slot, grad_x, n_tokens, top_k, width, stream);
}

extern "C" int b200moe_moe_combine(const void* y, int fp32, const float* weight, const int32_t* slot, void* out, int64_t n_tokens,
                                   int64_t top_k, int64_t width, void* stream) {
    if (!mp::row_sizes_ok(n_tokens, top_k, width)) return B200MOE_ERR_SHAPE;
    if (fp32 != 0 && fp32 != 1) return B200MOE_ERR_ARGUMENT;
    if (n_tokens == 0) return B200MOE_OK;
    if (!y || !weight || !slot || !out) return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(y) || !aligned16(out)) return B200MOE_ERR_ALIGNMENT;
    return mp::launch_sum(y, fp32, weight, slot, out, n_tokens, top_k, width, stream);
}

extern "C" int b200moe_moe_combine_grad(const void* y, int fp32, const float* weight, const int32_t* token_of, const int32_t* slot,
                                        const void* grad_out, void* grad_y, float* grad_weight, int64_t n_tokens, int64_t top_k,
                                        int64_t width, void* stream) {
    if (!mp::row_sizes_ok(n_tokens, top_k, width)) return B200MOE_ERR_SHAPE;
    if (fp32 != 0 && fp32 != 1) return B200MOE_ERR_ARGUMENT;
    if (n_tokens == 0 || (!grad_y && !grad_weight)) return B200MOE_OK;
    if (!y || !weight || !token_of || !slot || !grad_out) return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(y) || !aligned16(grad_out) || !aligned16(grad_y)) return B200MOE_ERR_ALIGNMENT;
    const int w16 = mp::width16_of(width, fp32);
    const auto run = [&](auto zero) {
        using T = decltype(zero);
        void (*kernel)(const uint4*, const float*, const int32_t*, const int32_t*, const uint4*, uint4*, float*, int, int);
        if (grad_y) kernel = grad_weight ? mp::combine_grad_kernel<T, true, true> : mp::combine_grad_kernel<T, true, false>;
        else kernel = mp::combine_grad_kernel<T, false, true>;
        // (one CTA a token: it adds up the token's products)
        kernel<<<(unsigned)n_tokens, mp::kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const uint4*>(y), weight, token_of, slot, static_cast<const uint4*>(grad_out), static_cast<uint4*>(grad_y),
            grad_weight, (int)top_k, w16);
    };
    if (fp32) run(float());
    else run(__nv_bfloat16());
    B200MOE_CUDA_TRY(cudaGetLastError());
    return B200MOE_OK;
}

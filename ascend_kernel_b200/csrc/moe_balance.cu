// Balance loss of the MoE router, the pairs per expert, and the loss's gradient.
//
// The tokens form sequences (a list of cumulative ends; without one, a single sequence).  For sequence s with T_s tokens that the
// mask leaves, p_t the softmax of a token's logits and c_se the number of its (token, j) pairs on expert e:
//
//   loss_s = E / (k T_s) sum_e c_se (1 / T_s sum_t p_te)                     (1 where the load is even)
//   d loss_s / d logit_te = p_te / T_s (F_se - sum_j F_sj p_tj),   F_se = E c_se / (k T_s) - 1
//
// (the 1 cancels in the difference; taking it out first keeps the digits that an almost even load leaves).  The counts are piecewise
// constant and have no gradient.
//
// Forward: a CTA takes a range of tokens, a warp (or a group of 8 or 16 lanes, where a row needs no more) a row at a time, its lanes
// adding the probabilities of their experts up in registers, and counts the range's pairs in shared memory; what a CTA has of a sequence goes
// to row (range + sequence) of the scratch (going on by a range or by a sequence raises that sum by one, so no two pieces share a row), and
// a second kernel adds a sequence's rows in their order: no floating-point atomics, the same bits each time.  Backward: the
// softmax again from the logits.  Each reads the logits once.
//
// Measured, forward (both kernels) | backward, rows larger than L2 among them, us: 4096 fp32 rows of 256: 9.0 | 5.9 (launches);
// 65536: 21 | 24; 262144: 55 | 90 (4.9 and 6.0 TB/s); 262144 bf16 rows of 256: 51 | 67; of 64: 25 | 19.  Memory bounds the fp32 backward, the
// latency of the loads the fp32 forward (two rows of each of 32 warps under way), instructions the others: a probability at a time and
// a warp for every row, the five were 9.8 | 6.4, 27 | 25, 74 | 87, 75 | 80 and 72 | 75.
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace b200moe {
namespace mb {

constexpr int kMaxTopK = 32;

template <class T>
struct Logit;
template <>
struct Logit<__nv_bfloat16> {
    static constexpr int kVec = 8;
    template <int VEC>
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[VEC]) {
        if constexpr (VEC == 8) {
            const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        } else {
            v[0] = __bfloat162float(*p);
        }
    }
    template <int VEC>
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[VEC]) {
        if constexpr (VEC == 8)
            *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                                      pack_bf16x2(v[6], v[7]));
        else
            *p = __float2bfloat16_rn(v[0]);
    }
};
template <>
struct Logit<float> {
    static constexpr int kVec = 4;
    template <int VEC>
    static __device__ __forceinline__ void load(const float* p, float (&v)[VEC]) {
        if constexpr (VEC == 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(p));
            v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        } else {
            v[0] = __ldg(p);
        }
    }
    // VEC values of a table whose rows are as wide as the logits': 16 bytes at a time where VEC says that these are aligned
    template <int VEC>
    static __device__ __forceinline__ void load_row(const float* p, float (&v)[VEC]) {
        if constexpr (VEC == 8) {
            float a[4], b[4];
            load<4>(p, a);
            load<4>(p + 4, b);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else {
            load<VEC>(p, v);
        }
    }
    template <int VEC>
    static __device__ __forceinline__ void store(float* p, const float (&v)[VEC]) {
        if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else *p = v[0];
    }
};

struct Args {
    const void* logits;
    const int32_t* idx;
    const int64_t* seq_list;  // cumulative ends, or NULL: one sequence of all tokens
    const uint8_t* mask;      // NULL: every token counts
    int T, E, k, S, chunk;    // chunk: tokens a CTA takes
    int pitch;                // floats of a scratch row: E rounded up to 4
    float* psum;              // [rows][pitch]
    int32_t* csum;            // [rows][pitch]
    int32_t* nsum;            // [rows]
};

// [a, b) of sequence s, inside the tokens whatever the list holds
__device__ __forceinline__ int seq_end(const Args& a, int s) {
    if (a.seq_list == nullptr) return a.T;
    const long long v = __ldg(a.seq_list + s);
    return (int)(v < 0 ? 0 : (v > a.T ? a.T : v));
}
__device__ __forceinline__ int seq_start(const Args& a, int s) { return s == 0 ? 0 : seq_end(a, s - 1); }
// the first sequence that ends behind token t (a.S if none does)
__device__ __forceinline__ int seq_of(const Args& a, int t) {
    if (a.seq_list == nullptr) return 0;
    int lo = 0, hi = a.S;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (seq_end(a, mid) > t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The largest of the values of a group of LANES lanes (NaN where all are NaN).
template <int LANES>
__device__ __forceinline__ float group_max(float v) {
    if constexpr (LANES == 32) {
        float r;
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
        return r;
    } else {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
}
// 2^v, results below 2^-126 as 0: of a row's largest probability that is none.
__device__ __forceinline__ float exp2_flushed(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// exp(logit - the row's largest) of U tokens and the reciprocals of the rows' sums, their chains of loads and reductions side by
// side.  LANES lanes take a row, lane l of them experts (c * LANES + l) * VEC + j; where that is no whole warp, its groups have rows of their own.  A row of nothing but -infinity has no probability (all 0), a NaN or +infinity makes the
// row NaN.  A row that is not `on` is not read.  Instructions are what these kernels cost, so the arithmetic is two-wide.
template <class T, int VEC, int CHUNKS, int LANES, int U>
__device__ __forceinline__ void softmax_rows(const T* const (&row)[U], const bool (&on)[U], int E, f32x2 (&p)[U][VEC * CHUNKS / 2],
                                             float (&inv)[U]) {
    constexpr int N = VEC * CHUNKS;
    const int lane = threadIdx.x & (LANES - 1);
    float m[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float z[CHUNKS][VEC];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int e = (c * LANES + lane) * VEC;
            if (on[u] && e < E) {
                Logit<T>::template load<VEC>(row[u] + e, z[c]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) z[c][j] = -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) p[u][i] = pack_f32x2(z[2 * i / VEC][2 * i % VEC], z[(2 * i + 1) / VEC][(2 * i + 1) % VEC]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        m[u] = -INFINITY;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) m[u] = fmaxf(m[u], fmaxf(f32x2_lo(p[u][i]), f32x2_hi(p[u][i])));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) m[u] = group_max<LANES>(m[u]);
    float sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        // (a difference first: logits of the type's lowest value times log2(e) would overflow)
        const float base = m[u] == -INFINITY ? 0.f : m[u];
        const f32x2 base2 = pack_f32x2(base, base), log2e = pack_f32x2(1.44269504f, 1.44269504f);
        f32x2 total = 0ull;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const f32x2 x = mul_f32x2(sub_f32x2(p[u][i], base2), log2e);
            p[u][i] = pack_f32x2(exp2_flushed(f32x2_lo(x)), exp2_flushed(f32x2_hi(x)));
            total = add_f32x2(total, p[u][i]);
        }
        sum[u] = f32x2_lo(total) + f32x2_hi(total);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
#pragma unroll
    for (int u = 0; u < U; ++u) inv[u] = sum[u] == 0.f ? 0.f : __fdividef(1.f, sum[u]);  // (the sum is 1 .. 1024)
}
// Tokens a warp has side by side: what 16 values a lane hold.
template <int VEC, int CHUNKS>
constexpr int kTokens = VEC * CHUNKS <= 8 ? 2 : 1;

// Warps of a CTA of the forward pass: half as many where a lane's experts fill its registers.
template <int VEC, int CHUNKS>
constexpr int kForwardWarps = VEC * CHUNKS <= 16 ? 32 : 16;

template <class T, int VEC, int CHUNKS, int LANES>
__global__ void __launch_bounds__(32 * kForwardWarps<VEC, CHUNKS>, 1) forward_kernel(const Args a) {
    constexpr int U = kTokens<VEC, CHUNKS>, kWarps = kForwardWarps<VEC, CHUNKS>, kThreads = 32 * kWarps, kGroups = 32 / LANES;
    extern __shared__ float smem[];  // [kWarps][pitch] probabilities, [pitch] counts, 1 number of tokens
    int* hist = reinterpret_cast<int*>(smem + kWarps * a.pitch);
    int* n_tokens = hist + a.pitch;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & (LANES - 1), group = (threadIdx.x & 31) / LANES;
    const int t0 = blockIdx.x * a.chunk, t1 = min(t0 + a.chunk, a.T);
    const T* logits = static_cast<const T*>(a.logits);
    const auto counts = [&](int t) { return a.mask == nullptr || __ldg(a.mask + t) != 0; };
    for (int s = seq_of(a, t0); s < a.S; ++s) {
        const int start = seq_start(a, s);
        if (start >= t1) break;
        const int lo = max(start, t0), hi = min(seq_end(a, s), t1);
        if (lo >= hi) continue;
        for (int e = threadIdx.x; e <= a.pitch; e += kThreads) hist[e] = 0;  // (and the number of tokens behind them)
        __syncthreads();
        // the pairs, all threads side by side
        const int32_t* idx = a.idx + (size_t)lo * a.k;
        const int pairs = (hi - lo) * a.k;
#pragma unroll 4
        for (int i = threadIdx.x; i < pairs; i += kThreads) {
            const int e = __ldg(idx + i);
            if ((unsigned)e < (unsigned)a.E && counts(lo + i / a.k)) atomicAdd(&hist[e], 1);
        }
        f32x2 acc[VEC * CHUNKS / 2] = {};
        int n = 0;
        for (int t = lo + warp * kGroups; t < hi; t += kWarps * U * kGroups) {
            const T* row[U];
            bool on[U];
            f32x2 p[U][VEC * CHUNKS / 2];
            float inv[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int tu = t + u * kWarps * kGroups + group;
                on[u] = tu < hi && counts(tu);
                row[u] = logits + (size_t)(on[u] ? tu : t) * a.E;
                n += on[u];
            }
            softmax_rows<T, VEC, CHUNKS, LANES, U>(row, on, a.E, p, inv);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < VEC * CHUNKS / 2; ++i) acc[i] = fma_f32x2(p[u][i], pack_f32x2(inv[u], inv[u]), acc[i]);
        }
        if (lane == 0 && n) atomicAdd(n_tokens, n);
        // the groups of a warp, then the warps in their order
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
            for (int i = 0; i < VEC * CHUNKS / 2; ++i) acc[i] = add_f32x2(acc[i], __shfl_xor_sync(0xffffffffu, acc[i], o));
#pragma unroll
        for (int i = 0; i < VEC * CHUNKS; ++i) {
            const int e = (i / VEC * LANES + lane) * VEC + i % VEC;
            if (group == 0 && e < a.pitch) smem[warp * a.pitch + e] = i & 1 ? f32x2_hi(acc[i >> 1]) : f32x2_lo(acc[i >> 1]);
        }
        __syncthreads();
        const size_t row = (size_t)blockIdx.x + s;
        for (int e = threadIdx.x; e < a.pitch; e += kThreads) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) sum += smem[w * a.pitch + e];
            a.psum[row * a.pitch + e] = sum;
            a.csum[row * a.pitch + e] = hist[e];
        }
        if (threadIdx.x == 0) a.nsum[row] = *n_tokens;
        __syncthreads();
    }
    grid_dep_launch();
}

// A CTA per sequence and 128 experts, the CTAs of a sequence as a cluster: a warp takes every 32nd of the sequence's rows, what the
// warps have is added in their order, and the first CTA adds up the parts of the loss.  (One CTA of a sequence for all experts, in 64
// bits: 21 us for 296 rows of 256.)
constexpr int kJoinThreads = 1024;
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Args a, float* __restrict__ loss, long long* __restrict__ counts,
                                                            float* __restrict__ load, float* __restrict__ inv_n, int* findings) {
    __shared__ alignas(16) float s_p[32][128];
    __shared__ alignas(16) int s_c[32][128];
    __shared__ int s_n[32];
    __shared__ int s_tokens;
    __shared__ float s_part[4], s_loss;
    const int s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int start = seq_start(a, s), end = seq_end(a, s);
    if (threadIdx.x == 0 && blockIdx.x == 0) {
        const long long given = a.seq_list ? a.seq_list[s] : a.T;
        if (given != end || end < start) keep_finding(findings, kDevBadGroupList, s);
    }
    const int e = blockIdx.x * 128 + lane * 4;
    float4 p = make_float4(0.f, 0.f, 0.f, 0.f);
    int4 c = make_int4(0, 0, 0, 0);
    int n = 0;
    grid_dep_wait();
    if (end > start) {
        const int last = (end - 1) / a.chunk;
#pragma unroll 8
        for (int r = start / a.chunk + warp; r <= last; r += 32) {
            const size_t row = (size_t)r + s;
            if (e < a.pitch) {
                const float4 q = __ldcg(reinterpret_cast<const float4*>(a.psum + row * a.pitch + e));
                const int4 d = __ldcg(reinterpret_cast<const int4*>(a.csum + row * a.pitch + e));
                p.x += q.x; p.y += q.y; p.z += q.z; p.w += q.w;
                c.x += d.x; c.y += d.y; c.z += d.z; c.w += d.w;
            }
            n += __ldcg(a.nsum + row);
        }
    }
    reinterpret_cast<float4*>(s_p[warp])[lane] = p;
    reinterpret_cast<int4*>(s_c[warp])[lane] = c;
    if (lane == 0) s_n[warp] = n;
    __syncthreads();
    if (warp < 4) {
        const int tokens = __reduce_add_sync(0xffffffffu, s_n[lane]), x = (int)threadIdx.x, expert = blockIdx.x * 128 + x;
        const long long pairs = (long long)tokens * a.k;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        int count = 0;
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            sum[r & 3] += s_p[r][x];
            count += s_c[r][x];
        }
        float part = 0.f;
        if (expert < a.E) {
            const size_t o = (size_t)s * a.E + expert;
            counts[o] = count;
            // (the difference is of whole numbers)
            load[o] = tokens ? (float)((long long)count * a.E - pairs) / (float)pairs : 0.f;
            if (tokens) part = (float)count * ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        }
        part = warp_sum(part);
        if (lane == 0) s_part[warp] = part;
        if (threadIdx.x == 0) s_tokens = tokens;
        if (threadIdx.x == 0 && blockIdx.x == 0) inv_n[s] = tokens ? 1.f / (float)tokens : 0.f;
    }
    __syncthreads();
    if (threadIdx.x == 0) s_loss = (s_part[0] + s_part[1]) + (s_part[2] + s_part[3]);
    ptx::cluster_sync();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        float sum = 0.f;
        for (unsigned r = 0; r < gridDim.x; ++r) sum += ptx::ld_cluster_f32(ptx::map_rank(ptx::smem_u32(&s_loss), r));
        const float tokens = (float)s_tokens;
        loss[s] = s_tokens ? sum / (tokens * (float)a.k) * ((float)a.E / tokens) : 0.f;
    }
    ptx::cluster_sync();  // (the other CTAs' shared memory has been read)
}

template <class T, int VEC, int CHUNKS, int LANES>
__global__ void __launch_bounds__(256) backward_kernel(const Args a, const float* __restrict__ load, const float* __restrict__ inv_n,
                                                       const float* __restrict__ grad, T* __restrict__ out) {
    constexpr int U = kTokens<VEC, CHUNKS>, kGroups = 32 / LANES;
    const int lane = threadIdx.x & (LANES - 1), t = (blockIdx.x * 8 + (threadIdx.x >> 5)) * (U * kGroups);
    if (t >= a.T) return;
    const int first = t + (threadIdx.x & 31) / LANES;  // of the lane's tokens, every kGroups-th
    const T* row[U];
    const float* f[U];
    bool on[U];
    float g[U], mean[U], inv[U];
    f32x2 p[U][VEC * CHUNKS / 2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        // a token of no sequence, or one that the mask takes out, has no part in any loss (what its logits hold is not read)
        const int tu = first + u * kGroups, s = tu < a.T ? seq_of(a, tu) : a.S;
        on[u] = s < a.S && tu >= seq_start(a, s) && (a.mask == nullptr || __ldg(a.mask + tu) != 0);
        row[u] = static_cast<const T*>(a.logits) + (size_t)(on[u] ? tu : t) * a.E;
        f[u] = load + (size_t)(on[u] ? s : 0) * a.E;
        g[u] = on[u] ? __ldg(grad + s) * __ldg(inv_n + s) : 0.f;
        mean[u] = 0.f;
    }
    softmax_rows<T, VEC, CHUNKS, LANES, U>(row, on, a.E, p, inv);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int e = (c * LANES + lane) * VEC;
            if (e < a.E) {
                float fv[VEC];
                Logit<float>::template load_row<VEC>(f[u] + e, fv);
                if constexpr (VEC == 1) {
                    mean[u] = fmaf(fv[0], c & 1 ? f32x2_hi(p[u][c / 2]) : f32x2_lo(p[u][c / 2]), mean[u]);
                } else {
                    f32x2 sum = 0ull;
#pragma unroll
                    for (int j = 0; j < VEC; j += 2) sum = fma_f32x2(pack_f32x2(fv[j], fv[j + 1]), p[u][(c * VEC + j) / 2], sum);
                    mean[u] += f32x2_lo(sum) + f32x2_hi(sum);
                }
            }
        }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) mean[u] += __shfl_xor_sync(0xffffffffu, mean[u], o);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (first + u * kGroups >= a.T) break;
        const float of = -mean[u] * inv[u], by = g[u] * inv[u];
        T* dst = out + (size_t)(first + u * kGroups) * a.E;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int e = (c * LANES + lane) * VEC;
            if (e < a.E) {
                float fv[VEC];
                Logit<float>::template load_row<VEC>(f[u] + e, fv);  // (again, from L1)
                // (a token that is not on has by = 0 and probabilities of 0)
                if constexpr (VEC == 1) {
                    fv[0] = ((c & 1 ? f32x2_hi(p[u][c / 2]) : f32x2_lo(p[u][c / 2])) * by) * (fv[0] + of);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; j += 2) {
                        const f32x2 d = mul_f32x2(mul_f32x2(p[u][(c * VEC + j) / 2], pack_f32x2(by, by)),
                                                  add_f32x2(pack_f32x2(fv[j], fv[j + 1]), pack_f32x2(of, of)));
                        fv[j] = f32x2_lo(d);
                        fv[j + 1] = f32x2_hi(d);
                    }
                }
                Logit<T>::template store<VEC>(dst + e, fv);
            }
        }
    }
}

// Tokens a CTA of the forward pass takes: about a CTA a multiprocessor, a token a warp at least.
static int chunk_of(int64_t T) {
    const int64_t ctas = 148;  // (not the device's own number: the scratch size is a function of the sizes alone)
    int64_t c = (T + ctas - 1) / ctas;
    return (int)(c < 32 ? 32 : c);
}
static int64_t scratch_rows(int64_t T, int64_t S) { return (T + chunk_of(T) - 1) / chunk_of(T) + S; }
static int pitch_of(int64_t E) { return (int)((E + 3) & ~3LL); }

static bool sizes_ok(int64_t T, int64_t E, int64_t k, int64_t S) {
    return T >= 0 && T <= 0x3FFFFFFFLL && E > 0 && E <= 1024 && k > 0 && k <= kMaxTopK && k <= E && S > 0 && S <= 65535 && T * k <= 0x3FFFFFFFLL;
}

// Calls fn(VEC, CHUNKS, LANES) with the widest loads that E and the pointers allow and as many of them as E needs; rows that need half
// the lanes of a warp or fewer get a group of 16 or 8.
template <class T, class F>
static void pick(int E, bool aligned, F&& fn) {
    constexpr int V = Logit<T>::kVec;
    constexpr std::integral_constant<int, V> wide;
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::integral_constant<int, 32> warp;
    if (aligned && E % V == 0) {
        const int n = E / V;
        if (n <= 8) fn(wide, one, std::integral_constant<int, 8>());
        else if (n <= 16) fn(wide, one, std::integral_constant<int, 16>());
        else if (n <= 32) fn(wide, one, warp);
        else if (n <= 64) fn(wide, std::integral_constant<int, 2>(), warp);
        else if (V == 8 || n <= 128) fn(wide, four, warp);  // (E is 1024 at most)
        else if constexpr (V == 4) fn(wide, std::integral_constant<int, 8>(), warp);
    } else {
        if (E <= 128) fn(one, four, warp);
        else if (E <= 512) fn(one, std::integral_constant<int, 16>(), warp);
        else fn(one, warp, warp);
    }
}

}  // namespace mb
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_moe_balance_scratch_bytes(int64_t n_tokens, int64_t n_experts, int64_t n_seqs) {
    if (!mb::sizes_ok(n_tokens, n_experts, 1, n_seqs)) return 0;
    return (size_t)mb::scratch_rows(n_tokens, n_seqs) * (8u * (size_t)mb::pitch_of(n_experts) + 4u);
}

extern "C" int b200moe_moe_balance_loss_findings(const void* logits, int logits_fp32, const int32_t* idx, const int64_t* seq_list,
                                                 const uint8_t* token_mask, int64_t n_tokens, int64_t n_experts, int64_t top_k,
                                                 int64_t n_seqs, float* loss, int64_t* counts, float* load, float* inv_tokens,
                                                 void* scratch, size_t scratch_bytes, int32_t* findings, void* stream) {
    if (!mb::sizes_ok(n_tokens, n_experts, top_k, n_seqs) || (!seq_list && n_seqs != 1)) return B200MOE_ERR_SHAPE;
    if (logits_fp32 != 0 && logits_fp32 != 1) return B200MOE_ERR_ARGUMENT;
    if ((n_tokens > 0 && (!logits || !idx)) || !loss || !counts || !load || !inv_tokens) return B200MOE_ERR_NULL_POINTER;
    if (!scratch || scratch_bytes < b200moe_moe_balance_scratch_bytes(n_tokens, n_experts, n_seqs)) return B200MOE_ERR_WORKSPACE;
    if (!aligned16(scratch)) return B200MOE_ERR_ALIGNMENT;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    mb::Args a;
    a.logits = logits;
    a.idx = idx;
    a.seq_list = seq_list;
    a.mask = token_mask;
    a.T = (int)n_tokens; a.E = (int)n_experts; a.k = (int)top_k; a.S = (int)n_seqs;
    a.chunk = mb::chunk_of(n_tokens);
    a.pitch = mb::pitch_of(n_experts);
    const size_t cells = (size_t)mb::scratch_rows(n_tokens, n_seqs) * a.pitch;
    a.psum = static_cast<float*>(scratch);
    a.csum = reinterpret_cast<int32_t*>(a.psum + cells);
    a.nsum = a.csum + cells;
    if (a.T > 0) {
        const unsigned grid = (unsigned)((a.T + a.chunk - 1) / a.chunk);
        cudaError_t err = cudaSuccess;
        const auto run = [&](auto vec, auto chunks, auto lanes, auto zero) {
            auto* k = mb::forward_kernel<decltype(zero), decltype(vec)::value, decltype(chunks)::value, decltype(lanes)::value>;
            constexpr int warps = mb::kForwardWarps<decltype(vec)::value, decltype(chunks)::value>;
            const size_t smem = (size_t)(warps + 1) * a.pitch * 4 + 4;
            if (smem > 48 * 1024) err = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 140 * 1024);
            if (err == cudaSuccess) {
                k<<<grid, 32 * warps, smem, st>>>(a);
                err = cudaGetLastError();
            }
        };
        if (logits_fp32) mb::pick<float>(a.E, aligned16(logits), [&](auto v, auto c, auto l) { run(v, c, l, float()); });
        else mb::pick<__nv_bfloat16>(a.E, aligned16(logits), [&](auto v, auto c, auto l) { run(v, c, l, __nv_bfloat16()); });
        B200MOE_CUDA_TRY(err);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.pitch + 127) / 128), (unsigned)a.S);
    cfg.blockDim = dim3(mb::kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cfg.gridDim.x;  // 8 at most
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    // (the list is read before the wait for the kernel ahead, so that must be the forward kernel, which began when the list was there)
    cfg.numAttrs = a.T > 0 ? 2 : 1;
    B200MOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, mb::join_kernel, a, loss, reinterpret_cast<long long*>(counts), load, inv_tokens,
                                        findings != nullptr ? findings : findings_words()));
    return B200MOE_OK;
}

extern "C" int b200moe_moe_balance_loss(const void* logits, int logits_fp32, const int32_t* idx, const int64_t* seq_list,
                                        const uint8_t* token_mask, int64_t n_tokens, int64_t n_experts, int64_t top_k, int64_t n_seqs,
                                        float* loss, int64_t* counts, float* load, float* inv_tokens, void* scratch,
                                        size_t scratch_bytes, void* stream) {
    return b200moe_moe_balance_loss_findings(logits, logits_fp32, idx, seq_list, token_mask, n_tokens, n_experts, top_k, n_seqs, loss, counts,
                                             load, inv_tokens, scratch, scratch_bytes, nullptr, stream);
}

extern "C" int b200moe_moe_balance_loss_grad(const void* logits, int logits_fp32, const int64_t* seq_list, const uint8_t* token_mask,
                                             const float* load, const float* inv_tokens, const float* grad_loss, int64_t n_tokens,
                                             int64_t n_experts, int64_t n_seqs, void* grad_logits, void* stream) {
    if (!mb::sizes_ok(n_tokens, n_experts, 1, n_seqs) || (!seq_list && n_seqs != 1)) return B200MOE_ERR_SHAPE;
    if (logits_fp32 != 0 && logits_fp32 != 1) return B200MOE_ERR_ARGUMENT;
    if (n_tokens == 0) return B200MOE_OK;
    if (!logits || !load || !inv_tokens || !grad_loss || !grad_logits) return B200MOE_ERR_NULL_POINTER;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    mb::Args a = {};
    a.logits = logits;
    a.seq_list = seq_list;
    a.mask = token_mask;
    a.T = (int)n_tokens; a.E = (int)n_experts; a.S = (int)n_seqs;
    const bool aligned = aligned16(logits) && aligned16(grad_logits) && aligned16(load);
    const auto run = [&](auto vec, auto chunks, auto lanes, auto zero) {
        using T = decltype(zero);
        const int64_t per_cta = 8 * mb::kTokens<decltype(vec)::value, decltype(chunks)::value> * (32 / decltype(lanes)::value);
        const unsigned grid = (unsigned)((n_tokens + per_cta - 1) / per_cta);
        mb::backward_kernel<T, decltype(vec)::value, decltype(chunks)::value, decltype(lanes)::value>
            <<<grid, 256, 0, st>>>(a, load, inv_tokens, grad_loss, static_cast<T*>(grad_logits));
    };
    if (logits_fp32) mb::pick<float>(a.E, aligned, [&](auto v, auto c, auto l) { run(v, c, l, float()); });
    else mb::pick<__nv_bfloat16>(a.E, aligned, [&](auto v, auto c, auto l) { run(v, c, l, __nv_bfloat16()); });
    B200MOE_CUDA_TRY(cudaGetLastError());
    return B200MOE_OK;
}

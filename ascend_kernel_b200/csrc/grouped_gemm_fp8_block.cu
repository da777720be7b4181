// Grouped GEMM whose two operands are 8-bit floats with one scale per block of 128:
//
//   y[m, n] = sum over blocks kb of 128 k:  x_scale[m, kb] * weight_scale[g, kb, n / 128] * sum_{k in kb} x[m, k] * w[g, k, n]
//
// x e4m3 [M, K] with fp32 scales per row and 128 k, weights e4m3 [G, K, N] with fp32 scales per 128 x 128.
//
// Persistent kernel on pairs of CTAs.  The operands are swapped: the 256 lanes of a pair's MMA (tcgen05 kind::f8f6f4, M = 256) are
// weight columns, 128 to a CTA, and its N extent is the tile's token rows rounded up to 32 (32 .. 160), so an expert with 130 rows costs
// 160 columns, and a decode step's few rows cost 32.  The weights enter as they are stored: a TMA box of 128 k x 128 columns is
// the MN-major A operand.  The rows of x are split between the two CTAs' shared memory and read by both.
//
// An arbitrary fp32 scale cannot ride in the MMA, so a block of 128 k is a sum of its own: the MMA warps write it to one
// of the 3 .. 8 tensor-memory buffers that fit, and the epilogue warps add it, times scale, to the tile's sums in their registers (one
// fused multiply-add per two elements).  Blocks being independent, two warps issue them in turn.
//
// Gate/up: a stage holds 128 gate columns and the 128 up columns of the same indices for the same rows of x, two blocks, and a thread
// has both sums of its columns and tokens: silu(gate) * up in fp32, the largest magnitude over the 128 columns, e4m3.
//
// Warp roles: 0 loads (and, in the pair's first CTA, deals out the tiles); 1 and 2 MMA issue (first CTA); 3 scales; from 4 on epilogue.
// The shared-memory ring holds as many stages as the call's widest tile leaves room for.  Every wait is bounded.
//
// Few tiles: the k range is split into parts whose fp32 sums go to the workspace, and a second kernel adds them in their order.
//
// What bounds it.  Few rows: the weights' bytes (256 experts of a row, 2048 x 7168: 523 us, 7.2 TB/s, 549 in a steady loop; 8 experts: 25 us,
// 1.5 waves of the pairs; gate/up of one token, 7168 x 4096: 45 us, 128 units and their join for 36 us of bytes).
// Many rows: the way of a block through the epilogue -- wait for the commit, loads from tensor memory, multiply-adds, the buffer handed
// back -- whose latencies two warps a scheduler do not cover: with the weights in L2 (8 experts of 640 rows) the tensor pipe is active 35 % of the
// cycles, issue slots 36 to 42 %, and no pipe is near its limit.  A block of 256 x 160 x 128 is 320 cycles of a pair's MMA; a call
// takes a pair 664 (Zipf rows, 7168 x 4096) to 875 cycles a block, the ends of its tiles included.  Short bursts run at a higher clock than
// the 1.25 to 1.42 GHz that the power limit leaves a steady loop, burst | steady: 256 experts of 256 rows, 2048 x 7168: 1.39 | 1.65 ms (1.17
// PFLOP/s); gate/up of 256 experts of 128 rows each, 7168 x 4096: 1.49 | 1.80 ms.  That is the favourable split: of a routed batch of the same
// mean half the experts have 129 to 160 rows, which cost a tile 160 and the whole call a fourth buffer (1.93 ms steady).
// Tiles of at most 160 rows leave three buffers of tensor memory: with 256 rows there are two, with 128 four, both slower.  Two groups of
// four epilogue warps: with four groups 37 tokens x 8 on 256 experts of 2048 x 7168 took 396 us for 372, 4096 x 8 rows 886 for 783.
#include <algorithm>

#include "common.cuh"
#include "fp8_block.cuh"
#include "ptx.cuh"
#include "tile_ring.h"
#include "token_slots.h"

namespace b200moe {
namespace fb {

constexpr int kWarpLoad = 0, kWarpMma0 = 1, kWarpScale = 3, kWarpEpi0 = 4;
constexpr int kMaxR = kTileTokens;     // token rows of a tile
constexpr int kABytes = 128 * 128;     // 128 weight columns of a stage
constexpr int kMaxSlots = 10, kMaxBufs = 8;
constexpr uint32_t kTmemCols = 512;
constexpr int kStripBytes = 2048;      // of an epilogue warp
// The epilogue's warps come in groups of four (128 weight columns), which share the tile's tokens.
constexpr int kGroups = 2, kEpiWarps = 4 * kGroups, kThreads = (kWarpEpi0 + kEpiWarps) * 32;
static_assert(kGroups * kGroupTokens == kMaxR, "token slots");
constexpr int kBigBox = 64, kSmallBox = 16;
constexpr int kScaleRingBytes = (int)kTmemCols * 4;  // a scale for every accumulator column
constexpr int kBarrierBytes = 2048;
constexpr int kSmemBytes = 227 * 1024;

// What a tile is: the number of blocks of a stage (128 weight columns of a CTA each) and whether they are gate and up columns.
template <int HALVES, bool GATE>
struct Mode {
    static constexpr int kHalves = HALVES;
    static constexpr bool kGate = GATE;
    // columns of a tile: what a pair advances by (gate/up: 256 of each), the CTA's first and the distance of its second block
    static constexpr int kTileColumns = GATE ? 256 : 256 * HALVES;
    static __device__ __forceinline__ int first_column(int nt, uint32_t rank) { return nt * kTileColumns + (int)rank * (kTileColumns / 2); }
    static __device__ __forceinline__ int block_step(int N) { return GATE ? N >> 1 : 128; }
    static constexpr int kTopBytes = GATE ? kMaxR * 16 : 0;  // [tokens][4 warps] magnitudes, and less for what they give
    static constexpr int kFixedBytes = 1024 + kBarrierBytes + kScaleRingBytes + kEpiWarps * kStripBytes + 2 * kTopBytes + 2 * (kMaxExperts + 4) * 4;
    static constexpr int kRingBytes = kSmemBytes - kFixedBytes;
    static_assert(kRingBytes % 16 == 0 && kRingBytes >= 4 * (HALVES * kABytes + kMaxR * 64), "stages");
    static_assert(kRingBytes / (HALVES * kABytes + 32 * 64) <= kMaxSlots, "barriers of every stage");
};
using One = Mode<1, false>;
using Two = Mode<2, false>;
using GateUp = Mode<2, true>;

struct Args {
    const float* x_scale;
    const float* w_scale;
    const int64_t* group_list;
    void* out;
    float* out_scale;
    float* parts;      // [max_parts][M][N], or NULL
    int max_parts;
    int M, K, N, G, gl_type, KB, NB;
    int dynamic;       // whether the pairs draw their units (from the ticket) or take every n-th
    int* words;        // the workspace's first: kWord*
    int* findings;
};
constexpr int kWordTicket = 0, kWordParts = 1, kWordRows = 2, kWordBytes = 256;

struct Sync {
    uint64_t full[kMaxSlots];    // first CTA: the bytes of both CTAs' loads
    uint64_t empty[kMaxSlots];   // each CTA: commit of the stage's blocks
    uint64_t t_full[kMaxBufs];   // each CTA: commit, and the buffer's scales are written
    uint64_t t_empty[kMaxBufs];  // first CTA: the epilogue warps of the pair have the buffer's sums
    uint64_t s_empty[kMaxBufs];  // each CTA: its epilogue warps have done with the buffer's scales
    uint64_t wg[4];              // the four epilogue warps of a group among themselves
    uint64_t drain[2];
    uint32_t tmem_base;
    int abort;
    int n_units, parts, width;   // width: token rows of the widest tile, rounded up to 32
    alignas(16) TileEntry ring[kTileRing];
};
static_assert(sizeof(Sync) <= kBarrierBytes, "barrier block");

struct Tile {
    int g, row0, rows, n, nt, kb0, kb1, part;  // n: rows rounded up to 32; nt: 256 columns (gate/up: 256 of each)
};

// Waits and tile look-ups are a whole warp's: it votes at every poll and so leaves them together (instructions for the whole warp
// follow; with lanes that left at different times these ran in halves).
__device__ __forceinline__ bool all(bool v) { return __all_sync(0xffffffffu, v); }
// Whether a poll that has failed `spins` times gives up: the other roles have, or the time is over.
__device__ __forceinline__ bool give_up(uint32_t spins, uint64_t& t0, Sync* sy, int* findings, int id) {
    if ((spins & 0xFF) != 0) return false;
    if (spins == 0) {
        t0 = ptx::globaltimer_ns();
        return false;
    }
    bool out = *reinterpret_cast<volatile int*>(&sy->abort) != 0;
    if (!out && ptx::globaltimer_ns() - t0 > ptx::kWaitLimitNs) {
        *reinterpret_cast<volatile int*>(&sy->abort) = 1;
        keep_finding(findings, kDevWaitExpired, id);
        out = true;
    }
    return !all(!out);
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Sync* sy, int* findings, int id) {
    const uint32_t b = ptx::smem_u32(bar);
    uint64_t t0 = 0;
    for (uint32_t spins = 0; !all(ptx::mbar_try_wait(b, parity)); ++spins)
        if (give_up(spins, t0, sy, findings, id)) return false;
    return true;
}

// The seq-th tile of the pair (seq is advanced); false when the schedule has ended, a wait expired or another role aborted.
__device__ __forceinline__ bool next_tile(Sync* sy, uint32_t& seq, Tile& t, const Args& a, int parts) {
    const TileEntry* e = &sy->ring[seq % kTileRing];
    const uint32_t want = seq + 1;
    TileEntry v;
    uint64_t t0 = 0;
    for (uint32_t spins = 0; !all(tile_entry_is(v = ring_load(e), want)); ++spins)
        if (give_up(spins, t0, sy, a.findings, 90)) return false;
    ++seq;
    t.rows = tile_entry_rows(v);
    if (t.rows == 0) return false;
    t.row0 = tile_entry_row0(v);
    t.g = tile_entry_expert(v);
    t.n = (t.rows + 31) & ~31;
    const int c = tile_entry_column(v);
    if (parts == 1) {
        t.nt = c;
        t.part = 0;
        t.kb0 = 0;
        t.kb1 = a.KB;
    } else {
        t.nt = c / parts;
        t.part = c - t.nt * parts;
        t.kb0 = (int)((long long)t.part * a.KB / parts);
        t.kb1 = (int)((long long)(t.part + 1) * a.KB / parts);
    }
    return true;
}

// An expert's rows are cut into the fewest tiles, of equal size rounded up to 32.
__device__ __forceinline__ int tiles_of(int rows) { return (rows + kMaxR - 1) / kMaxR; }
__device__ __forceinline__ int tile_rows_of(int rows, int tiles) { return ((rows + tiles - 1) / tiles + 31) & ~31; }

// unit -> ring entry; inside an expert the row tiles of a weight column run together, so that they share the weights in L2
__device__ __forceinline__ TileEntry locate(uint32_t seq, int unit, int parts, const int* prefix, const int* row_start, int G, int n_nt) {
    const int t = unit / parts, part = unit - t * parts;
    int lo = 0, hi = G;  // largest g with prefix[g] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int j = t - prefix[lo], mt = (prefix[lo + 1] - prefix[lo]) / n_nt;
    const int nt = j / mt, m = j - nt * mt;
    const int rows = row_start[lo + 1] - row_start[lo], tr = tile_rows_of(rows, mt);
    return tile_entry(seq, (uint32_t)(row_start[lo] + m * tr), (uint32_t)min(tr, rows - m * tr), (uint32_t)lo, (uint32_t)(nt * parts + part));
}

__device__ __forceinline__ float silu(float g) {
    const float e = __expf(-fabsf(g));  // (at most 1: nothing overflows)
    return g * __fdividef(g < 0.f ? e : 1.f, 1.f + e);
}
// Of two values, with one reciprocal for both denominators, which are at most 2.  A NaN in one makes the other NaN: for two columns of a row
// in the same block of 128, which has no finite scale then anyway, never for two rows.
__device__ __forceinline__ void silu2(float& g0, float& g1) {
    const float e0 = __expf(-fabsf(g0)), e1 = __expf(-fabsf(g1)), d0 = 1.f + e0, d1 = 1.f + e1, r = __fdividef(1.f, d0 * d1);
    g0 *= (g0 < 0.f ? e0 : 1.f) * (r * d1);
    g1 *= (g1 < 0.f ? e1 : 1.f) * (r * d0);
}

// What an epilogue warp carries from tile to tile.
struct Epilogue {
    int warp, parts;
    uint32_t rank, buf, ph, wg_ph, n_bufs, width, tmem, t_empty;
    float* scales;
    uint8_t* strip;
    float *tops, *quantizers;
};

// One block into the warp's sums.  The warp holds 32 weight columns (tensor-memory lanes) x NP patches of 8 tokens:
// acc[patch][16 lanes][8 lanes], two tokens to a register pair: lane (g8, q) has columns g8, g8 + 8, .. and tokens 2q, 2q + 1.  The number
// of patches is a constant: a warp passes here once a block of 128 k, and its instructions are what a block costs (with a
// test at every patch, 1000 cycles a block instead of 600).  It is even.
template <int NP>
__device__ __forceinline__ bool add_block(f32x2 (&acc)[NP][2][2], Epilogue& e, uint32_t first, Sync* sy, const Args& a) {
    static_assert(NP % 2 == 0, "patches go in twos");
    const int lane = threadIdx.x & 31, q = lane & 3;
    const uint32_t column = e.buf * e.width + first, td = e.tmem + column;
    const float2* sv = reinterpret_cast<const float2*>(e.scales + column) + q;
    if (!wait(&sy->t_full[e.buf], e.ph, sy, a.findings, 50)) return false;
    ptx::tc_fence_after();
    uint32_t v[2][2][8];  // two patches are fetched while the two before them are added
    const auto fetch = [&](int p, uint32_t(&d)[2][8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) ptx::tmem_ld_16x16(td + (uint32_t)(p * 8) + ((uint32_t)(h * 16) << 16), d[h]);
    };
    fetch(0, v[0]);
#pragma unroll
    for (int p = 0; p < NP; p += 2) {
        ptx::tmem_ld_wait();
        if (p + 2 < NP) {
            fetch(p + 2, v[(p / 2 + 1) & 1]);
        } else {
            // all is in registers: the buffer goes back
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_remote(e.t_empty + e.buf * 8);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 s = sv[(p + j) * 4];
            const f32x2 s2 = pack_f32x2(s.x, s.y);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t(&d)[8] = v[(p / 2) & 1][h];
                    acc[p + j][h][i] = fma_f32x2(pack_u32x2(d[4 * j + 2 * i], d[4 * j + 2 * i + 1]), s2, acc[p + j][h][i]);
                }
        }
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sy->s_empty[e.buf]));
    if (++e.buf == e.n_bufs) { e.buf = 0; e.ph ^= 1; }
    return true;
}

// A part's sums as they are, [part][row][column]; `columns`: how many from `col` on the tile has.
template <int NP>
__device__ __forceinline__ void store_part(const f32x2 (&acc)[NP][2][2], const Tile& t, int first, int col, int columns, const Args& a) {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3;
    float* dst = a.parts + ((size_t)t.part * a.M + t.row0) * a.N + col;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int token = first + p * 8 + 2 * q, c = h * 16 + i * 8 + g8;
                if (c < columns) {
                    if (token < t.rows) dst[(size_t)token * a.N + c] = f32x2_lo(acc[p][h][i]);
                    if (token + 1 < t.rows) dst[(size_t)(token + 1) * a.N + c] = f32x2_hi(acc[p][h][i]);
                }
            }
}

// bf16 rows, 16 tokens x 32 columns at a time through the warp's strip: the transposing store gives 16-byte pieces of eight columns,
// 64 contiguous bytes of a row.  The strip's halves take turns, and a chunk is on its way out while the next one is transposed.
template <int NP>
__device__ __forceinline__ void store_rows(const f32x2 (&acc)[NP][2][2], const Tile& t, const Epilogue& e, int first, int col, const Args& a) {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3;
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (size_t)(t.row0 + first) * a.N + col + q * 8;
    const bool inside = col + q * 8 < a.N;
    uint4 out[2];
    const auto send = [&](int p) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int token = p * 8 + j * 8 + g8;
            if (first + token < t.rows && inside) *reinterpret_cast<uint4*>(dst + (size_t)token * a.N) = out[j];
        }
    };
#pragma unroll
    for (int p = 0; p < NP; p += 2) {
        uint8_t* half = e.strip + (p & 2) * 512;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t o[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) o[m] = pack_bf16x2(f32x2_lo(acc[p + j][m >> 1][m & 1]), f32x2_hi(acc[p + j][m >> 1][m & 1]));
            const int token = j * 8 + (lane & 7);  // row lane % 8 of piece lane / 8
            ptx::stmatrix_x4_trans(ptx::smem_u32(half) + (uint32_t)(token * 64 + (((lane >> 3) ^ (token >> 1)) & 3) * 16), o[0], o[1], o[2], o[3]);
        }
        __syncwarp();
        if (p > 0) send(p - 2);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int token = j * 8 + g8;
            out[j] = *reinterpret_cast<const uint4*>(half + token * 64 + ((q ^ (token >> 1)) & 3) * 16);
        }
    }
    send(NP - 2);
    __syncwarp();
}

// silu(gate) * up of the thread's columns and tokens, quantised by the rows' 128 columns: the warps of a group put what their 32
// columns have as largest magnitudes together, a thread per token makes the scale, and the codes leave through the strip.
template <int NP>
__device__ __forceinline__ bool store_quantized(f32x2 (&gate)[NP][2][2], const f32x2 (&up)[NP][2][2], const Tile& t, Epilogue& e, int first,
                                                int block, Sync* sy, const Args& a) {
    static_assert(NP * 8 <= kGroupTokens, "token slots");
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3, quarter = e.warp & 3, wg = e.warp >> 2;
    const int slots = token_slot(wg, 0);  // of the group's tokens in `tops` and `quantizers`
    const int inter = a.N >> 1, blocks = inter >> 7;
    const bool inside = block < blocks;  // (an odd number of blocks leaves the pair's last CTA without one)
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        uint32_t m0 = 0, m1 = 0;  // magnitudes order as their bits do, infinities and NaN last
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float lo[2] = {f32x2_lo(gate[p][h][0]), f32x2_lo(gate[p][h][1])}, hi[2] = {f32x2_hi(gate[p][h][0]), f32x2_hi(gate[p][h][1])};
            silu2(lo[0], lo[1]);
            silu2(hi[0], hi[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                lo[i] *= f32x2_lo(up[p][h][i]);
                hi[i] *= f32x2_hi(up[p][h][i]);
                m0 = max(m0, __float_as_uint(lo[i]) & 0x7FFFFFFFu);
                m1 = max(m1, __float_as_uint(hi[i]) & 0x7FFFFFFFu);
                gate[p][h][i] = pack_f32x2(lo[i], hi[i]);
            }
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            m0 = max(m0, __shfl_xor_sync(0xffffffffu, m0, o));
            m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, o));
        }
        if (g8 < 2) e.tops[(slots + p * 8 + 2 * q + g8) * 4 + quarter] = __uint_as_float(g8 ? m1 : m0);
    }
    const auto meet = [&]() {
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sy->wg[wg]));
        const bool ok = wait(&sy->wg[wg], e.wg_ph, sy, a.findings, 62);
        e.wg_ph ^= 1;
        return ok;
    };
    if (!meet()) return false;
    const int mine = quarter * 32 + lane;
    if (mine < NP * 8) {
        const int token = first + mine;
        const uint4 m = reinterpret_cast<const uint4*>(e.tops)[slots + mine];
        const fp8_block::Quantizer qz(__uint_as_float(max(max(m.x, m.y), max(m.z, m.w))));
        reinterpret_cast<float2*>(e.quantizers)[slots + mine] = qz.packed();
        if (inside && token < t.rows) a.out_scale[(size_t)(t.row0 + token) * blocks + block] = qz.scale;
    }
    if (!meet()) return false;
    uint8_t* dst = static_cast<uint8_t*>(a.out) + (size_t)t.row0 * inter + block * 128 + quarter * 32 + (lane & 1) * 16;
#pragma unroll
    for (int p = 0; p < NP; p += 2) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const fp8_block::Quantizer qz(reinterpret_cast<const float2*>(e.quantizers)[slots + (p + j) * 8 + 2 * q + b]);
                float h[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) h[m] = b ? f32x2_hi(gate[p + j][m >> 1][m & 1]) : f32x2_lo(gate[p + j][m >> 1][m & 1]);
                const uint32_t o = qz.finite() ? qz.codes2(pack_f32x2(h[0], h[1])) | (qz.codes2(pack_f32x2(h[2], h[3])) << 16) : 0u;
                uint8_t* at = e.strip + (j * 8 + 2 * q + b) * 32 + g8;
                at[0] = (uint8_t)o;
                at[8] = (uint8_t)(o >> 8);
                at[16] = (uint8_t)(o >> 16);
                at[24] = (uint8_t)(o >> 24);
            }
        __syncwarp();
        const int token = first + p * 8 + (lane >> 1);
        if (inside && token < t.rows) *reinterpret_cast<uint4*>(dst + (size_t)token * inter) = *reinterpret_cast<const uint4*>(e.strip + lane * 16);
        __syncwarp();
    }
    return true;
}

// A tile's sums and what becomes of them; NP: patches of 8 tokens a warp has.
template <class M, int NP>
__device__ __forceinline__ bool finish_tile(const Tile& t, Epilogue& e, Sync* sy, const Args& a) {
    constexpr int kHalves = M::kHalves;
    const int first = (e.warp >> 2) * (NP * 8), quarter = e.warp & 3;
    f32x2 acc[kHalves][NP][2][2];
#pragma unroll
    for (int u = 0; u < kHalves; ++u)
#pragma unroll
        for (int p = 0; p < NP; ++p) acc[u][p][0][0] = acc[u][p][0][1] = acc[u][p][1][0] = acc[u][p][1][1] = 0ull;
    const int col = M::first_column(t.nt, e.rank) + quarter * 32;
    for (int kb = t.kb0; kb < t.kb1; ++kb)
#pragma unroll
        for (int u = 0; u < kHalves; ++u) {
            if (!add_block<NP>(acc[u], e, (uint32_t)first, sy, a)) return false;
            // (the first block's rows go out while the second one's last sum is made)
            if (!M::kGate && u + 1 < kHalves && kb + 1 == t.kb1 && e.parts == 1) store_rows<NP>(acc[u], t, e, first, col + u * 128, a);
        }
    if (e.parts > 1) {
        const int step = M::block_step(a.N), end = M::kGate ? step : a.N;  // (a block's columns end there)
#pragma unroll
        for (int u = 0; u < kHalves; ++u) store_part<NP>(acc[u], t, first, u * step + col, end - col - (M::kGate ? 0 : u * step), a);
        return true;
    }
    if constexpr (M::kGate) {
        return store_quantized<NP>(acc[0], acc[1], t, e, first, col >> 7, sy, a);
    } else {
        store_rows<NP>(acc[kHalves - 1], t, e, first, col + (kHalves - 1) * 128, a);
        return true;
    }
}

template <class M>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    grouped_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x64,
                   const __grid_constant__ CUtensorMap map_x16, const Args a) {
    constexpr int kHalves = M::kHalves;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
    Sync* sy = reinterpret_cast<Sync*>(ring + M::kRingBytes);
    float* scales = reinterpret_cast<float*>(ring + M::kRingBytes + kBarrierBytes);
    uint8_t* strips = reinterpret_cast<uint8_t*>(scales) + kScaleRingBytes;
    float* tops = reinterpret_cast<float*>(strips + kEpiWarps * kStripBytes);
    int* row_start = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(tops) + 2 * M::kTopBytes);
    int* prefix = row_start + kMaxExperts + 4;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_rank();
    const int n_nt = ((M::kGate ? a.N >> 1 : a.N) + M::kTileColumns - 1) / M::kTileColumns;

    // what needs nothing from memory comes first: the kernel may have started beside the end of the one before it
    if (threadIdx.x == kThreads - 32) {
        sy->abort = 0;
        for (int i = 0; i < kTileRing; ++i) sy->ring[i] = tile_entry(0u, 0u, 0u, 0u, 0u);
        const auto init = [](uint64_t* b, int n, uint32_t count) {
            for (int i = 0; i < n; ++i) ptx::mbar_init(ptx::smem_u32(b + i), count);
        };
        init(sy->full, kMaxSlots, 1);
        init(sy->empty, kMaxSlots, kHalves);
        init(sy->t_full, kMaxBufs, 2);
        init(sy->t_empty, kMaxBufs, 2 * kEpiWarps);
        init(sy->s_empty, kMaxBufs, kEpiWarps);
        init(sy->wg, kGroups, 4);
        init(sy->drain, 2, 1);
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&map_w);
        ptx::prefetch_tensormap(&map_x64);
        ptx::prefetch_tensormap(&map_x16);
    }
    if (warp == kWarpMma0) {
        ptx::tmem_alloc_pair(ptx::smem_u32(&sy->tmem_base), kTmemCols);
        ptx::tmem_relinquish_pair();
    }
    grid_dep_wait();
    grid_dep_launch();
    load_row_starts(a.group_list, a.G, a.M, a.gl_type, row_start, nullptr, blockIdx.x == 0 ? a.findings : nullptr);
    if (warp == 0) {
        int lo, hi, mine = 0, total, wide = 0;
        lane_experts(a.G, lo, hi);
        for (int g = lo; g < hi; ++g) {
            const int rows = row_start[g + 1] - row_start[g], mt = tiles_of(rows);
            mine += mt;
            if (mt) wide = max(wide, tile_rows_of(rows, mt));
        }
        int at = warp_exclusive_sum(mine, total);
        wide = __reduce_max_sync(0xffffffffu, wide);
        for (int g = lo; g < hi; ++g) {
            prefix[g] = at * n_nt;
            at += tiles_of(row_start[g + 1] - row_start[g]);
        }
        if (lane == 0) {
            const int tiles = total * n_nt, pairs = (int)gridDim.x / 2;
            prefix[a.G] = tiles;
            int parts = 1;
            if (a.parts != nullptr && tiles > 0 && tiles < pairs) parts = min(a.max_parts, (pairs + tiles - 1) / tiles);
            sy->parts = parts;
            sy->n_units = tiles * parts;
            sy->width = max(wide, 32);
            if (blockIdx.x == 0) {
                a.words[kWordParts] = parts;
                a.words[kWordRows] = row_start[a.G];
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();
    ptx::tc_fence_after();

    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&sy->tmem_base);
    const int parts = sy->parts, n_units = sy->n_units, width = sy->width;
    const int slot_bytes = kHalves * kABytes + width * 64;
    const int n_slots = min(kMaxSlots, M::kRingBytes / slot_bytes);
    const int n_bufs = min(kMaxBufs, (int)kTmemCols / width);

    if (warp < kWarpEpi0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == kWarpLoad) {
            // ------------------------------ loads ------------------------------
            // The warp walks together and one lane issues (a lane on its own took 550 cycles a stage).
            const bool leader = ptx::elect_one();
            uint32_t seq = 0, published = 0, it = 0, slot = 0, ph = 0;
            const int pairs = (int)gridDim.x / 2;
            int unit = (int)blockIdx.x / 2;
            bool live = true, ok = true;
            const uint32_t ring_there = ptx::map_rank(ptx::smem_u32(sy->ring), 1);
            const uint32_t full0 = ptx::map_rank(ptx::smem_u32(sy->full), 0), full_here = ptx::smem_u32(sy->full);
            const auto publish = [&]() {
                if (rank != 0 || !live) return;
                live = unit < n_units;
                const TileEntry e = live ? locate(published + 1, unit, parts, prefix, row_start, a.G, n_nt)
                                         : tile_entry(published + 1, 0u, 0u, 0u, 0u);  // rows 0: the schedule has ended
                int drawn = 0;
                if (leader) {
                    const uint32_t at = (published % kTileRing) * (uint32_t)sizeof(TileEntry);
                    ring_store(&sy->ring[published % kTileRing], e);
                    ptx::st_cluster_u64(ring_there + at, e.a);
                    ptx::st_cluster_u64(ring_there + at + 8, e.b);
                    if (live && a.dynamic) drawn = atomicAdd(a.words + kWordTicket, 1);
                }
                if (a.dynamic) unit = pairs + __reduce_add_sync(0xffffffffu, drawn);
                else unit += pairs;
                ++published;
            };
            publish();
            Tile t;
            while (ok) {
                publish();  // (a tile ahead: the other roles find it there)
                if (!next_tile(sy, seq, t, a, parts)) break;
                const int half = t.n >> 1, n_big = half / kBigBox, n_small = (half % kBigBox) / kSmallBox;
                const uint32_t bytes = 2u * (uint32_t)(kHalves * kABytes + half * 128);
                const int col = M::first_column(t.nt, rank);
                const int row = t.row0 + (int)rank * half;
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                    if (it >= (uint32_t)n_slots && !wait(&sy->empty[slot], ph ^ 1, sy, a.findings, 10)) { ok = false; break; }
                    if (leader) {
                        const uint32_t bar0 = full0 + slot * 8, dst = ptx::smem_u32(ring) + slot * (uint32_t)slot_bytes;
                        if (rank == 0) ptx::mbar_arrive_expect_tx(full_here + slot * 8, bytes);
#pragma unroll
                        for (int u = 0; u < kHalves; ++u)
                            ptx::tma_load_3d_pair(dst + u * kABytes, &map_w, bar0, col + u * M::block_step(a.N), kb * 128, t.g);
                        uint32_t at = dst + kHalves * kABytes;
                        int r = row;
                        for (int b = 0; b < n_big; ++b, at += kBigBox * 128, r += kBigBox)
                            ptx::tma_load_2d_pair(at, &map_x64, bar0, kb * 128, r);
                        for (int b = 0; b < n_small; ++b, at += kSmallBox * 128, r += kSmallBox)
                            ptx::tma_load_2d_pair(at, &map_x16, bar0, kb * 128, r);
                    }
                    __syncwarp();
                    if (++slot == (uint32_t)n_slots) { slot = 0; ph ^= 1; }
                }
            }
            // The commits that give the last stages back have arrived before the CTA ends: those for the second CTA's barriers come from the
            // first one, and nothing else there waits for them.
            for (uint32_t i = it; ok && i < it + (uint32_t)n_slots; ++i) {
                if (i >= (uint32_t)n_slots) ok = wait(&sy->empty[slot], ph ^ 1, sy, a.findings, 11);
                if (++slot == (uint32_t)n_slots) { slot = 0; ph ^= 1; }
            }
            if (leader && *reinterpret_cast<volatile int*>(&sy->abort)) {
                // copies in flight land before the shared memory goes (those of both CTAs are counted in the first one)
                if (rank == 0) {
                    const uint32_t from = it > (uint32_t)n_slots ? it - n_slots : 0;
                    for (uint32_t j = from; j < it; ++j)
                        (void)ptx::mbar_wait(ptx::smem_u32(&sy->full[j % n_slots]), (j / n_slots) & 1);
                }
                const uint64_t t0 = ptx::globaltimer_ns();
                while (ptx::globaltimer_ns() - t0 < 10000000ull) {}
            }
            __syncwarp();
        } else if (warp == kWarpScale) {
            // ------------------------------ scales ------------------------------
            // Row scale times the block's weight scale, with ordinary loads: the kernel ahead may have written either.
            uint32_t seq = 0, it = 0, buf = 0, ph = 0;
            bool ok = true;
            Tile t;
            while (ok && next_tile(sy, seq, t, a, parts)) {
                const float* ws = a.w_scale + (size_t)t.g * a.KB * a.NB;
                int nb[kHalves];
#pragma unroll
                for (int u = 0; u < kHalves; ++u) nb[u] = min(a.NB - 1, (M::first_column(t.nt, rank) + u * M::block_step(a.N)) >> 7);
                const float* xs = a.x_scale + (size_t)(t.row0 + lane) * a.KB;
                const size_t group = (size_t)a.KB * 32;
                for (int kb = t.kb0; kb < t.kb1 && ok; kb += 4) {  // (four stages' loads in flight)
                    float w[4][kHalves], v[kMaxR / 32][4];
                    const int last = t.kb1 - 1 - kb;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
#pragma unroll
                        for (int u = 0; u < kHalves; ++u) w[b][u] = __ldca(ws + (size_t)(kb + min(b, last)) * a.NB + nb[u]);
#pragma unroll
                    for (int g = 0; g < kMaxR / 32; ++g)
                        if (g * 32 < t.n) {
                            const bool row = g * 32 + lane < t.rows;
#pragma unroll
                            for (int b = 0; b < 4; ++b) v[g][b] = row ? __ldca(xs + g * group + kb + min(b, last)) : 0.f;
                        }
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        if (b > last || !ok) break;
#pragma unroll
                        for (int u = 0; u < kHalves; ++u) {
                            if (ok && it >= (uint32_t)n_bufs) ok = wait(&sy->s_empty[buf], ph ^ 1, sy, a.findings, 20);
                            if (!ok) break;
                            float* dst = scales + buf * (uint32_t)width + lane;
#pragma unroll
                            for (int g = 0; g < kMaxR / 32; ++g)
                                if (g * 32 < t.n) dst[g * 32] = v[g][b] * w[b][u];
                            __syncwarp();
                            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sy->t_full[buf]));
                            ++it;
                            if (++buf == (uint32_t)n_bufs) { buf = 0; ph ^= 1; }
                        }
                    }
                }
            }
        } else if (rank == 0) {
            // ------------------------------ MMA issue ------------------------------
            // The warp walks together, one lane issues; this warp takes every other block.
            const uint32_t turn = (uint32_t)(warp - kWarpMma0);
            const bool leader = ptx::elect_one();
            uint32_t seq = 0, it = 0, slot = 0, ph = 0, buf = 0, tph = 0;
            bool ok = true;
            const uint64_t da0 = ptx::umma_desc_sw128(ptx::smem_u32(ring), kABytes, 1024);
            const uint64_t db0 = ptx::umma_desc_sw128(ptx::smem_u32(ring) + kHalves * kABytes, 0, 1024);
            Tile t;
            while (ok && next_tile(sy, seq, t, a, parts)) {
                const uint32_t idesc = ptx::umma_idesc_e4m3_mn_k(256, t.n);
                for (int kb = t.kb0; kb < t.kb1 && ok; ++kb) {
#pragma unroll
                    for (int u = 0; u < kHalves; ++u, ++it) {
                        if ((it & 1) == turn) {
                            // the epilogue of both CTAs has taken what the buffer held
                            if (it >= (uint32_t)n_bufs && !wait(&sy->t_empty[buf], tph ^ 1, sy, a.findings, 30)) { ok = false; break; }
                            if (!wait(&sy->full[slot], ph, sy, a.findings, 40)) { ok = false; break; }
                            ptx::tc_fence_after();
                            if (leader) {
                                const uint64_t at = (uint64_t)(slot * (uint32_t)slot_bytes >> 4);
#pragma unroll
                                for (int k32 = 0; k32 < 4; ++k32)
                                    ptx::umma_f8_pair(tmem_base + buf * (uint32_t)width, da0 + at + (uint64_t)(u * (kABytes >> 4) + k32 * 256),
                                                      db0 + at + (uint64_t)(k32 * 2), idesc, (uint32_t)(k32 != 0));
                                ptx::umma_commit_pair(ptx::smem_u32(&sy->t_full[buf]));
                                ptx::umma_commit_pair(ptx::smem_u32(&sy->empty[slot]));
                            }
                            __syncwarp();
                        }
                        if (++buf == (uint32_t)n_bufs) { buf = 0; tph ^= 1; }
                    }
                    if (++slot == (uint32_t)n_slots) { slot = 0; ph ^= 1; }
                }
            }
            // every MMA issued here must have completed before tensor and shared memory go
            if (leader) {
                ptx::umma_commit_pair(ptx::smem_u32(&sy->drain[turn]));
                (void)ptx::mbar_wait(ptx::smem_u32(&sy->drain[turn]), 0);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ------------------------------ epilogue ------------------------------
        Epilogue e;
        e.warp = warp - kWarpEpi0;
        e.parts = parts;
        e.rank = rank;
        e.buf = e.ph = e.wg_ph = 0;
        e.n_bufs = (uint32_t)n_bufs;
        e.width = (uint32_t)width;
        e.tmem = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        e.t_empty = ptx::map_rank(ptx::smem_u32(sy->t_empty), 0);
        e.scales = scales;
        e.strip = strips + e.warp * kStripBytes;
        e.tops = tops;
        e.quantizers = tops + M::kTopBytes / 4;
        uint32_t seq = 0;
        bool ok = true;
        Tile t;
        while (ok && next_tile(sy, seq, t, a, parts)) {
            switch (t.n >> 5) {
                case 1: ok = finish_tile<M, 1 * 2>(t, e, sy, a); break;
                case 2: ok = finish_tile<M, 2 * 2>(t, e, sy, a); break;
                case 3: ok = finish_tile<M, 3 * 2>(t, e, sy, a); break;
                case 4: ok = finish_tile<M, 4 * 2>(t, e, sy, a); break;
                default: ok = finish_tile<M, 5 * 2>(t, e, sy, a); break;
            }
        }
    }

    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    // (so have the last commits of both MMA warps, which arrive here too; the first CTA's warps waited for theirs)
    if (rank != 0 && (warp == kWarpMma0 || warp == kWarpMma0 + 1)) (void)ptx::mbar_wait(ptx::smem_u32(&sy->drain[warp - kWarpMma0]), 0);
    __syncwarp();
    ptx::cluster_sync();  // (what one CTA sends the other, loads and MMAs of the pair among it, has arrived)
    if (warp == kWarpMma0) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// The parts of a split k range, added in their order.  A warp takes 128 columns of a row.
template <bool GATE_UP>
__global__ void __launch_bounds__(256) join_kernel(const Args a) {
    grid_dep_wait();
    const int parts = __ldcg(a.words + kWordParts), rows = __ldcg(a.words + kWordRows);
    if (parts == 1) return;
    const int lane = threadIdx.x & 31, out_n = GATE_UP ? a.N >> 1 : a.N, blocks = (out_n + 127) / 128;
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = (int)(unit / blocks), nb = (int)(unit % blocks), col = nb * 128 + lane * 4;
    if (row >= rows) return;
    float4 s[2] = {};
    for (int p = 0; p < parts; ++p)
#pragma unroll
        for (int u = 0; u < (GATE_UP ? 2 : 1); ++u)
            if (col < out_n) {
                const float4 v = __ldcg(reinterpret_cast<const float4*>(a.parts + ((size_t)p * a.M + row) * a.N + u * out_n + col));
                s[u].x += v.x; s[u].y += v.y; s[u].z += v.z; s[u].w += v.w;
            }
    if constexpr (!GATE_UP) {
        if (col < out_n)
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (size_t)row * a.N + col) =
                make_uint2(pack_bf16x2(s[0].x, s[0].y), pack_bf16x2(s[0].z, s[0].w));
    } else {
        const float h[4] = {silu(s[0].x) * s[1].x, silu(s[0].y) * s[1].y, silu(s[0].z) * s[1].z, silu(s[0].w) * s[1].w};
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(h[i]) & 0x7FFFFFFFu);
        const fp8_block::Quantizer q(__uint_as_float(__reduce_max_sync(0xffffffffu, m)));
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + (size_t)row * out_n + col) =
            q.finite() ? q.codes2(pack_f32x2(h[0], h[1])) | (q.codes2(pack_f32x2(h[2], h[3])) << 16) : 0u;
        if (lane == 0) a.out_scale[(size_t)row * blocks + nb] = q.scale;
    }
}

static bool sizes_ok(int64_t M, int64_t K, int64_t N, int64_t G) {
    constexpr int64_t kMost = 0x3FFFFFFF;  // (products of two sizes stay in 64 bits)
    return M >= 0 && M <= kMost && K > 0 && K <= kMost && N > 0 && N <= kMost && G > 0 && G <= kMaxExperts;
}

constexpr int64_t kPairs = 74;  // of a B200's multiprocessors (rules and sizes go by the sizes of a call alone)

// Whether a tile's stage holds two blocks of 128 columns a CTA: a pair then reads 512 contiguous bytes of a weight row and the rows of x
// half as often, but has four or five stages in flight instead of seven to ten.  One | two blocks, us (experts, tokens x
// top_k, K x N): 256, 37 x 8, 2048 x 7168: 445 | 376; 256, 1024 x 8, 7168 x 4096: 1325 | 1138; 256, 2048 x 8, 2048 x 7168: 851 | 662, of 80 rows
// an expert 840 | 772, of 96 rows 810 | 924, of 128 rows 966 | 1148.  Where the tiles are a few waves of the pairs, the cut that
// fills its last wave better: 8 experts of a row, 2048 x 7168: 29.8 | 27.2; 64 experts of 64 rows, 2048 x 2048: 58.6 | 65.5.
static bool two_blocks(int64_t M, int64_t N, int64_t G) {
    if (N < 1024 || M > 80 * G) return false;
    const int64_t tiles = std::min(G, M) * ((N + Two::kTileColumns - 1) / Two::kTileColumns);
    if (tiles < kPairs || tiles >= 7 * kPairs) return true;
    return 2 * ((tiles + kPairs - 1) / kPairs) <= (2 * tiles + kPairs - 1) / kPairs;
}
static int64_t tiles_across(int64_t M, int64_t N, int64_t G, int gate_up) {
    const int64_t columns = gate_up ? 2 * GateUp::kTileColumns : two_blocks(M, N, G) ? Two::kTileColumns : One::kTileColumns;
    return (N + columns - 1) / columns;
}

// Whether a call can have fewer tiles than there are pairs of multiprocessors, and in how many parts its k range is cut at most: parts of
// four blocks or more, sums of 32 MB or less.
static int max_parts(int64_t M, int64_t K, int64_t N, int64_t G, int gate_up) {
    const int64_t n_nt = tiles_across(M, N, G, gate_up), experts = std::min(G, M);
    if (experts * n_nt >= kPairs) return 1;
    const int64_t kb = (K + 127) / 128, room = (32ll << 20) / (M * N * 4);
    return (int)std::max<int64_t>(1, std::min<int64_t>({16, kb / 4, room}));
}

}  // namespace fb
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_grouped_gemm_fp8_block_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t G, int gate_up_silu) {
    if (!fb::sizes_ok(M, K, N, G) || M == 0) return fb::kWordBytes;
    const int parts = fb::max_parts(M, K, N, G, gate_up_silu);
    return fb::kWordBytes + (parts > 1 ? (size_t)parts * (size_t)M * (size_t)N * 4 : 0);
}

extern "C" int b200moe_grouped_gemm_fp8_block_findings(const void* x, const float* x_scale, const void* weight, const float* weight_scale,
                                                       const int64_t* group_list, void* out, float* out_scale, int64_t M, int64_t K,
                                                       int64_t N, int64_t G, int group_list_type, int gate_up_silu, void* workspace,
                                                       size_t workspace_bytes, int32_t* findings, void* stream) {
    if (!fb::sizes_ok(M, K, N, G) || (K % 16) != 0 || (N % 16) != 0 || (gate_up_silu && (N % 256) != 0))
        return B200MOE_ERR_SHAPE;
    if (group_list_type != B200MOE_GROUP_LIST_CUMSUM && group_list_type != B200MOE_GROUP_LIST_COUNTS) return B200MOE_ERR_ARGUMENT;
    if (gate_up_silu != 0 && gate_up_silu != 1) return B200MOE_ERR_ARGUMENT;
    if (M == 0) return B200MOE_OK;
    // (unit numbers and ring entries)
    if ((M / fb::kMaxR + G) * ((N + 255) / 256) > 0x3FFFFFFLL) return B200MOE_ERR_SHAPE;
    if (!x || !x_scale || !weight || !weight_scale || !group_list || !out || (gate_up_silu && !out_scale))
        return B200MOE_ERR_NULL_POINTER;
    if (!aligned16(x) || !aligned16(weight) || !aligned16(out)) return B200MOE_ERR_ALIGNMENT;
    if (!workspace || workspace_bytes < b200moe_grouped_gemm_fp8_block_workspace_bytes(M, K, N, G, gate_up_silu))
        return B200MOE_ERR_WORKSPACE;
    if (!aligned16(workspace)) return B200MOE_ERR_ALIGNMENT;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    fb::Args a = {};
    a.x_scale = x_scale;
    a.w_scale = weight_scale;
    a.group_list = group_list;
    a.out = out;
    a.out_scale = out_scale;
    a.M = (int)M; a.K = (int)K; a.N = (int)N; a.G = (int)G;
    a.gl_type = group_list_type;
    a.KB = (int)((K + 127) / 128);
    a.NB = (int)((N + 127) / 128);
    a.words = static_cast<int*>(workspace);
    a.findings = findings != nullptr ? findings : findings_words();
    a.max_parts = fb::max_parts(M, K, N, G, gate_up_silu);
    if (a.max_parts > 1) a.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + fb::kWordBytes);
    CUtensorMap map_w, map_x64, map_x16;
    int rc = make_tensor_map_3d_u8(&map_w, weight, (uint64_t)G, (uint64_t)K, (uint64_t)N, 128, 128);
    if (rc == B200MOE_OK) rc = make_tensor_map_2d(&map_x64, x, 1, (uint64_t)M, (uint64_t)K, fb::kBigBox, 128, true);
    if (rc == B200MOE_OK) rc = make_tensor_map_2d(&map_x16, x, 1, (uint64_t)M, (uint64_t)K, fb::kSmallBox, 128, true);
    if (rc != B200MOE_OK) return rc;
    const unsigned grid = (unsigned)(sm_count() / 2 * 2);
    const auto kernel = gate_up_silu ? fb::grouped_kernel<fb::GateUp> : fb::two_blocks(M, N, G) ? fb::grouped_kernel<fb::Two> : fb::grouped_kernel<fb::One>;
    B200MOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, fb::kSmemBytes));
    a.dynamic = fb::tiles_across(M, N, G, gate_up_silu) * std::min(G, M) >= 16 * fb::kPairs;
    if (a.dynamic) B200MOE_CUDA_TRY(cudaMemsetAsync(workspace, 0, fb::kWordBytes, st));
    B200MOE_CUDA_TRY(launch_dependent(kernel, grid, fb::kThreads, fb::kSmemBytes, st, map_w, map_x64, map_x16, a));
    if (a.max_parts > 1) {
        const int64_t out_n = gate_up_silu ? N / 2 : N;
        const unsigned blocks = (unsigned)((M * ((out_n + 127) / 128) + 7) / 8);
        B200MOE_CUDA_TRY(launch_dependent(gate_up_silu ? fb::join_kernel<true> : fb::join_kernel<false>, blocks, 256, 0, st, a));
    }
    return B200MOE_OK;
}

extern "C" int b200moe_grouped_gemm_fp8_block(const void* x, const float* x_scale, const void* weight, const float* weight_scale,
                                              const int64_t* group_list, void* out, float* out_scale, int64_t M, int64_t K, int64_t N,
                                              int64_t G, int group_list_type, int gate_up_silu, void* workspace,
                                              size_t workspace_bytes, void* stream) {
    return b200moe_grouped_gemm_fp8_block_findings(x, x_scale, weight, weight_scale, group_list, out, out_scale, M, K, N, G, group_list_type,
                                                   gate_up_silu, workspace, workspace_bytes, nullptr, stream);
}

// Grouped GEMM whose two operands are 4-bit floats with one power-of-two scale per 32 k:
//
//   y[m, n] = sum_k x[m, k] * w[g, n, k],  both e2m1 with an e8m0 scale per 32 k along their rows
//
// Persistent kernel on pairs of CTAs, tcgen05 kind::mxf4: the tensor core multiplies the codes, applies both scales and keeps the sums of the whole k
// range in fp32.  The operands are swapped: the 256 lanes of a pair's MMA are weight columns, two blocks of 128 to a CTA's tile, and its N extent
// is the tile's token rows rounded up to 16 (16 .. 192), so an expert's weights pass once where it has up to 192 rows.  The rows of x are split
// between the two CTAs' shared memory and read by both.  Codes enter by TMA as they are stored.  Scales come through registers, 16 bytes (512 k of a
// row) at a time, and are written to tensor memory by the warps that fetch them.
//
// Gate/up: a CTA's two blocks are 128 gate columns and the up columns of the same indices; silu(gate) * up in fp32, a warp's 32 columns
// are a block of the result: its largest magnitude, its scale and codes are the warp's own business.
//
// Warp roles: 0 loads codes, 1 and 2 issue the MMAs of a block of columns each (first CTA), 4 .. 7 bring scales, 8 .. 15 epilogue.  Every wait
// is bounded.  A tile's sums are single in tensor memory where it has more than 96 rows, so the epilogue takes them to registers (silu and the product
// made on the way) before it quantises or stores.
//
// What bounds it, measured alone | in a steady loop (which runs at 1.2 to 1.45 GHz, at the power limit), us: 256 experts, 4096 x 8 rows: 2048 x
// 7168 386 | 416, of 381 for its 2.5 GB; gate/up 7168 x 4096 683 | 766, of 634; 8192 x 8 Zipf rows, gate/up 1085 to 1111 | 1260, of 658 for its bytes and 450 of
// MMA at the nominal rate; 37 x 8 rows, 2048 x 7168 229 of 213; 32 x 8 rows, gate/up 395 of 388; one token's 8 experts 25 (2048 x 7168) and 41 (gate/up, of
// 19: 64 tiles on 74 pairs, each a walk over all of k; 8 are launch and set-up, and the 128 CTAs in use could read the bytes in 22: the rest is not
// explained).  So: memory, then power; Zipf rows, whose experts with thousands of rows read the weights from L2 again and again: loads into the
// multiprocessors (without the epilogue 1069, with MMAs of 16 columns 1050, of both 978), and behind them the MMAs (without loads 647).
//
// Steps, us (gate/up 4096 x 8 | Zipf rows): scales gathered by cp.async, handed over two stages late 3137 Zipf; on arrival 1063 | 1872; through registers
// 795 | 1405; sums to registers first 739 | 1296; scales written to tensor memory instead of copied there (tcgen05.cp goes in turn with the
// MMAs) and an MMA warp for each block 684 | 1149; pairs 683 | 1107.  Tried and not kept: copies of the next stage's scales ahead of the
// MMAs (813), weight scales prefetched to L2 a tile ahead (833), one reciprocal for two values of silu (706 | 1152), tiles drawn from a counter (below).
#include <algorithm>

#include "common.cuh"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace b200moe {
namespace mf {

constexpr int kWarpLoad = 0, kWarpMma0 = 1, kWarpScale0 = 4, kScaleWarps = 4, kWarpEpi0 = 8, kEpiWarps = 8;
constexpr int kThreads = (kWarpEpi0 + kEpiWarps) * 32;
constexpr int kMaxR = 192;               // token rows of a tile
constexpr int kBlocks = 2;               // of 128 weight columns, of a CTA's tile
constexpr int kBlockBytes = 128 * 128;   // 128 weight columns x 256 k
constexpr int kStageK = 256;             // 128 bytes of a row
constexpr int kWords = 2;                // of scales of a stage (a word: 128 k)
constexpr int kChunkWords = 4;           // of scales: 16 bytes, 512 k of a row
constexpr int kMaxSlots = 10, kMaxBufs = 4;
constexpr uint32_t kTmemCols = 512;
constexpr int kStripBytes = 1024;        // of an epilogue warp: 16 tokens x 32 columns in bf16
constexpr int kBoxes[4] = {64, 32, 16, 8};  // rows of x that a load takes
constexpr int kScaleRows = 2 * 128 + kMaxR;
constexpr int kExchangeBytes = 2 * kScaleRows * 16;
constexpr int kBarrierBytes = 1024;
constexpr int kSmemBytes = 227 * 1024;

// What a tile is: two blocks of 128 weight columns to a CTA, neighbours, or gate columns and the up columns of the same indices.
template <bool GATE>
struct Mode {
    static constexpr bool kGate = GATE;
    // columns that a tile advances by (gate/up: of each), the CTA's first, and how far its second block is
    static constexpr int kTileColumns = GATE ? 256 : 512;
    static __device__ __forceinline__ int first_column(int nt, uint32_t rank) { return nt * kTileColumns + (int)rank * (kTileColumns / 2); }
    static __device__ __forceinline__ int block_step(int N) { return GATE ? N >> 1 : 128; }
    // neighbours come in one load
    static constexpr int kLoads = GATE ? 2 : 1, kLoadColumns = 256 / kLoads;
};
using Plain = Mode<false>;
using GateUp = Mode<true>;
constexpr int kFixedBytes = 1024 + kBarrierBytes + kEpiWarps * kStripBytes + kExchangeBytes + 2 * (kMaxExperts + 4) * 4;
constexpr int kRingBytes = kSmemBytes - kFixedBytes;
// A stage: the CTA's two blocks, and its half of the tile's rows.
__host__ __device__ constexpr int slot_bytes_of(int width) { return kBlocks * kBlockBytes + width * 64; }
constexpr int kScaleColumns = kChunkWords * 4 * (kBlocks + 2);  // tensor-memory columns of a chunk of scales
static_assert(kRingBytes % 16 == 0 && kRingBytes / slot_bytes_of(kMaxR) >= 3, "stages");
static_assert(kBlocks * kMaxR + 2 * kScaleColumns <= (int)kTmemCols, "tensor memory");

struct Args {
    const uint8_t* x_scale;
    const uint8_t* w_scale;
    const int64_t* group_list;
    void* out;
    uint8_t* out_scale;
    int M, K, N, G, gl_type;
    int words;         // of a row of scales
    int* findings;
};

struct Sync {
    uint64_t full[kMaxSlots];    // first CTA: the bytes of both CTAs' codes
    uint64_t empty[kMaxSlots];   // each CTA: commits of the stage's MMAs, one for each block of columns
    uint64_t s_full[2];          // first CTA: the scale warps of both have written their lanes' copy of a chunk
    uint64_t s_empty[2];         // each CTA: commits of its last MMAs
    uint64_t exchange;           // the CTA's scale warps among themselves
    uint64_t d_full[kMaxBufs];   // each CTA: commits of a tile's MMAs
    uint64_t d_empty[kMaxBufs];  // first CTA: the epilogue warps of both have the tile's sums
    uint64_t drain[2];
    uint32_t tmem_base;
    int abort;
    int n_tiles, width;          // width: token rows of the widest tile, rounded up to 16
};
static_assert(sizeof(Sync) <= kBarrierBytes, "barrier block");

struct Tile {
    int g, row0, rows, n, nt;  // n: rows rounded up to 16
};

// Waits and tile look-ups are a whole warp's: it votes at every poll and so leaves them together.
__device__ __forceinline__ bool all(bool v) { return __all_sync(0xffffffffu, v); }
// A value that every lane has, in a form that shows it.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
// Whether a poll that has failed `spins` times gives up: the other roles have, or the time is over.
__device__ __forceinline__ bool give_up(uint32_t spins, uint64_t& t0, Sync* sy, int* findings, int id) {
    if ((spins & 0xFF) != 0xFF) return false;  // (the clock is not read in a wait that ends soon)
    if (t0 == 0) {
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

// An expert's rows are cut into the fewest tiles, of equal size rounded up to 16.
__device__ __forceinline__ int tiles_of(int rows) { return (rows + kMaxR - 1) / kMaxR; }
__device__ __forceinline__ int tile_rows_of(int rows, int tiles) { return ((rows + tiles - 1) / tiles + 15) & ~15; }

// Inside an expert the row tiles of a weight column run together, so that they share the weights in L2.
struct Tiles {
    const int *prefix, *row_start;
    int G, n_nt, n, pairs;
};
__device__ __forceinline__ Tile locate(const Tiles& s, int tile) {
    int lo = 0, hi = s.G;  // largest g with prefix[g] <= tile
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s.prefix[mid] <= tile) lo = mid;
        else hi = mid;
    }
    const int j = tile - s.prefix[lo], mt = (s.prefix[lo + 1] - s.prefix[lo]) / s.n_nt;
    const int nt = j / mt, m = j - nt * mt;
    const int rows = s.row_start[lo + 1] - s.row_start[lo], tr = tile_rows_of(rows, mt);
    Tile t;
    t.g = lo;
    t.nt = nt;
    t.row0 = s.row_start[lo] + m * tr;
    t.rows = min(tr, rows - m * tr);
    t.n = (t.rows + 15) & ~15;
    return t;
}

// The pair's next tile, every n-th of all, which each role finds by itself; false at the end.  (Drawing tiles from a counter costs a call that clears it
// and a ring between the roles, and a steady loop, which the power limit bounds, gains nothing: 256 experts, 4096 x 8 rows, 2048 x
// 7168: alone 386 | drawn 377, in a loop 416 | 430.)
__device__ __forceinline__ bool next_tile(const Tiles& s, int& tile, Tile& t) {
    if (tile >= s.n) return false;
    t = locate(s, tile);
    tile += s.pairs;
    return true;
}

// 2^v and 1 / v; what is below 2^-126 as 0 (the first of these is then added to 1, the second multiplies what it divides)
__device__ __forceinline__ float exp2_flushed(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float reciprocal_flushed(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// g / (1 + e^-g), for g down to kTail: from -87 on the reciprocal would be below the smallest normal number, and up, which multiplies it, may be large
constexpr float kTail = -80.f;
__device__ __forceinline__ float silu(float g) { return g * reciprocal_flushed(1.f + exp2_flushed(-1.44269504f * g)); }
// silu(g) * up for every g.  Under kTail silu is g e^g (to 2^-115), and either factor takes half of the exponent.  e^(g / 2) is 0 from g = -174 on, where
// what it stands for is below 2^-116 for every up; half of the smallest code of the smallest scale is 2^-102.
__device__ __forceinline__ float silu_times(float g, float up) {
    if (!(g < kTail)) return silu(g) * up;
    const float r = exp2_flushed(0.72134752f * g);
    return (g * r) * (up * r);
}

// What an epilogue warp works on: its 32 columns from `col` on (tensor-memory lanes) of the tile's sums at `tmem`.
struct Share {
    Tile t;
    uint32_t tmem, width;
    int group, col;
    uint32_t d_empty;  // in the first CTA
    uint8_t* strip;
};
// The sums are in registers: the buffer goes back, unless they are needed once more.
__device__ __forceinline__ void release(const Share& e, bool now = true) {
    ptx::tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0 && now) ptx::mbar_arrive_remote(e.d_empty);
}

// Sixteen tokens x the warp's 32 columns in bf16 through the warp's strip: the transposing store gives 16-byte pieces of eight columns, 64
// contiguous bytes of a row.  d[4 j + 2 h + i]: columns 16 h + 8 i + g8 and tokens 8 j + 2 q, + 1 of lane (g8, q).
__device__ __forceinline__ void store_rows(const uint32_t (&d)[8], const Tile& t, int token0, int col, uint8_t* strip, const Args& a) {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, q = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int token = j * 8 + (lane & 7);  // row lane % 8 of piece lane / 8
        ptx::stmatrix_x4_trans(ptx::smem_u32(strip) + (uint32_t)(token * 64 + (((lane >> 3) ^ (token >> 1)) & 3) * 16), d[4 * j], d[4 * j + 1],
                               d[4 * j + 2], d[4 * j + 3]);
    }
    __syncwarp();
    const bool inside = col + q * 8 < a.N;
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (size_t)(t.row0 + token0) * a.N + col + q * 8;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int token = j * 8 + g8;
        const uint4 v = *reinterpret_cast<const uint4*>(strip + token * 64 + ((q ^ (token >> 1)) & 3) * 16);
        if (token0 + token < t.rows && inside) *reinterpret_cast<uint4*>(dst + (size_t)token * a.N) = v;
    }
    __syncwarp();
}

// Block `group` of the tile's 128 columns in bf16: NC pieces of 16 tokens at most, all in registers before the first is stored.
template <int NC>
__device__ __forceinline__ void finish_rows(const Share& e, const Args& a) {
    const uint32_t td = e.tmem + e.group * e.width;
    uint32_t v[2][2][8], o[NC][8];
    const auto fetch = [&](int c, uint32_t(&d)[2][8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) ptx::tmem_ld_16x16(td + (uint32_t)(c * 16) + ((uint32_t)(h * 16) << 16), d[h]);
    };
    fetch(0, v[0]);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        ptx::tmem_ld_wait();
        if (c + 1 < NC) fetch(c + 1, v[(c + 1) & 1]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const uint32_t(&d)[8] = v[c & 1][m >> 1];
                o[c][4 * j + m] = pack_bf16x2(__uint_as_float(d[4 * j + 2 * (m & 1)]), __uint_as_float(d[4 * j + 2 * (m & 1) + 1]));
            }
    }
    release(e);
#pragma unroll
    for (int c = 0; c < NC; ++c) store_rows(o[c], e.t, c * 16, e.col + e.group * 128, e.strip, a);
}

// Nibble i of lane j of every eight lanes becomes nibble j of lane i.
__device__ __forceinline__ uint32_t transpose_nibbles(uint32_t v) {
    const int lane = threadIdx.x & 31;
    uint32_t r = __shfl_xor_sync(0xffffffffu, v, 4);
    v = (lane & 4) ? (v & 0xFFFF0000u) | (r >> 16) : (v & 0x0000FFFFu) | (r << 16);
    r = __shfl_xor_sync(0xffffffffu, v, 2);
    v = (lane & 2) ? (v & 0xFF00FF00u) | ((r >> 8) & 0x00FF00FFu) : (v & 0x00FF00FFu) | ((r & 0x00FF00FFu) << 8);
    r = __shfl_xor_sync(0xffffffffu, v, 1);
    return (lane & 1) ? (v & 0xF0F0F0F0u) | ((r >> 4) & 0x0F0F0F0Fu) : (v & 0x0F0F0F0Fu) | ((r & 0x0F0F0F0Fu) << 4);
}

// The lane's column of sixteen tokens, quantised by the warp's 32 columns.
__device__ __forceinline__ void store_quantized(float (&h)[16], const Tile& t, int token0, int col, const Args& a) {
    const int lane = threadIdx.x & 31, inter = a.N >> 1;
    const bool inside = col < inter;  // (an odd number of blocks leaves the pair's last CTA without one)
    uint32_t top = 0;  // lane i: the largest magnitude of token i (magnitudes order as their bits do, infinities and NaN last)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(h[i]) & 0x7FFFFFFFu);
        if (lane == i) top = m;
    }
    const uint32_t byte = mxfp4::scale_byte(top);
    const float inv = mxfp4::inverse(byte);
#pragma unroll
    for (int i = 0; i < 16; ++i) h[i] *= __shfl_sync(0xffffffffu, inv, i);
    const uint32_t bad = __ballot_sync(0xffffffffu, byte == mxfp4::kNaN);
    if (bad != 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((bad >> i) & 1) h[i] = 0.f;
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const float v[8] = {h[8 * p], h[8 * p + 1], h[8 * p + 2], h[8 * p + 3], h[8 * p + 4], h[8 * p + 5], h[8 * p + 6], h[8 * p + 7]};
        const uint32_t codes = transpose_nibbles(mxfp4::codes8(v));  // lane % 8's token, eight columns
        const int token = token0 + 8 * p + (lane & 7);
        if (token < t.rows && inside)
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + (size_t)(t.row0 + token) * (inter >> 1) + (col >> 1) + (lane >> 3) * 4) = codes;
    }
    if (lane < 16 && token0 + lane < t.rows && inside) a.out_scale[(size_t)(t.row0 + token0 + lane) * (inter >> 5) + (col >> 5)] = (uint8_t)byte;
}

// silu(gate) * up of every other piece of 16 tokens, NC at most, in registers before the first is quantised.  false: a gate is under kTail, and the buffer
// is kept for finish_tail.  (A piece behind the tile's rows counts too: whatever it holds costs time alone.  To leave here in that case, before the
// buffer goes back, costs every tile: Zipf rows 1081 us without a look at the gates, 1085 so, 1105 with a branch.)
template <int NC>
__device__ __forceinline__ bool finish_quantized(const Share& e, const Args& a) {
    uint32_t v[2][2][8];
    float h[NC][16], low = 0.f;
    const auto fetch = [&](int s, uint32_t(&d)[2][8]) {  // half a piece
        const uint32_t at = e.tmem + (uint32_t)(((s & ~1) + e.group) * 16 + (s & 1) * 8);
        ptx::tmem_ld_32x8(at, d[0]);
        ptx::tmem_ld_32x8(at + e.width, d[1]);
    };
    fetch(0, v[0]);
#pragma unroll
    for (int s = 0; s < 2 * NC; ++s) {
        ptx::tmem_ld_wait();
        if (s + 1 < 2 * NC) fetch(s + 1, v[(s + 1) & 1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float g = __uint_as_float(v[s & 1][0][i]);
            low = fminf(low, g);
            h[s >> 1][(s & 1) * 8 + i] = silu(g) * __uint_as_float(v[s & 1][1][i]);
        }
    }
    const bool done = all(!(low < kTail));
    release(e, done);
#pragma unroll
    for (int c = 0; c < NC; ++c) store_quantized(h[c], e.t, (2 * c + e.group) * 16, e.col, a);
    return done;
}

// The same, piece by piece, whatever the gates are; every thread stores over what it has stored.
__device__ __forceinline__ void finish_tail(const Share& e, const Args& a) {
#pragma unroll 1
    for (int token0 = e.group * 16; token0 < e.t.n; token0 += 32) {
        float h[16];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint32_t g[8], up[8];
            ptx::tmem_ld_32x8(e.tmem + (uint32_t)(token0 + 8 * s), g);
            ptx::tmem_ld_32x8(e.tmem + (uint32_t)(token0 + 8 * s) + e.width, up);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) h[8 * s + i] = silu_times(__uint_as_float(g[i]), __uint_as_float(up[i]));
        }
        store_quantized(h, e.t, token0, e.col, a);
    }
    release(e);
}

template <class M>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    grouped_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x64,
                   const __grid_constant__ CUtensorMap map_x32, const __grid_constant__ CUtensorMap map_x16, const __grid_constant__ CUtensorMap map_x8, const Args a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
    Sync* sy = reinterpret_cast<Sync*>(ring + kRingBytes);
    uint8_t* strips = ring + kRingBytes + kBarrierBytes;
    uint8_t* exchange = strips + kEpiWarps * kStripBytes;
    int* row_start = reinterpret_cast<int*>(exchange + kExchangeBytes);
    int* prefix = row_start + kMaxExperts + 4;

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_rank();
    const int pairs = (int)gridDim.x / 2, pair = (int)blockIdx.x / 2;
    const int n_nt = ((M::kGate ? a.N >> 1 : a.N) + M::kTileColumns - 1) / M::kTileColumns;

    // what needs nothing from memory comes first: the kernel may have started beside the end of the one before it
    if (threadIdx.x == kThreads - 32) {
        sy->abort = 0;
        const auto init = [](uint64_t* b, int n, uint32_t count) {
            for (int i = 0; i < n; ++i) ptx::mbar_init(ptx::smem_u32(b + i), count);
        };
        init(sy->full, kMaxSlots, 1);
        init(sy->empty, kMaxSlots, kBlocks);
        init(sy->s_full, 2, 2 * kScaleWarps);
        init(sy->s_empty, 2, kBlocks);
        init(&sy->exchange, 1, kScaleWarps);
        init(sy->d_full, kMaxBufs, kBlocks);
        init(sy->d_empty, kMaxBufs, 2 * kEpiWarps);
        init(sy->drain, 2, 1);
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&map_w);
        ptx::prefetch_tensormap(&map_x64);
        ptx::prefetch_tensormap(&map_x32);
        ptx::prefetch_tensormap(&map_x16);
        ptx::prefetch_tensormap(&map_x8);
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
            prefix[a.G] = total * n_nt;
            sy->n_tiles = total * n_nt;
            sy->width = max(wide, 16);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();
    ptx::tc_fence_after();

    const uint32_t tmem_base = (uint32_t)uniform((int)*reinterpret_cast<volatile uint32_t*>(&sy->tmem_base));
    const int n_tiles = uniform(sy->n_tiles), width = uniform(sy->width);
    const int slot_bytes = slot_bytes_of(width), n_slots = min(kMaxSlots, kRingBytes / slot_bytes);
    // tensor memory: the sums of one to four tiles from the start, two chunks of scales at the end
    constexpr int kXScaleAt = kChunkWords * 4 * kBlocks;
    const int n_bufs = min(kMaxBufs, ((int)kTmemCols - 2 * kScaleColumns) / (kBlocks * width));
    const uint32_t scale0 = tmem_base + kTmemCols - 2 * kScaleColumns;
    constexpr int x_at = kBlocks * kBlockBytes;  // of a stage: the codes of the weights, then those of x
    const Tiles tiles = {prefix, row_start, a.G, n_nt, n_tiles, pairs};
    const int words = a.words, stages = (a.K + kStageK - 1) / kStageK;

    // registers of a lane: 48, 112 and twice 176 for the four warps of each kind, together as many as the launch has (with 56 and 104 the
    // down projection spills in a loop: 386 -> 428 us)
    if (warp < kWarpScale0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == kWarpLoad) {
            // ------------------------------ codes ------------------------------
            // The warp walks together and one lane issues.
            const bool leader = ptx::elect_one();
            uint32_t it = 0, slot = 0, ph = 0;
            int tile = pair;
            bool ok = true;
            const uint32_t full0 = ptx::map_rank(ptx::smem_u32(sy->full), 0);
            Tile t;
            while (ok && next_tile(tiles, tile, t)) {
                const int half = t.n >> 1;
                const int col = M::first_column(t.nt, rank), row = t.row0 + (int)rank * half;
                for (int kb = 0; kb < stages; ++kb, ++it) {
                    if (it >= (uint32_t)n_slots && !wait(&sy->empty[slot], ph ^ 1, sy, a.findings, 10)) { ok = false; break; }
                    if (leader) {
                        const uint32_t bar0 = full0 + slot * 8, dst = ptx::smem_u32(ring) + slot * (uint32_t)slot_bytes;
                        if (rank == 0) ptx::mbar_arrive_expect_tx(ptx::smem_u32(&sy->full[slot]), 2u * (uint32_t)(kBlocks * kBlockBytes + half * 128));
                        const int x = kb * 128;
#pragma unroll
                        for (int u = 0; u < M::kLoads; ++u)
                            ptx::tma_load_3d_pair(dst + u * kBlockBytes, &map_w, bar0, x, col + u * M::block_step(a.N), t.g);
                        uint32_t at = dst + x_at;
                        int r = row;
                        if (half & 64) ptx::tma_load_2d_pair(at, &map_x64, bar0, x, r), at += 64 * 128, r += 64;
                        if (half & 32) ptx::tma_load_2d_pair(at, &map_x32, bar0, x, r), at += 32 * 128, r += 32;
                        if (half & 16) ptx::tma_load_2d_pair(at, &map_x16, bar0, x, r), at += 16 * 128, r += 16;
                        if (half & 8) ptx::tma_load_2d_pair(at, &map_x8, bar0, x, r);
                    }
                    __syncwarp();
                    if (++slot == (uint32_t)n_slots) { slot = 0; ph ^= 1; }
                }
            }
            // the commits that give the last stages back have arrived before the CTA ends (the second CTA's come from the first one)
            for (uint32_t i = it; ok && i < it + (uint32_t)n_slots; ++i) {
                if (i >= (uint32_t)n_slots) ok = wait(&sy->empty[slot], ph ^ 1, sy, a.findings, 11);
                if (++slot == (uint32_t)n_slots) { slot = 0; ph ^= 1; }
            }
            if (leader && *reinterpret_cast<volatile int*>(&sy->abort)) {
                // copies in flight land before the shared memory goes
                const uint64_t t0 = ptx::globaltimer_ns();
                while (ptx::globaltimer_ns() - t0 < 10000000ull) {}
            }
            __syncwarp();
        } else if (warp < kWarpMma0 + kBlocks && rank == 0) {
            // ------------------------------ MMA issue ------------------------------
            // A warp for each block of columns: it walks together and one lane issues.  Of the descriptors only the address, in the low
            // word, changes.
            const int u = warp - kWarpMma0;
            const bool leader = ptx::elect_one();
            uint32_t slot = 0, ph = 0, buf = 0, bph = 0, n = 0, cb = 0, cph = 0;
            bool ok = true;
            const uint64_t desc = ptx::umma_desc_sw128(0, 0, 1024);
            const uint32_t desc_hi = (uint32_t)(desc >> 32);
            const uint32_t a0 = (uint32_t)desc + ((ptx::smem_u32(ring) + (uint32_t)(u * kBlockBytes)) >> 4);
            const uint32_t x0 = (uint32_t)desc + ((ptx::smem_u32(ring) + (uint32_t)x_at) >> 4);
            const uint32_t slot_step = (uint32_t)slot_bytes >> 4;
            int tile = pair;
            Tile t;
            for (; ok && next_tile(tiles, tile, t); ++n) {
                const int cols = uniform(t.n), x_words = cols > 128 ? 8 : 4;
                const uint32_t idesc = ptx::umma_idesc_mxf4(256, cols), d = tmem_base + (buf * kBlocks + u) * (uint32_t)width;
                // the epilogue has taken what the buffer held
                if (n >= (uint32_t)n_bufs && !wait(&sy->d_empty[buf], bph ^ 1, sy, a.findings, 30)) break;
                uint32_t more = 0;
                for (int kb = 0; kb < stages; ++kb) {
                    if (!wait(&sy->full[slot], ph, sy, a.findings, 40)) { ok = false; break; }
                    const uint32_t al = a0 + slot * slot_step, xl = x0 + slot * slot_step;
                    const int here = min(kWords, words - kb * kWords);
#pragma unroll
                    for (int w = 0; w < kWords; ++w) {
                        if (w >= here) break;
                        const int cw = (kb * kWords + w) & (kChunkWords - 1);  // the word's place in its chunk
                        if (cw == 0 && !wait(&sy->s_full[cb], cph, sy, a.findings, 41)) { ok = false; break; }
                        if (w == 0 || cw == 0) ptx::tc_fence_after();
                        if (leader) {
                            const uint32_t ws = scale0 + cb * kScaleColumns + (uint32_t)((u * kChunkWords + cw) * 4);
                            const uint32_t xs = scale0 + cb * kScaleColumns + (uint32_t)(kXScaleAt + cw * x_words);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t step = (uint32_t)((w * 2 + h) * 2);  // 64 k: 32 bytes
                                ptx::umma_mxf4_pair(d, al + step, xl + step, desc_hi, idesc | ptx::umma_scale_half(h), ws, xs, h == 0 ? more : 1u);
                            }
                        }
                        more = 1;
                        if (cw == kChunkWords - 1 || kb * kWords + w + 1 == words) {
                            if (leader) ptx::umma_commit_pair(ptx::smem_u32(&sy->s_empty[cb]));
                            cb ^= 1;
                            cph ^= cb == 0;
                        }
                    }
                    if (leader && ok) {
                        ptx::umma_commit_pair(ptx::smem_u32(&sy->empty[slot]));
                        if (kb + 1 == stages) ptx::umma_commit_pair(ptx::smem_u32(&sy->d_full[buf]));
                    }
                    __syncwarp();
                    if (!ok) break;
                    if (++slot == (uint32_t)n_slots) { slot = 0; ph ^= 1; }
                }
                if (++buf == (uint32_t)n_bufs) { buf = 0; bph ^= 1; }
            }
            // every MMA issued here must have completed before tensor and shared memory go
            if (leader) {
                ptx::umma_commit_pair(ptx::smem_u32(&sy->drain[u]));
                (void)ptx::mbar_wait(ptx::smem_u32(&sy->drain[u]), 0);
            }
            __syncwarp();
        }
    } else if (warp < kWarpEpi0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        // ------------------------------ scales ------------------------------
        // A thread fetches a row of every block of 128, 16 bytes (512 k) of each; the warps exchange them through shared memory, since each
        // writes all rows to its quarter of the lanes: row r in lane r % 32 of column r / 32, four columns for a word (128 k) of 128 rows.
        const int q = warp - kWarpScale0, row = q * 32 + lane, chunks = (words + kChunkWords - 1) / kChunkWords;
        const bool whole = (words & 3) == 0 && ((reinterpret_cast<uintptr_t>(a.w_scale) | reinterpret_cast<uintptr_t>(a.x_scale)) & 15) == 0;
        struct Chunk {
            uint4 v[kBlocks + 2];  // of the weights' blocks and the two of x
            int cols;              // token rows of the tile rounded up; 0: the schedule has ended
        };
        int at = chunks, cols = 0;
        int tile = pair;
        bool live = true;
        const uint32_t* src[kBlocks + 2];  // NULL: no row there, zeros
        const auto fetch = [&](Chunk& c) {
            if (at == chunks) {
                Tile t;
                if (live) live = next_tile(tiles, tile, t);
                if (!live) {
                    c.cols = 0;
                    return;
                }
                cols = t.n;
#pragma unroll
                for (int u = 0; u < kBlocks; ++u) {
                    const int n = M::first_column(t.nt, rank) + u * M::block_step(a.N) + row;
                    src[u] = n < a.N ? reinterpret_cast<const uint32_t*>(a.w_scale) + ((size_t)t.g * a.N + n) * (size_t)words : nullptr;
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    src[kBlocks + b] = b * 128 + row < t.rows
                                           ? reinterpret_cast<const uint32_t*>(a.x_scale) + (size_t)(t.row0 + b * 128 + row) * (size_t)words
                                           : nullptr;
                at = 0;
            }
            c.cols = cols;
            const int here = words - kChunkWords * at;
#pragma unroll
            for (int b = 0; b < kBlocks + 2; ++b) {
                const uint32_t* p = src[b] + kChunkWords * at;
                c.v[b] = make_uint4(0u, 0u, 0u, 0u);
                if (src[b] != nullptr) {
                    // (ordinary loads: the kernel ahead may have written either operand's scales)
                    if (whole) {
                        c.v[b] = __ldca(reinterpret_cast<const uint4*>(p));
                    } else {
                        c.v[b].x = __ldca(p);
                        if (here > 1) c.v[b].y = __ldca(p + 1);
                        if (here > 2) c.v[b].z = __ldca(p + 2);
                        if (here > 3) c.v[b].w = __ldca(p + 3);
                    }
                }
            }
            ++at;
        };
        uint32_t n = 0, cb = 0, cph = 0;
        const uint32_t s_full0 = ptx::map_rank(ptx::smem_u32(sy->s_full), 0);
        const uint32_t quarter = scale0 + ((uint32_t)(q * 32) << 16);
        const auto put = [&](const Chunk& c) {
            uint4* room = reinterpret_cast<uint4*>(exchange) + cb * kScaleRows;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) room[b * 128 + row] = c.v[b];
            room[kBlocks * 128 + row] = c.v[kBlocks];
            if (128 + row < kMaxR) room[kBlocks * 128 + 128 + row] = c.v[kBlocks + 1];
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sy->exchange));
            if (!wait(&sy->exchange, n & 1, sy, a.findings, 21)) return false;
            if (n >= 2 && !wait(&sy->s_empty[cb], cph ^ 1, sy, a.findings, 20)) return false;
            ptx::tc_fence_after();
            const uint32_t to = quarter + cb * kScaleColumns;
            // four rows of a block, word by word
            const auto rows4 = [&](const uint4* r, uint32_t(&o)[16]) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 v = r[i * 32 + lane];
                    o[i] = v.x; o[4 + i] = v.y; o[8 + i] = v.z; o[12 + i] = v.w;
                }
            };
            uint32_t o[16];
#pragma unroll
            for (int u = 0; u < kBlocks; ++u) {
                rows4(room + u * 128, o);
                ptx::tmem_st_32x16(to + u * (kChunkWords * 4), o);
            }
            rows4(room + kBlocks * 128, o);
            if (c.cols <= 128) {
                ptx::tmem_st_32x16(to + kXScaleAt, o);
            } else {
                uint32_t p[8];
#pragma unroll
                for (int i = 0; i < (kMaxR - 128) / 32; ++i) {
                    const uint4 v = room[kBlocks * 128 + 128 + i * 32 + lane];
                    p[i] = v.x; p[2 + i] = v.y; p[4 + i] = v.z; p[6 + i] = v.w;
                }
#pragma unroll
                for (int w = 0; w < kChunkWords; ++w) {
                    const uint32_t r[8] = {o[4 * w], o[4 * w + 1], o[4 * w + 2], o[4 * w + 3], p[2 * w], p[2 * w + 1], 0u, 0u};
                    ptx::tmem_st_32x8(to + kXScaleAt + w * 8, r);
                }
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_remote(s_full0 + cb * 8);
            ++n;
            cb ^= 1;
            cph ^= cb == 0;
            return true;
        };
        static_assert(kMaxR == 192, "two rows of the second block of x");
        Chunk c0, c1;
        bool ok = true;
        fetch(c0);
        while (true) {
            fetch(c1);
            if (c0.cols == 0 || !(ok = put(c0))) break;
            fetch(c0);
            if (c1.cols == 0 || !(ok = put(c1))) break;
        }
        // (the commits of the last chunks have arrived before the CTA ends)
        for (uint32_t i = n < 2 ? n : 2; ok && i > 0; --i) {
            if (n < 2 && i == n) cb = 0, cph = 1;  // (one chunk alone: the first buffer's first phase)
            ok = wait(&sy->s_empty[cb], cph ^ 1, sy, a.findings, 22);
            cb ^= 1;
            cph ^= cb == 0;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        // ------------------------------ epilogue ------------------------------
        Share e;
        e.group = (warp - kWarpEpi0) >> 2;
        e.strip = strips + (warp - kWarpEpi0) * kStripBytes;
        e.width = (uint32_t)width;
        const int quarter = warp & 3;
        const uint32_t d_empty0 = ptx::map_rank(ptx::smem_u32(sy->d_empty), 0);
        uint32_t buf = 0, ph = 0;
        int tile = pair;
        while (next_tile(tiles, tile, e.t)) {
            e.tmem = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * (uint32_t)(kBlocks * width);
            e.col = M::first_column(e.t.nt, rank) + quarter * 32;
            e.d_empty = d_empty0 + buf * 8;
            if (!wait(&sy->d_full[buf], ph, sy, a.findings, 50)) break;
            ptx::tc_fence_after();
            // (the number of pieces is a constant, so that they stay in registers)
            if constexpr (M::kGate) {
                bool done;
                switch ((e.t.n + 31) / 32) {
                    case 1: done = finish_quantized<1>(e, a); break;
                    case 2: done = finish_quantized<2>(e, a); break;
                    case 3: done = finish_quantized<3>(e, a); break;
                    case 4: done = finish_quantized<4>(e, a); break;
                    case 5: done = finish_quantized<5>(e, a); break;
                    default: done = finish_quantized<6>(e, a); break;
                }
                if (!done) finish_tail(e, a);
            } else {
                switch ((e.t.n + 31) / 32) {
                    case 1: finish_rows<2>(e, a); break;
                    case 2: finish_rows<4>(e, a); break;
                    case 3: finish_rows<6>(e, a); break;
                    case 4: finish_rows<8>(e, a); break;
                    case 5: finish_rows<10>(e, a); break;
                    default: finish_rows<12>(e, a); break;
                }
            }
            if (++buf == (uint32_t)n_bufs) { buf = 0; ph ^= 1; }
        }
    }

    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    // (so have the last commits of the MMA warps, which arrive here too; the first CTA's warps waited for theirs)
    if (rank != 0 && warp >= kWarpMma0 && warp < kWarpMma0 + kBlocks) (void)ptx::mbar_wait(ptx::smem_u32(&sy->drain[warp - kWarpMma0]), 0);
    __syncwarp();
    ptx::cluster_sync();  // (what one CTA sends the other, loads and MMAs of the pair among it, has arrived)
    if (warp == kWarpMma0) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

static bool sizes_ok(int64_t M, int64_t K, int64_t N, int64_t G) {
    constexpr int64_t kMost = 0x3FFFFFFF;  // (products of two sizes stay in 64 bits)
    return M >= 0 && M <= kMost && K > 0 && K <= kMost && N > 0 && N <= kMost && G > 0 && G <= kMaxExperts;
}

}  // namespace mf
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_grouped_gemm_mxfp4(const void* x, const uint8_t* x_scale, const void* weight, const uint8_t* weight_scale,
                                          const int64_t* group_list, void* out, uint8_t* out_scale, int64_t M, int64_t K, int64_t N,
                                          int64_t G, int group_list_type, int gate_up_silu, int32_t* findings, void* stream) {
    if (!mf::sizes_ok(M, K, N, G) || (K % 32) != 0 || (N % 16) != 0 || (gate_up_silu && (N % 256) != 0)) return B200MOE_ERR_SHAPE;
    if (group_list_type != B200MOE_GROUP_LIST_CUMSUM && group_list_type != B200MOE_GROUP_LIST_COUNTS) return B200MOE_ERR_ARGUMENT;
    if (gate_up_silu != 0 && gate_up_silu != 1) return B200MOE_ERR_ARGUMENT;
    if (M == 0) return B200MOE_OK;
    // (unit numbers)
    if ((M / mf::kMaxR + G) * ((N + 255) / 256) > 0x3FFFFFFLL) return B200MOE_ERR_SHAPE;
    if (!x || !x_scale || !weight || !weight_scale || !group_list || !out || (gate_up_silu && !out_scale)) return B200MOE_ERR_NULL_POINTER;
    const auto aligned4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
    if (!aligned16(x) || !aligned16(weight) || !aligned16(out) || !aligned4(x_scale) || !aligned4(weight_scale) || !aligned4(out_scale))
        return B200MOE_ERR_ALIGNMENT;
    mf::Args a = {};
    a.x_scale = x_scale;
    a.w_scale = weight_scale;
    a.group_list = group_list;
    a.out = out;
    a.out_scale = out_scale;
    a.M = (int)M; a.K = (int)K; a.N = (int)N; a.G = (int)G;
    a.gl_type = group_list_type;
    a.words = (int)(mxfp4::scale_width(K) / 4);
    a.findings = findings != nullptr ? findings : findings_words();
    CUtensorMap map_w, map_x[4];
    int rc = make_tensor_map_3d_u8(&map_w, weight, (uint64_t)G, (uint64_t)N, (uint64_t)(K / 2), gate_up_silu ? mf::GateUp::kLoadColumns : mf::Plain::kLoadColumns, 128);
    for (int i = 0; i < 4 && rc == B200MOE_OK; ++i)
        rc = make_tensor_map_2d(&map_x[i], x, 1, (uint64_t)M, (uint64_t)(K / 2), mf::kBoxes[i], 128, true);
    if (rc != B200MOE_OK) return rc;
    const auto kernel = gate_up_silu ? mf::grouped_kernel<mf::GateUp> : mf::grouped_kernel<mf::Plain>;
    B200MOE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, mf::kSmemBytes));
    B200MOE_CUDA_TRY(launch_dependent(kernel, (unsigned)(sm_count() / 2 * 2), mf::kThreads, mf::kSmemBytes, static_cast<cudaStream_t>(stream), map_w,
                                      map_x[0], map_x[1], map_x[2], map_x[3], a));
    return B200MOE_OK;
}

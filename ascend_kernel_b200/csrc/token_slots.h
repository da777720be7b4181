// Where the two epilogue groups of the gate/up product keep what belongs to a token (magnitudes, then what the codes are made
// with): every group has room of its own, whatever the tile's size.  A group has half of a tile's tokens, and a group may be
// a tile ahead of the other one where a tile has no more blocks than there are tensor-memory buffers; numbered by the token's place in the tile,
// 16 .. 31 of a tile of 32 tokens (the second group's) would be the first group's in a tile of 64.
// Plain C++ as well: the CPU tests compile it.
#pragma once

#ifdef __CUDACC__
#define B200MOE_SLOTS_HD __host__ __device__ __forceinline__
#else
#define B200MOE_SLOTS_HD inline
#endif

namespace b200moe {

constexpr int kTileTokens = 160;                // of the widest tile
constexpr int kGroupTokens = kTileTokens / 2;   // of a group in it

// Token `i` of those that group `group` has in the tile.
B200MOE_SLOTS_HD constexpr int token_slot(int group, int i) { return group * kGroupTokens + i; }

}  // namespace b200moe

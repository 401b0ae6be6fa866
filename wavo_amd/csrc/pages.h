// Caches in pages (include/wavo_hip.h, wh_pages): where a position's keys and values stand.
//
// A page holds, key head by key head, tiles of 32 positions in the order in which the matrix cores take them
// (v_mfma_f32_16x16x32_f16: lane 16g + m holds row m's 8 elements from 8g on).  A tile's words of 8 values, for every
// chunk c of 32 values of a head:
//   K, word (c, u) of lane 16g + m: values 32c + 8g .. + 7 of position 16u + m, an operand row of K Q^T;
//   V, word (c, x) of lane 16g + m: value 32c + 2m + x of positions 16 (e / 4) + 4g + e % 4, e < 8, an operand row of
//     V^T P^T: those are the positions whose scores lane 16g + i holds after K Q^T, in that order, so that softmax
//     weights never leave their lane.
// 16 bits: a word is 8 halfs, word (c, u) of lane l at half ((2c + u) * 64 + l) * 8; K's 32 hd halfs, then V's.
// 4 bits (Q4_0): value (nibble - 8) * d with one f16 factor d per position and chunk.  Element e is nibble
// e / 2 + 4 (e % 2), so that two neighbours come out of one mask as a pair of halfs.  A lane's words stand next to each
// other in fours, the last two where hd / 16 is no multiple of four; factors [g][c][e] for the positions of V's words,
// 16 bytes that a lane takes at once.  K's words and factors, then V's: 9 hd words in all.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pages {

constexpr int TILE = 32;  // positions

struct Pages {
  uint32_t *pool;
  const int32_t *table;
  size_t table_stride;
  int pages, shift, room, kv_heads, hd;  // positions of a page: 1 << shift; of a sequence, at most: room
  size_t page_words;
};

constexpr __host__ __device__ int tile_words(bool q4, int hd) { return q4 ? 9 * hd : 32 * hd; }

// The first word of a sequence's tile of key head kh, or nullptr where its page is not there.
__device__ __forceinline__ uint32_t *tile_at(const Pages &p, bool q4, int b, int tile, int kh) {
  const int slot = p.shift - 5, id = p.table[(size_t)b * p.table_stride + (tile >> slot)];
  if ((uint32_t)id >= (uint32_t)p.pages) return nullptr;
  return p.pool + (size_t)id * p.page_words + (size_t)((kh << slot) + (tile & ((1 << slot) - 1))) * tile_words(q4, p.hd);
}

// The position (of its tile) of element e of group g, and the group and element of a position.
__device__ __forceinline__ int position_of(int g, int e) { return 16 * (e >> 2) + 4 * g + (e & 3); }

// Where word t = 2c + u of a lane stands in 4 bits, T of them a lane.
__device__ __forceinline__ int word_at(int t, int lane, int T) {
  const int whole = T & ~3;
  return t < whole ? (t >> 2) * 256 + lane * 4 + (t & 3) : whole * 64 + lane * 2 + (t - whole);
}
__device__ __forceinline__ constexpr int nibble_of(int e) { return 4 * (e / 2 + 4 * (e % 2)); }

}  // namespace pages

// The cache of keys and values in MX4 (include/tetris_attention.h): how a page is laid out.
//
// A page holds for each kv head its granules of 16 tokens one after another; a granule of heads of D elements is 17 D bytes:
//   keys' codes    8 D      for a product of 16 tokens by 16 rows of q over 32 elements (v_mfma_f32_16x16x32) a lane holds 8 elements of
//                           one token.  Lane 16 g + t has token t and the elements from g D / 4 on, D / 4 of them: D / 8 bytes, read in one piece.
//                           (Which elements a step of the product takes is free, as long as q's are the same.)
//   values' codes  8 D      for the product of values (as rows: elements) by softmax weights (as columns) over tokens lane 16 g + m holds
//                           tokens 4 g .. 4 g + 3, which are those whose scores the first product leaves in lanes 16 g ..: no exchange
//                           between lanes.  Of each of the four it has D / 16 elements, D / 32 bytes, so again D / 8 bytes in one piece.  Byte c of
//                           a token is elements m D / 16 + 2 c and the next one where D is 32, 64, 128 or 256: all of a lane's lie in
//                           one block, with one scale a token.  Else it is elements 32 c + m and 32 c + 16 + m, of block c.
//   keys' scales   D / 2    [token][block]
//   values' scales D / 2    [token / 4][block][token % 4]
// A token is written without reading what is there, whatever its neighbours are.
#ifndef TETRIS_CSRC_CACHE_H_
#define TETRIS_CSRC_CACHE_H_

#include "mx4.h"
#include "tetris_attention.h"

namespace tetris {

constexpr int kGranule = 16;  // tokens
constexpr int kCacheHead = 256, kCachePage = 4096, kCacheHeads = 1024;

// whether a lane's elements of a value are neighbours
constexpr bool neighbours(int head) { return (head & (head - 1)) == 0; }

}  // namespace tetris

struct tetris_cache {
  int kv_heads = 0, head = 0, page = 0, pages = 0, device = 0;
  int64_t page_bytes = 0;
  uint8_t* data = nullptr;
  tetris::Workspaces space;
};

namespace tetris {
// The handle's device is the current one.
int check_cache(const tetris_cache* c);
}  // namespace tetris

#endif  // TETRIS_CSRC_CACHE_H_

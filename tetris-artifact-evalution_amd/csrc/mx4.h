// Internal declarations of the operators on MX4 weights (include/tetris_mx4.h).
//
// Layout for the matrix cores.  Rows are taken in tiles of 32, columns in tiles of 64 (two blocks); a tile's codes are 1 KiB,
// lane l of a wave holding the 16 bytes of row l % 32, block l / 32: what one lane feeds to a 32 x 32 x 64 product of 4-bit
// numbers, and to four 32 x 32 x 16 products of bf16 (product j takes elements 8j .. 8j + 7 of the lane's block, on both sides).
//   codes  [matrix][row tile][column tile][64 lanes][16 bytes]
//   scales [matrix][row tile][pair of column tiles][64 lanes][2 bytes]
// Columns are padded to 128 with zero codes of scale 1.  In a gated matrix row tile t is rows 16 t .. 16 t + 15 of the
// gate and then the same rows of what it gates, so that a lane of a product holds both.
#ifndef TETRIS_CSRC_MX4_H_
#define TETRIS_CSRC_MX4_H_

#include "common.h"
#include "tetris_mx4.h"

namespace tetris {

constexpr int kMxPad = 128;  // columns of a laid-out matrix and of staged rows are padded to this
constexpr int kMxSide = 1 << 21;           // most rows and columns of a matrix, and most elements from one row to the next of rows read as they lie
constexpr int64_t kMxReach = 0x7fff0000;   // bytes that a kernel's 32-bit offsets reach

template <int TYPE>
struct Elem;
template <>
struct Elem<TETRIS_F32> { using type = float; };
template <>
struct Elem<TETRIS_F16> { using type = _Float16; };
template <>
struct Elem<TETRIS_BF16> { using type = __bf16; };

inline int elem_size(int type) { return type == TETRIS_F32 ? 4 : 2; }
inline bool bad_type(int type) { return type != TETRIS_F32 && type != TETRIS_F16 && type != TETRIS_BF16; }
inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
// how many bf16 numbers hold one of `type` exactly (8 bits of significand each)
inline int parts_of(int type) { return type == TETRIS_BF16 ? 1 : type == TETRIS_F16 ? 2 : 3; }

// Where quantised rows go: as MX4 rows; in the layout above (rows of the last tile past `rows` and columns to kMxPad filled);
// or as the values they stand for, in bf16 rows of kMxPad columns' multiple.
enum { kMxRows = 0, kMxTiles = 1, kMxValues = 2 };
int mx4_quantize_to(int kind, const void* d_x, int type, int64_t rows, int cols, int64_t ld, void* d_codes, uint8_t* d_scales,
                    hipStream_t stream);

// Rows of any alignment copied to rows of round_up(cols, kMxPad) elements filled with zeros: of the same type (parts = 0), or
// as `parts` arrays of bf16 that add up to the numbers, one after another.
int stage_rows(const void* d_x, int type, int64_t rows, int cols, int64_t ld, int parts, void* d_out, hipStream_t stream);

}  // namespace tetris

struct tetris_mx4 {
  int experts = 0, n = 0, k = 0;
  bool gated = false;
  bool half = false;                 // every weight is exact in f16
  int row_tiles = 0, col_tiles = 0;  // of one matrix
  uint8_t* codes = nullptr;
  uint8_t* scales = nullptr;
  std::mutex mu;
  struct Space { void* ptr = nullptr; size_t bytes = 0; };
  std::map<std::pair<hipStream_t, uint64_t>, Space> space;  // the number: of the thread, for hipStreamPerThread, which is one value for many streams
  std::vector<void*> retired;  // replaced by larger ones; a captured graph may hold their addresses
};

#endif  // TETRIS_CSRC_MX4_H_

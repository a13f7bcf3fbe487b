// Rows read by pieces of eight elements, a piece a lane.
#ifndef TETRIS_CSRC_ROWS_H_
#define TETRIS_CSRC_ROWS_H_

#include "mx4.h"

namespace tetris {

// Eight elements of a row from element `at`, those from `cols` on zero.  VEC: the row starts on 16 bytes and `at` is a
// multiple of eight.
template <typename T, bool VEC>
__device__ inline void load8(const T* row, int at, int cols, float (&v)[8]) {
  if (VEC && at + 8 <= cols) {
    T t[8];
    const int4* src = reinterpret_cast<const int4*>(row + at);
    int4* dst = reinterpret_cast<int4*>(t);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) dst[i] = src[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at + i < cols ? (float)row[at + i] : 0.f;
  }
}

// A lane's place in a matrix of `per_row` pieces of eight elements a row, the pieces numbered through: wave w of the grid takes
// pieces 64 w .. 64 w + 63, so the division is the wave's, on the scalar unit, and a lane only steps over row ends.
struct Place { int64_t row; int piece; };
__device__ inline Place place_of(int64_t wave, unsigned per_row) {
  const int64_t first = wave * 64;
  Place p;
  p.row = first / per_row;
  unsigned piece = (unsigned)(first - p.row * per_row) + (threadIdx.x & 63);
  if (piece >= per_row) {
    const unsigned over = per_row >= 64 ? 1 : piece / per_row;
    piece -= over * per_row;
    p.row += over;
  }
  p.piece = (int)piece;
  return p;
}

__device__ inline int64_t wave_of() {
  return (int64_t)blockIdx.x * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}

// Largest magnitude of the four lanes that share a block, as bits: those of non-negative numbers order like the numbers, and
// an infinity or a NaN comes out as 0x7f800000 or more.
__device__ inline unsigned quad_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));  // lanes 2 3 0 1
}

}  // namespace tetris

#endif  // TETRIS_CSRC_ROWS_H_

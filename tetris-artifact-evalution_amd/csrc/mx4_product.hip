// Products with weights in MX4 (csrc/mx4.h has their layout): y = x W^T, and the experts' products of tokens routed to them.
//
// A weight is a 4-bit code times a power of two: exact in bf16, which the matrix cores multiply at full rate with sums
// in 32 bits.  Activations are taken as one, two or three bf16 numbers each (bf16, f16, f32: 8, 11, 24 bits of
// significand in parts of 8), so every product is exact in every type.  Codes become bf16 pairs with one instruction a pair, which
// also multiplies by the scale, in the registers of the wave that uses them: what comes from memory is 17 bytes for 32 weights.
#include <algorithm>
#include <atomic>
#include <new>
#include <type_traits>

#include "mx4.h"

namespace tetris {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// What a launch writes: numbers of a type, or (between the experts' products) bf16 parts of numbers.
enum { kOutF32 = TETRIS_F32, kOutF16 = TETRIS_F16, kOutBF16 = TETRIS_BF16, kOutParts2, kOutParts3 };

struct Product {
  const uint8_t* x_scales;  // of rows in MX4
  const void* x;         // rows of ldx elements that start on 16 bytes; elements k .. k8 - 1 of a row are zero
  int64_t ldx, part;     // part: elements between the parts' arrays
  int parts, k8, rows;   // rows of all groups together
  const i32x4* codes;    // laid-out weights
  const uint8_t* scales;
  int row_tiles, col_tiles, n;
  // Rows in groups, one for each expert: positions offsets[e] .. offsets[e + 1] - 1 are expert e's, position p standing for slot
  // order[p].  NULL: one group, position = row.
  const int* offsets;
  const int* order;
  const int* index;      // of up to 64 slots, in place of offsets and order
  int experts;
  int from_div;          // > 0: position p reads row order[p] / from_div; 0: row p
  int to_slot;           // position p writes row order[p], else row p
  int max_tiles;         // of rows, over all groups
  void* y;
  int64_t ldy, y_part;
  int vec_out;           // rows of outputs start on 16 bytes
  const float* bias;
};

// Which rows a workgroup has: tile `tile` of the groups' tiles of `size` rows, numbered through.  Every wave finds it for itself.
__device__ inline bool find_tile(const Product& a, int tile, int size, int* expert, int* first, int* count) {
  if (!a.offsets) {
    *expert = 0;
    *first = tile * size;
    *count = min(size, a.rows - tile * size);
    return *count > 0;
  }
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < a.experts; base += 64) {
    const int e = base + lane;
    const int lo = a.offsets[min(e, a.experts)], hi = a.offsets[min(e + 1, a.experts)];
    const int tiles = (hi - lo + size - 1) / size;
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned long long here = __ballot(tile < before + sum);
    if (here) {
      const int l = __builtin_ctzll(here);
      const int t = tile - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));
      *expert = base + l;
      *first = __builtin_amdgcn_readlane(lo, l) + t * size;
      *count = min(size, __builtin_amdgcn_readlane(hi, l) - *first);
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// The same for tiles of sixteen rows, and the lane's row of the tile (that of lane % 16; the last one past the end).  Up to 64 slots
// need no sorting: workgroup `tile` looks for the slots that name the same expert as slot `tile`, and goes on if there are a multiple of sixteen
// of them before it.
__device__ inline bool find_rows(const Product& a, int tile, int* expert, int* first, int* count, int* from, int* to) {
  const int lane = threadIdx.x & 63, r16 = lane & 15;
  if (a.index) {
    const int mine = lane < a.rows ? a.index[lane] : -1;
    const int e = __builtin_amdgcn_readlane(mine, tile);
    if (e < 0 || e >= a.experts) return false;
    const unsigned long long same = __ballot(mine == e);
    const int rank = __builtin_popcountll(same & ((1ull << lane) - 1)), before = __builtin_amdgcn_readlane(rank, tile);
    if (before & 15) return false;
    *expert = e;
    *first = 0;
    *count = min(16, __builtin_popcountll(same) - before);
    const int place = rank - before;
    const int slot = __builtin_amdgcn_ds_permute((mine == e && place >= 0 && place < 16 ? place : 63) * 4, lane);
    *to = __shfl(slot, min(r16, *count - 1));
    *from = *to / a.from_div;
    return true;
  }
  if (!find_tile(a, tile, 16, expert, first, count)) return false;
  const int p = *first + min(r16, *count - 1);
  *from = a.from_div ? a.order[p] / a.from_div : p;
  *to = a.to_slot ? a.order[p] : p;
  return true;
}

// Eight codes and their scale's exponent bits to bf16.
__device__ inline bf16x8 weights8(int codes, float scale) {
  i32x4 v;
  v.x = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)codes, scale, 0));
  v.y = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)codes, scale, 1));
  v.z = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)codes, scale, 2));
  v.w = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)codes, scale, 3));
  return __builtin_bit_cast(bf16x8, v);
}

// The i-th pair of eight codes to bf16, or to f16.
template <bool HALF>
__device__ inline int pair_of(int codes, float scale, int i) {
  const unsigned c = (unsigned)codes;
  if constexpr (HALF) {
    switch (i) {  // (a constant where this is used)
      case 0: return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0));
      case 1: return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1));
      case 2: return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2));
      default: return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3));
    }
  } else {
    switch (i) {
      case 0: return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
      case 1: return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
      case 2: return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
      default: return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
    }
  }
}
template <bool HALF>
__device__ inline f32x16 product32(i32x4 w, i32x4 x, f32x16 acc) {
  if constexpr (HALF)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
}

__device__ inline float silu(float v) { return v / (1.f + expf(-v)); }

// the leading 16 bits of v that are a bf16 number, and what is left (csrc/mx4_quantize.hip, split)
__device__ inline unsigned leading(float& v) {
  unsigned u = __float_as_uint(v);
  if ((u & 0x7f800000u) == 0x7f800000u) {
    if (u & 0x007fffffu) u |= 0x00400000u;
    v = 0.f;
  } else {
    v -= __uint_as_float(u & 0xffff0000u);
  }
  return u >> 16;
}

template <int OUT>
__device__ inline void store1(const Product& a, int64_t at, float v) {
  if constexpr (OUT <= kOutBF16) {
    static_cast<typename Elem<OUT>::type*>(a.y)[at] = (typename Elem<OUT>::type)v;
  } else {
#pragma unroll
    for (int p = 0; p < (OUT == kOutParts2 ? 2 : 3); ++p) static_cast<unsigned short*>(a.y)[at + p * a.y_part] = (unsigned short)leading(v);
  }
}

// Four outputs of one row from feature f on, at the edge of a matrix or where rows lie badly.
template <int OUT>
__device__ inline void put4(const Product& a, int64_t row, int f, f32x4 v) {
  const int64_t at = row * a.ldy + f;
  const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (f + i < a.n) store1<OUT>(a, at + i, w[i] + (a.bias ? a.bias[f + i] : 0.f));
}

// What a wave has of a tile: 32 WT rows from row0 of the workgroup's on, two row tiles of features from row_tile0 on.  Whole
// tiles go through 4 KiB of LDS of the wave's own, 32 rows of 128 bytes at a time, so that a store writes whole lines: stored from
// the sums' layout, 16 bytes of a row at once, 4096 x 8192 outputs took 20 us of a product of 190.  A 16-byte piece of row r lies at
// piece ^ (r / 2 % 8).
template <int WT, int OUT, bool GATED>
__device__ inline void put_tile(const Product& a, const f32x16 (&acc)[WT][2], int row0, int first, int count, int row_tile0, i32x4* stage) {
  constexpr bool kWide = OUT == kOutF32;                         // four bytes an output
  constexpr int kParts = OUT == kOutParts2 ? 2 : OUT == kOutParts3 ? 3 : 1;
  constexpr int kQuads = GATED ? 2 : 4;                          // of outputs a lane has in a row tile
  constexpr int kTimes = (kWide ? 2 : 1) * kParts;               // through LDS for 32 rows
  constexpr int kWidth = GATED ? 32 : kWide ? 32 : 64;           // features at a time
  constexpr int kPieces = kWidth * (kWide ? 4 : 2) / 16, kEach = 64 / kPieces;
  static_assert(!(GATED && kWide), "what a gated product writes has 16 bits");
  const int lane = threadIdx.x & 63, half = lane >> 5, n = GATED ? a.n / 2 : a.n, f0 = row_tile0 * (GATED ? 16 : 32);
  const bool whole = GATED || (a.vec_out && f0 + 64 <= n);
  f32x4 bias[GATED ? 1 : 2][GATED ? 1 : 4] = {};
  if constexpr (!GATED) {
    if (whole && a.bias) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) bias[r][q][i] = a.bias[f0 + r * 32 + q * 8 + half * 4 + i];
    }
  }
#pragma unroll
  for (int t = 0; t < WT; ++t) {
    f32x4 v[2][kQuads];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const f32x16& u = acc[t][r];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (GATED)
            v[r][q][i] = f0 + r * 16 + q * 8 + half * 4 + i < n ? silu(u[q * 4 + i]) * u[8 + q * 4 + i] : 0.f;
          else
            v[r][q][i] = u[q * 4 + i] + bias[r][q][i];
        }
      }
    if constexpr (!GATED) {
      if (!whole) {
        const int r_in = row0 + t * 32 + (lane & 31);
        if (r_in < count) {
          const int64_t row = a.to_slot ? a.order[first + r_in] : first + r_in;
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int q = 0; q < kQuads; ++q) put4<OUT>(a, row, f0 + r * 32 + q * 8 + half * 4, v[r][q]);
        }
        continue;
      }
    }
#pragma unroll
    for (int c = 0; c < kTimes; ++c) {
      const int row = lane & 31, turn = (row >> 1) & 7;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
          if constexpr (kWide) {
            if (r == c) stage[row * 8 + ((q * 2 + half) ^ turn)] = __builtin_bit_cast(i32x4, v[r][q]);
          } else {
            const int piece = r * kQuads + q;
            uint2 u;
            if constexpr (kParts > 1) {
              float w[4] = {v[r][q].x, v[r][q].y, v[r][q].z, v[r][q].w};
              u.x = leading(w[0]); u.x |= leading(w[1]) << 16;
              u.y = leading(w[2]); u.y |= leading(w[3]) << 16;
              v[r][q] = f32x4{w[0], w[1], w[2], w[3]};
            } else {
              using T = typename Elem<OUT == kOutF16 ? TETRIS_F16 : TETRIS_BF16>::type;
              typedef T T4 __attribute__((ext_vector_type(4)));
              u = __builtin_bit_cast(uint2, T4{(T)v[r][q].x, (T)v[r][q].y, (T)v[r][q].z, (T)v[r][q].w});
            }
            reinterpret_cast<uint2*>(stage)[(row * 8 + (piece ^ turn)) * 2 + half] = u;
          }
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < 32 / kEach; ++i) {
        const int out_row = i * kEach + lane / kPieces, piece = lane % kPieces;
        const i32x4 u = stage[out_row * 8 + (piece ^ ((out_row >> 1) & 7))];
        const int r_in = row0 + t * 32 + out_row, f = f0 + (kWide ? c * 32 + piece * 4 : piece * 8);
        if (r_in < count && f < a.row_tiles * (GATED ? 16 : 32)) {
          const int64_t to = (a.to_slot ? a.order[first + r_in] : first + r_in) * a.ldy + f;
          if constexpr (kWide)
            *reinterpret_cast<i32x4*>(static_cast<float*>(a.y) + to) = u;
          else
            *reinterpret_cast<i32x4*>(static_cast<unsigned short*>(a.y) + to + (kParts > 1 ? c * a.y_part : 0)) = u;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// Which tile a workgroup has.  Workgroups go to the eight L2s in turn; runs of 32 tiles, one for each of its compute units, stay on one of them
// and share weights between kBand tiles of rows.  (Eighths of the whole grid would leave the last L2 the groups' empty tiles.)
__device__ inline bool place_tile(const Product& a, int row_tiles_each, int* block, int* tile) {
  constexpr int kBand = 4;
  const int row_blocks = (a.row_tiles + row_tiles_each - 1) / row_tiles_each;
  const int id = (((blockIdx.x >> 8) * 8 + (blockIdx.x & 7)) << 5) + ((blockIdx.x >> 3) & 31);
  if (id >= row_blocks * a.max_tiles) return false;
  const int band = id / (row_blocks * kBand), in_band = id - band * row_blocks * kBand;
  const int wide = min(kBand, a.max_tiles - band * kBand);
  *block = in_band / wide;
  *tile = band * kBand + in_band - *block * wide;
  return true;
}

// Memory as the buffer loads see it: a base and offsets below 2^31 bytes; at kNowhere they read zeros.  (Loads by pointer that write LDS
// make the compiler wait for every LDS read under way, these do not; and their addresses cost no vector instructions.)
constexpr int kNowhere = 0x7fffffff;
__device__ inline __amdgpu_buffer_rsrc_t buffer(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, kNowhere, 0x00020000);
}
// Sixteen bytes a lane to LDS, to `to` (the same for the whole wave) + lane.
__device__ inline void to_lds(__amdgpu_buffer_rsrc_t from, int at, int offset, i32x4* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, at, offset, 0, 0);
}

// Nothing may be on its way to LDS when a workgroup gives it back.
__device__ inline void loads_have_ended() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// What is loaded before it is asked for before what is loaded behind it: the counts below rest on the order of the issue, which nothing else holds where
// loads do not depend on each other.
__device__ inline void in_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A barrier behind which the LDS of the whole workgroup may be read and written over: this wave's reads of it have ended, and all its loads
// have arrived but the N issued last.  (__syncthreads would wait for those as well.)
template <int N>
__device__ inline void barrier_but() {
  static_assert(N < 64, "a six-bit counter");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0070);  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- many rows: tiles through LDS ---------------------------------------------------------------------------------
//
// A workgroup computes 32 WT rows by 32 WR WN features (KS: column tiles a step, PI: parts of the rows taken in one step, each with the weights made once).
// Bound by the matrix cores: 4096 x 4096 x 8192 of bf16 in 193 us (1.42 PFLOP/s), their pipes 83 % busy at the clock that power leaves; by the
// weights' bytes where groups are small: 4.2 TB/s in the first product of 200 tokens of 8 of 64 experts of 2048 x 1000.  Rows come in steps of 64 KS columns, 128 KS bytes of each
// row in one stretch, straight to one of two LDS buffers while the other is multiplied; weights come straight
// from memory to the registers that use them, a step ahead, once for all parts of the rows.  A row's 16-byte pieces are permuted in LDS
// (by turn_of, exclusive or) so that the sixteen lanes that an LDS read serves at once touch all 64 banks.
template <int KS>
__device__ inline int turn_of(int row) { return KS == 1 ? (row >> 1) & 7 : row & 15; }

template <int WT, int WR, int WN, int KS, int PI, bool HALF, int OUT, bool GATED>
__global__ __launch_bounds__(64 * WN, 2) void tile_kernel(Product a) {
  constexpr int kRows = 32 * WT, kThreads = 64 * WN, kPieces = 8 * KS, kLoads = kRows * kPieces / kThreads;
  static_assert(kThreads / kPieces % 16 == 0, "a thread's pieces lie in the same columns");
  constexpr int kBuffer = PI * kRows * kPieces;
  __shared__ i32x4 lds0[kBuffer], lds1[kBuffer], stage[WN][256];  // (two arrays, so that the compiler can tell a load to one from reads of the other)
  auto buffer_of = [&](int i) -> i32x4* { return i ? lds1 : lds0; };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int block, tile;
  if (!place_tile(a, WR * WN, &block, &tile)) return;
  int expert, first, count;
  if (!find_tile(a, tile, kRows, &expert, &first, &count)) return;

  const int column = ((threadIdx.x % kPieces) ^ turn_of<KS>(threadIdx.x / kPieces)) * 8;
  __amdgpu_buffer_rsrc_t codes[WR], scales[WR];
#pragma unroll
  for (int r = 0; r < WR; ++r) {
    const int64_t t = (int64_t)expert * a.row_tiles + min((block * WN + wave) * WR + r, a.row_tiles - 1);
    codes[r] = buffer(a.codes + t * a.col_tiles * 64);
    scales[r] = buffer(a.scales + t * a.col_tiles * 64);
  }

  f32x16 acc[WT][WR];
#pragma unroll
  for (int t = 0; t < WT; ++t)
#pragma unroll
    for (int r = 0; r < WR; ++r) acc[t][r] = f32x16{};

  // Steps alternate between two LDS buffers and two sets of registers for weights, so that nothing is copied.
  i32x4 w[2][WR][KS];
  unsigned s[2][WR];
  int w_step = 0, x_col = 0, x_part = 0, w_col = 0;
  auto fetch_weights = [&](int set) {  // past the last step that one's again
    const int c0 = min(w_col, a.col_tiles - KS);
#pragma unroll
    for (int r = 0; r < WR; ++r) {
#pragma unroll
      for (int c = 0; c < KS; ++c) w[set][r][c] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(codes[r], lane * 16, (c0 + c) * 1024, 0));
      if constexpr (KS == 1)
        s[set][r] = __builtin_amdgcn_raw_buffer_load_b8(scales[r], lane * 2, (c0 >> 1) * 128 + (c0 & 1), 0);
      else
        s[set][r] = __builtin_amdgcn_raw_buffer_load_b16(scales[r], lane * 2, c0 * 64, 0);
    }
    w_step += PI;
    if (w_step == a.parts) w_step = 0, w_col += KS;
  };
  fetch_weights(0);  // on their way while the tile's rows are looked up
  fetch_weights(1);
  in_order();

  const __amdgpu_buffer_rsrc_t rows = buffer(static_cast<const __bf16*>(a.x) + (a.from_div ? 0 : first * a.ldx));
  int from[kLoads];  // bytes
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int p = min((int)(i * kThreads + threadIdx.x) / kPieces, count - 1);
    from[i] = (a.from_div ? a.order[first + p] / a.from_div : p) * (int)a.ldx * 2 + column * 2;
  }
  auto fetch_rows = [&](int set) {  // straight to LDS; zeros past a row's end, and past the last step, where nobody reads them (the barriers count them)
    const bool in = x_col * 64 + column < a.k8;
#pragma unroll
    for (int p = 0; p < PI; ++p)
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        to_lds(rows, in ? from[i] : kNowhere, (x_part + p) * (int)a.part * 2 + x_col * 128, buffer_of(set) + (p * kLoads + i) * kThreads + wave * 64);
    x_part += PI;
    if (x_part == a.parts) x_part = 0, x_col += KS;
  };
  constexpr int kWeightLoads = WR * (KS + 1), kRowLoads = PI * kLoads;

  const int steps = a.col_tiles / KS * (a.parts / PI);
  const int row_in = lane & 31, turn = turn_of<KS>(row_in), half = lane >> 5;
  constexpr int kRounds = 4 * KS * PI, kProducts = WT * WR, kPairs = 4 * WR;
  i32x4 xs[2][WT], ws[2][WR];
  auto read = [&](int buffer, int round) {  // the rows' share in a round of a step's products: PI parts of the same columns after another
    const int j = round / PI, p = round % PI;
    const i32x4* in = buffer_of(buffer) + (p * kRows + row_in) * kPieces + (((j >> 2) * 8 + half * 4 + (j & 3)) ^ turn);
#pragma unroll
    for (int t = 0; t < WT; ++t) xs[round & 1][t] = in[t * 32 * kPieces];
  };
  auto convert = [&](int set, int j, int i) {  // (the sign bit of a scale is not looked at)
    const float scale = __uint_as_float((s[set][i >> 2] >> (8 * (j >> 2))) << 23);
    ws[j & 1][i >> 2][i & 3] = pair_of<HALF>(w[set][i >> 2][j >> 2][j & 3], scale, i & 3);
  };
  // The weights' pairs of the next round are made between the products of this one.  A step's last round runs behind the barrier, while the
  // next step's first reads are under way.  All reads of a buffer have ended when its step's barrier is passed: the rows of the step after
  // the next are asked for there, and with that step's weights have a step to arrive.  Loads arrive in the order of their issue, so the barrier
  // lets the weights be that were asked for last.  (Three and four buffers, for one workgroup alone some 15 % faster, leave room for fewer: 79 us
  // instead of 69 on 200 tokens of 8 of 64 experts, 198 instead of 193 on 4096 x 4096 x 8192.)
  auto multiply = [&](int set) {
    const int next = set ^ 1;
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
      const bool last = round + 1 == kRounds;
      const int j = round / PI;
      if (last) {
        fetch_weights(set);
        barrier_but<kWeightLoads>();  // the rows of the next step are there
        fetch_rows(set);
      }
      read(last ? next : set, last ? 0 : round + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        const int t = i / WR, r = i % WR;
        acc[t][r] = product32<HALF>(ws[j & 1][r], xs[round & 1][t], acc[t][r]);
        if (round % PI == PI - 1) {
#pragma unroll
          for (int c = i * kPairs / kProducts; c < (i + 1) * kPairs / kProducts; ++c) convert(last ? next : set, last ? 0 : j + 1, c);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  fetch_rows(0);
  in_order();
  fetch_rows(1);
  in_order();
  barrier_but<kRowLoads>();
  read(0, 0);
#pragma unroll
  for (int c = 0; c < kPairs; ++c) convert(0, 0, c);
  for (int step = 0; step + 1 < steps; step += 2) {
    multiply(0);
    multiply(1);
  }
  if (steps & 1) multiply(0);
  put_tile<WT, OUT, GATED>(a, acc, 0, first, count, (block * WN + wave) * WR, stage[wave]);
  loads_have_ended();
}

// The same for rows that are in MX4 as well, in the weights' layout (csrc/mx4.h): products of 4-bit numbers with both blocks' scales
// applied by the matrix cores, four times the rate of bf16.  8192^3 in 262 us behind 41 for the rows' quantisation (4.2 PFLOP/s), pipes 57 % busy: for each 128
// columns a CU loads 48 KiB, some 750 cycles, beside 1024 of products; and every third step waits for all loads under way, as the scales, loaded in 16 bits,
// are widened to 32 behind the last of them.  Rows come in steps of 128 columns through LDS, as they lie; a wave's
// reads of it are one contiguous kilobyte.
template <int WT, int WR, int WM, int WN, int OUT>
__global__ __launch_bounds__(64 * WM * WN) void rounded_kernel(Product a) {
  constexpr int D = 3;  // LDS buffers and sets of registers; with two of them 8192^3 takes 2 % longer
  constexpr int kTiles = WT * WM, kThreads = 64 * WM * WN, kLoads = kTiles * 128 / kThreads;
  __shared__ i32x4 lds0[kTiles * 128], lds1[kTiles * 128], lds2[kTiles * 128], stage[WM * WN][256];
  auto buffer_of = [&](int i) -> i32x4* { return i == 0 ? lds0 : i == 1 ? lds1 : lds2; };  // (i is a constant where this is used)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  int block, tile;
  if (!place_tile(a, WR * WN, &block, &tile)) return;
  const int first = tile * kTiles * 32, count = min(kTiles * 32, a.rows - first);
  const int last = (a.rows - 1) >> 5, tile0 = first >> 5;

  const __amdgpu_buffer_rsrc_t rows = buffer(static_cast<const i32x4*>(a.x) + (int64_t)tile0 * a.col_tiles * 64);
  int from[kLoads];  // bytes
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int q = i * kThreads + threadIdx.x;
    from[i] = min(q >> 7, last - tile0) * a.col_tiles * 1024 + (q & 127) * 16;
  }
  __amdgpu_buffer_rsrc_t codes[WR], scales[WR], x_scales[WT];
#pragma unroll
  for (int t = 0; t < WT; ++t) x_scales[t] = buffer(a.x_scales + (int64_t)min(tile0 + wm * WT + t, last) * a.col_tiles * 64);
#pragma unroll
  for (int r = 0; r < WR; ++r) {
    const int64_t t = min((block * WN + wn) * WR + r, a.row_tiles - 1);
    codes[r] = buffer(a.codes + t * a.col_tiles * 64);
    scales[r] = buffer(a.scales + t * a.col_tiles * 64);
  }
  f32x16 acc[WT][WR];
#pragma unroll
  for (int t = 0; t < WT; ++t)
#pragma unroll
    for (int r = 0; r < WR; ++r) acc[t][r] = f32x16{};

  const int steps = a.col_tiles >> 1;
  i32x4 w[D][WR][2], xs[2][WT];
  int w_scale[D][WR], x_scale[D][WT];
  int row_step = 0, weight_step = 0;
  auto fetch_rows = [&](int set) {  // past the last step that one again, into a buffer that nobody reads
    const int at = min(row_step++, steps - 1) * 2048;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) to_lds(rows, from[i], at, buffer_of(set) + i * kThreads + wave * 64);
  };
  auto fetch_weights = [&](int set) {  // past the last step that one's again
    const int at = min(weight_step++, steps - 1) * 2048;
#pragma unroll
    for (int r = 0; r < WR; ++r) {
      w[set][r][0] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(codes[r], lane * 16, at, 0));
      w[set][r][1] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(codes[r], lane * 16, at + 1024, 0));
      w_scale[set][r] = __builtin_amdgcn_raw_buffer_load_b16(scales[r], lane * 2, at >> 4, 0);
    }
#pragma unroll
    for (int t = 0; t < WT; ++t) x_scale[set][t] = __builtin_amdgcn_raw_buffer_load_b16(x_scales[t], lane * 2, at >> 4, 0);
  };
  constexpr int kWeightLoads = WR * 3 + WT;
  auto wide = [](i32x4 v) { return i32x8{v.x, v.y, v.z, v.w, 0, 0, 0, 0}; };
  auto read = [&](int buffer, int j) {
    const i32x4* in = buffer_of(buffer) + wm * WT * 128 + lane + j * 64;
#pragma unroll
    for (int t = 0; t < WT; ++t) xs[j][t] = in[t * 128];
  };
  // as in tile_kernel, with two rounds of products a step
  auto multiply = [&](int set) {
    const int next = set + 1 == D ? 0 : set + 1;
    read(set, 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < WT; ++t)
#pragma unroll
      for (int r = 0; r < WR; ++r)
        acc[t][r] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(w[set][r][0]), wide(xs[0][t]), acc[t][r], 4, 4, 0, w_scale[set][r], 0, x_scale[set][t]);
    __builtin_amdgcn_sched_barrier(0);
    barrier_but<(D - 2) * kLoads + (D - 1) * kWeightLoads>();
    fetch_rows(set);
    read(next, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < WT; ++t)
#pragma unroll
      for (int r = 0; r < WR; ++r)
        acc[t][r] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(w[set][r][1]), wide(xs[1][t]), acc[t][r], 4, 4, 1, w_scale[set][r], 1, x_scale[set][t]);
    __builtin_amdgcn_sched_barrier(0);
    fetch_weights(set);
  };
#pragma unroll
  for (int i = 0; i < D; ++i) {
    fetch_rows(i);
    in_order();
    fetch_weights(i);
    in_order();
  }
  barrier_but<(D - 1) * kLoads + D * kWeightLoads>();
  read(0, 0);
  int step = 0;
  for (; step + D <= steps; step += D) {
#pragma unroll
    for (int i = 0; i < D; ++i) multiply(i);
  }
#pragma unroll
  for (int i = 0; i < D - 1; ++i)
    if (step + i < steps) multiply(i);
  put_tile<WT, OUT, false>(a, acc, wm * WT * 32, first, count, (block * WN + wn) * WR, stage[wave]);
  loads_have_ended();
}

// ---- few rows: weights streamed once -----------------------------------------------------------------------------------
//
// A workgroup computes 16 RT features for up to 16 rows; its waves take turns at stretches of 128 columns and add their sums
// in LDS at the end, in the order of the waves.  Bound by the weights' bytes and, for small matrices, by the latency of one pass through the
// memory: a lane loads 16 bytes of codes, whose 32 weights feed four 16 x 16 x 32 products, and the rows' numbers come from the
// caches, split into parts in registers.  4096 weights for each of 4096 features and one row: 4.3 us (2.1 TB/s); 16384 features 8.8 us as a
// call (4 TB/s).  Two stretches a wave under way: more of them is more code to fetch than it hides.

template <int TYPE>
constexpr int kPartsOf = TYPE == TETRIS_F32 ? 3 : TYPE == TETRIS_F16 ? 2 : 1;

// Eight numbers of a row, as they lie, and as parts.
template <int TYPE>
struct Eight {
  i32x4 raw[TYPE == TETRIS_F32 ? 2 : 1];
  __device__ inline void load(const typename Elem<TYPE>::type* p, bool in) {
#pragma unroll
    for (int i = 0; i < (TYPE == TETRIS_F32 ? 2 : 1); ++i) raw[i] = in ? reinterpret_cast<const i32x4*>(p)[i] : i32x4{0, 0, 0, 0};
  }
  // Parts by truncation.  What is left of an infinity is NaN here, where it has to be nothing: lanes that hold one take the longer way.
  __device__ inline void split(bf16x8 (&out)[kPartsOf<TYPE>]) const {
    if constexpr (TYPE == TETRIS_BF16) {
      out[0] = __builtin_bit_cast(bf16x8, raw[0]);
    } else {
      float v[8];
      if constexpr (TYPE == TETRIS_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __int_as_float(raw[i >> 2][i & 3]);
      } else {
        typedef _Float16 half8 __attribute__((ext_vector_type(8)));
        const half8 u = __builtin_bit_cast(half8, raw[0]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)u[i];
      }
      float most = fabsf(v[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
      i32x4 o[kPartsOf<TYPE>];
      if (most == __builtin_inff()) {
#pragma unroll
        for (int q = 0; q < kPartsOf<TYPE>; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned lo = leading(v[2 * i]), hi = leading(v[2 * i + 1]);
            o[q][i] = (int)(lo | hi << 16);
          }
      } else {
#pragma unroll
        for (int q = 0; q < kPartsOf<TYPE>; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned lo = __float_as_uint(v[2 * i]), hi = __float_as_uint(v[2 * i + 1]);
            o[q][i] = (int)__builtin_amdgcn_perm(hi, lo, 0x07060302);  // the upper halves
            v[2 * i] -= __uint_as_float(lo & 0xffff0000u);
            v[2 * i + 1] -= __uint_as_float(hi & 0xffff0000u);
          }
      }
#pragma unroll
      for (int q = 0; q < kPartsOf<TYPE>; ++q) out[q] = __builtin_bit_cast(bf16x8, o[q]);
    }
  }
};

// The products of U stretches of 128 columns, c, c + step, ...: all of their loads first.
template <int TYPE, int RT, int U>
__device__ inline void stretch(const typename Elem<TYPE>::type* from, bool have, const i32x4* const (&codes)[RT], const uint8_t* const (&scales)[RT],
                               int c, int step, int end, int column, int k8, f32x4 (&acc)[RT]) {
  i32x4 w[U][RT];
  unsigned s[U][RT];
  Eight<TYPE> x[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = min(c + u * step, end - 1);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      w[u][r] = codes[r][(int64_t)at * 128];
      s[u][r] = scales[r][(int64_t)at * 128];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x[u][j].load(from + at * 128 + j * 8, have && c + u * step < end && at * 128 + column + j * 8 < k8);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 xs[kPartsOf<TYPE>];
      x[u][j].split(xs);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const bf16x8 ws = weights8(w[u][r][j], __uint_as_float(s[u][r] << 23));
#pragma unroll
        for (int q = 0; q < kPartsOf<TYPE>; ++q) acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ws, xs[q], acc[r], 0, 0, 0);
      }
    }
}

// All stretches c, c + step, ... before end, U at a time while there are as many.
template <int TYPE, int RT, int U>
__device__ inline void stretches(const typename Elem<TYPE>::type* from, bool have, const i32x4* const (&codes)[RT], const uint8_t* const (&scales)[RT],
                                 int c, int step, int end, int column, int k8, f32x4 (&acc)[RT]) {
  for (; c + (U - 1) * step < end; c += U * step) stretch<TYPE, RT, U>(from, have, codes, scales, c, step, end, column, k8, acc);
  if constexpr (U > 1) stretches<TYPE, RT, U / 2>(from, have, codes, scales, c, step, end, column, k8, acc);
}

// Where a lane's codes and scales of 16-row half `half` of an expert's matrix begin.
__device__ inline void half_of(const Product& a, int expert, int half, int lane, const i32x4** codes, const uint8_t** scales) {
  const int r16 = lane & 15, g = lane >> 4;
  const int64_t t = ((int64_t)expert * a.row_tiles + (half >> 1)) * a.col_tiles;
  const int l = (g & 1) * 32 + (half & 1) * 16 + r16;
  *codes = a.codes + (t + (g >> 1)) * 64 + l;
  *scales = a.scales + t * 64 + l * 2 + (g >> 1);
}

template <int TYPE, int RT, int OUT, bool GATED>
__global__ __launch_bounds__(1024) void stream_kernel(Product a) {
  using T = typename Elem<TYPE>::type;
  extern __shared__ float sums[];  // [wave][RT][4][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int halves = a.row_tiles * 2, blocks = (halves + RT - 1) / RT;
  const int tile = blockIdx.x / blocks, block = blockIdx.x - tile * blocks;
  int expert, first, count, my_row, my_slot;  // of the lane's row of the tile
  if (!find_rows(a, tile, &expert, &first, &count, &my_row, &my_slot)) return;

  const int r16 = lane & 15, g = lane >> 4;
  const T* from = static_cast<const T*>(a.x) + (int64_t)my_row * a.ldx + 32 * g;
  const i32x4* codes[RT];
  const uint8_t* scales[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) half_of(a, expert, min(block * RT + r, halves - 1), lane, &codes[r], &scales[r]);
  f32x4 acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int chunks = a.col_tiles >> 1;
  stretches<TYPE, RT, TYPE == TETRIS_F32 ? 1 : 2>(from, r16 < count, codes, scales, wave, waves, chunks, 32 * g, a.k8, acc);
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[((wave * RT + r) * 4 + i) * 64 + lane] = acc[r][i];
  __syncthreads();

  const int n = GATED ? a.n / 2 : a.n;
  auto sum = [&](int r, int row, int f) {
    const int at = (r * 4 + (f & 3)) * 64 + (f >> 2) * 16 + row;
    float v = 0.f;
    for (int w = 0; w < waves; ++w) v += sums[w * (RT * 256) + at];
    return v;
  };
  constexpr int kWidth = GATED ? 16 : 16 * RT;
  for (int i = threadIdx.x; i < 16 * kWidth; i += blockDim.x) {  // (whole waves: the rows' numbers are passed between lanes)
    const int row = i / kWidth, f = i % kWidth, feature = block * kWidth + f;
    const int to = __shfl(my_slot, row);
    if (row >= count) continue;
    if constexpr (GATED) {
      static_assert(RT == 2, "a gate's rows and what they gate");
      store1<OUT>(a, (int64_t)to * a.ldy + feature, feature < n ? silu(sum(0, row, f)) * sum(1, row, f) : 0.f);
    } else if (feature < n) {
      store1<OUT>(a, (int64_t)to * a.ldy + feature, sum(f >> 4, row, f & 15) + (a.bias ? a.bias[feature] : 0.f));
    }
  }
}

// The second product of the experts for up to 64 slots in all, and the weighted sum of each token's.  A workgroup has 16 features and goes
// through every expert that is named; its waves share (expert, stretch of columns) pairs evenly, in runs of neighbouring ones.  A wave's sums for one
// expert are kept at place (number of the expert + number of the wave): along the runs each step raises one of the two, so
// no two share a place.  Bound by latency: the slots, then weights, then the sums; 9.7 us for four tokens of 4 of 64 experts of 1024 x 2048
// (16 MB of codes and scales).  Each output is then added up by one thread, slots in their order, waves in theirs.
//
// Rows of an operator of 16 bits come as two bf16 parts, in two arrays: eight slots' leading parts are columns 0 to 7 of the products, what they leave is
// columns 8 to 15, as few experts have more than eight of 64 slots.  So the numbers between the two products are off by 2^-14 at most, at the price of one
// part (for both products, before slots were found by bits, 19.8 us; 19.4 with one, rounded to bf16; 22.4 with two parts in a lane, 28.0 with 32 bits split here).  With them rounded
// to bf16, one token of 5 experts of 64 numbers each was off by 0.0026; 0.0017 is the rounding of the output itself.
template <int OUT>
__global__ __launch_bounds__(1024) void down_kernel(Product a, const float* __restrict__ weight, int top) {
  constexpr int TYPE = OUT == kOutF32 ? TETRIS_F32 : TETRIS_BF16;
  constexpr int kSlots = OUT == kOutF32 ? 16 : 8;  // in a tile
  using T = typename Elem<TYPE>::type;
  extern __shared__ float sums[];  // [places][4][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r16 = lane & 15, g = lane >> 4, block = blockIdx.x;
  const int mine = lane < a.rows ? a.index[lane] : -1;
  const bool named = mine >= 0 && mine < a.experts;
  const float my_weight = lane < a.rows ? weight[lane] : 0.f;
  // Tiles of up to kSlots slots of one expert, numbered by their first slots; a lane knows its slot's tile and place in it.  Which slots name the same expert
  // is found a bit of its number at a time (a loop over the experts named took 1.1 us more of sixteen slots of as many experts).
  unsigned long long same = __ballot(named);
  for (int bit = 0; (1 << bit) < a.experts; ++bit) {
    const bool set = mine >> bit & 1;
    const unsigned long long those = __ballot(set);
    same &= set ? those : ~those;
  }
  const int rank = __builtin_popcountll(same & ((1ull << lane) - 1)), my_column = rank % kSlots;
  const unsigned long long starts = __ballot(named && my_column == 0);
  const int tiles = __builtin_popcountll(starts);
  const int number = __builtin_popcountll(starts & ((1ull << lane) - 1));  // of the tile that starts here
  unsigned long long from_mine = same;
  for (int i = rank - my_column; i > 0; --i) from_mine &= from_mine - 1;
  const int its = __shfl(number, __builtin_ctzll(from_mine | 1ull << 63));
  const int my_tile = named ? its : -1;
  // lane t: the expert of tile t (lane 63 takes what starts no tile, unless every lane starts one)
  const int expert_of = __builtin_amdgcn_ds_permute((named && my_column == 0 ? number : 63) * 4, mine);
  const int chunks = a.col_tiles >> 1, items = tiles * chunks, each = (items + waves - 1) / waves;
  const int begin = min(wave * each, items), end = min(begin + each, items);
  for (int at = begin; at < end;) {
    const int tile = at / chunks, c0 = at - tile * chunks, c1 = min(chunks, c0 + end - at);
    const int expert = __builtin_amdgcn_readlane(expert_of, tile);
    const unsigned long long in = __ballot(my_tile == tile);
    const int count = __builtin_popcountll(in);
    // lane with column q of the tile -> every lane with r16 % kSlots == q
    const int slot = __builtin_amdgcn_ds_permute((my_tile == tile ? my_column : 63) * 4, lane);
    const int row = __shfl(slot, min(r16 % kSlots, count - 1));
    const T* from = static_cast<const T*>(a.x) + (r16 / kSlots) * a.part + (int64_t)row * a.ldx + 32 * g;
    const i32x4* codes[1];
    const uint8_t* scales[1];
    half_of(a, expert, block, lane, &codes[0], &scales[0]);
    f32x4 acc[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
    stretches<TYPE, 1, 2>(from, r16 % kSlots < count, codes, scales, c0, 1, c1, 32 * g, a.k8, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[((tile + wave) * 4 + i) * 64 + lane] = acc[0][i];
    at += c1 - c0;
  }
  __syncthreads();
  const int tokens = a.rows / top;
  for (int i = threadIdx.x; i < ((tokens * 16 + 63) & ~63); i += blockDim.x) {
    const int token = i >> 4, f = i & 15, feature = block * 16 + f;
    float y = 0.f;
    for (int j = 0; j < top; ++j) {
      const int slot = token * top + j;
      const int tile = __shfl(my_tile, slot & 63), column = __shfl(my_column, slot & 63);
      const float by = __shfl(my_weight, slot & 63);
      if (token >= tokens || tile < 0) continue;
      float v = 0.f;
      for (int w = tile * chunks / each; w <= ((tile + 1) * chunks - 1) / each; ++w)
#pragma unroll
        for (int p = 0; p < 16; p += kSlots) v += sums[((tile + w) * 4 + (f & 3)) * 64 + (f >> 2) * 16 + p + column];
      y = fmaf(by, v, y);
    }
    if (token < tokens && feature < a.n) store1<OUT>(a, (int64_t)token * a.ldy + feature, y);
  }
}

// ---- routed rows ---------------------------------------------------------------------------------------------------------

// Slots (token, j) in the order of their experts, those of one expert in the order of the slots.  Workgroup e finds expert e's: it
// counts the slots of lower experts, which is where its own begin, and the matches in each wave's stretch of the slots,
// then goes through them again and writes.  16384 slots of 32 experts: 11.9 us, 1600 of 64: 4.7, both latency.  Slots of no expert are in no group.  No atomics: the order is always the same.
__global__ __launch_bounds__(1024) void plan_kernel(const int* __restrict__ index, int slots, int experts, int* __restrict__ offsets,
                                                    int* __restrict__ order) {
  __shared__ int lower_of[16], match_of[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, e = blockIdx.x;
  const int stretch = ((slots + waves - 1) / waves + 63) & ~63;
  const int begin = min(wave * stretch, slots), end = min(begin + stretch, slots);
  int lower = 0, match = 0;
  for (int i = begin + lane; i < end; i += 64) {
    const int v = index[i];
    lower += v >= 0 && v < e;
    match += v == e;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    lower += __shfl_xor(lower, d);
    match += __shfl_xor(match, d);
  }
  if (lane == 0) lower_of[wave] = lower, match_of[wave] = match;
  __syncthreads();
  int at = 0, all = 0;
  for (int w = 0; w < waves; ++w) {
    at += lower_of[w] + (w < wave ? match_of[w] : 0);
    all += lower_of[w] + match_of[w];
  }
  if (threadIdx.x == 0) {
    if (e == 0) offsets[0] = 0;
    offsets[e + 1] = all;
  }
  for (int i = begin; i < end; i += 64) {
    const bool mine = i + lane < end && index[i + lane] == e;
    const unsigned long long found = __ballot(mine);
    if (mine) order[at + __builtin_popcountll(found & ((1ull << lane) - 1))] = i + lane;
    at += __builtin_popcountll(found);
  }
}

// y[t] = sum over j of weight[t][j] rows[t top + j], four columns a thread; bound by the rows' bytes: 4096 tokens of
// four rows of 4096 in 46.4 us (302 MB, 6.5 TB/s, half of the rows still in the last-level cache).
template <int TYPE>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ rows, int64_t ld_rows, const int* __restrict__ index,
                                                      const float* __restrict__ weight, int tokens, int top, int experts, int width,
                                                      typename Elem<TYPE>::type* __restrict__ y, int64_t ldy, int vec) {
  using T = typename Elem<TYPE>::type;
  const int quads = (width + 3) / 4;
  const int64_t total = (int64_t)tokens * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / quads;
    const int c = (int)(i - t * quads) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < top; j0 += 4) {  // four rows under way; those of no expert were never written and count for nothing
      f32x4 r[4];
      float w[4];
      bool in[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t slot = t * top + min(j0 + q, top - 1);
        const int e = index[slot];
        in[q] = j0 + q < top && e >= 0 && e < experts;
        w[q] = weight[slot];
        r[q] = *reinterpret_cast<const f32x4*>(rows + slot * ld_rows + c);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = in[q] ? fmaf(w[q], r[q][i], v[i]) : v[i];
    }
    T* out = y + t * ldy + c;
    if (vec && c + 4 <= width) {
      typedef T T4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<T4*>(out) = T4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
      for (int q = 0; q < 4 && c + q < width; ++q) out[q] = (T)v[q];
    }
  }
}

// ---- launches ------------------------------------------------------------------------------------------------------------

// Waves that share a row of `chunks` stretches of 128 columns.
int stream_waves(int chunks, int64_t workgroups) {
  int waves = workgroups <= 512 ? 16 : 4;
  while (waves > 1 && waves > chunks) waves >>= 1;
  return waves;
}

template <int WT, int WR, int WN, int KS, int PI, bool HALF, int OUT, bool GATED>
int launch_tile(Product& a, hipStream_t stream) {
  const int size = 32 * WT, row_blocks = ceil_div(a.row_tiles, WR * WN);
  a.max_tiles = a.offsets ? std::min(a.rows, a.rows / size + std::min(a.experts, a.rows)) : ceil_div(a.rows, size);
  const int64_t blocks = round_up((int64_t)row_blocks * a.max_tiles, 256);
  if (blocks > 0x7fffffff / 2) return fail(TETRIS_EINVAL, "%d rows by %d features are too many for one launch", a.rows, a.n);
  hipLaunchKernelGGL((tile_kernel<WT, WR, WN, KS, PI, HALF, OUT, GATED>), dim3((unsigned)blocks), dim3(64 * WN), 0, stream, a);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

template <int WT, int WR, int WM, int WN, int OUT>
int launch_rounded(Product& a, hipStream_t stream) {
  a.max_tiles = ceil_div(a.rows, 32 * WT * WM);
  const int64_t blocks = round_up((int64_t)ceil_div(a.row_tiles, WR * WN) * a.max_tiles, 256);
  if (blocks > 0x7fffffff / 2) return fail(TETRIS_EINVAL, "%d rows by %d features are too many for one launch", a.rows, a.n);
  hipLaunchKernelGGL((rounded_kernel<WT, WR, WM, WN, OUT>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, stream, a);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

// The rows of `a` are of TYPE.
template <int TYPE, int OUT, bool GATED>
int launch_stream(Product& a, hipStream_t stream) {
  constexpr int RT = GATED ? 2 : 1;
  const int blocks = ceil_div(a.row_tiles * 2, RT);
  a.max_tiles = a.index ? a.rows : a.offsets ? std::min(a.rows, a.rows / 16 + std::min(a.experts, a.rows)) : ceil_div(a.rows, 16);
  const int64_t grid = (int64_t)blocks * a.max_tiles;
  if (grid > 0x7fffffff / 2) return fail(TETRIS_EINVAL, "%d rows by %d features are too many for one launch", a.rows, a.n);
  const int waves = stream_waves(a.col_tiles / 2, grid);
  hipLaunchKernelGGL((stream_kernel<TYPE, RT, OUT, GATED>), dim3((unsigned)grid), dim3(64 * waves), (size_t)waves * RT * 1024, stream, a);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

template <int TYPE>
int launch_down(Product& a, const float* weight, int top, hipStream_t stream) {
  const int waves = 16;
  const size_t lds = (size_t)(std::min(a.rows, a.rows / (TYPE == TETRIS_F32 ? 16 : 8) + a.experts) + waves) * 1024;  // at most 80 KiB
  static const hipError_t room = hipFuncSetAttribute(reinterpret_cast<const void*>(down_kernel<TYPE>), hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024);
  TETRIS_HIP(room);
  hipLaunchKernelGGL((down_kernel<TYPE>), dim3(ceil_div(a.n, 16)), dim3(64 * waves), lds, stream, a, weight, top);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

// Tiles of `size` rows that the groups make: one half more each than their mean number of rows fills.
double tiles_of(const Product& a, int size) {
  if (!a.offsets && !a.index) return ceil_div(a.rows, size);
  const double named = std::min(a.experts, a.rows), mean = a.rows / named;
  return mean <= size / 2 ? named : named * (mean / size + 0.5);
}
// What a product takes in tiles of `size` rows, in units of what a workgroup of 32 rows takes; a workgroup has 256 features, and each of the 256 compute
// units needs one at a time to be full.  Measured, 4096 columns of bf16: 18, 27 and 51 us a workgroup of 32, 64 and 128 rows.
double tile_cost(const Product& a, int size) {
  const double each = size == 32 ? 1.0 : size == 64 ? 1.55 : 2.9;
  return each * std::max(1.0, tiles_of(a, size) * ceil_div(a.row_tiles, 8) / 256);
}
// The same for streaming, whose workgroups have up to 16 rows and 16 features (a gated product 32, for a third more): 4 us, and for each 256 of them 1.2 us
// with one row to 3.8 with sixteen.
double stream_cost(const Product& a, bool gated) {
  const bool groups = a.offsets || a.index;
  const double rows = std::min(16.0, groups ? (double)a.rows / std::min(a.experts, a.rows) : (double)a.rows);
  return 0.2 + (0.06 + 0.0095 * rows) * (gated ? 0.65 : 1.0) * tiles_of(a, 16) * a.row_tiles * 2 / 256;
}

// P: the rows' parts.  HALF: rows and weights in f16.
template <int OUT, bool GATED, int P, bool HALF = false>
int tile_rows(Product& a, hipStream_t stream) {
  const double small = tile_cost(a, 32), middle = tile_cost(a, 64), large = tile_cost(a, 128);
  if (small <= middle && small <= large) return launch_tile<1, 2, 4, P == 3 ? 1 : 2, P, HALF, OUT, GATED>(a, stream);
  if (middle < large) return launch_tile<2, 2, 4, P == 2 ? 1 : 2, P == 2 ? 2 : 1, HALF, OUT, GATED>(a, stream);
  return launch_tile<4, 2, 4, 1, 1, HALF, OUT, GATED>(a, stream);
}

void set_weights(Product* a, const tetris_mx4* w) {
  a->codes = reinterpret_cast<const i32x4*>(w->codes);
  a->scales = w->scales;
  a->row_tiles = w->row_tiles;
  a->col_tiles = w->col_tiles;
  a->n = w->n;
}

// Whether the kernels can read rows as they lie.
bool lies_well(const void* x, int64_t ld, int k, int type) {
  return (reinterpret_cast<size_t>(x) & 15) == 0 && (ld * elem_size(type)) % 16 == 0 && k % 8 == 0 && ld <= kMxSide;
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// A number of the calling thread, never given to another one.
uint64_t thread_number() {
  static std::atomic<uint64_t> threads{0};
  static thread_local const uint64_t mine = ++threads;
  return mine;
}

// The workspace of (handle, stream), at least `need` bytes.  A buffer that has to grow is replaced and kept until the handle goes: a
// captured graph may hold its address.  It at least doubles, so that those kept are together no larger than the last one.
int workspace(tetris_mx4* w, hipStream_t stream, size_t need, uint8_t** out) {
  *out = nullptr;
  if (!need) return TETRIS_OK;
  try {
    std::lock_guard<std::mutex> lock(w->mu);
    tetris_mx4::Space& s = w->space[{stream, stream == hipStreamPerThread ? thread_number() : 0}];
    if (s.bytes < need) {
      hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
      if (hipStreamIsCapturing(stream, &cap) == hipSuccess && cap != hipStreamCaptureStatusNone)
        return fail(TETRIS_EINVAL, "this launch would allocate its workspace: prepare it before capturing");
      w->retired.reserve(w->retired.size() + 1);
      void* d = nullptr;
      size_t bytes = std::max(need, 2 * s.bytes);
      if (bytes > need && hipMalloc(&d, bytes) != hipSuccess) {
        (void)hipGetLastError();  // no room for twice as much
        d = nullptr;
      }
      if (!d) TETRIS_HIP(hipMalloc(&d, bytes = need));
      if (s.ptr) w->retired.push_back(s.ptr);
      s.ptr = d;
      s.bytes = bytes;
    }
    *out = static_cast<uint8_t*>(s.ptr);
    return TETRIS_OK;
  } catch (const std::exception& e) {
    return fail(TETRIS_EINVAL, "%s", e.what());
  }
}

constexpr int kFewSlots = 64;      // the experts' slots that down_kernel takes, a lane each
constexpr int kStreamMost = 1024;  // more rows are not streamed, whatever the matrix

// Whether a product's rows are streamed.  Decided by its sizes alone, so that a workspace can be made ahead.
bool streams(const tetris_mx4* w, int rows) {
  Product a{};
  a.rows = rows;
  a.row_tiles = w->row_tiles;
  return rows <= kStreamMost && stream_cost(a, false) < tile_cost(a, 32);
}
// The experts': of the first product, for both; up to 64 slots always are.
bool streams_slots(const tetris_mx4* up, int tokens, int top) {
  const int64_t slots = (int64_t)tokens * top;
  if (slots <= kFewSlots) return true;
  if (slots > kStreamMost) return false;
  Product a{};
  a.rows = (int)slots;
  a.experts = up->experts;
  a.row_tiles = up->row_tiles;
  static const int some = 0;
  a.offsets = &some;
  return stream_cost(a, true) < tile_cost(a, 32);
}

// Whether rows of `type` are multiplied in f16: where the weights are exact in it.  Others of f16 are taken in two bf16 parts.
bool in_half(int type, const tetris_mx4* w) { return type == TETRIS_F16 && w->half; }

// Whether a product reads them so.
bool as_they_lie(const void* x, int type, int k, int64_t ld, bool rounded, bool stream, bool half) {
  return !rounded && (stream || half || type == TETRIS_BF16) && lies_well(x, ld, k, type);
}

// bytes that rows made ready for a product take at most
size_t staged_bytes(int rows, int k, int type, bool rounded, bool stream, bool half) {
  const size_t padded = (size_t)rows * round_up(k, kMxPad);
  if (rounded) return stream ? padded * 2 : (size_t)round_up(rows, 32) * round_up(k, kMxPad) / 32 * 17;
  return padded * (stream || half ? elem_size(type) : 2 * parts_of(type));
}

// Points `a` at rows x of `type`, made ready in d_ready where they have to be.  *as: the type the product reads.
int ready_rows(Product* a, const void* x, int type, int rows, int k, int64_t ld, bool rounded, bool stream, bool half, uint8_t* d_ready, int* as,
               hipStream_t s) {
  const int64_t padded = round_up(k, kMxPad);
  a->rows = rows;
  a->parts = 1;
  a->part = 0;
  *as = type;
  if (rounded) {
    a->x = d_ready;
    a->ldx = padded;
    a->k8 = (int)padded;
    *as = TETRIS_BF16;
    if (stream) return mx4_quantize_to(kMxValues, x, type, rows, k, ld, d_ready, nullptr, s);
    uint8_t* scales = d_ready + round_up(rows, 32) * padded / 2;
    a->x_scales = scales;
    return mx4_quantize_to(kMxTiles, x, type, rows, k, ld, d_ready, scales, s);
  }
  if (as_they_lie(x, type, k, ld, rounded, stream, half)) {
    a->x = x;
    a->ldx = ld;
    a->k8 = k;
    return TETRIS_OK;
  }
  a->x = d_ready;
  a->ldx = padded;
  a->k8 = (int)padded;
  if (stream || half || type == TETRIS_BF16) return stage_rows(x, type, rows, k, ld, 0, d_ready, s);
  a->parts = parts_of(type);
  a->part = rows * padded;
  *as = TETRIS_BF16;
  return stage_rows(x, type, rows, k, ld, a->parts, d_ready, s);
}

// Which of the three products it is: numbers of a type; the gated product of the experts, which writes what the next
// reads; and that one, which writes numbers of 32 bits.  Beyond 64 slots what lies between those two is, of f32, all of its 24 bits; of f16, whose range a product
// of two sums may leave, two bf16 parts, or 32 bits where rows are streamed (in f16 200 tokens of 8 of 64 experts take 77 us instead of 84, 4096 of 4 of 16 322
// instead of 405, but a number above 65504 there makes the output infinite or NaN); of bf16, which has the range, bf16: one rounding of 2^-9, where the output's is
// one as well (in two parts 4096 tokens of 4 of 32 experts take 983 us instead of 777).
enum Role { kLinear, kUp, kDown };

// `as`: the type of the rows; `type`: that of the operator.
int launch_product(Product& a, Role role, int as, int type, bool stream, hipStream_t s) {
  if (stream) {
    if (as == TETRIS_F32)
      return role == kUp ? launch_stream<TETRIS_F32, kOutF32, true>(a, s) : launch_stream<TETRIS_F32, kOutF32, false>(a, s);
    if (role == kUp && a.index && type != TETRIS_F32)
      return as == TETRIS_F16 ? launch_stream<TETRIS_F16, kOutParts2, true>(a, s) : launch_stream<TETRIS_BF16, kOutParts2, true>(a, s);
    if (as == TETRIS_F16)
      return role == kUp ? launch_stream<TETRIS_F16, kOutF32, true>(a, s) : launch_stream<TETRIS_F16, kOutF16, false>(a, s);
    if (role == kUp) return launch_stream<TETRIS_BF16, kOutBF16, true>(a, s);
    if (role == kDown || type == TETRIS_F32) return launch_stream<TETRIS_BF16, kOutF32, false>(a, s);
    if (type == TETRIS_F16) return launch_stream<TETRIS_BF16, kOutF16, false>(a, s);
    return launch_stream<TETRIS_BF16, kOutBF16, false>(a, s);
  }
  if (a.x_scales) {
    if (type == TETRIS_F32) return launch_rounded<4, 2, 2, 4, kOutF32>(a, s);
    if (type == TETRIS_F16) return launch_rounded<4, 2, 2, 4, kOutF16>(a, s);
    return launch_rounded<4, 2, 2, 4, kOutBF16>(a, s);
  }
  if (type == TETRIS_F32) return role == kUp ? tile_rows<kOutParts3, true, 3>(a, s) : tile_rows<kOutF32, false, 3>(a, s);
  if (as == TETRIS_F16) return role == kUp ? tile_rows<kOutParts2, true, 1, true>(a, s) : tile_rows<kOutF16, false, 1, true>(a, s);
  if (type == TETRIS_F16)
    return role == kUp     ? tile_rows<kOutParts2, true, 2>(a, s)
           : role == kDown ? tile_rows<kOutF32, false, 2>(a, s)
                           : tile_rows<kOutF16, false, 2>(a, s);
  return role == kUp     ? tile_rows<kOutBF16, true, 1>(a, s)
         : role == kDown ? tile_rows<kOutF32, false, 1>(a, s)
                         : tile_rows<kOutBF16, false, 1>(a, s);
}

int check_rows(const void* x, int type, int rows, int64_t ld, int k, const char* what) {
  if (!x) return fail(TETRIS_EINVAL, "null argument");
  if (ld < k) return fail(TETRIS_EINVAL, "%s: leading dimension %lld below the %d columns", what, (long long)ld, k);
  if (reinterpret_cast<size_t>(x) % elem_size(type)) return fail(TETRIS_EINVAL, "%s not aligned to its elements", what);
  return TETRIS_OK;
}

}  // namespace
}  // namespace tetris

using namespace tetris;

namespace {

// rows of a linear product that a launch takes: those made ready in parts lie within a kernel's reach
int rows_at_once(const tetris_mx4* w, int m, int type, bool rounded) {
  if (rounded || streams(w, m) || parts_of(type) == 1 || in_half(type, w)) return m;
  return (int)std::min<int64_t>(m, kMxReach / (2 * parts_of(type) * round_up(w->k, kMxPad)));
}

int linear_rows(tetris_mx4* w, const void* d_x, int type, int m, int64_t ldx, void* d_y, int64_t ldy, const float* d_bias, bool rounded, hipStream_t s) {
  const bool stream_it = streams(w, m), half = in_half(type, w);
  uint8_t* d = nullptr;
  int rc;
  if (!as_they_lie(d_x, type, w->k, ldx, rounded, stream_it, half) && (rc = workspace(w, s, staged_bytes(m, w->k, type, rounded, stream_it, half), &d))) return rc;
  Product a{};
  set_weights(&a, w);
  int as;
  if ((rc = ready_rows(&a, d_x, type, m, w->k, ldx, rounded, stream_it, half, d, &as, s))) return rc;
  a.y = d_y;
  a.ldy = ldy;
  a.vec_out = ldy * elem_size(type) % 16 == 0 && (reinterpret_cast<size_t>(d_y) & 15) == 0;
  a.bias = d_bias;
  return launch_product(a, kLinear, as, type, stream_it, s);
}

}  // namespace

extern "C" int tetris_mx4_prepare(tetris_mx4* w, int m, int type, int mx4_input, void* stream) {
  if (!w) return fail(TETRIS_EINVAL, "null argument");
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (m < 0) return fail(TETRIS_EINVAL, "%d rows", m);
  uint8_t* d;
  const int rows = rows_at_once(w, m, type, mx4_input);
  const bool half = in_half(type, w);
  // fewer rows may be streamed where these are not, and rounded ones then take more room each
  const size_t need = std::max(staged_bytes(rows, w->k, type, mx4_input, streams(w, m), half), staged_bytes(std::min(m, kStreamMost), w->k, type, mx4_input, true, half));
  return workspace(w, static_cast<hipStream_t>(stream), need, &d);
}

extern "C" int tetris_mx4_linear(tetris_mx4* w, const void* d_x, int type, int m, int64_t ldx, void* d_y, int64_t ldy,
                                 const float* d_bias, int mx4_input, void* stream) {
  if (!w) return fail(TETRIS_EINVAL, "null argument");
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (w->gated || w->experts != 1) return fail(TETRIS_EINVAL, "one matrix that is not gated is needed, these are %d%s", w->experts, w->gated ? ", gated" : "");
  if (m < 0) return fail(TETRIS_EINVAL, "%d rows", m);
  if (m == 0) return TETRIS_OK;
  int rc = check_rows(d_x, type, m, ldx, w->k, "input");
  if (!rc) rc = check_rows(d_y, type, m, ldy, w->n, "output");
  if (rc) return rc;
  if (reinterpret_cast<size_t>(d_bias) & 3) return fail(TETRIS_EINVAL, "bias not aligned to its elements");
  const int each = rows_at_once(w, m, type, mx4_input);
  for (int64_t from = 0; from < m; from += each) {
    rc = linear_rows(w, static_cast<const char*>(d_x) + from * ldx * elem_size(type), type, (int)std::min<int64_t>(each, m - from), ldx,
                     static_cast<char*>(d_y) + from * ldy * elem_size(type), ldy, d_bias, mx4_input != 0, static_cast<hipStream_t>(stream));
    if (rc) return rc;
  }
  return TETRIS_OK;
}

namespace {

struct ExpertSpace {
  size_t offsets, order, hidden, rows, ready, all;
};

ExpertSpace expert_space(const tetris_mx4* up, const tetris_mx4* down, int tokens, int top, int type, bool stream) {
  const size_t slots = (size_t)tokens * top;
  const int between = slots <= kFewSlots || (stream && type == TETRIS_F16) ? 4 : stream ? elem_size(type) : 2 * parts_of(type);
  ExpertSpace e;
  e.offsets = 0;
  e.order = up256(e.offsets + 4 * ((size_t)up->experts + 1));
  e.hidden = up256(e.order + 4 * slots);
  e.rows = up256(e.hidden + slots * round_up(down->k, kMxPad) * between);
  e.ready = up256(e.rows + slots * round_up(down->n, 4) * 4);
  e.all = e.ready + staged_bytes(tokens, up->k, type, false, stream, in_half(type, up));
  return e;
}

int experts_check(const tetris_mx4* up, const tetris_mx4* down, int tokens, int top, int type) {
  if (!up || !down) return fail(TETRIS_EINVAL, "null argument");
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (!up->gated || down->gated || up->experts != down->experts || up->n != 2 * down->k || up->k != down->n)
    return fail(TETRIS_EINVAL, "experts of %d x %d x %d%s and %d x %d x %d%s do not follow each other", up->experts, up->n, up->k,
                up->gated ? " gated" : "", down->experts, down->n, down->k, down->gated ? " gated" : "");
  if (tokens < 0 || top <= 0 || top > 1024 || (int64_t)tokens * top > (1 << 28)) return fail(TETRIS_EINVAL, "%d tokens of %d experts each", tokens, top);
  return TETRIS_OK;
}


}  // namespace

namespace {

// slots whose numbers between the products, all parts of them, lie within a kernel's reach; 341 at least
int64_t slots_at_once(const tetris_mx4* down, int type) { return kMxReach / (round_up(down->k, kMxPad) * 2 * parts_of(type)); }

// tokens that one pass takes: their rows, and those between the products, lie within a kernel's reach (unless one token has too many), and the
// rows before the weighted sum, 4 bytes a number, take no more memory than that
int tokens_at_once(const tetris_mx4* up, const tetris_mx4* down, int tokens, int top, int type, int64_t ldx) {
  const bool half = in_half(type, up);
  const int64_t row = std::max<int64_t>(std::min<int64_t>(ldx, kMxSide) * elem_size(type), round_up(up->k, kMxPad) * (half ? 2 : 2 * parts_of(type)));
  const int64_t sums = top * round_up(down->n, 4) * 4;
  return (int)std::min<int64_t>(tokens, std::max<int64_t>(1, std::min({kMxReach / row, slots_at_once(down, type) / top, kMxReach / sums})));
}

}  // namespace

extern "C" int tetris_experts_prepare(tetris_mx4* up, tetris_mx4* down, int tokens, int top, int type, void* stream) {
  const int rc = experts_check(up, down, tokens, top, type);
  if (rc || tokens == 0) return rc;
  uint8_t* d;
  const int once = tokens_at_once(up, down, tokens, top, type, up->k), few = std::min(once, kFewSlots / top);
  size_t need = expert_space(up, down, once, top, type, streams_slots(up, once, top)).all;
  if (few) need = std::max(need, expert_space(up, down, few, top, type, true).all);  // a few tokens' numbers between the products take more
  return workspace(up, static_cast<hipStream_t>(stream), need, &d);
}

namespace {

// Both products of the slots of `tokens` rows, sorted by expert first: slot i's numbers of 32 bits to row i of `out`.
int expert_products(tetris_mx4* up, tetris_mx4* down, const void* d_x, int type, int tokens, int64_t ldx, int top, const int32_t* d_index,
                    bool stream_it, const ExpertSpace& e, uint8_t* d, float* out, int64_t ld_out, hipStream_t s) {
  int rc;
  const int slots = tokens * top;
  const bool half = in_half(type, up);
  int* offsets = reinterpret_cast<int*>(d + e.offsets);
  int* order = reinterpret_cast<int*>(d + e.order);
  const int threads = std::min(1024, (int)round_up(slots, 64));
  hipLaunchKernelGGL(plan_kernel, dim3(up->experts), dim3(threads), 0, s, d_index, slots, up->experts, offsets, order);
  TETRIS_HIP(hipGetLastError());

  Product a{};
  set_weights(&a, up);
  int as;
  if ((rc = ready_rows(&a, d_x, type, tokens, up->k, ldx, false, stream_it, half, d + e.ready, &as, s))) return rc;
  a.rows = slots;
  a.offsets = offsets;
  a.order = order;
  a.experts = up->experts;
  a.from_div = top;
  a.y = d + e.hidden;
  a.ldy = round_up(down->k, kMxPad);
  a.y_part = (int64_t)slots * a.ldy;
  if ((rc = launch_product(a, kUp, as, type, stream_it, s))) return rc;

  Product b{};
  set_weights(&b, down);
  b.x = d + e.hidden;
  b.ldx = a.ldy;
  b.part = a.y_part;
  b.parts = stream_it ? 1 : parts_of(type);
  b.k8 = (int)round_up(down->k, 8);
  b.rows = slots;
  b.experts = up->experts;
  b.offsets = offsets;
  b.order = order;
  b.to_slot = 1;
  b.y = out;
  b.ldy = ld_out;
  b.vec_out = 1;
  const int between = !stream_it ? TETRIS_BF16 : type == TETRIS_F16 ? TETRIS_F32 : type;
  return launch_product(b, kDown, between, type, stream_it, s);
}

// The same for up to 64 slots: no sorting, two launches, the weighted sum in the second.
int few_slots(tetris_mx4* up, tetris_mx4* down, const void* d_x, int type, int tokens, int64_t ldx, int top, const int32_t* d_index,
              const float* d_weight, void* d_y, int64_t ldy, const ExpertSpace& e, uint8_t* d, hipStream_t s) {
  int rc;
  const int slots = tokens * top;
  Product a{};
  set_weights(&a, up);
  int as;
  if ((rc = ready_rows(&a, d_x, type, tokens, up->k, ldx, false, true, false, d + e.ready, &as, s))) return rc;
  a.rows = slots;
  a.index = d_index;
  a.experts = up->experts;
  a.from_div = top;
  a.y = d + e.hidden;
  a.ldy = round_up(down->k, kMxPad);
  a.y_part = (int64_t)slots * a.ldy;
  if ((rc = launch_product(a, kUp, as, type, true, s))) return rc;

  Product b{};
  set_weights(&b, down);
  b.x = d + e.hidden;
  b.ldx = a.ldy;
  b.part = a.y_part;
  b.parts = 1;
  b.k8 = (int)round_up(down->k, 8);
  b.rows = slots;
  b.experts = up->experts;
  b.index = d_index;
  b.y = d_y;
  b.ldy = ldy;
  return type == TETRIS_F32   ? launch_down<TETRIS_F32>(b, d_weight, top, s)
         : type == TETRIS_F16 ? launch_down<TETRIS_F16>(b, d_weight, top, s)
                              : launch_down<TETRIS_BF16>(b, d_weight, top, s);
}

int expert_tokens(tetris_mx4* up, tetris_mx4* down, const void* d_x, int type, int tokens, int64_t ldx, int top, const int32_t* d_index,
                  const float* d_weight, void* d_y, int64_t ldy, hipStream_t s) {
  int rc;
  const int slots = tokens * top;
  const bool stream_it = streams_slots(up, tokens, top);
  const ExpertSpace e = expert_space(up, down, tokens, top, type, stream_it);
  uint8_t* d;
  if ((rc = workspace(up, s, as_they_lie(d_x, type, up->k, ldx, false, stream_it, in_half(type, up)) ? e.ready : e.all, &d))) return rc;
  if (slots <= kFewSlots) return few_slots(up, down, d_x, type, tokens, ldx, top, d_index, d_weight, d_y, ldy, e, d, s);

  float* rows = reinterpret_cast<float*>(d + e.rows);
  const int64_t ld_rows = round_up(down->n, 4);
  // One token may still have more slots than tile_kernel's 32-bit offsets reach between the products: they are taken in several passes.
  const int each = tokens == 1 && !stream_it ? (int)std::min<int64_t>(top, slots_at_once(down, type)) : top;
  for (int from = 0; from < top; from += each) {
    rc = expert_products(up, down, d_x, type, tokens, ldx, std::min(each, top - from), d_index + from, stream_it, e, d, rows + from * ld_rows, ld_rows, s);
    if (rc) return rc;
  }

  const int vec = ldy % 4 == 0 && (reinterpret_cast<size_t>(d_y) & (4 * elem_size(type) - 1)) == 0;
  const dim3 grid((unsigned)std::min<int64_t>(((int64_t)tokens * ceil_div(down->n, 4) + 255) / 256, 256 * 64));
  if (type == TETRIS_F32)
    hipLaunchKernelGGL(combine_kernel<TETRIS_F32>, grid, dim3(256), 0, s, rows, ld_rows, d_index, d_weight, tokens, top, up->experts, down->n,
                       static_cast<float*>(d_y), ldy, vec);
  else if (type == TETRIS_F16)
    hipLaunchKernelGGL(combine_kernel<TETRIS_F16>, grid, dim3(256), 0, s, rows, ld_rows, d_index, d_weight, tokens, top, up->experts, down->n,
                       static_cast<_Float16*>(d_y), ldy, vec);
  else
    hipLaunchKernelGGL(combine_kernel<TETRIS_BF16>, grid, dim3(256), 0, s, rows, ld_rows, d_index, d_weight, tokens, top, up->experts, down->n,
                       static_cast<__bf16*>(d_y), ldy, vec);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

}  // namespace

extern "C" int tetris_experts(tetris_mx4* up, tetris_mx4* down, const void* d_x, int type, int tokens, int64_t ldx, int top,
                              const int32_t* d_index, const float* d_weight, void* d_y, int64_t ldy, void* stream) {
  int rc = experts_check(up, down, tokens, top, type);
  if (rc) return rc;
  if (tokens == 0) return TETRIS_OK;
  if ((rc = check_rows(d_x, type, tokens, ldx, up->k, "input"))) return rc;
  if ((rc = check_rows(d_y, type, tokens, ldy, down->n, "output"))) return rc;
  if (!d_index || !d_weight) return fail(TETRIS_EINVAL, "null argument");
  if ((reinterpret_cast<size_t>(d_index) | reinterpret_cast<size_t>(d_weight)) & 3) return fail(TETRIS_EINVAL, "index or weights not aligned to their elements");
  const int each = tokens_at_once(up, down, tokens, top, type, ldx);
  for (int64_t from = 0; from < tokens; from += each) {
    rc = expert_tokens(up, down, static_cast<const char*>(d_x) + from * ldx * elem_size(type), type, (int)std::min<int64_t>(each, tokens - from), ldx, top,
                       d_index + from * top, d_weight + from * top, static_cast<char*>(d_y) + from * ldy * elem_size(type), ldy, static_cast<hipStream_t>(stream));
    if (rc) return rc;
  }
  return TETRIS_OK;
}

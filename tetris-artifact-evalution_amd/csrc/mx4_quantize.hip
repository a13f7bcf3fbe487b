// MX4: numbers to 4-bit codes with a shared power-of-two scale for each block of 32, and back; rows made ready for the
// products (csrc/mx4_product.hip).  All of it is one pass over memory, bound by HBM.
#include <algorithm>

#include "mx4.h"
#include "rows.h"

namespace tetris {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// A piece of eight elements a lane, four lanes a block: loads and stores of a wave are contiguous (1 or 2 KiB in, 256 bytes
// of codes out).  The scale's exponent is the largest magnitude's, less two (6 = 1.5 * 2^2 is the largest code); the
// instruction that makes codes divides by the scale, rounds to nearest even and saturates.  8192 x 8200 of f32 in 57 us (304 MB, 5.4 TB/s, half of them found in the last-level cache), 8192 x 8192
// of bf16 to the products' layout in 42 (4.1 TB/s: 16 bytes of a line at a time).
template <int TYPE, int KIND, bool VEC>
__global__ __launch_bounds__(256) void quantize_kernel(const typename Elem<TYPE>::type* __restrict__ x, int64_t rows, int cols,
                                                       int64_t ld, unsigned per_row, void* __restrict__ codes,
                                                       uint8_t* __restrict__ scales) {
  const int64_t out_rows = KIND == kMxTiles ? (rows + 31) / 32 * 32 : rows;
  const int64_t waves = (out_rows * per_row + 63) / 64;
  for (int64_t w = wave_of(); w < waves; w += (int64_t)gridDim.x * (blockDim.x >> 6)) {
    const Place p = place_of(w, per_row);
    const bool in = p.row < out_rows;  // the four lanes of a block are in or out together: per_row is a multiple of four
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (p.row < rows) load8<typename Elem<TYPE>::type, VEC>(x + p.row * ld, p.piece * 8, cols, v);
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = quad_max(top);
    const bool fine = top < 0x7f800000u;
    const int scale = max((int)(top >> 23) - 2, 0);
    const float by = __uint_as_float((unsigned)scale << 23);
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], by, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], by, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], by, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], by, 3);
    if (!fine) c = 0;
    const unsigned byte = fine ? (unsigned)scale : 255u;
    if (!in) continue;
    if (KIND == kMxRows) {
      reinterpret_cast<unsigned*>(codes)[p.row * per_row + p.piece] = c;
      if ((p.piece & 3) == 0) scales[p.row * (per_row >> 2) + (p.piece >> 2)] = (uint8_t)byte;
    } else if (KIND == kMxTiles) {
      const int col_tiles = (int)(per_row >> 3), tile = p.piece >> 3, lane = (int)(p.row & 31) + ((p.piece >> 2) & 1) * 32;
      const int64_t at = ((p.row >> 5) * col_tiles + tile) * 64 + lane;
      reinterpret_cast<unsigned*>(codes)[at * 4 + (p.piece & 3)] = c;
      if ((p.piece & 3) == 0)
        scales[(((p.row >> 5) * (col_tiles >> 1) + (tile >> 1)) * 64 + lane) * 2 + (tile & 1)] = (uint8_t)byte;
    } else {
      int4 out;
      const float s = __uint_as_float(byte << 23);
      out.x = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0));
      out.y = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1));
      out.z = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2));
      out.w = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3));
      reinterpret_cast<int4*>(codes)[p.row * per_row + p.piece] = out;
    }
  }
}

// The way back, by the same pieces: 8192 x 8200 to bf16 in 26.6 us (170 MB, 6.4 TB/s with the codes still in the last-level cache).
template <int TYPE, bool VEC>
__global__ __launch_bounds__(256) void dequantize_kernel(const unsigned* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                         int64_t rows, int cols, unsigned per_row,
                                                         typename Elem<TYPE>::type* __restrict__ y, int64_t ld) {
  using T = typename Elem<TYPE>::type;
  const int64_t waves = (rows * per_row + 63) / 64;
  for (int64_t w = wave_of(); w < waves; w += (int64_t)gridDim.x * (blockDim.x >> 6)) {
    const Place p = place_of(w, per_row);
    if (p.row >= rows) continue;
    const int at = p.piece * 8;
    if (at >= cols) continue;
    const unsigned c = codes[p.row * per_row + p.piece];
    const unsigned byte = scales[p.row * (per_row >> 2) + (p.piece >> 2)];
    const float s = __uint_as_float(byte << 23);
    T t[8];
    if (TYPE == TETRIS_BF16) {
      int* o = reinterpret_cast<int*>(t);
      o[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0));
      o[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1));
      o[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2));
      o[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3));
    } else {
      const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
      const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
      t[0] = (T)a.x; t[1] = (T)a.y; t[2] = (T)b.x; t[3] = (T)b.y;
      t[4] = (T)d.x; t[5] = (T)d.y; t[6] = (T)e.x; t[7] = (T)e.y;
    }
    T* out = y + p.row * ld + at;
    if (VEC && at + 8 <= cols) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<int4*>(out)[i] = reinterpret_cast<const int4*>(t)[i];
    } else {
      const int n = min(8, cols - at);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) out[i] = t[i];
    }
  }
}

// A number as bf16 parts: each takes the leading 8 bits of what is left, by truncation, so that what is left is exact
// and three parts hold the 24 bits of any number whose smallest part is not below bf16's range.  The parts after an
// infinity or a NaN are zero: inf - inf would turn an infinite sum into NaN.
template <int P>
__device__ inline void split(float v, unsigned short (&part)[P]) {
  const bool fine = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
  unsigned u = __float_as_uint(v);
  if (!fine && (u & 0x007fffffu)) u |= 0x00400000u;  // NaN stays NaN
#pragma unroll
  for (int i = 0; i < P; ++i) {
    part[i] = (unsigned short)(u >> 16);
    v -= __uint_as_float(u & 0xffff0000u);
    u = fine ? __float_as_uint(v) : 0u;
  }
}

// Rows to rows of a multiple of kMxPad columns, zeros behind them: of the same type (P = 0) or as P arrays of parts.  One pass over memory.
template <int TYPE, int P, bool VEC>
__global__ __launch_bounds__(256) void stage_kernel(const typename Elem<TYPE>::type* __restrict__ x, int64_t rows, int cols,
                                                    int64_t ld, unsigned per_row, void* __restrict__ out) {
  using T = typename Elem<TYPE>::type;
  const int64_t waves = (rows * per_row + 63) / 64;
  for (int64_t w = wave_of(); w < waves; w += (int64_t)gridDim.x * (blockDim.x >> 6)) {
    const Place p = place_of(w, per_row);
    if (p.row >= rows) continue;
    float v[8];
    load8<T, VEC>(x + p.row * ld, p.piece * 8, cols, v);
    const int64_t at = p.row * per_row + p.piece;
    if (P == 0) {
      T t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
      int4* dst = reinterpret_cast<int4*>(out) + at * (sizeof(T) / 2);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) dst[i] = reinterpret_cast<const int4*>(t)[i];
    } else {
      unsigned short part[8][P ? P : 1];
#pragma unroll
      for (int i = 0; i < 8; ++i) split<P ? P : 1>(v[i], part[i]);
#pragma unroll
      for (int q = 0; q < P; ++q) {
        int4 o;
        o.x = part[0][q] | part[1][q] << 16;
        o.y = part[2][q] | part[3][q] << 16;
        o.z = part[4][q] | part[5][q] << 16;
        o.w = part[6][q] | part[7][q] << 16;
        reinterpret_cast<int4*>(out)[q * rows * per_row + at] = o;
      }
    }
  }
}

// MX4 rows to the layout of csrc/mx4.h: one thread moves one block (16 bytes and a scale).  range: the least and the largest scale of
// blocks that hold a number other than zero (kept by minimum and maximum, so the order of the atomics does not show).
__global__ __launch_bounds__(256) void layout_kernel(const int4* __restrict__ codes, const uint8_t* __restrict__ scales, int n, int k,
                                                     int gated, int row_tiles, int col_tiles, int64_t total,
                                                     int4* __restrict__ out, uint8_t* __restrict__ out_scales, int* __restrict__ range) {
  const int blocks = (k + 31) / 32;
  int least = 255, most = 0;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int lane = (int)(i & 63);
    const int64_t tile = i >> 6, row_tile = tile / col_tiles, matrix = row_tile / row_tiles;
    const int col_tile = (int)(tile - row_tile * col_tiles), t = (int)(row_tile - matrix * row_tiles);
    const int r = lane & 31, b = col_tile * 2 + (lane >> 5);
    int row = t * 32 + r;
    bool in = row < n;
    if (gated) {
      const int half = n / 2, f = t * 16 + (r & 15);
      in = f < half;
      row = r < 16 ? f : half + f;
    }
    in = in && b < blocks;
    const int64_t from = (matrix * n + row) * blocks + b;
    int4 c = in ? codes[from] : int4{0, 0, 0, 0};
    if (in && b == blocks - 1 && (k & 31)) {  // codes past the end of the row count as zeros, whatever they are
      unsigned* u = reinterpret_cast<unsigned*>(&c);
      const int left = k & 31;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int have = min(max(left - 8 * q, 0), 8);
        u[q] &= have == 8 ? 0xffffffffu : (1u << (4 * have)) - 1u;
      }
    }
    out[i] = c;
    if (in && ((c.x | c.y | c.z | c.w) & 0x77777777) && scales[from] != 255) {
      least = min(least, (int)scales[from]);
      most = max(most, (int)scales[from]);
    }
    out_scales[((row_tile * (col_tiles >> 1) + (col_tile >> 1)) * 64 + lane) * 2 + (col_tile & 1)] = in ? scales[from] : 127;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    least = min(least, __shfl_xor(least, d));
    most = max(most, __shfl_xor(most, d));
  }
  if ((threadIdx.x & 63) == 0) {
    atomicMin(&range[0], least);
    atomicMax(&range[1], most);
  }
}

template <typename T>
bool on16(const T* p, int64_t ld, int type) {
  return (reinterpret_cast<size_t>(p) & 15) == 0 && (ld * elem_size(type)) % 16 == 0;
}

// workgroups of 256 for `pieces` lanes of work: enough to fill the chip eight waves deep, then loops
unsigned blocks_for(int64_t pieces) { return (unsigned)std::min<int64_t>((pieces + 255) / 256, 256 * 64); }

template <int TYPE, int KIND>
int quantize_typed(const void* d_x, int64_t rows, int cols, int64_t ld, void* d_codes, uint8_t* d_scales, hipStream_t stream) {
  const auto* x = static_cast<const typename Elem<TYPE>::type*>(d_x);
  const unsigned per_row = KIND == kMxRows ? (unsigned)((cols + 31) / 32 * 4) : (unsigned)(round_up(cols, kMxPad) / 8);
  const int64_t out_rows = KIND == kMxTiles ? round_up(rows, 32) : rows;
  const dim3 grid(blocks_for(out_rows * per_row));
  if (on16(x, ld, TYPE))
    hipLaunchKernelGGL((quantize_kernel<TYPE, KIND, true>), grid, dim3(256), 0, stream, x, rows, cols, ld, per_row, d_codes, d_scales);
  else
    hipLaunchKernelGGL((quantize_kernel<TYPE, KIND, false>), grid, dim3(256), 0, stream, x, rows, cols, ld, per_row, d_codes, d_scales);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

template <int KIND>
int quantize_kind(const void* d_x, int type, int64_t rows, int cols, int64_t ld, void* d_codes, uint8_t* d_scales, hipStream_t s) {
  if (type == TETRIS_F32) return quantize_typed<TETRIS_F32, KIND>(d_x, rows, cols, ld, d_codes, d_scales, s);
  if (type == TETRIS_F16) return quantize_typed<TETRIS_F16, KIND>(d_x, rows, cols, ld, d_codes, d_scales, s);
  return quantize_typed<TETRIS_BF16, KIND>(d_x, rows, cols, ld, d_codes, d_scales, s);
}

template <int TYPE>
int dequantize_typed(const uint8_t* d_codes, const uint8_t* d_scales, int64_t rows, int cols, void* d_y, int64_t ld, hipStream_t stream) {
  auto* y = static_cast<typename Elem<TYPE>::type*>(d_y);
  const unsigned per_row = (unsigned)((cols + 31) / 32 * 4);
  const dim3 grid(blocks_for(rows * per_row));
  const auto* codes = reinterpret_cast<const unsigned*>(d_codes);
  if (on16(y, ld, TYPE))
    hipLaunchKernelGGL((dequantize_kernel<TYPE, true>), grid, dim3(256), 0, stream, codes, d_scales, rows, cols, per_row, y, ld);
  else
    hipLaunchKernelGGL((dequantize_kernel<TYPE, false>), grid, dim3(256), 0, stream, codes, d_scales, rows, cols, per_row, y, ld);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

template <int TYPE, int P>
int stage_typed(const void* d_x, int64_t rows, int cols, int64_t ld, void* d_out, hipStream_t stream) {
  const auto* x = static_cast<const typename Elem<TYPE>::type*>(d_x);
  const unsigned per_row = (unsigned)(round_up(cols, kMxPad) / 8);
  const dim3 grid(blocks_for(rows * per_row));
  if (on16(x, ld, TYPE))
    hipLaunchKernelGGL((stage_kernel<TYPE, P, true>), grid, dim3(256), 0, stream, x, rows, cols, ld, per_row, d_out);
  else
    hipLaunchKernelGGL((stage_kernel<TYPE, P, false>), grid, dim3(256), 0, stream, x, rows, cols, ld, per_row, d_out);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

int bad_matrix(int64_t rows, int cols, int64_t ld, int type) {
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (rows < 0 || cols <= 0 || cols > (1 << 30)) return fail(TETRIS_EINVAL, "bad matrix of %lld x %d", (long long)rows, cols);
  if (ld < cols) return fail(TETRIS_EINVAL, "leading dimension %lld below the %d columns", (long long)ld, cols);
  if (rows > (int64_t)1 << 40) return fail(TETRIS_EINVAL, "%lld rows", (long long)rows);
  return TETRIS_OK;
}

}  // namespace

int mx4_quantize_to(int kind, const void* d_x, int type, int64_t rows, int cols, int64_t ld, void* d_codes, uint8_t* d_scales,
                    hipStream_t stream) {
  if (rows == 0) return TETRIS_OK;
  if (kind == kMxRows) return quantize_kind<kMxRows>(d_x, type, rows, cols, ld, d_codes, d_scales, stream);
  if (kind == kMxTiles) return quantize_kind<kMxTiles>(d_x, type, rows, cols, ld, d_codes, d_scales, stream);
  return quantize_kind<kMxValues>(d_x, type, rows, cols, ld, d_codes, d_scales, stream);
}

int stage_rows(const void* d_x, int type, int64_t rows, int cols, int64_t ld, int parts, void* d_out, hipStream_t stream) {
  if (rows == 0) return TETRIS_OK;
  if (type == TETRIS_F32)
    return parts ? stage_typed<TETRIS_F32, 3>(d_x, rows, cols, ld, d_out, stream) : stage_typed<TETRIS_F32, 0>(d_x, rows, cols, ld, d_out, stream);
  if (type == TETRIS_F16)
    return parts ? stage_typed<TETRIS_F16, 2>(d_x, rows, cols, ld, d_out, stream) : stage_typed<TETRIS_F16, 0>(d_x, rows, cols, ld, d_out, stream);
  return stage_typed<TETRIS_BF16, 0>(d_x, rows, cols, ld, d_out, stream);
}

}  // namespace tetris

using namespace tetris;

extern "C" size_t tetris_mx4_code_bytes(int cols) { return cols <= 0 ? 0 : ((size_t)cols + 31) / 32 * 16; }
extern "C" size_t tetris_mx4_scale_bytes(int cols) { return cols <= 0 ? 0 : ((size_t)cols + 31) / 32; }

extern "C" int tetris_mx4_quantize(const void* d_x, int type, int64_t rows, int cols, int64_t ld, uint8_t* d_codes,
                                   uint8_t* d_scales, void* stream) {
  if (const int rc = bad_matrix(rows, cols, ld, type)) return rc;
  if (rows == 0) return TETRIS_OK;
  if (!d_x || !d_codes || !d_scales) return fail(TETRIS_EINVAL, "null argument");
  if (reinterpret_cast<size_t>(d_codes) & 15) return fail(TETRIS_EINVAL, "codes must lie on 16 bytes");
  if (reinterpret_cast<size_t>(d_x) % elem_size(type)) return fail(TETRIS_EINVAL, "input not aligned to its elements");
  return mx4_quantize_to(kMxRows, d_x, type, rows, cols, ld, d_codes, d_scales, static_cast<hipStream_t>(stream));
}

extern "C" int tetris_mx4_dequantize(const uint8_t* d_codes, const uint8_t* d_scales, int64_t rows, int cols, void* d_y, int type,
                                     int64_t ld, void* stream) {
  if (const int rc = bad_matrix(rows, cols, ld, type)) return rc;
  if (rows == 0) return TETRIS_OK;
  if (!d_codes || !d_scales || !d_y) return fail(TETRIS_EINVAL, "null argument");
  if (reinterpret_cast<size_t>(d_codes) & 15) return fail(TETRIS_EINVAL, "codes must lie on 16 bytes");
  if (reinterpret_cast<size_t>(d_y) % elem_size(type)) return fail(TETRIS_EINVAL, "output not aligned to its elements");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (type == TETRIS_F32) return dequantize_typed<TETRIS_F32>(d_codes, d_scales, rows, cols, d_y, ld, s);
  if (type == TETRIS_F16) return dequantize_typed<TETRIS_F16>(d_codes, d_scales, rows, cols, d_y, ld, s);
  return dequantize_typed<TETRIS_BF16>(d_codes, d_scales, rows, cols, d_y, ld, s);
}

extern "C" void tetris_mx4_destroy(tetris_mx4* w) {
  if (!w) return;
  if (w->codes) (void)hipFree(w->codes);
  if (w->scales) (void)hipFree(w->scales);
  w->space.release();
  delete w;
}

namespace {

int create_check(int experts, int n, int k, int gated, tetris_mx4** out) {
  if (!out) return fail(TETRIS_EINVAL, "null argument");
  *out = nullptr;
  if (experts <= 0 || experts > 1024 || n <= 0 || n > kMxSide || k <= 0 || k > kMxSide)
    return fail(TETRIS_EINVAL, "bad weights: %d matrices of %d x %d (at most 1024, sides up to 2^21)", experts, n, k);
  if (gated && (n & 1)) return fail(TETRIS_EINVAL, "a gated matrix has an even number of rows, got %d", n);
  return TETRIS_OK;
}

int lay_out(tetris_mx4* w, const uint8_t* d_codes, const uint8_t* d_scales, hipStream_t stream) {
  w->row_tiles = w->gated ? ceil_div(w->n / 2, 16) : ceil_div(w->n, 32);
  w->col_tiles = (int)(round_up(w->k, kMxPad) / 64);
  const int64_t tiles = (int64_t)w->experts * w->row_tiles * w->col_tiles;
  TETRIS_HIP(hipMalloc(&w->codes, (size_t)tiles * 1024));
  TETRIS_HIP(hipMalloc(&w->scales, (size_t)tiles * 64 + sizeof(int[2])));
  const int64_t total = tiles * 64;
  int range[2] = {255, 0};
  int* d_range = reinterpret_cast<int*>(w->scales + tiles * 64);
  TETRIS_HIP(hipMemcpyAsync(d_range, range, sizeof range, hipMemcpyHostToDevice, stream));
  hipLaunchKernelGGL(layout_kernel, dim3(blocks_for(total)), dim3(256), 0, stream, reinterpret_cast<const int4*>(d_codes), d_scales, w->n,
                     w->k, w->gated ? 1 : 0, w->row_tiles, w->col_tiles, total, reinterpret_cast<int4*>(w->codes), w->scales, d_range);
  TETRIS_HIP(hipGetLastError());
  TETRIS_HIP(hipMemcpyAsync(range, d_range, sizeof range, hipMemcpyDeviceToHost, stream));
  TETRIS_HIP(hipStreamSynchronize(stream));
  // f16 holds multiples of 2^-24 up to 65504: half a unit of the least scale, six of the largest
  w->half = range[0] >= 127 - 23 && range[1] <= 127 + 13;
  return TETRIS_OK;
}

int not_captured(hipStream_t stream) {
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &cap) == hipSuccess && cap != hipStreamCaptureStatusNone)
    return fail(TETRIS_EINVAL, "weights are laid out outside of a graph capture");
  return TETRIS_OK;
}

}  // namespace

extern "C" int tetris_mx4_create(const uint8_t* d_codes, const uint8_t* d_scales, int experts, int n, int k, int gated, void* stream,
                                 tetris_mx4** out) {
  int rc = create_check(experts, n, k, gated, out);
  if (rc) return rc;
  if (!d_codes || !d_scales) return fail(TETRIS_EINVAL, "null argument");
  if (reinterpret_cast<size_t>(d_codes) & 15) return fail(TETRIS_EINVAL, "codes must lie on 16 bytes");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if ((rc = not_captured(s))) return rc;
  std::unique_ptr<tetris_mx4, void (*)(tetris_mx4*)> w(new (std::nothrow) tetris_mx4, tetris_mx4_destroy);
  if (!w) return fail(TETRIS_EINVAL, "no host memory for a handle");
  w->experts = experts; w->n = n; w->k = k; w->gated = gated != 0;
  if ((rc = lay_out(w.get(), d_codes, d_scales, s))) return rc;
  *out = w.release();
  return TETRIS_OK;
}

extern "C" int tetris_mx4_create_values(const void* d_w, int type, int experts, int n, int k, int64_t ld, int gated, void* stream,
                                        tetris_mx4** out) {
  int rc = create_check(experts, n, k, gated, out);
  if (rc) return rc;
  const int64_t rows = (int64_t)experts * n;
  if ((rc = bad_matrix(rows, k, ld, type))) return rc;
  if (!d_w) return fail(TETRIS_EINVAL, "null argument");
  if (reinterpret_cast<size_t>(d_w) % elem_size(type)) return fail(TETRIS_EINVAL, "weights not aligned to their elements");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if ((rc = not_captured(s))) return rc;
  const size_t code_bytes = (size_t)rows * tetris_mx4_code_bytes(k), scale_bytes = (size_t)rows * tetris_mx4_scale_bytes(k);
  uint8_t* d = nullptr;
  TETRIS_HIP(hipMalloc(&d, code_bytes + scale_bytes));
  rc = mx4_quantize_to(kMxRows, d_w, type, rows, k, ld, d, d + code_bytes, s);
  if (!rc) rc = tetris_mx4_create(d, d + code_bytes, experts, n, k, gated, stream, out);
  const hipError_t e = hipFree(d);
  if (!rc && e != hipSuccess) {
    tetris_mx4_destroy(*out);
    *out = nullptr;
    return fail(TETRIS_EHIP, "hipFree failed: %s", hipGetErrorString(e));
  }
  return rc;
}

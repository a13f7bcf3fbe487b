// The residual's addition with a root-mean-square norm: s = x + r, y = s / sqrt(mean(s^2) + eps) * w.  A workgroup has a row, which
// stays in registers between the sum of squares and the outputs, so that memory is passed once; bound by HBM, and for few rows by
// the launch.
#include <algorithm>

#include "mx4.h"
#include "tetris_attention.h"

namespace tetris {
namespace {

constexpr int kNormMost = 1 << 20;  // columns

struct NormRows {
  const void* x;
  const void* residual;
  const float* weight;
  void* sum;
  void* y;
  int64_t ldx, ldr, lds, ldy;
  int cols;
  float eps;
};

// Eight elements of a thread: neighbours where rows lie on 16 bytes (VEC), else every THREADS-th, so that a wave's loads are whole lines.
template <int THREADS, bool VEC>
__device__ inline int first_of(int piece) {
  return VEC ? (piece * THREADS + (int)threadIdx.x) * 8 : piece * THREADS * 8 + (int)threadIdx.x;
}
template <typename T, int THREADS, bool VEC>
__device__ inline void load_piece(const T* row, int at, int cols, float (&v)[8]) {
  if constexpr (VEC) {
    if (at < cols) {
      int4 raw[sizeof(T) / 2];
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const int4*>(row + at)[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)reinterpret_cast<const T*>(raw)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at + i * THREADS < cols ? (float)row[at + i * THREADS] : 0.f;
  }
}
template <typename T, int THREADS, bool VEC>
__device__ inline void store_piece(T* row, int at, int cols, const float (&v)[8]) {
  if constexpr (VEC) {
    if (at >= cols) return;
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<int4*>(row + at)[i] = reinterpret_cast<const int4*>(t)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i * THREADS < cols) row[at + i * THREADS] = (T)v[i];
  }
}

// The sum of v over the workgroup, in all threads, always added in the same order.
template <int THREADS>
__device__ inline float sum_of_all(float v, float* shared) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v += shared[w];
  }
  return v;
}

// KEPT pieces a thread stay in registers; those of wider rows are made again from x and r after the sum.
template <int TYPE, int THREADS, int KEPT, bool VEC>
__global__ __launch_bounds__(THREADS) void rms_norm_kernel(NormRows a) {
  using T = typename Elem<TYPE>::type;
  __shared__ float shared[THREADS / 64];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
  T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.lds : nullptr;
  T* y = static_cast<T*>(a.y) + row * a.ldy;
  const int pieces = (a.cols + THREADS * 8 - 1) / (THREADS * 8);
  auto total = [&](int piece, float (&v)[8]) {
    const int at = first_of<THREADS, VEC>(piece);
    load_piece<T, THREADS, VEC>(x, at, a.cols, v);
    if (r) {
      float u[8];
      load_piece<T, THREADS, VEC>(r, at, a.cols, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += u[i];
    }
  };
  float kept[KEPT][8], squares = 0.f;
#pragma unroll
  for (int p = 0; p < KEPT; ++p) total(p, kept[p]);
#pragma unroll
  for (int p = 0; p < KEPT; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) squares = fmaf(kept[p][i], kept[p][i], squares);
  for (int p = KEPT; p < pieces; ++p) {
    float v[8];
    total(p, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) squares = fmaf(v[i], v[i], squares);
  }
  const float by = 1.f / sqrtf(sum_of_all<THREADS>(squares, shared) / (float)a.cols + a.eps);
  auto finish = [&](int piece, const float (&v)[8]) {
    const int at = first_of<THREADS, VEC>(piece);
    if (sum) store_piece<T, THREADS, VEC>(sum, at, a.cols, v);
    float w[8], out[8];
    if (a.weight) load_piece<float, THREADS, VEC>(a.weight, at, a.cols, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = a.weight ? v[i] * by * w[i] : v[i] * by;
    store_piece<T, THREADS, VEC>(y, at, a.cols, out);
  };
#pragma unroll
  for (int p = 0; p < KEPT; ++p) finish(p, kept[p]);
  for (int p = KEPT; p < pieces; ++p) {
    float v[8];
    total(p, v);
    finish(p, v);
  }
}

template <int TYPE, bool VEC>
void launch(const NormRows& a, int64_t rows, hipStream_t s) {
  constexpr int64_t kMost = 1 << 30;  // rows of a launch
  constexpr int size = TYPE == TETRIS_F32 ? 4 : 2;
  for (int64_t from = 0; from < rows; from += kMost) {
    NormRows b = a;
    b.x = static_cast<const char*>(a.x) + from * a.ldx * size;
    if (a.residual) b.residual = static_cast<const char*>(a.residual) + from * a.ldr * size;
    if (a.sum) b.sum = static_cast<char*>(a.sum) + from * a.lds * size;
    b.y = static_cast<char*>(a.y) + from * a.ldy * size;
    const dim3 grid((unsigned)std::min(kMost, rows - from));
    if (a.cols <= 512) hipLaunchKernelGGL((rms_norm_kernel<TYPE, 64, 1, VEC>), grid, dim3(64), 0, s, b);
    else if (a.cols <= 2048) hipLaunchKernelGGL((rms_norm_kernel<TYPE, 256, 1, VEC>), grid, dim3(256), 0, s, b);
    else if (a.cols <= 4096) hipLaunchKernelGGL((rms_norm_kernel<TYPE, 256, 2, VEC>), grid, dim3(256), 0, s, b);
    else hipLaunchKernelGGL((rms_norm_kernel<TYPE, 256, 4, VEC>), grid, dim3(256), 0, s, b);
  }
}

int check_norm(const void* p, int type, int64_t ld, int cols, const char* what) {
  if (ld < cols) return fail(TETRIS_EINVAL, "%s: leading dimension %lld below the %d columns", what, (long long)ld, cols);
  if (reinterpret_cast<size_t>(p) % elem_size(type)) return fail(TETRIS_EINVAL, "%s not aligned to its elements", what);
  return TETRIS_OK;
}

}  // namespace
}  // namespace tetris

using namespace tetris;

extern "C" int tetris_rms_norm(const void* d_x, int type, int64_t rows, int cols, int64_t ldx, const void* d_residual, int64_t ld_residual,
                               const float* d_weight, float eps, void* d_sum, int64_t ld_sum, void* d_y, int64_t ldy, void* stream) {
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (rows < 0 || rows > (int64_t)1 << 40) return fail(TETRIS_EINVAL, "%lld rows", (long long)rows);
  if (cols <= 0 || cols > kNormMost) return fail(TETRIS_EINVAL, "%d columns (1 to %d)", cols, kNormMost);
  if (!(eps >= 0.f)) return fail(TETRIS_EINVAL, "eps %g is negative or no number", (double)eps);
  if (rows == 0) return TETRIS_OK;
  if (!d_x || !d_y) return fail(TETRIS_EINVAL, "null argument");
  int rc = check_norm(d_x, type, ldx, cols, "input");
  if (!rc && d_residual) rc = check_norm(d_residual, type, ld_residual, cols, "residual");
  if (!rc && d_sum) rc = check_norm(d_sum, type, ld_sum, cols, "sum");
  if (!rc) rc = check_norm(d_y, type, ldy, cols, "output");
  if (rc) return rc;
  if (reinterpret_cast<size_t>(d_weight) & 3) return fail(TETRIS_EINVAL, "weight not aligned to its elements");
  if (d_y == d_x || d_y == d_residual || d_y == d_sum || d_sum == d_x) return fail(TETRIS_EINVAL, "an output is another argument (only the sum may be the residual)");
  if (d_sum && d_sum == d_residual && ld_sum != ld_residual) return fail(TETRIS_EINVAL, "the sum takes the residual's place with another leading dimension");
  const NormRows a{d_x, d_residual, d_weight, d_sum, d_y, ldx, ld_residual, ld_sum, ldy, cols, eps};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t size = elem_size(type);
  auto whole = [&](const void* p, int64_t ld) { return !p || ((reinterpret_cast<size_t>(p) & 15) == 0 && ld * size % 16 == 0); };
  const bool vec = cols % 8 == 0 && whole(d_x, ldx) && whole(d_residual, ld_residual) && whole(d_sum, ld_sum) && whole(d_y, ldy) && whole(d_weight, 4);
  if (type == TETRIS_F32) vec ? launch<TETRIS_F32, true>(a, rows, s) : launch<TETRIS_F32, false>(a, rows, s);
  else if (type == TETRIS_F16) vec ? launch<TETRIS_F16, true>(a, rows, s) : launch<TETRIS_F16, false>(a, rows, s);
  else vec ? launch<TETRIS_BF16, true>(a, rows, s) : launch<TETRIS_BF16, false>(a, rows, s);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

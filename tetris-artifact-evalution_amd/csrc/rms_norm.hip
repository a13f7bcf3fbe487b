// The residual's addition with a root-mean-square norm: s = x + r, y = s / sqrt(mean(s^2) + eps) * w.  A workgroup has a row, which
// stays in registers between the sum of squares and the outputs up to 8192 columns, so that memory is passed once (what lies beyond is read twice, mostly from the caches: 8192
// rows of 16384 bf16 193 us, 5.6 TB/s of what has to pass); bound by HBM (8192 rows of 4096 bf16, with
// residual and sum: 50 us for 268 MB, 5.4 TB/s, some of it from the last-level cache), for few rows by the launch (8 rows: 3.3 us), and for rows of a head by a workgroup's
// beginning (262144 of 128: 80 us, 3.4 TB/s).
#include <algorithm>
#include <type_traits>

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

// Eight elements of a thread: neighbours where rows lie on 16 bytes (VEC), else every THREADS-th, so that a wave's loads are whole lines.  All loads of a
// row are asked for before any is used: those past its end read its last elements, which count as zeros then.
template <typename T, int THREADS, bool VEC>
struct Piece {
  static constexpr int Q = sizeof(T) / 2;
  int4 raw[VEC ? Q : 1];
  T one[VEC ? 1 : 8];
  __device__ static inline int first(int piece) { return VEC ? (piece * THREADS + (int)threadIdx.x) * 8 : piece * THREADS * 8 + (int)threadIdx.x; }
  __device__ inline void load(const T* row, int piece, int cols) {
    if constexpr (VEC) {
      const int4* from = reinterpret_cast<const int4*>(row + min(first(piece), cols - 8));
#pragma unroll
      for (int i = 0; i < Q; ++i) raw[i] = from[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) one[i] = row[min(first(piece) + i * THREADS, cols - 1)];
    }
  }
  __device__ inline float at(int i) const {
    if constexpr (VEC) return (float)reinterpret_cast<const T*>(raw)[i];
    else return (float)one[i];
  }
  __device__ static inline bool in(int piece, int i, int cols) { return VEC ? first(piece) < cols : first(piece) + i * THREADS < cols; }
  __device__ static inline void store(T* row, int piece, int cols, const float (&v)[8]) {
    if constexpr (VEC) {
      if (first(piece) >= cols) return;
      T t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
#pragma unroll
      for (int i = 0; i < Q; ++i) reinterpret_cast<int4*>(row + first(piece))[i] = reinterpret_cast<const int4*>(t)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (first(piece) + i * THREADS < cols) row[first(piece) + i * THREADS] = (T)v[i];
    }
  }
};

// The sum of v over the workgroup, in all threads, always added in the same order.
template <int THREADS>
__device__ inline float sum_of_all(float v, float* shared) {
  auto step = [&](auto ctrl, auto rows) {
    v += __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // from 1, 2, 4 and 8 lanes below in rows of sixteen
  step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // a row's last to the next row, the second row's to the upper half
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  v = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
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
  using P = Piece<T, THREADS, VEC>;
  using W = Piece<float, THREADS, VEC>;
  __shared__ float shared[THREADS / 64];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
  T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.lds : nullptr;
  T* y = static_cast<T*>(a.y) + row * a.ldy;
  const int pieces = (a.cols + THREADS * 8 - 1) / (THREADS * 8);
  P xs[KEPT], rs[KEPT];
  W ws[KEPT];
#pragma unroll
  for (int p = 0; p < KEPT; ++p) xs[p].load(x, p, a.cols);
  if (r) {
#pragma unroll
    for (int p = 0; p < KEPT; ++p) rs[p].load(r, p, a.cols);
  }
  if (a.weight) {
#pragma unroll
    for (int p = 0; p < KEPT; ++p) ws[p].load(a.weight, p, a.cols);
  }
  auto total = [&](const P& u, const P& v, int p, float (&out)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = P::in(p, i, a.cols) ? (r ? u.at(i) + v.at(i) : u.at(i)) : 0.f;
  };
  float kept[KEPT][8], squares = 0.f;
#pragma unroll
  for (int p = 0; p < KEPT; ++p) {
    total(xs[p], rs[p], p, kept[p]);
#pragma unroll
    for (int i = 0; i < 8; ++i) squares = fmaf(kept[p][i], kept[p][i], squares);
  }
  for (int p = KEPT; p < pieces; ++p) {
    P u, v;
    float t[8];
    u.load(x, p, a.cols);
    if (r) v.load(r, p, a.cols);
    total(u, v, p, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) squares = fmaf(t[i], t[i], squares);
  }
  const float under = sum_of_all<THREADS>(squares, shared) / (float)a.cols + a.eps;
  if (__builtin_expect(!(under >= 0x1p-100f && under < __builtin_inff()), 0)) {
    // Squares that 32 bits do not hold are taken of the row scaled by a power of two: elements up to 2^128 by 2^-80, and where what is under the root is
    // below 2^-100, elements from 2^-149 on by 2^96.  The row is read again for that, so that the registers of ordinary ones are what they were.
    const bool small = under < 1.f;
    const float scale = small ? 0x1p96f : 0x1p-80f;
    auto again = [&](auto each) {
#pragma unroll 1
      for (int p = 0; p < pieces; ++p) {
        P u, v;
        float t[8];
        u.load(x, p, a.cols);
        if (r) v.load(r, p, a.cols);
        total(u, v, p, t);
        each(p, t);
      }
    };
    if constexpr (THREADS > 64) __syncthreads();  // (the waves' sums have been read)
    float scaled = 0.f;
    again([&](int, const float (&t)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) scaled = fmaf(t[i] * scale, t[i] * scale, scaled);
    });
    const float by = 1.f / sqrtf(sum_of_all<THREADS>(scaled, shared) / (float)a.cols + a.eps * scale * scale);
    const float first = small ? scale : by, second = small ? by : scale;  // (in this order products of elements that matter stay within 32 bits' range)
    again([&](int p, const float (&t)[8]) {
      W w;
      float out[8];
      if (a.weight) w.load(a.weight, p, a.cols);
      if (sum) P::store(sum, p, a.cols, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = a.weight ? t[i] * first * second * w.at(i) : t[i] * first * second;
      P::store(y, p, a.cols, out);
    });
    return;
  }
  const float by = 1.f / sqrtf(under);
  auto finish = [&](int p, const W& w, const float (&v)[8]) {
    if (sum) P::store(sum, p, a.cols, v);
    float out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = a.weight ? v[i] * by * w.at(i) : v[i] * by;
    P::store(y, p, a.cols, out);
  };
#pragma unroll
  for (int p = 0; p < KEPT; ++p) finish(p, ws[p], kept[p]);
  for (int p = KEPT; p < pieces; ++p) {
    P u, v;
    W w;
    float t[8];
    u.load(x, p, a.cols);
    if (r) v.load(r, p, a.cols);
    if (a.weight) w.load(a.weight, p, a.cols);
    total(u, v, p, t);
    finish(p, w, t);
  }
}

template <int TYPE, bool VEC>
void launch(const NormRows& a, int64_t rows, hipStream_t s) {
  constexpr int64_t kMost = 1 << 21;  // rows of a launch, which has fewer than 2^32 threads
  constexpr int size = TYPE == TETRIS_F32 ? 4 : 2;
  for (int64_t from = 0; from < rows; from += kMost) {
    NormRows b = a;
    b.x = static_cast<const char*>(a.x) + from * a.ldx * size;
    if (a.residual) b.residual = static_cast<const char*>(a.residual) + from * a.ldr * size;
    if (a.sum) b.sum = static_cast<char*>(a.sum) + from * a.lds * size;
    b.y = static_cast<char*>(a.y) + from * a.ldy * size;
    const dim3 grid((unsigned)std::min(kMost, rows - from));
#define TETRIS_NORM(THREADS, KEPT) hipLaunchKernelGGL((rms_norm_kernel<TYPE, THREADS, KEPT, VEC>), grid, dim3(THREADS), 0, s, b)
    // Many rows: fewer threads with two pieces each, so that a compute unit has several rows under way.  512 rows of 4096 bf16 4.95 us against 5.5 with 1024 threads, 2048
    // 12.4 against 14.2, 2048 of f32 27.9 against 29.4, 1024 of 8192 bf16 13.1 against 14.0; at 64 rows the two are as fast.
    if (a.cols <= 512) TETRIS_NORM(64, 1);
    else if (a.cols <= 2048) TETRIS_NORM(256, 1);
    else if (a.cols <= 4096 && rows >= 512) TETRIS_NORM(256, 2);
    else if (a.cols <= 8192 && rows >= 512) TETRIS_NORM(512, 2);
    else TETRIS_NORM(1024, 1);  // all of a row's loads at once
#undef TETRIS_NORM
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
  const bool vec = cols % 8 == 0 && whole(d_x, ldx) && whole(d_residual, ld_residual) && whole(d_sum, ld_sum) && whole(d_y, ldy) && (reinterpret_cast<size_t>(d_weight) & 15) == 0;
  if (type == TETRIS_F32) vec ? launch<TETRIS_F32, true>(a, rows, s) : launch<TETRIS_F32, false>(a, rows, s);
  else if (type == TETRIS_F16) vec ? launch<TETRIS_F16, true>(a, rows, s) : launch<TETRIS_F16, false>(a, rows, s);
  else vec ? launch<TETRIS_BF16, true>(a, rows, s) : launch<TETRIS_BF16, false>(a, rows, s);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

// Rotary positions: pairs of a head's elements turned by position * rate, each pair by the position of its section's axis.  A workgroup
// makes the cosines and sines of a few tokens once, in LDS, and turns all heads of these tokens with them; one pass over memory, which
// bounds it: 4096 tokens of 32 heads of 128 f32 29 us (134 MB, 4.7 TB/s), 15000 of 16 of 80 f16 with three axes 14.7 (77 MB, 5.2 TB/s); 8 tokens
// are a launch, 3.3 us.
//
// A pair's angle in turns is formed in 64 bits and its whole turns taken off, which leaves a far position's angle exact to about
// 2^-49 of the position.  What is left goes to 32 bits as t + d with |d| at most 2^-25 (half turns, |t| at most 1), and cos(t + d) = cos t - d sin t, so that the cosine is
// as near as one rounded from 64 bits.
#include <algorithm>
#include <cmath>

#include "mx4.h"
#include "tetris_attention.h"

namespace tetris {
namespace {

constexpr int kRotaryHead = 1024;     // most elements of a head
constexpr int kRotaryEntries = 1024;  // cosines and sines of a workgroup

struct Rotary {
  const void* x;
  void* y;
  const int* position;
  int64_t ldx, ldy, ldp;
  int tokens, heads, head, half;  // half: pairs of a head
  int start[5];                   // first pair of each section, and the end
  int halves, by_axis, backward;
  int each;    // tokens of a workgroup
  int splits;  // workgroups that share a token's heads
  double turns;  // log2 of the base
};

// Eight elements as they lie.
template <typename T>
struct Eight {
  int4 raw[sizeof(T) / 2];
  __device__ inline void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const int4*>(p)[i];
  }
  __device__ inline void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<int4*>(p)[i] = raw[i];
  }
  __device__ inline float get(int i) const { return (float)reinterpret_cast<const T*>(raw)[i]; }
  __device__ inline void set(int i, float v) { reinterpret_cast<T*>(raw)[i] = (T)v; }
};

// VEC: rows lie on 16 bytes, and a unit of work is eight elements, or eight pairs of halves.  Otherwise it is a pair, or an element past the pairs.
template <int TYPE, bool VEC, bool HALVES>
__global__ __launch_bounds__(256) void rotary_kernel(Rotary a) {
  using T = typename Elem<TYPE>::type;
  __shared__ float2 table[kRotaryEntries];  // cosine and sine of a token's pairs
  const int group = blockIdx.x / a.splits, split = blockIdx.x - group * a.splits;
  const int first = group * a.each, count = min(a.each, a.tokens - first);
  for (int e = threadIdx.x; e < count * a.half; e += 256) {
    const int token = e / a.half, pair = e - token * a.half;
    int axis = 0;
#pragma unroll
    for (int k = 1; k < 4; ++k) axis += pair >= a.start[k] ? 1 : 0;
    int from = 0, of = a.half;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (a.by_axis && axis == k) from = a.start[k], of = a.start[k + 1] - a.start[k];
    const double rate = exp2(-(double)(pair - from) * a.turns / (double)of);
    const int position = a.position[axis * a.ldp + first + token];
    double t = (double)position * (rate * 0.15915494309189533577);  // 1 / (2 pi)
    t = 2.0 * (t - rint(t));
    const float near = (float)t, left = (float)((t - (double)near) * 3.14159265358979323846);
    float s, c;
    sincospif(near, &s, &c);
    const float sine = fmaf(left, c, s);
    table[e] = make_float2(fmaf(-left, s, c), a.backward ? -sine : sine);
  }
  __syncthreads();
  const int dims = 2 * a.half, tail = a.head - dims;
  const int turned = VEC ? (HALVES ? a.half / 8 : a.half / 4) : a.half, units = turned + (VEC ? tail / 8 : tail);  // of a head
  const int h0 = (int)((int64_t)a.heads * split / a.splits), heads = (int)((int64_t)a.heads * (split + 1) / a.splits) - h0;
  const int all = heads * units;
  if constexpr (VEC) {
    // two tokens' loads are under way together
    for (int t0 = 0; t0 < count; t0 += 2) {
      const T* x = static_cast<const T*>(a.x) + (int64_t)(first + t0) * a.ldx;
      T* y = static_cast<T*>(a.y) + (int64_t)(first + t0) * a.ldy;
      const int more = min(count - t0, 2);
      for (int w = threadIdx.x; w < all; w += 256) {
        const int h = w / units, u = w - h * units;
        const int64_t head = (int64_t)(h0 + h) * a.head;
        const bool copied = u >= turned;
        const int64_t at = head + (copied ? dims + (u - turned) * 8 : u * 8);
        Eight<T> p[2], q[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const T* from = x + (k < more ? k : 0) * a.ldx + at;
          p[k].load(from);
          if (HALVES) q[k].load(from + (copied ? 0 : a.half));
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (k >= more) break;
          T* to = y + k * a.ldy + at;
          if (!copied) {
            const float2* angle = table + (t0 + k) * a.half + u * (HALVES ? 8 : 4);
#pragma unroll
            for (int i = 0; i < (HALVES ? 8 : 4); ++i) {
              const float2 cs = angle[i];
              const float v = HALVES ? p[k].get(i) : p[k].get(2 * i), z = HALVES ? q[k].get(i) : p[k].get(2 * i + 1);
              const float f = v * cs.x - z * cs.y, g = v * cs.y + z * cs.x;
              if (HALVES) p[k].set(i, f), q[k].set(i, g);
              else p[k].set(2 * i, f), p[k].set(2 * i + 1, g);
            }
            if (HALVES) q[k].store(to + a.half);
          }
          p[k].store(to);
        }
      }
    }
  } else {
    for (int token = 0; token < count; ++token) {
      const T* x = static_cast<const T*>(a.x) + (int64_t)(first + token) * a.ldx;
      T* y = static_cast<T*>(a.y) + (int64_t)(first + token) * a.ldy;
      const float2* angle = table + token * a.half;
      for (int w = threadIdx.x; w < all; w += 256) {
        const int h = w / units, u = w - h * units;
        const int64_t at = (int64_t)(h0 + h) * a.head;
        if (u >= turned) {
          y[at + dims + u - turned] = x[at + dims + u - turned];
        } else {
          const int64_t i = at + (HALVES ? u : 2 * u), j = HALVES ? i + a.half : i + 1;
          const float p = (float)x[i], q = (float)x[j];
          const float2 cs = angle[u];
          y[i] = (T)(p * cs.x - q * cs.y);
          y[j] = (T)(p * cs.y + q * cs.x);
        }
      }
    }
  }
}

template <int TYPE>
void launch(Rotary a, bool vec, int64_t groups, hipStream_t s) {
  const dim3 grid((unsigned)groups), block(256);
  if (vec && a.halves) hipLaunchKernelGGL((rotary_kernel<TYPE, true, true>), grid, block, 0, s, a);
  else if (vec) hipLaunchKernelGGL((rotary_kernel<TYPE, true, false>), grid, block, 0, s, a);
  else if (a.halves) hipLaunchKernelGGL((rotary_kernel<TYPE, false, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((rotary_kernel<TYPE, false, false>), grid, block, 0, s, a);
}

}  // namespace
}  // namespace tetris

using namespace tetris;

extern "C" int tetris_rotate(const tetris_rotary* r, const void* d_x, int type, int tokens, int heads, int64_t ldx, const int32_t* d_position,
                             int64_t ld_position, int backward, void* d_y, int64_t ldy, void* stream) {
  if (!r) return fail(TETRIS_EINVAL, "null argument");
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (r->head <= 0 || r->head > kRotaryHead) return fail(TETRIS_EINVAL, "heads of %d elements (1 to %d)", r->head, kRotaryHead);
  if (r->dims <= 0 || r->dims > r->head || (r->dims & 1)) return fail(TETRIS_EINVAL, "%d elements of %d to turn (an even number of them)", r->dims, r->head);
  if (r->axes < 1 || r->axes > 4) return fail(TETRIS_EINVAL, "%d axes (1 to 4)", r->axes);
  Rotary a{};
  a.half = r->dims / 2;
  for (int k = 0; k < 4; ++k) {
    const int n = k < r->axes ? r->sections[k] : 0;
    if (n < 0 || n > a.half) return fail(TETRIS_EINVAL, "a section of %d pairs", n);
    a.start[k + 1] = a.start[k] + n;
  }
  if (a.start[4] != a.half) return fail(TETRIS_EINVAL, "sections of %d pairs together where %d are turned", a.start[4], a.half);
  if (r->pairing != TETRIS_PAIR_HALVES && r->pairing != TETRIS_PAIR_NEIGHBOURS) return fail(TETRIS_EINVAL, "pairing %d", r->pairing);
  if (r->rate != TETRIS_RATE_HEAD && r->rate != TETRIS_RATE_AXIS) return fail(TETRIS_EINVAL, "rate %d", r->rate);
  if (!(r->base > 0.0) || !std::isfinite(r->base)) return fail(TETRIS_EINVAL, "base %g is not positive and finite", r->base);
  if (tokens < 0 || heads < 0 || heads > (1 << 20)) return fail(TETRIS_EINVAL, "%d tokens of %d heads", tokens, heads);
  const int64_t width = (int64_t)heads * r->head;
  if (ldx < width || ldy < width) return fail(TETRIS_EINVAL, "leading dimension %lld below the %lld elements of a token", (long long)(ldx < ldy ? ldx : ldy), (long long)width);
  if (r->axes > 1 && ld_position < tokens) return fail(TETRIS_EINVAL, "positions: leading dimension %lld below the %d tokens", (long long)ld_position, tokens);
  if (tokens == 0 || heads == 0) return TETRIS_OK;
  if (!d_x || !d_y || !d_position) return fail(TETRIS_EINVAL, "null argument");
  if ((reinterpret_cast<size_t>(d_x) | reinterpret_cast<size_t>(d_y)) % elem_size(type)) return fail(TETRIS_EINVAL, "rows not aligned to their elements");
  if (reinterpret_cast<size_t>(d_position) & 3) return fail(TETRIS_EINVAL, "positions not aligned to their elements");
  if (d_x == d_y && ldx != ldy) return fail(TETRIS_EINVAL, "in place with another leading dimension");
  a.x = d_x; a.y = d_y; a.position = d_position;
  a.ldx = ldx; a.ldy = ldy; a.ldp = ld_position;
  a.tokens = tokens; a.heads = heads; a.head = r->head;
  a.halves = r->pairing == TETRIS_PAIR_HALVES;
  a.by_axis = r->rate == TETRIS_RATE_AXIS;
  a.backward = backward != 0;
  a.turns = std::log2(r->base);
  const int size = elem_size(type);
  const bool vec = ((reinterpret_cast<size_t>(d_x) | reinterpret_cast<size_t>(d_y)) & 15) == 0 && ldx * size % 16 == 0 && ldy * size % 16 == 0 &&
                   r->head % 8 == 0 && a.half % (a.halves ? 8 : 4) == 0;
  // Few tokens: a workgroup each, or several that share its heads.  Many: as many as fill the table, so that every thread makes an angle or two.
  a.each = 1;
  while (a.each * 2 * a.half <= kRotaryEntries / 2 && tokens / (a.each * 2) >= 2048) a.each *= 2;
  constexpr int kMost = 1 << 22;  // tokens of a launch, which has fewer than 2^32 threads
  const int64_t groups = ceil_div(std::min(tokens, kMost), a.each);
  a.splits = 1;
  while (a.splits * 2 <= heads && groups * a.splits < 512 && width / (a.splits * 2) >= 1024) a.splits *= 2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int from = 0; from < tokens; from += std::min(kMost, tokens - from)) {
    Rotary b = a;
    b.x = static_cast<const char*>(d_x) + from * ldx * size;
    b.y = static_cast<char*>(d_y) + from * ldy * size;
    b.position = d_position + from;
    b.tokens = std::min(kMost, tokens - from);
    const int64_t grid = (int64_t)ceil_div(b.tokens, b.each) * b.splits;
    if (type == TETRIS_F32) launch<TETRIS_F32>(b, vec, grid, s);
    else if (type == TETRIS_F16) launch<TETRIS_F16>(b, vec, grid, s);
    else launch<TETRIS_BF16>(b, vec, grid, s);
  }
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

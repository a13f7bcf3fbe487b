// Attention over a cache of keys and values in MX4 (include/tetris_attention.h), one pass over the cache with a running maximum and sum.
//
// A wave takes steps of 32 tokens of one kv head, for up to 16 NT rows: pairs (query token, head) that read this kv head.
//   scores    S^T [32 tokens][rows] = K q^T       v_mfma_f32_16x16x32_bf16 of keys made bf16 in registers, one instruction for two of them
//   weights   P = 2^(S - m), m a bound of the row's scores so far
//   outputs   O^T [elements][rows] += V^T P^T     the same instruction; the page's layout (csrc/cache.h) gives a lane the values of the tokens whose
//                                               weights it holds, so that weights go from one product to the next without leaving the lane
// A key or value has two significant bits and its scale's exponent: exact in bf16.  q comes in 1, 2 or 3 bf16 parts (bf16, f16, f32), which hold
// all of its bits, and P in two (16 bits; f32: three), so outputs are those of 32-bit arithmetic rounded once.
// m is raised only to a score that is more than 8 above it (weights are at most 2^8, far from overflow); most steps need no exchange
// between lanes for it.  A row's sum stays apart in four lanes until the end.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache.h"

namespace tetris {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 32;  // tokens
constexpr float kRoom = 8.f;
constexpr int kCacheLength = 1 << 28;  // tokens of a sequence: granules that page_magic divides exactly

struct Attend {
  const uint8_t* data;
  const void* q;
  void* y;
  const int* first;
  const int* length;
  const int* table;
  float* part;  // of chunks: maximum and sum [chunk][row][head][2], then outputs [chunk][row][head][elements]
  int64_t page_bytes, ldt, ldq, ldy;
  int pages, page, granules, kv_heads, heads, group, sequences, rows, most_rows, most_length, window;
  int blocks;  // of rows
  int chunk, chunks;  // tokens of a workgroup; most of them in a sequence
  int whole;   // rows of q lie on 16 bytes
  unsigned page_magic;  // to divide by granules (0 where that is one)
  float scale;  // to powers of two, not negative
  float sign;  // what q is multiplied by: scale's sign, or zero where scale is
};

// What a sequence is: its rows and tokens, whatever the arrays hold.
struct Sequence { int begin, rows, length, base; };
__device__ inline Sequence sequence_of(const Attend& a, int s) {
  Sequence q;
  q.begin = a.first ? min(max(a.first[s], 0), a.rows) : s;
  const int end = a.first ? min(max(a.first[s + 1], q.begin), a.rows) : s + 1;
  q.rows = end - q.begin;
  q.length = min(max(a.length[s], 0), a.most_length);
  // the first token that any row sees, down to a whole step
  q.base = a.window ? max(q.length - q.rows - a.window + 1, 0) & ~(kStep - 1) : 0;
  return q;
}

template <int TYPE>
constexpr int kParts = TYPE == TETRIS_BF16 ? 1 : TYPE == TETRIS_F16 ? 2 : 3;
template <int TYPE>
constexpr int kWeightParts = TYPE == TETRIS_F32 ? 3 : 2;

// the i-th pair of the codes in a word to bf16
template <int I>
__device__ inline unsigned pair(unsigned codes, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, I));
}
__device__ inline unsigned pair_at(unsigned codes, float scale, int i) {  // (i a constant where this is used)
  switch (i) {
    case 0: return pair<0>(codes, scale);
    case 1: return pair<1>(codes, scale);
    case 2: return pair<2>(codes, scale);
    default: return pair<3>(codes, scale);
  }
}
__device__ inline float scale_of(unsigned word, int byte) { return __uint_as_float((word >> (8 * byte) & 255u) << 23); }
__device__ inline f32x4 product(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// the leading 16 bits of v, and what they leave of it; nothing of an infinity or NaN
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
// A pair of weights to PARTS pairs of bf16: the leading 8 bits by truncation, so that what is left is exact, and the last part rounded
// (two parts are within 2^-16 of the weight, three hold all of it).  Weights are finite or NaN, and a NaN stays one in every part.
template <int PARTS>
__device__ inline void split_pair(float u, float v, unsigned (&out)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS - 1; ++i) {
    out[i] = __builtin_amdgcn_perm(__float_as_uint(v), __float_as_uint(u), 0x07060302u);
    u -= __uint_as_float(__float_as_uint(u) & 0xffff0000u);
    v -= __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  }
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  out[PARTS - 1] = __builtin_bit_cast(unsigned, bf16x2{(__bf16)u, (__bf16)v});
}

__device__ inline float max_of_row(float v) {  // over lanes l, l + 16, l + 32, l + 48
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float sum_of_row(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// What a lane reads of a granule.
template <int D>
struct Granule {
  static constexpr int N = D / 32;                          // words of codes, of a key and of four values
  static constexpr int KS = neighbours(D) ? (D + 127) / 128 : N;  // scales of a key
  static constexpr int VS = neighbours(D) ? 1 : N;           // words of values' scales
  unsigned k[N], v[N], ks[KS], vs[VS];
  __device__ inline void load(const uint8_t* g, int lane) {
    const int r = lane & 15, q = lane >> 4;
    const unsigned* from = reinterpret_cast<const unsigned*>(g) + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) k[i] = from[i];
    from += 2 * D;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from[i];
    const uint8_t* scales = g + 16 * D;
#pragma unroll
    for (int i = 0; i < KS; ++i) ks[i] = scales[r * N + (neighbours(D) ? q * D / 128 + i : (q * (D / 4) + 8 * i) / 32)];
    const unsigned* vscales = reinterpret_cast<const unsigned*>(scales + D / 2);
#pragma unroll
    for (int i = 0; i < VS; ++i) vs[i] = vscales[q * N + (neighbours(D) ? r * (D / 16) / 32 : i)];
  }
  __device__ inline i32x4 key(int w) const {  // the w-th word's eight elements
    const float s = __uint_as_float(ks[neighbours(D) ? w / 4 : w] << 23);
    return i32x4{(int)pair<0>(k[w], s), (int)pair<1>(k[w], s), (int)pair<2>(k[w], s), (int)pair<3>(k[w], s)};
  }
  // elements 2 c and 2 c + 1 of the lane's (its c-th byte) of its four tokens: to words 0 and 1 of `even` and `odd`, from `at` on
  __device__ inline void values(int c, int at, i32x4& even, i32x4& odd) const {
    unsigned t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = i * N + c;
      t[i] = pair_at(v[b / 4], scale_of(vs[neighbours(D) ? 0 : c], i), b % 4);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      even[at + i] = (int)__builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x05040100u);
      odd[at + i] = (int)__builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x07060302u);
    }
  }
};

// which element row i of an output's j-th product is
template <int D>
__device__ inline int element_of(int j, int i) { return neighbours(D) ? i * (D / 16) + j : j * 16 + i; }

// The rows of a wave: their queries, and outputs so far.
template <int TYPE, int D, int NT>
struct Rows {
  static constexpr int QP = kParts<TYPE>, PP = kWeightParts<TYPE>, N = D / 32, S = D / 16;
  i32x4 q[QP][NT][N];
  f32x4 o[NT][S];
  float m[NT], l[NT];
  int last[NT];  // the newest token that the lane's row sees

  __device__ inline void begin(const Attend& a, const Sequence& seq, int kv, int r0, int all, int lane) {
    using T = typename Elem<TYPE>::type;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + n * 16 + (lane & 15), t = r / a.group, h = kv * a.group + r - t * a.group;
      last[n] = seq.length - seq.rows + t;
      const T* row = static_cast<const T*>(a.q) + (int64_t)(seq.begin + t) * a.ldq + (int64_t)h * D + (lane >> 4) * (D / 4);
#pragma unroll
      for (int w = 0; w < N; ++w) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        if (r < all) {
          if (a.whole) {
            int4 raw[sizeof(T) / 2];
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const int4*>(row + 8 * w)[i];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)reinterpret_cast<const T*>(raw)[i];
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)row[8 * w + i];
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= a.sign;
#pragma unroll
        for (int p = 0; p < QP; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned low = leading(v[2 * i]);
            q[p][n][w][i] = (int)(low | leading(v[2 * i + 1]) << 16);
          }
      }
      m[n] = -__builtin_inff();
      l[n] = 0.f;
#pragma unroll
      for (int j = 0; j < S; ++j) o[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // 32 tokens from `at` on, upto[u] of granule u's 16 in the sequence.  EDGE: some row does not see all of them.
  template <bool EDGE>
  __device__ inline void step(const Attend& a, Granule<D> (&g)[2], int at, const int (&upto)[2], int lane) {
    constexpr int VS = Granule<D>::VS;
    const int quad = lane >> 4;
    bool nan = false;  // the lane has a value that is NaN
    if constexpr (EDGE) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < VS; ++c) {
            const unsigned byte = g[u].vs[c] >> (8 * i) & 255u;
            const bool there = 4 * quad + i < upto[u];
            nan = nan || (byte == 255u && there);
            if (!there) g[u].vs[c] = (g[u].vs[c] & ~(255u << (8 * i))) | 127u << (8 * i);  // whatever lies there, it counts as a number
          }
    }
    i32x4 p[PP][NT], seen[NT];
    f32x4 x[NT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int w = 0; w < N; ++w) {
        const i32x4 key = g[u].key(w);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = QP - 1; i >= 0; --i) x[n][u] = product(key, q[i][n][w], w == 0 && i == QP - 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : x[n][u]);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (EDGE) {
            const int place = 4 * quad + i, j = at + 16 * u + place;
            const bool see = place < upto[u] && j <= last[n] && (!a.window || j > last[n] - a.window);
            x[n][u][i] = see ? x[n][u][i] : -__builtin_inff();
            const int one = see ? 0x3f80 : 0, k = 2 * u + i / 2;
            seen[n][k] = i & 1 ? seen[n][k] | one << 16 : one;
          }
          top = fmaxf(top, x[n][u][i]);
        }
      top *= a.scale;
      // Taken before the branch: where a branch comes between a matrix instruction and the first use of its result, the compiler has left out
      // the wait that the instruction needs (tests/test_matrix_waits.py looks for that in the built library).
      asm volatile("" : "+v"(top));
      if (__ballot(top > m[n] + kRoom)) {
        const float best = max_of_row(top), higher = best > m[n] + kRoom ? best : m[n];  // (a row's own matter, whatever its neighbours do)
        const float by = m[n] == higher ? 1.f : __builtin_amdgcn_exp2f(m[n] - higher);
        m[n] = higher;
        l[n] *= by;
#pragma unroll
        for (int j = 0; j < S; ++j) o[n][j] *= by;
      }
      const float base = m[n] == -__builtin_inff() ? 0.f : -m[n];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[n][u][i] = __builtin_amdgcn_exp2f(fmaf(x[n][u][i], a.scale, base));
          l[n] += x[n][u][i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          unsigned parts[PP];
          split_pair<PP>(x[n][u][2 * i], x[n][u][2 * i + 1], parts);
#pragma unroll
          for (int k = 0; k < PP; ++k) p[k][n][2 * u + i] = (int)parts[k];
        }
      }
    }
    if constexpr (EDGE) {
      if (__ballot(nan)) {
        // A NaN that some rows see and others do not: rows that see it get it by a product of their own (a one for each
        // NaN value by a one for each token that is seen), and the value counts as zero below.
#pragma unroll
        for (int c = 0; c < N; ++c) {
          i32x4 is_nan{};
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              is_nan[2 * u + i / 2] |= (g[u].vs[neighbours(D) ? 0 : c] >> (8 * i) & 255u) == 255u ? 0x3f80 << (16 * (i & 1)) : 0;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const f32x4 hit = product(is_nan, seen[n], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float add = hit[i] > 0.f ? __builtin_nanf("") : 0.f;
              o[n][2 * c][i] += add;
              o[n][2 * c + 1][i] += add;
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int c = 0; c < VS; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if ((g[u].vs[c] >> (8 * i) & 255u) == 255u) g[u].vs[c] = (g[u].vs[c] & ~(255u << (8 * i))) | 127u << (8 * i);
      }
    }
#pragma unroll
    for (int c = 0; c < N; ++c) {
      i32x4 even, odd;
      g[0].values(c, 0, even, odd);
      g[1].values(c, 2, even, odd);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = PP - 1; k >= 0; --k) {
          o[n][2 * c] = product(even, p[k][n], o[n][2 * c]);
          o[n][2 * c + 1] = product(odd, p[k][n], o[n][2 * c + 1]);
        }
    }
  }
};

// The pages of a step's two granules: -1 for one behind the newest token or outside of the pool.
struct Pages { int page[2]; };
__device__ inline unsigned page_index(const Attend& a, unsigned granule) { return a.page_magic ? __umulhi(granule, a.page_magic) : granule; }

// SHARED: the workgroup's waves take the steps of one block of rows in turn and join their outputs; else each has its own block.
// (Two waves a SIMD at least: with 256 registers or fewer the products' sums stay in ordinary registers, not in those that have to be copied for the rest.)
template <int TYPE, int D, int NT, bool SHARED>
__global__ __launch_bounds__(256, 2) void attend_kernel(Attend a) {
  using T = typename Elem<TYPE>::type;
  constexpr int S = D / 16, W = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, quad = lane >> 4;
  int id = blockIdx.x;
  const int chunk = id % a.chunks;
  id /= a.chunks;
  // (kv heads first: the blocks of rows of one kv head are a multiple of 8 workgroups apart where there are 8, 16, .. kv heads, on one of the eight
  // dies, whose cache then holds this kv head's tokens; the last rows first, which see the most)
  const int kv = id % a.kv_heads;
  id /= a.kv_heads;
  const int s = id % a.sequences, group = id / a.sequences;
  const int block = SHARED ? group : ((a.blocks + W - 1) / W - 1 - group) * W + wave;
  const Sequence seq = sequence_of(a, s);
  const int all = min(seq.rows, a.most_rows) * a.group, r0 = block * (16 * NT);
  const int left = all - r0;  // rows of this block and those behind it
  if (SHARED && (left <= 0 || (chunk > 0 && seq.base + chunk * a.chunk >= seq.length))) return;
  if (!SHARED && left <= 0) return;

  // the block's query tokens, and the tokens that some of its rows sees
  const int t0 = r0 / a.group, t1 = min(r0 + 16 * NT - 1, all - 1) / a.group;
  const int p0 = seq.length - seq.rows;  // position of row 0
  int from = seq.base + chunk * a.chunk, to = min(from + a.chunk, min(p0 + t1, seq.length - 1) + 1);
  if (a.window) from = max(from, max(p0 + t0 - a.window + 1, 0) & ~(kStep - 1));

  Rows<TYPE, D, NT> rows;
  rows.begin(a, seq, kv, r0, all, lane);

  const int* table = a.table + s * a.ldt;
  const uint8_t* head = a.data + (int64_t)kv * a.granules * (17 * D);
  auto pages_of = [&](int at) {
    Pages p;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      p.page[u] = -1;
      if (at + 16 * u < seq.length) {
        const int page = table[page_index(a, (unsigned)at / 16 + u)];
        if ((unsigned)page < (unsigned)a.pages) p.page[u] = page;
      }
    }
    return p;
  };
  auto load = [&](Granule<D> (&g)[2], int at, const Pages& p) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const unsigned granule = (unsigned)at / 16 + u, in_page = granule - page_index(a, granule) * a.granules;
      g[u].load(head + (int64_t)max(p.page[u], 0) * a.page_bytes + in_page * (17 * D), lane);
    }
  };
  constexpr int kStride = SHARED ? W * kStep : kStep;
  const int start = from + (SHARED ? wave * kStep : 0);
  // First the steps whose tokens all rows of the block see, as long as their pages are in the pool: two in turn, so that one's loads are under way while
  // the other is worked on, and the pages' numbers for the next while these loads are asked for.
  int at = start;
  if (a.window && at <= p0 + t1 - a.window) at += (p0 + t1 - a.window - at) / kStride * kStride + kStride;
  const int first = at, end = min(to, p0 + t0 + 1) - kStep;  // the last of these steps begins there or before
  if (at <= end) {
    Granule<D> even[2], odd[2];
    Pages pages = pages_of(at);
    const int full[2] = {16, 16};
    auto good = [](const Pages& p) { return p.page[0] >= 0 && p.page[1] >= 0; };
    if (good(pages)) {
      load(even, at, pages);
      pages = pages_of(at + kStride);
      for (;;) {
        const bool more = at + kStride <= end && good(pages);
        if (more) {
          load(odd, at + kStride, pages);
          pages = pages_of(at + 2 * kStride);
        }
        rows.template step<false>(a, even, at, full, lane);
        at += kStride;
        if (!more) break;
        const bool again = at + kStride <= end && good(pages);
        if (again) {
          load(even, at + kStride, pages);
          pages = pages_of(at + 2 * kStride);
        }
        rows.template step<false>(a, odd, at, full, lane);
        at += kStride;
        if (!again) break;
      }
    }
  }
  // Then the others: at the rows' newest tokens, where a window begins, and all that come behind a page that is not in the pool.
  for (int rest = start; rest < to; rest += kStride) {
    if (rest >= first && rest < at) {
      rest = at - kStride;
      continue;
    }
    Granule<D> g[2];
    const Pages pages = pages_of(rest);
    load(g, rest, pages);
    int upto[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) upto[u] = pages.page[u] < 0 ? 0 : min(seq.length - rest - 16 * u, 16);
    rows.template step<true>(a, g, rest, upto, lane);
  }

#pragma unroll
  for (int n = 0; n < NT; ++n) rows.l[n] = sum_of_row(rows.l[n]);

  // outputs of row r of the block: of this workgroup's chunk or, if that is all, finished
  auto finish = [&](int r, int element, float v, float top, float sum) {
    const int t = (r0 + r) / a.group, h = kv * a.group + r0 + r - t * a.group;
    if (SHARED && a.part) {
      const int64_t row = (int64_t)(seq.begin + t) * a.heads + h, at = row * a.chunks + chunk;
      a.part[2 * (int64_t)a.chunks * a.rows * a.heads + at * D + element] = v;
      if (element == 0) a.part[2 * at] = top, a.part[2 * at + 1] = sum;
    } else {
      static_cast<T*>(a.y)[(int64_t)(seq.begin + t) * a.ldy + (int64_t)h * D + element] = (T)(sum == 0.f ? 0.f : v / sum);
    }
  };
  if constexpr (SHARED) {
    __shared__ float out[W][NT * 16][D + 1];
    __shared__ float tops[W][NT * 16], sums[W][NT * 16];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (quad == 0) tops[wave][n * 16 + r16] = rows.m[n], sums[wave][n * 16 + r16] = rows.l[n];
#pragma unroll
      for (int j = 0; j < S; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) out[wave][n * 16 + r16][element_of<D>(j, 4 * quad + i)] = rows.o[n][j][i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < min(left, 16 * NT) * D; e += 256) {
      const int r = e / D, element = e - r * D;
      float top = tops[0][r];
#pragma unroll
      for (int w = 1; w < W; ++w) top = fmaxf(top, tops[w][r]);
      float v = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float by = tops[w][r] == top ? 1.f : __builtin_amdgcn_exp2f(tops[w][r] - top);
        v += out[w][r][element] * by;
        sum += sums[w][r] * by;
      }
      finish(r, element, v, top, sum);
    }
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n)
      if (n * 16 + r16 < left) {
#pragma unroll
        for (int j = 0; j < S; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) finish(n * 16 + r16, element_of<D>(j, 4 * quad + i), rows.o[n][j][i], rows.m[n], rows.l[n]);
      }
  }
}

// Chunks' outputs joined: a workgroup has a row and head, a wave of it every fourth chunk.
template <int TYPE>
__global__ __launch_bounds__(256) void join_kernel(Attend a, int head) {
  using T = typename Elem<TYPE>::type;
  constexpr int W = 4;
  __shared__ float out[W][kCacheHead];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int each = a.most_rows * a.heads, s = blockIdx.x / each, t = (blockIdx.x - s * each) / a.heads, h = blockIdx.x - s * each - t * a.heads;
  const Sequence seq = sequence_of(a, s);
  if (t >= seq.rows) return;
  const int64_t row = (int64_t)(seq.begin + t) * a.heads + h;
  // (chunks past the sequence's newest token are not written)
  const int chunks = min(a.chunks, (max(seq.length - seq.base, 0) + a.chunk - 1) / a.chunk);
  const float2* tops = reinterpret_cast<const float2*>(a.part) + row * a.chunks;
  const float* part = a.part + 2 * (int64_t)a.chunks * a.rows * a.heads + row * a.chunks * head;
  float top = -__builtin_inff();
  for (int c = lane; c < chunks; c += 64) top = fmaxf(top, tops[c].x);
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    float by = 0.f;
    if (c0 + lane < chunks) {
      const float2 of = tops[c0 + lane];
      by = of.x == top ? 1.f : __builtin_amdgcn_exp2f(of.x - top);
      sum += of.y * by;
    }
    const int end = min(chunks - c0, 64);
    for (int c = wave; c < end; c += W) {
      const float w = __shfl(by, c);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < head) v[i] += part[(int64_t)(c0 + c) * head + lane + 64 * i] * w;
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < head) out[wave][lane + 64 * i] = v[i];
  __syncthreads();
  T* y = static_cast<T*>(a.y) + (int64_t)(seq.begin + t) * a.ldy + (int64_t)h * head;
  if ((int)threadIdx.x < head) {
    float all = out[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < W; ++w) all += out[w][threadIdx.x];
    y[threadIdx.x] = (T)(sum == 0.f ? 0.f : all / sum);
  }
}

// Most row tiles of a wave: as many as its registers hold (q and outputs of a tile).
constexpr int most_tiles(int parts, int head) { return head <= 128 && parts * head / 8 + head / 4 <= 64 ? 2 : 1; }
template <int TYPE, int D>
constexpr int kMostTiles = most_tiles(kParts<TYPE>, D);

// How a call is cut: by its sizes alone, so that its workspace can be made ahead.
struct Cut { int tiles; bool shared; int blocks, chunk, chunks; size_t space; };
Cut cut_of(const tetris_cache* c, const tetris_attention* a, int type) {
  Cut k{};
  const int group = a->heads / c->kv_heads;
  const int64_t rows = (int64_t)std::min(a->most_rows, a->rows) * group, units = (int64_t)a->sequences * c->kv_heads;
  k.tiles = most_tiles(parts_of(type), c->head);
  const int64_t own = (rows + 64 * k.tiles - 1) / (64 * k.tiles);  // workgroups of four blocks
  k.shared = rows <= 32 || units * own < 256;
  if (rows <= 16) k.tiles = 1;
  k.blocks = (int)((rows + 16 * k.tiles - 1) / (16 * k.tiles));
  const int64_t span = a->window ? std::min<int64_t>(a->most_length, (int64_t)a->window + a->most_rows + kStep) : a->most_length;
  int64_t chunks = 1;
  // about 1024 workgroups, of at least two steps a wave
  if (k.shared) chunks = std::max<int64_t>(1, std::min<int64_t>(1024 / std::max<int64_t>(units * k.blocks, 1), (span + 8 * kStep - 1) / (8 * kStep)));
  k.chunk = (int)(((span + chunks - 1) / chunks + 4 * kStep - 1) / (4 * kStep) * (4 * kStep));
  if (k.chunk == 0) k.chunk = 4 * kStep;
  k.chunks = (int)std::max<int64_t>(1, (span + k.chunk - 1) / k.chunk);
  if (k.chunks > 1) k.space = (size_t)k.chunks * a->rows * a->heads * (c->head + 2) * sizeof(float);
  return k;
}

template <int TYPE, int D>
int launch(Attend a, const Cut& k, hipStream_t s) {
  const int64_t groups = (int64_t)k.chunks * a.kv_heads * a.sequences * (k.shared ? k.blocks : ceil_div(k.blocks, 4));
  const int64_t joined = k.chunks > 1 ? (int64_t)a.sequences * a.most_rows * a.heads : 0;
  if (std::max(groups, joined) > 0x7fffffff) return fail(TETRIS_EUNSUPPORTED, "%lld workgroups are more than a launch has", (long long)std::max(groups, joined));
  const dim3 grid((unsigned)groups), block(256);
  if (!k.shared) hipLaunchKernelGGL((attend_kernel<TYPE, D, kMostTiles<TYPE, D>, false>), grid, block, 0, s, a);
  else if (k.tiles == 1) hipLaunchKernelGGL((attend_kernel<TYPE, D, 1, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((attend_kernel<TYPE, D, kMostTiles<TYPE, D>, true>), grid, block, 0, s, a);
  TETRIS_HIP(hipGetLastError());
  if (joined) {
    hipLaunchKernelGGL((join_kernel<TYPE>), dim3((unsigned)joined), block, 0, s, a, D);
    TETRIS_HIP(hipGetLastError());
  }
  return TETRIS_OK;
}
template <int TYPE>
int by_head(int head, const Attend& a, const Cut& k, hipStream_t s) {
  switch (head) {
    case 32: return launch<TYPE, 32>(a, k, s);
    case 64: return launch<TYPE, 64>(a, k, s);
    case 96: return launch<TYPE, 96>(a, k, s);
    case 128: return launch<TYPE, 128>(a, k, s);
    case 160: return launch<TYPE, 160>(a, k, s);
    case 192: return launch<TYPE, 192>(a, k, s);
    case 224: return launch<TYPE, 224>(a, k, s);
    default: return launch<TYPE, 256>(a, k, s);
  }
}

int check_attention(const tetris_cache* c, const tetris_attention* a, int type) {
  if (!c || !a) return fail(TETRIS_EINVAL, "null argument");
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (a->heads <= 0 || a->heads % c->kv_heads || a->heads > kCacheHeads)
    return fail(TETRIS_EINVAL, "%d heads over %d kv heads (a multiple of them, up to %d)", a->heads, c->kv_heads, kCacheHeads);
  if (a->sequences < 0 || a->rows < 0 || a->most_rows < 0 || a->most_length < 0 || a->window < 0)
    return fail(TETRIS_EINVAL, "%d sequences, %d rows (at most %d each), %d tokens, window %d", a->sequences, a->rows, a->most_rows, a->most_length, a->window);
  if (a->most_length > kCacheLength || a->rows > 0x40000000 / a->heads) return fail(TETRIS_EINVAL, "%d rows of %d heads, %d tokens (up to 2^30 and 2^28)", a->rows, a->heads, a->most_length);
  return TETRIS_OK;
}

}  // namespace
}  // namespace tetris

using namespace tetris;

extern "C" int tetris_cache_prepare(tetris_cache* c, const tetris_attention* a, int type, void* stream) {
  int rc = check_attention(c, a, type);
  if (!rc) rc = check_cache(c);
  if (rc) return rc;
  uint8_t* d;
  return c->space.get(static_cast<hipStream_t>(stream), cut_of(c, a, type).space, &d);
}

extern "C" int tetris_cache_attend(tetris_cache* c, const tetris_attention* a, const void* d_q, int64_t ldq, int type, const int32_t* d_first,
                                   const int32_t* d_length, const int32_t* d_table, int64_t ld_table, void* d_y, int64_t ldy, void* stream) {
  int rc = check_attention(c, a, type);
  if (rc) return rc;
  const int64_t width = (int64_t)a->heads * c->head;
  if (ldq < width || ldy < width)
    return fail(TETRIS_EINVAL, "leading dimension %lld below the %lld elements of a row", (long long)std::min(ldq, ldy), (long long)width);
  if (!d_first && a->rows != a->sequences) return fail(TETRIS_EINVAL, "%d rows of %d sequences without their offsets", a->rows, a->sequences);
  if (a->rows == 0 || a->sequences == 0 || a->most_rows == 0) return TETRIS_OK;
  const int entries = ceil_div(a->most_length, c->page);
  if (ld_table < entries) return fail(TETRIS_EINVAL, "table: leading dimension %lld below the %d pages of %d tokens", (long long)ld_table, entries, a->most_length);
  if (!d_q || !d_y || !d_length || (!d_table && entries)) return fail(TETRIS_EINVAL, "null argument");
  if ((reinterpret_cast<size_t>(d_q) | reinterpret_cast<size_t>(d_y)) % elem_size(type)) return fail(TETRIS_EINVAL, "rows not aligned to their elements");
  if ((reinterpret_cast<size_t>(d_first) | reinterpret_cast<size_t>(d_length) | reinterpret_cast<size_t>(d_table)) & 3)
    return fail(TETRIS_EINVAL, "offsets, lengths or table not aligned to their elements");
  if (d_q == d_y) return fail(TETRIS_EINVAL, "the output is the input");
  if ((rc = check_cache(c))) return rc;
  const Cut k = cut_of(c, a, type);
  uint8_t* d = nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if ((rc = c->space.get(s, k.space, &d))) return rc;
  Attend t{};
  t.data = c->data; t.q = d_q; t.y = d_y;
  t.first = d_first; t.length = d_length; t.table = d_table;
  t.part = reinterpret_cast<float*>(d);
  t.page_bytes = c->page_bytes; t.ldt = ld_table; t.ldq = ldq; t.ldy = ldy;
  t.pages = c->pages; t.page = c->page; t.granules = c->page / kGranule;
  t.kv_heads = c->kv_heads; t.heads = a->heads; t.group = a->heads / c->kv_heads;
  t.sequences = a->sequences; t.rows = a->rows; t.most_rows = std::min(a->most_rows, a->rows); t.most_length = a->most_length;
  t.window = std::min(a->window, a->most_length);
  t.blocks = k.blocks; t.chunk = k.chunk; t.chunks = k.chunks;
  const int size = elem_size(type);
  t.whole = (reinterpret_cast<size_t>(d_q) & 15) == 0 && ldq * size % 16 == 0;
  t.scale = a->scale == 0.f ? 1.f : std::fabs(a->scale) * 1.44269504088896340736f;
  t.sign = a->scale == 0.f ? 0.f : a->scale < 0.f ? -1.f : 1.f;
  t.page_magic = magic_reciprocal(t.granules);
  if (type == TETRIS_F32) return by_head<TETRIS_F32>(c->head, t, k, s);
  if (type == TETRIS_F16) return by_head<TETRIS_F16>(c->head, t, k, s);
  return by_head<TETRIS_BF16>(c->head, t, k, s);
}

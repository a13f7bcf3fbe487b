// Attention over a cache of keys and values in MX4 (include/tetris_attention.h), one pass over the cache with a running maximum and sum.
//
// A wave takes steps of 32 tokens of one kv head, for up to 16 NT rows: pairs (query token, head) that read this kv head.
//   scores    S^T [32 tokens][rows] = K q^T       v_mfma_f32_16x16x32_bf16 of keys made bf16 in registers, one instruction for two of them
//   weights   P = 2^(S - m), m a bound of the row's scores so far
//   outputs   O^T [elements][rows] += V^T P^T     the same instruction; the page's layout (csrc/cache.h) gives a lane the values of the tokens whose
//                                               weights it holds, so that weights go from one product to the next without leaving the lane
// A key or value has two significant bits and its scale's exponent: exact in bf16.  q comes in 1, 2 or 3 bf16 parts (bf16, f16, f32), which hold
// all of its bits.  P comes in three for f32, which hold all of it, else in two, within 2^-16 of it (attend_prompt_kernel has one f16 for bf16, within 2^-11):
// a product an output costs less, and an output of f16 or bf16 is rounded by up to 2^-11 or 2^-8.  Sums, the softmax's statistics and outputs are of 32 bits until then.
// m is raised only to a score that is more than 8 above it (weights are at most 2^8, far from overflow); most steps need no exchange
// between lanes for it.  A row's sum stays apart in four lanes until the end.
//
// One token a sequence is bound by the cache's bytes: 64 sequences of 8192 tokens by 8 kv heads of 128 (570 MB) take 122 us with the joining, 4.7 TB/s, where a
// copy reaches 4.9; of up to 8192 tokens, 3700 on average (259 MB), 61.  Small calls are bound by their chain: page number, granule, two products with the
// softmax between them, the waves' join, the chunks' join: 4000 tokens 7 + 4 us.
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
  float* part;  // [2 workgroups][16 NT rows]: maximum and sum, then outputs (struct Slot)
  int2* shares; // of a unit: the first workgroup that has some of it, and how many have
  int64_t page_bytes, ldt, ldq, ldy;
  int pages, granules, kv_heads, group, sequences, rows, most_rows, most_length, window;
  int tiles;   // NT
  int blocks;  // most blocks of 16 NT rows of a sequence and kv head
  int workgroups;
  int chunk, chunks;  // quanta of a workgroup, or zero for equal shares; most chunks of a unit
  int whole, y_whole;  // rows of q, of y lie on 16 bytes
  unsigned page_magic;  // to divide by granules (0 where that is one)
  float scale;  // to powers of two, not negative
  float sign;  // what q is multiplied by: scale's sign, or zero where scale is
};

// What nothing writes while a kernel runs, from an address that is the wave's: by the scalar unit, also behind barriers and stores, where the compiler
// would not take it for unchanged.
template <typename V>
__device__ inline V fixed(const V* p) { return *(const __attribute__((address_space(4))) V*)(reinterpret_cast<uintptr_t>(p)); }

// What a sequence is: its rows and tokens, whatever the arrays hold.
struct Sequence { int begin, rows, length, base; };
__device__ inline Sequence sequence_from(const Attend& a, int s, int first, int behind, int length) {
  Sequence q;
  q.begin = a.first ? min(max(first, 0), a.rows) : s;
  const int end = a.first ? min(max(behind, q.begin), a.rows) : s + 1;
  q.rows = end - q.begin;
  q.length = min(max(length, 0), a.most_length);
  // the first token that any row sees, down to a whole step
  q.base = a.window ? max(q.length - q.rows - a.window + 1, 0) & ~(kStep - 1) : 0;
  return q;
}
__device__ inline Sequence sequence_of(const Attend& a, int s) {  // the wave's
  return sequence_from(a, s, a.first ? fixed(a.first + s) : 0, a.first ? fixed(a.first + s + 1) : 0, fixed(a.length + s));
}
__device__ inline Sequence sequence_of_lane(const Attend& a, int s) {
  return sequence_from(a, s, a.first ? a.first[s] : 0, a.first ? a.first[s + 1] : 0, a.length[s]);
}

template <int TYPE>
constexpr int kParts = TYPE == TETRIS_BF16 ? 1 : TYPE == TETRIS_F16 ? 2 : 3;
template <int TYPE>
constexpr int kWeightParts = TYPE == TETRIS_F32 ? 3 : 2;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

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
__device__ inline unsigned half_at(unsigned codes, float scale, int i) {  // to f16
  switch (i) {
    case 0: return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0));
    case 1: return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1));
    case 2: return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2));
    default: return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3));
  }
}
__device__ inline float scale_of(unsigned word, int byte) { return __uint_as_float((word >> (8 * byte) & 255u) << 23); }
__device__ inline f32x4 product(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ inline f32x4 half_product(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
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
  f32x4 sums[NT];  // of weights multiplied as f16, the whole row's in every element
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
    }
    reset();
  }
  __device__ inline void reset() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -__builtin_inff();
      l[n] = 0.f;
      sums[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < S; ++j) o[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // whether the lane's row sees token 4 (lane / 16) + i of granule u
  template <int G>
  __device__ inline bool sees(const Attend& a, int n, int u, int i, int at, const int (&upto)[G], int lane) const {
    const int place = 4 * (lane >> 4) + i, j = at + 16 * u + place;
    return place < upto[u] && j <= last[n] && (!a.window || j > last[n] - a.window);
  }
  // what the rows do not see of G granules out of their scores
  template <int G>
  __device__ inline void mask(const Attend& a, f32x4 (&x)[NT][G], int at, const int (&upto)[G], int lane) const {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int u = 0; u < G; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][u][i] = sees(a, n, u, i, at, upto, lane) ? x[n][u][i] : -__builtin_inff();
  }
  // ones for what they see of granules 2 h and 2 h + 1, in the form of a product's second operand
  template <int G>
  __device__ inline i32x4 seen(const Attend& a, int n, int h, int at, const int (&upto)[G], int lane) const {
    i32x4 ones{};
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) ones[2 * u + i / 2] |= sees(a, n, 2 * h + u, i, at, upto, lane) ? 0x3f80 << (16 * (i & 1)) : 0;
    return ones;
  }

  // Scores of 32 tokens (lane 16 g + r has tokens 4 g .. 4 g + 3 of each granule for row r) to weights in parts, with the sums and the bounds m brought up to
  // date.
  __device__ inline void weights(const Attend& a, f32x4 (&x)[NT][2], i32x4 (&p)[PP][NT]) {
    raise(a, x);
    parts(a, x, p);
  }
  __device__ inline void parts(const Attend& a, f32x4 (&x)[NT][2], i32x4 (&p)[PP][NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
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
  }
  // the bounds m up to these scores, and the sums and outputs to the bounds
  template <int G>
  __device__ inline void raise(const Attend& a, const f32x4 (&x)[NT][G]) {
    float top[NT];
    bool above = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      top[n] = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < G; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[n] = fmaxf(top[n], x[n][u][i]);
      top[n] *= a.scale;
      // Taken before the branch: where a branch comes between a matrix instruction and the first use of its result, the compiler has left out
      // the wait that the instruction needs (tests/test_matrix_waits_of_every_kernel.py looks for that in the built library).
      asm volatile("" : "+v"(top[n]));
      above = above || top[n] > m[n] + kRoom;
    }
    if (__ballot(above)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float best = max_of_row(top[n]), higher = best > m[n] + kRoom ? best : m[n];  // (a row's own matter, whatever its neighbours do)
        const float by = m[n] == higher ? 1.f : __builtin_amdgcn_exp2f(m[n] - higher);
        m[n] = higher;
        l[n] *= by;
        sums[n] *= by;
#pragma unroll
        for (int j = 0; j < S; ++j) o[n][j] *= by;
      }
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
    i32x4 p[PP][NT];
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
    if constexpr (EDGE) mask(a, x, at, upto, lane);
    weights(a, x, p);
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
            const f32x4 hit = product(is_nan, seen(a, n, 0, at, upto, lane), f32x4{0.f, 0.f, 0.f, 0.f});
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

// How the work is dealt out.  A unit is a block of 16 NT rows of a sequence and kv head; it is as many quanta of four steps as its sequence
// tokens that its rows see (one at least: rows that see nothing become zeros).  What a workgroup does of a unit that it does not do all of it leaves to join_kernel.
//   little work     a.chunk quanta of one unit each; chunks that a sequence is too short for end at once.  It begins without looking at the
//                   other sequences: one token of 4000 tokens by 32 heads takes 11 us in place of 13.  A chunk goes by most_length, which
//                   may be far more than there is: the same in a call made for 131072 tokens takes 17, with 32 kv heads 36 in place of 12.
//   much work       the units' quanta, sequence after sequence, in equal shares, whatever the lengths are: 64 sequences of up to 8192 tokens, 3700 on
//                   average, take 61 us (68 in place of 86 when both were measured).
constexpr int kQuantum = 4 * kStep;
constexpr int kBegin = 3;  // quanta's time that a unit takes besides: queries, the first loads, joining the waves' outputs
struct Units { int quanta, blocks; };
__device__ inline Units units_of(const Attend& a, const Sequence& q) {
  const int count = min(q.rows, a.most_rows), rows = count * a.group, size = 16 * a.tiles;
  const int seen = q.length - q.rows + count - q.base;  // (up to the last row that is worked on: no more than the launch is cut for, with a window too)
  return {max((seen + kQuantum - 1) / kQuantum, 1), (rows + size - 1) / size};
}
__device__ inline int quanta_of(const Attend& a, int s) {
  if (s >= a.sequences) return 0;
  const Units u = units_of(a, sequence_of_lane(a, s));
  return (u.quanta + kBegin) * u.blocks * a.kv_heads;
}

// the sums of v over the lanes up to this one
__device__ inline int sums_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // from 1, 2, 4 and 8 lanes below in rows of sixteen
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // a row's last to the next row, the second row's to the upper half
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

// Where a workgroup leaves a unit's rows: its last unit, if that goes on behind it, has slot 2 w + 1, and one that began before it 2 w.
struct Slot {
  float* top;  // [rows][2]
  float* out;  // [rows][elements]
};
__device__ inline Slot slot_of(const Attend& a, int slot, int head) {
  const int rows = 16 * a.tiles;
  return {a.part + (int64_t)slot * rows * 2, a.part + 4 * (int64_t)a.workgroups * rows + (int64_t)slot * rows * head};
}

// `count` quanta of a unit from its quantum `skip` on, by a workgroup; parts: how many workgroups have some of the unit.
template <int TYPE, int D, int NT>
__device__ inline void attend_unit(const Attend& a, const Sequence& seq, int quanta, int s, int kv, int block, int skip, int count, int parts) {
  using T = typename Elem<TYPE>::type;
  constexpr int S = D / 16, W = 4, kStride = W * kStep;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (what is computed from it is computed here, and not kept in registers from one unit to the next)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, quad = lane >> 4;
  __shared__ float out[W][NT * 16][D + 1];
  __shared__ float tops[W][NT * 16], sums[W][NT * 16];
  const int all = min(seq.rows, a.most_rows) * a.group, r0 = block * (16 * NT);
  const int left = all - r0;  // rows of this block and those behind it

  // the block's query tokens, and the tokens that some of its rows sees
  const int t0 = r0 / a.group, t1 = min(r0 + 16 * NT - 1, all - 1) / a.group;
  const int p0 = seq.length - seq.rows;  // position of row 0
  int from = seq.base + skip * kQuantum;
  const int to = min(from + count * kQuantum, min(p0 + t1, seq.length - 1) + 1);
  if (a.window) from = max(from, max(p0 + t0 - a.window + 1, 0) & ~(kStep - 1));

  const int* table = a.table + s * a.ldt;
  const uint8_t* head = a.data + (int64_t)kv * a.granules * (17 * D);
  auto pages_of = [&](int at) {
    Pages p;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // (read wherever the table has an entry, so that it need not wait for the sequence's length)
      const int page = fixed(table + page_index(a, (unsigned)min(at + 16 * u, a.most_length - 1) / 16));
      p.page[u] = at + 16 * u < seq.length && (unsigned)page < (unsigned)a.pages ? page : -1;
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
  const int begin = from + wave * kStep;
  // First the steps whose tokens all rows of the block see, as long as their pages are in the pool: two in turn, so that one's loads are under way
  // while the other is worked on, and the pages' numbers for the next while these loads are asked for.  What comes behind them is loaded ahead as well.
  int now = begin;
  if (a.window && now <= p0 + t1 - a.window) now += (p0 + t1 - a.window - now) / kStride * kStride + kStride;
  const int first = now, end = min(to, p0 + t0 + 1) - kStep;  // the last of these steps begins there or before
  Granule<D> even[2], odd[2];
  Pages pages = {-1, -1}, ahead;  // of the step at `now`, of the next
  const int full[2] = {16, 16};
  auto good = [](const Pages& p) { return p.page[0] >= 0 && p.page[1] >= 0; };
  if (now < to) {
    pages = pages_of(now);
    load(even, now, pages);
  }
  Rows<TYPE, D, NT> rows;
  rows.begin(a, seq, kv, r0, all, lane);
  if (now <= end && good(pages)) {
    ahead = pages_of(now + kStride);
    for (;;) {
      if (now + kStride < to) load(odd, now + kStride, ahead);
      pages = ahead;
      ahead = pages_of(now + 2 * kStride);
      rows.template step<false>(a, even, now, full, lane);
      now += kStride;
      if (now > end || !good(pages)) {
        even[0] = odd[0];
        even[1] = odd[1];
        break;
      }
      if (now + kStride < to) load(even, now + kStride, ahead);
      pages = ahead;
      ahead = pages_of(now + 2 * kStride);
      rows.template step<false>(a, odd, now, full, lane);
      now += kStride;
      if (now > end || !good(pages)) break;
    }
  }
  // Then the others: at the rows' newest tokens, where a window begins, and all that come behind a page that is not in the pool.
  bool loaded = now < to, wrapped = false;
  for (;; now += kStride) {
    if (!wrapped && now >= to) wrapped = true, now = begin;
    if (wrapped && now >= min(first, to)) break;
    if (!loaded) {
      pages = pages_of(now);
      load(even, now, pages);
    }
    loaded = false;
    int upto[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) upto[u] = pages.page[u] < 0 ? 0 : min(seq.length - now - 16 * u, 16);
    rows.template step<true>(a, even, now, upto, lane);
  }

  // the waves' outputs joined, to the output or to a slot
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float sum = sum_of_row(rows.l[n]);
    if (quad == 0) tops[wave][n * 16 + r16] = rows.m[n], sums[wave][n * 16 + r16] = sum;
#pragma unroll
    for (int j = 0; j < S; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) out[wave][n * 16 + r16][element_of<D>(j, 4 * quad + i)] = rows.o[n][j][i];
  }
  __syncthreads();
  const bool whole = count == quanta;
  const Slot slot = slot_of(a, 2 * blockIdx.x + (skip == 0), D);
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
    if (whole) {
      const int t = (r0 + r) / a.group, h = kv * a.group + r0 + r - t * a.group;
      static_cast<T*>(a.y)[(int64_t)(seq.begin + t) * a.ldy + (int64_t)h * D + element] = (T)(sum == 0.f ? 0.f : v / sum);
    } else {
      slot.out[r * D + element] = v;
      if (element == 0) slot.top[2 * r] = top, slot.top[2 * r + 1] = sum;
    }
  }
  if (skip == 0 && threadIdx.x == 0) a.shares[((int64_t)s * a.kv_heads + kv) * a.blocks + block] = make_int2(blockIdx.x, parts);
}

// Waves of a SIMD, and so workgroups of a compute unit, that the registers of a wave leave room for.
constexpr int kResidentMost = 256 * 4;  // workgroups that run at once, for any of them
constexpr int waves_of(int parts, int head, int tiles) { return parts * tiles * head <= 64 ? 4 : tiles * head <= 128 && parts * tiles * head <= 256 ? 3 : 2; }
// (Two waves a SIMD at least: with 256 registers or fewer the products' sums stay in ordinary registers, not in those that have to be copied for the rest.
// 21 of the 94 forms keep some of theirs in memory for that: of f32 heads of 96 by two tiles and of 160 to 256, of f16 heads of 64 by two tiles (6 registers), of
// 192 to 256 and prompts of 128, of bf16 heads of 192 and 224.  f32 at 224 has the most, 263 and 320: 64 sequences of 4096 tokens by 4 kv heads take 309 us, at
// 256, with 105 and 43, 131, and 97 and 72 in bf16.)
template <int TYPE, int D, int NT>
__global__ __launch_bounds__(256, waves_of(kParts<TYPE>, D, NT)) void attend_chunks_kernel(Attend a) {
  int id = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x - id * a.chunks, s = id / (a.kv_heads * a.blocks);
  id -= s * (a.kv_heads * a.blocks);
  const int kv = id / a.blocks, block = id - kv * a.blocks, skip = chunk * a.chunk;
  const Sequence seq = sequence_of(a, s);
  const Units units = units_of(a, seq);
  if (block >= units.blocks || skip >= units.quanta) return;
  attend_unit<TYPE, D, NT>(a, seq, units.quanta, s, kv, block, skip, min(a.chunk, units.quanta - skip), (units.quanta + a.chunk - 1) / a.chunk);
}
template <int TYPE, int D, int NT>
__global__ __launch_bounds__(256, waves_of(kParts<TYPE>, D, NT)) void attend_shares_kernel(Attend a) {
  const int lane = threadIdx.x & 63;
  // this workgroup's share, and the sequence that it begins in
  const int mine = sums_upto(quanta_of(a, lane));
  int total = __builtin_amdgcn_readlane(mine, 63);
  for (int s0 = 64; s0 < a.sequences; s0 += 64) total += __builtin_amdgcn_readlane(sums_upto(quanta_of(a, s0 + lane)), 63);
  const int share = (total + a.workgroups - 1) / a.workgroups;
  int at = blockIdx.x * share;
  const int stop = min(at + share, total);
  if (at >= stop) return;
  int s = 0, start = 0;  // the sequence and its first quantum
  for (int s0 = 0; s0 < a.sequences; s0 += 64) {
    const int upto = s0 ? sums_upto(quanta_of(a, s0 + lane)) : mine;
    const unsigned long long behind = __ballot(start + upto > at);
    if (behind) {
      const int l = __builtin_ctzll(behind);
      s = s0 + l;
      start += l ? __builtin_amdgcn_readlane(upto, l - 1) : 0;
      break;
    }
    start += __builtin_amdgcn_readlane(upto, 63);
  }
  while (at < stop) {
    const Sequence seq = sequence_of(a, s);
    const Units units = units_of(a, seq);
    if (units.blocks) {
      const int cost = units.quanta + kBegin, unit = (at - start) / cost, into = at - start - unit * cost, kv = unit / units.blocks;
      const int mine = min(cost - into, stop - at), skip = max(into - kBegin, 0), count = max(into + mine - kBegin, 0) - skip;
      if (count > 0) {
        attend_unit<TYPE, D, NT>(a, seq, units.quanta, s, kv, unit - kv * units.blocks, skip, count, (at - into + cost - 1) / share - (int)blockIdx.x + 1);
        __syncthreads();
      }
      at += mine;
    }
    if (at - start == (units.quanta + kBegin) * units.blocks * a.kv_heads) start = at, ++s;
  }
}

// All waves' writes to LDS are done; loads from memory may be under way (__syncthreads would wait for them too).
__device__ inline void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Many rows of a sequence (prompts, drafts of many tokens).  Four waves, each with 16 NT rows of its own, share what is made of the keys and values of 64
// tokens: each makes a quarter of it bf16, in the form in which the products take it, and leaves it in LDS (8 KiB for 32 elements of a head, twice, so that
// one barrier a turn is enough).  Four prompts of 1030, 1791, 3917 and 4096 tokens, 32 by 8 heads of 128, take 373 us, 800 TFLOP/s of what their rows see.
// No unit is full: the products alone would take 145 us at the rate that a loop of them reaches, the vector instructions (softmax, conversions,
// addresses) 112, LDS 100; a wave needs them one after another, and the registers leave room for two waves a SIMD.
//
// A weight of bf16 operators enters the second product as f16, 2^7 as large as it is (2^15 at most), with values that are exact in f16: one
// product in place of two, and one conversion of a pair of weights in place of six instructions.  It is within 2^-11 of the weight, an eighth of what the
// output's own rounding may be off by, or within 2^-32 of the row's largest; a row's sum is of the weights as they are multiplied.  Where some
// values are beyond f16's range a workgroup begins again with bf16, and weights in two parts.
constexpr int kPromptWaves = 4, kTurn = 64, kShift = 7;
constexpr int kNan = 1, kBf16 = 2;
// Scales whose values are exact in f16: those are multiples of half the scale, and six times it at most; f16 has multiples of 2^-24 up to 65504.
constexpr unsigned kHalfLeast = 127 - 23, kHalfMost = 127 + 13;
__device__ inline bool has_nan(unsigned scales) { return (((scales & 0x7f7f7f7fu) + 0x01010101u) & scales & 0x80808080u) != 0; }
// whether one of four scales is outside of [kHalfLeast, kHalfMost]: bytes less kHalfLeast, and those above 36, by their borrows and carries
__device__ inline bool beyond_half(unsigned scales) {
  const unsigned low = (scales | 0x80808080u) - kHalfLeast * 0x01010101u;  // bit 7 stays where the low seven bits are not below 104
  const unsigned under = ~(low | scales) & 0x80808080u;                    // below 104
  const unsigned over = scales & ((scales & 0x7f7f7f7fu) + (0x7fu - (kHalfMost - 128)) * 0x01010101u) & 0x80808080u;  // above 140: 128 and more than 12
  return (under | over) != 0;
}
template <int D>
struct Share {
  static constexpr int N = D / 32, KS = neighbours(D) ? (D + 127) / 128 : N, VS = neighbours(D) ? 1 : N;
  static constexpr int VU = (N + 1) / 2;  // bytes of a token's values
  // the keys of granule `wave`; of the values of 32 tokens (the first or the last two granules, by the wave's lowest bit) every second byte from wave / 2 on
  unsigned k[N], ks[KS], v[2][N], vs[2][VS];

  __device__ inline void load(const uint8_t* g, const uint8_t* v0, const uint8_t* v1, int lane) {
    const int r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < N; ++i) k[i] = (reinterpret_cast<const unsigned*>(g) + i)[(unsigned)lane * N];
#pragma unroll
    for (int i = 0; i < KS; ++i) ks[i] = (g + 16 * D)[(unsigned)(r * N + (neighbours(D) ? q * D / 128 + i : (q * (D / 4) + 8 * i) / 32))];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t* from = u ? v1 : v0;
#pragma unroll
      for (int i = 0; i < N; ++i) v[u][i] = (reinterpret_cast<const unsigned*>(from + 8 * D) + i)[(unsigned)lane * N];
#pragma unroll
      for (int i = 0; i < VS; ++i) vs[u][i] = (reinterpret_cast<const unsigned*>(from + 16 * D + D / 2) + (neighbours(D) ? 0 : i))[(unsigned)(q * N + (neighbours(D) ? r * (D / 16) / 32 : 0))];
    }
  }
  // To LDS.  Values that are NaN are zeros there, and so are those behind the newest token, whatever they are.  forms: of 32 tokens, whether they have a NaN
  // (kNan; which ones: nan_of[token][block]) and whether values that are to be f16 (HALF) are not exact in it (kBf16).
  template <bool HALF>
  __device__ inline void store(i32x4* keys, i32x4* values, int* forms, uint8_t* nan_of, const int (&upto)[4], int wave, int lane) {
    const int half = wave & 1, c0 = wave >> 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = __uint_as_float(ks[neighbours(D) ? i / 4 : i] << 23);
      keys[(wave * N + i) * 64 + lane] = i32x4{(int)pair<0>(k[i], s), (int)pair<1>(k[i], s), (int)pair<2>(k[i], s), (int)pair<3>(k[i], s)};
    }
    const int there[2] = {half ? upto[2] : upto[0], half ? upto[3] : upto[1]};
    // whether some scale needs a closer look
    bool odd = false;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < VS; ++c) odd = odd || (HALF ? beyond_half(vs[u][c]) : has_nan(vs[u][c]));
    i32x4* to = values + half * 2 * N * 64 + lane;
    if (there[0] == 16 && there[1] == 16 && !__ballot(odd)) {
      if (c0 == 0 && lane == 0) forms[half] = 0;
      convert<false, HALF>(to, c0, {});
      return;
    }
    bool nan = false, wide = false;
    unsigned gone[2] = {};  // what counts as zero: bit 4 c + i for token i and the c-th word of scales
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < VS; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int token = 4 * (lane >> 4) + i;
          const unsigned scale = vs[u][c] >> (8 * i) & 255u;
          const bool in = token < there[u], is = in && scale == 255u;
          nan = nan || is;
          unsigned code = 0;  // (zeros have the least scale)
#pragma unroll
          for (int b = i * N + c; b < i * N + c + (VS > 1 ? 1 : N); ++b) code |= v[u][b / 4] >> (8 * (b % 4)) & 0x77u;
          wide = wide || (in && !is && code && (scale < kHalfLeast || scale > kHalfMost));
          if (c0 == 0) nan_of[(half * 32 + u * 16 + token) * N + (neighbours(D) ? (lane & 15) * (D / 16) / 32 : c)] = is;
          if (is || !in) gone[u] |= 1u << (4 * c + i);
        }
    const bool any = __ballot(nan) != 0, bf16 = HALF && __ballot(wide) != 0;  // (then what is left here is not read)
    if (c0 == 0 && lane == 0) forms[half] = (any ? kNan : 0) | (bf16 ? kBf16 : 0);
    convert<true, HALF>(to, c0, {gone[0], gone[1]});
  }
  template <bool SPECIAL, bool HALF>
  __device__ inline void convert(i32x4* to, int c0, uint2 gone) {
    unsigned codes[2][N];  // from byte c0 of the first token on
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) codes[u][i] = __builtin_amdgcn_alignbyte(i + 1 < N ? v[u][i + 1] : 0u, v[u][i], (unsigned)c0);
#pragma unroll
    for (int j = 0; j < VU; ++j) {
      const int c = c0 + 2 * j;
      if (c >= N) break;
      i32x4 even, odd;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned scales = neighbours(D) ? vs[u][0] : c0 && 2 * j + 1 < VS ? vs[u][2 * j + 1 < VS ? 2 * j + 1 : 0] : vs[u][2 * j];
        unsigned t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int b = i * N + 2 * j;
          const float scale = scale_of(scales, i);
          t[i] = HALF ? half_at(codes[u][b / 4], scale, b % 4) : pair_at(codes[u][b / 4], scale, b % 4);
          if (SPECIAL) t[i] = (u ? gone.y : gone.x) >> ((VS > 1 ? 4 * c : 0) + i) & 1u ? 0u : t[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          even[2 * u + i] = (int)__builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x05040100u);
          odd[2 * u + i] = (int)__builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x07060302u);
        }
      }
      to[2 * c * 64] = even;
      to[(2 * c + 1) * 64] = odd;
    }
  }
};

template <int TYPE, int D, int NT>
__global__ __launch_bounds__(64 * kPromptWaves, D <= 128 ? 2 : 1) void attend_prompt_kernel(Attend a) {
  using T = typename Elem<TYPE>::type;
  using R = Rows<TYPE, D, NT>;
  constexpr int N = D / 32, S = D / 16, W = kPromptWaves, QP = R::QP, PP = R::PP;
  __shared__ i32x4 keys[2][4 * N * 64], values[2][4 * N * 64];
  __shared__ int forms[2][2];
  __shared__ uint8_t nan_of[2][kTurn * N];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, quad = lane >> 4;
  // (kv heads first: the workgroups of one kv head are a multiple of 8 apart where there are 8, 16, .. kv heads, on one of the eight dies, whose cache then
  // holds this kv head's tokens; the last rows first, which see the most.  Sequences take turns in another order from one row of workgroups to the next: a die
  // deals its workgroups to its four shader engines in turn, each of which would have one sequence of four, however long they are)
  int id = blockIdx.x;
  const int kv = id % a.kv_heads;
  id /= a.kv_heads;
  const int turn = id / a.sequences, s = (int)((unsigned)(id + turn + turn / 4) % (unsigned)a.sequences), group = (a.blocks + W - 1) / W - 1 - turn;
  const Sequence seq = sequence_of(a, s);
  const int all = min(seq.rows, a.most_rows) * a.group, w0 = group * W * (16 * NT), r0 = w0 + wave * (16 * NT);
  if (w0 >= all) return;
  const int p0 = seq.length - seq.rows;
  // the tokens that some row of the workgroup sees, and of the wave
  auto span = [&](int first, int count, int& from, int& to) {
    const int t0 = first / a.group, t1 = min(first + count - 1, all - 1) / a.group;
    from = a.window ? max(p0 + t0 - a.window + 1, 0) : 0;
    to = first < all ? min(p0 + t1, seq.length - 1) + 1 : 0;
  };
  int from, to, mine_from, mine_to;
  span(w0, W * 16 * NT, from, to);
  span(r0, 16 * NT, mine_from, mine_to);
  from &= ~(kTurn - 1);
  const int t0 = r0 / a.group, t1 = min(r0 + 16 * NT - 1, all - 1) / a.group;

  const int* table = a.table + s * a.ldt;
  const uint8_t* head = a.data + (int64_t)kv * a.granules * (17 * D);
  Share<D> share;
  // Where 64 granules lie, a lane each, and which of them are there; and the pages of the 64 behind them, asked for early.
  int batch = 0, page_ahead = 0, offset_low = 0, offset_high = 0;
  unsigned long long there = 0;
  const int granules = (a.most_length + 15) / 16;  // that the table has pages for
  auto look_ahead = [&](int g) { page_ahead = table[page_index(a, (unsigned)min(g + lane, granules - 1))]; };
  auto turn_table = [&](int g0) {
    const int g = g0 + lane, index = (int)page_index(a, (unsigned)g);
    const bool good = g < granules && 16 * g < seq.length && (unsigned)page_ahead < (unsigned)a.pages;
    const int64_t offset = (good ? page_ahead : 0) * a.page_bytes + (g - index * a.granules) * (17 * D);
    offset_low = (int)offset;
    offset_high = (int)(offset >> 32);
    there = __ballot(good);
    batch = g0;
    look_ahead(g0 + 64);
  };
  auto ask = [&](int at) {  // for the wave's share of 64 tokens
    const int g = at / 16;
    if (g >= batch + 64) turn_table(g);
    auto granule = [&](int u) {
      const int l = g - batch + u;
      const int64_t offset = (int64_t)__builtin_amdgcn_readlane(offset_high, l) << 32 | (unsigned)__builtin_amdgcn_readlane(offset_low, l);
      return head + offset;
    };
    const int v = 2 * (wave & 1);
    share.load(granule(wave), granule(v), granule(v + 1), lane);
  };
  auto begin = [&] {
    if (from >= to) return;
    look_ahead(from / 16);
    turn_table(from / 16);
    ask(from);
  };
  begin();
  R rows;
  rows.begin(a, seq, kv, r0, all, lane);
  unsigned lost[NT] = {};  // outputs that are NaN: bit i for elements of row 4 (lane / 16) + i of all products, or 4 c + i for those of products 2 c and 2 c + 1
  // turns from plain_from on, up to plain_to, have tokens that all rows of the wave see
  const int plain_from = a.window ? p0 + t1 - a.window + 1 : 0, plain_to = p0 + t0 + 1 - kTurn;
  // All turns.  HALF: values and weights are multiplied as f16; false where some values are not exact in it.
  auto turns = [&](auto as_half) {
    constexpr bool HALF = decltype(as_half)::value;
    int buffer = 0;
    unsigned next = from < to ? (unsigned)(there >> (from / 16 - batch)) & 15u : 0u;  // which of the four granules asked for are there
    for (int at = from; at < to; at += kTurn, buffer ^= 1) {
      const unsigned here = next;
      const int behind = seq.length - at;
      int upto[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) upto[u] = here >> u & 1 ? min(behind - 16 * u, 16) : 0;
      share.template store<HALF>(keys[buffer], values[buffer], forms[buffer], nan_of[buffer], upto, wave, lane);
      if (at + kTurn < to) {
        ask(at + kTurn);
        next = (unsigned)(there >> ((at + kTurn) / 16 - batch)) & 15u;
      }
      lds_barrier();
      const int form[2] = {__builtin_amdgcn_readfirstlane(forms[buffer][0]), __builtin_amdgcn_readfirstlane(forms[buffer][1])};
      if (HALF && ((form[0] | form[1]) & kBf16)) return false;
      if (at >= mine_to || at + kTurn <= mine_from) continue;
      f32x4 x[NT][4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int w = 0; w < N; ++w) {
          const i32x4 key = keys[buffer][(u * N + w) * 64 + lane];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = QP - 1; i >= 0; --i) x[n][u] = product(key, rows.q[i][n][w], w == 0 && i == QP - 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : x[n][u]);
        }
      // (used before the branch: see Rows::raise)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int u = 0; u < 4; ++u) asm volatile("" : "+v"(x[n][u]));
      if (here != 15u || behind < kTurn || at < plain_from || at > plain_to) rows.mask(a, x, at, upto, lane);
      if ((form[0] | form[1]) & kNan) {
        // A NaN that some rows see and others do not: those that see it are found by a product of a one for each NaN value by a one for each token
        // that is seen.  The value itself is zero in LDS.
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (!(forms[buffer][h] & kNan)) continue;
          const int there[2] = {h ? upto[2] : upto[0], h ? upto[3] : upto[1]};
#pragma unroll
          for (int c = 0; c < (neighbours(D) ? 1 : N); ++c) {
            i32x4 ones{};
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                ones[2 * u + i / 2] |= nan_of[buffer][(h * 32 + u * 16 + 4 * quad + i) * N + (neighbours(D) ? r16 * (D / 16) / 32 : c)] ? 0x3f80 << (16 * (i & 1)) : 0;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const f32x4 hit = product(ones, rows.seen(a, n, 0, at + h * kStep, there, lane), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
              for (int i = 0; i < 4; ++i) lost[n] |= (hit[i] > 0.f ? 1u : 0u) << (4 * c + i);
            }
          }
        }
      }
      rows.raise(a, x);
      if constexpr (HALF) {
        i32x4 p[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float base = (float)kShift - (rows.m[n] == -__builtin_inff() ? 0.f : rows.m[n]);
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float v = __builtin_amdgcn_exp2f(fmaf(x[n][u][2 * i], a.scale, base)), w = __builtin_amdgcn_exp2f(fmaf(x[n][u][2 * i + 1], a.scale, base));
              p[n][u / 2][2 * (u % 2) + i] = __builtin_bit_cast(int, f16x2{(_Float16)v, (_Float16)w});
            }
        }
        const i32x4 ones = {0x3c003c00, 0x3c003c00, 0x3c003c00, 0x3c003c00};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int n = 0; n < NT; ++n) rows.sums[n] = half_product(ones, p[n][h], rows.sums[n]);
#pragma unroll
          for (int j = 0; j < S; ++j) {
            const i32x4 v = values[buffer][(h * S + j) * 64 + lane];
#pragma unroll
            for (int n = 0; n < NT; ++n) rows.o[n][j] = half_product(v, p[n][h], rows.o[n][j]);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x4 y[NT][2];
          i32x4 p[PP][NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) y[n][0] = x[n][2 * h], y[n][1] = x[n][2 * h + 1];
          rows.parts(a, y, p);
#pragma unroll
          for (int j = 0; j < S; ++j) {
            const i32x4 v = values[buffer][(h * S + j) * 64 + lane];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int k = PP - 1; k >= 0; --k) rows.o[n][j] = product(v, p[k][n], rows.o[n][j]);
          }
        }
      }
    }
    return true;
  };
  bool done = false;
  if constexpr (TYPE == TETRIS_BF16) {
    done = turns(std::true_type{});
    if (!done) {  // (all waves see the same forms, so they are all here)
      __syncthreads();
      rows.reset();
#pragma unroll
      for (int n = 0; n < NT; ++n) lost[n] = 0;
      begin();
    }
  }
  if (!done) turns(std::false_type{});

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float sum = sum_of_row(rows.l[n]) + rows.sums[n][0];
    const int r = r0 + n * 16 + r16;
    if (r >= all) continue;
    const int t = r / a.group, h = kv * a.group + r - t * a.group;
    T* y = static_cast<T*>(a.y) + (int64_t)(seq.begin + t) * a.ldy + (int64_t)h * D;
    auto output = [&](int j, int i) {
      const bool nan = lost[n] >> (neighbours(D) ? i : 4 * (j / 2) + i) & 1u;
      return (T)(nan ? __builtin_nanf("") : sum == 0.f ? 0.f : rows.o[n][j][i] / sum);
    };
    if (neighbours(D) && S * sizeof(T) >= 16 && a.y_whole) {  // a lane's S elements of a row lie together
      constexpr int V = S * (int)sizeof(T) / 16 ? S * (int)sizeof(T) / 16 : 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        T v[V * 16 / sizeof(T)];
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = output(j, i);
#pragma unroll
        for (int k = 0; k < V; ++k) reinterpret_cast<int4*>(y + element_of<D>(0, 4 * quad + i))[k] = reinterpret_cast<const int4*>(v)[k];
      }
    } else if (!neighbours(D) && a.y_whole) {  // four of them
      typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int j = 0; j < S; ++j) *reinterpret_cast<T4*>(y + element_of<D>(j, 4 * quad)) = T4{output(j, 0), output(j, 1), output(j, 2), output(j, 3)};
    } else {
#pragma unroll
      for (int j = 0; j < S; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[element_of<D>(j, 4 * quad + i)] = output(j, i);
    }
  }
}

// Units that several workgroups have parts of: a workgroup of W waves joins four rows, a wave of it every W-th part.  What the parts' weights are is known
// only with the last of their maxima, so a wave joins its own parts first, and all loads of a part are under way together.
template <int TYPE, int D, int W>
__global__ __launch_bounds__(64 * W) void join_kernel(Attend a) {
  using T = typename Elem<TYPE>::type;
  constexpr int R = 4, V = (R * D + 255) / 256, K = 4;  // rows; fours of a lane; parts that are loaded together
  __shared__ float4 out[W][V * 64];
  __shared__ float tops[W][R], sums[W][R];
  const int groups = 4 * a.tiles, g = blockIdx.x % groups;  // of a unit's rows
  const int64_t unit = blockIdx.x / groups;
  const int2 shares = a.shares[unit];
  const int block = (int)(unit % a.blocks), kv = (int)(unit / a.blocks % a.kv_heads), s = (int)(unit / a.blocks / a.kv_heads);
  const Sequence seq = sequence_of(a, s);
  const int all = min(seq.rows, a.most_rows) * a.group, r0 = block * 16 * a.tiles + g * R;
  if (r0 >= all || shares.y == 1) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float top[R], sum[R];
  float4 v[V];
#pragma unroll
  for (int r = 0; r < R; ++r) top[r] = -__builtin_inff(), sum[r] = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = wave; p0 < shares.y; p0 += W * K) {
    float4 of[K][2], x[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int p = min(p0 + k * W, shares.y - 1);
      const Slot slot = slot_of(a, 2 * (shares.x + p) + (p == 0), D);
      of[k][0] = reinterpret_cast<const float4*>(slot.top + 2 * g * R)[0];
      of[k][1] = reinterpret_cast<const float4*>(slot.top + 2 * g * R)[1];
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] = reinterpret_cast<const float4*>(slot.out + g * R * D)[min(lane + 64 * i, D - 1)];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (p0 + k * W >= shares.y) break;
      const float m[R] = {of[k][0].x, of[k][0].z, of[k][1].x, of[k][1].z}, l[R] = {of[k][0].y, of[k][0].w, of[k][1].y, of[k][1].w};
      float keep[R], take[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float most = fmaxf(top[r], m[r]);
        keep[r] = top[r] == most ? 1.f : __builtin_amdgcn_exp2f(top[r] - most);
        take[r] = m[r] == most ? 1.f : __builtin_amdgcn_exp2f(m[r] - most);
        top[r] = most;
        sum[r] = sum[r] * keep[r] + l[r] * take[r];
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int r = (lane + 64 * i) * 4 / D;
        const float f = r == 0 ? keep[0] : r == 1 ? keep[1] : r == 2 ? keep[2] : keep[3];
        const float t = r == 0 ? take[0] : r == 1 ? take[1] : r == 2 ? take[2] : take[3];
        v[i].x = v[i].x * f + x[k][i].x * t;
        v[i].y = v[i].y * f + x[k][i].y * t;
        v[i].z = v[i].z * f + x[k][i].z * t;
        v[i].w = v[i].w * f + x[k][i].w * t;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) out[wave][lane + 64 * i] = v[i];
  if (lane < R) tops[wave][lane] = lane == 0 ? top[0] : lane == 1 ? top[1] : lane == 2 ? top[2] : top[3];
  if (lane < R) sums[wave][lane] = lane == 0 ? sum[0] : lane == 1 ? sum[1] : lane == 2 ? sum[2] : sum[3];
  __syncthreads();
  for (int e = threadIdx.x; e < R * D; e += 64 * W) {
    const int r = e / D;
    if (r0 + r >= all) break;
    float most = tops[0][r], z = 0.f, y = 0.f;
#pragma unroll
    for (int w = 1; w < W; ++w) most = fmaxf(most, tops[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float by = tops[w][r] == most ? 1.f : __builtin_amdgcn_exp2f(tops[w][r] - most);
      z += sums[w][r] * by;
      y += reinterpret_cast<const float*>(out[w])[e] * by;
    }
    const int t = (r0 + r) / a.group, h = kv * a.group + r0 + r - t * a.group;
    static_cast<T*>(a.y)[(int64_t)(seq.begin + t) * a.ldy + (int64_t)h * D + e - r * D] = (T)(z == 0.f ? 0.f : y / z);
  }
}

// Most row tiles of a wave: as many as its registers hold (q and outputs of a tile).
constexpr int most_tiles(int parts, int head) { return head <= 128 && parts * head / 8 + head / 4 <= 64 ? 2 : 1; }
template <int TYPE, int D>
constexpr int kMostTiles = most_tiles(kParts<TYPE>, D);

// How a call is cut: by its sizes alone, so that its workspace can be made ahead.
struct Cut { bool prompt; int tiles, blocks, workgroups, chunk, chunks; int64_t units, most; size_t part, shares, space; };

// Whether rows share what is made of the values (attend_prompt_kernel) or each block of 16 NT rows makes its own (the others), by the microseconds that each is
// expected to take.  Measured, and what these fit within a fifth: 4 prompts of 300, 16 by 4 heads of 128: 19 us against 27; 16 of 128 16 against 30; 32 newest
// rows of 32 sequences of 4096 126 against 148; one prompt of 1024 of 8 by 8 heads, whose last workgroups are long alone, 38 against 28; 16 newest rows of 8
// sequences of 4096 120 against 36.
bool shares_values(const tetris_attention* a, int kv_heads, int head, int type, int64_t rows, int tiles) {
  if (rows <= 32) return false;
  const double parts = type == TETRIS_BF16 ? 1.0 : type == TETRIS_F16 ? 1.5 : 2.0, size = tiles * head / 128.0 * parts;
  const double length = a->window ? std::min<double>(a->most_length, (double)a->window + a->most_rows) : a->most_length;
  const double seen = std::max(length - std::min<double>(a->most_rows, length) / 2, 1.0), units = (double)a->sequences * kv_heads;
  // turns of 64 tokens: the longest workgroup's alone, all of them with two on a compute unit
  const double turn = (0.7 + 0.58 * size) * (head > 128 ? 1.4 : 1.0), groups = units * std::ceil(rows / (16.0 * tiles * kPromptWaves));
  const double prompt = 8 + std::max(turn * std::ceil(length / kTurn), groups * seen / kTurn * turn * 1.25 / (head > 128 ? 256 : 512));
  // steps of 32 tokens by a block, on 1024 SIMDs, and a workgroup's beginning and end
  const double blocks = units * std::ceil(rows / (16.0 * tiles));
  const double other = 8 + 8 * std::max(1.0, blocks / (256 * waves_of(parts_of(type), head, tiles))) + blocks * seen / kStep * (0.4 + 0.38 * size) / 1024;
  return prompt < other;
}

Cut cut_of(const tetris_cache* c, const tetris_attention* a, int type) {
  Cut k{};
  const int64_t rows = (int64_t)std::min(a->most_rows, a->rows) * (a->heads / c->kv_heads);
  k.tiles = rows <= 16 ? 1 : most_tiles(parts_of(type), c->head);
  k.blocks = (int)((rows + 16 * k.tiles - 1) / (16 * k.tiles));
  k.units = (int64_t)a->sequences * c->kv_heads * k.blocks;
  k.prompt = shares_values(a, c->kv_heads, c->head, type, rows, k.tiles);
  if (k.prompt) {
    k.most = (int64_t)a->sequences * c->kv_heads * ((k.blocks + kPromptWaves - 1) / kPromptWaves);
    k.workgroups = (int)std::min<int64_t>(k.most, 0x7fffffff);
    return k;
  }
  const int64_t span = a->window ? std::min<int64_t>(a->most_length, (int64_t)a->window + a->most_rows + kStep) : a->most_length;
  const int64_t quanta = std::max<int64_t>((span + kQuantum - 1) / kQuantum, 1);
  k.most = k.units > 0x7fffffff ? k.units : k.units * (quanta + kBegin);  // (a call of so many units is refused, and the product of both may pass 64 bits)
  const int resident = 256 * waves_of(parts_of(type), c->head, k.tiles);
  if (a->sequences > 1 && k.most >= 16 * (int64_t)resident) {
    k.workgroups = resident;
  } else {
    const int64_t chunks = std::min<int64_t>(std::max<int64_t>(resident / std::max<int64_t>(k.units, 1), 1), quanta);
    k.chunk = (int)((quanta + chunks - 1) / chunks);
    k.chunks = (int)((quanta + k.chunk - 1) / k.chunk);
    k.workgroups = (int)std::min<int64_t>(k.units * k.chunks, 0x7fffffff);
  }
  if (k.chunks != 1) k.part = ((size_t)k.workgroups * 2 * 16 * k.tiles * (c->head + 2) * sizeof(float) + 15) / 16 * 16;
  k.shares = (size_t)k.units * sizeof(int2);
  k.space = k.part + k.shares;
  return k;
}

template <int TYPE, int D>
int launch(Attend a, const Cut& k, hipStream_t s) {
  const dim3 grid((unsigned)k.workgroups), block(256);
  if (k.prompt) {
    hipLaunchKernelGGL((attend_prompt_kernel<TYPE, D, kMostTiles<TYPE, D>>), grid, dim3(64 * kPromptWaves), 0, s, a);
    TETRIS_HIP(hipGetLastError());
    return TETRIS_OK;
  }
  if (k.chunk) {
    if (k.tiles == 1) hipLaunchKernelGGL((attend_chunks_kernel<TYPE, D, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attend_chunks_kernel<TYPE, D, kMostTiles<TYPE, D>>), grid, block, 0, s, a);
  } else {
    if (k.tiles == 1) hipLaunchKernelGGL((attend_shares_kernel<TYPE, D, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attend_shares_kernel<TYPE, D, kMostTiles<TYPE, D>>), grid, block, 0, s, a);
  }
  TETRIS_HIP(hipGetLastError());
  if (k.chunks == 1) return TETRIS_OK;
  const dim3 joins((unsigned)(k.units * 4 * k.tiles));
  // Four waves to join the parts of rows that have few, sixteen for more: 64 sequences of up to 8192 tokens (768 workgroups of 512 units) 68 us against 75, 24 of
  // drafts (432 of 144) 26 against 29, 24 of 4000 (768 of 192) 32 against 34; two of 131072 (752 of 8) 50 against 44, one of 4000 (256 of 8) 12.3 against 11.1; as fast
  // either way where a unit has 6 (16 of 2048).
  if (k.workgroups <= 4 * k.units) hipLaunchKernelGGL((join_kernel<TYPE, D, 4>), joins, block, 0, s, a);
  else hipLaunchKernelGGL((join_kernel<TYPE, D, 16>), joins, dim3(1024), 0, s, a);
  TETRIS_HIP(hipGetLastError());
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
  if (!std::isfinite(a->scale * 1.44269504088896340736f)) return fail(TETRIS_EINVAL, "scale %g is not finite in powers of two", (double)a->scale);
  return TETRIS_OK;
}

}  // namespace
}  // namespace tetris

using namespace tetris;

extern "C" int tetris_cache_prepare(tetris_cache* c, const tetris_attention* a, int type, void* stream) {
  int rc = check_attention(c, a, type);
  if (!rc) rc = check_cache(c);
  if (rc) return rc;
  // what a call of these sizes or smaller ones may take: parts of as many workgroups as run at once
  size_t part = 0;
  for (int tiles = 1; tiles <= most_tiles(parts_of(type), c->head); ++tiles)
    part = std::max(part, (size_t)256 * waves_of(parts_of(type), c->head, tiles) * 2 * 16 * tiles * (c->head + 2) * sizeof(float));
  const int64_t rows = (int64_t)std::min(a->most_rows, a->rows) * (a->heads / c->kv_heads);
  uint8_t* d;
  return c->space.get(static_cast<hipStream_t>(stream), part + (size_t)a->sequences * c->kv_heads * ((rows + 15) / 16) * sizeof(int2), &d);
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
  const Cut k = cut_of(c, a, type);
  // a launch has fewer than 2^32 threads; attend_shares_kernel's quanta are numbered in 31 bits, up to its last workgroup's share, which may pass their end
  if (k.most > 0x7fffffff - kResidentMost || k.workgroups >= 1 << 24 || (!k.prompt && k.chunks != 1 && k.units * 4 * k.tiles >= 1 << 24))
    return fail(TETRIS_EUNSUPPORTED, "%d sequences of up to %d rows and %d tokens are more than a launch has", a->sequences, a->most_rows, a->most_length);
  if ((rc = check_cache(c))) return rc;
  uint8_t* d = nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if ((rc = c->space.get(s, k.space, &d))) return rc;
  Attend t{};
  t.data = c->data; t.q = d_q; t.y = d_y;
  t.first = d_first; t.length = d_length; t.table = d_table;
  t.part = reinterpret_cast<float*>(d);
  t.shares = reinterpret_cast<int2*>(d + k.part);
  t.page_bytes = c->page_bytes; t.ldt = ld_table; t.ldq = ldq; t.ldy = ldy;
  t.pages = c->pages; t.granules = c->page / kGranule;
  t.kv_heads = c->kv_heads; t.group = a->heads / c->kv_heads;
  t.sequences = a->sequences; t.rows = a->rows; t.most_rows = std::min(a->most_rows, a->rows); t.most_length = a->most_length;
  t.window = std::min(a->window, a->most_length);
  t.tiles = k.tiles; t.blocks = k.blocks; t.workgroups = k.workgroups; t.chunk = k.chunk; t.chunks = k.chunks;
  const int size = elem_size(type);
  t.whole = (reinterpret_cast<size_t>(d_q) & 15) == 0 && ldq * size % 16 == 0;
  t.y_whole = (reinterpret_cast<size_t>(d_y) & 15) == 0 && ldy * size % 16 == 0;
  t.scale = a->scale == 0.f ? 1.f : std::fabs(a->scale) * 1.44269504088896340736f;
  t.sign = a->scale == 0.f ? 0.f : a->scale < 0.f ? -1.f : 1.f;
  t.page_magic = magic_reciprocal(t.granules);
  if (type == TETRIS_F32) return by_head<TETRIS_F32>(c->head, t, k, s);
  if (type == TETRIS_F16) return by_head<TETRIS_F16>(c->head, t, k, s);
  return by_head<TETRIS_BF16>(c->head, t, k, s);
}

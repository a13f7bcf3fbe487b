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
#include <type_traits>

#include "cache.h"

namespace tetris {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 32;  // tokens
constexpr float kRoom = 8.f;

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
  float scale;  // to powers of two
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

// SHARED: the workgroup's waves take the steps of one block of rows in turn and join their outputs; else each has its own block.
template <int TYPE, int D, int NT, bool SHARED>
__global__ __launch_bounds__(256) void attend_kernel(Attend a) {
  using T = typename Elem<TYPE>::type;
  constexpr int QP = kParts<TYPE>, PP = kWeightParts<TYPE>, N = D / 32, S = D / 16, W = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, quad = lane >> 4;
  int id = blockIdx.x;
  const int chunk = id % a.chunks;
  id /= a.chunks;
  const int kv = id % a.kv_heads;
  id /= a.kv_heads;
  const int s = id % a.sequences, block = SHARED ? id / a.sequences : id / a.sequences * W + wave;
  const Sequence seq = sequence_of(a, s);
  const int all = min(seq.rows, a.most_rows) * a.group, r0 = block * (16 * NT);
  const int left = all - r0;  // rows of this block and those behind it
  if (SHARED && (left <= 0 || (chunk > 0 && seq.base + chunk * a.chunk >= seq.length))) return;

  // the block's query tokens, and the tokens that some of its rows sees
  const int t0 = r0 / a.group, t1 = min(r0 + 16 * NT - 1, max(all - 1, 0)) / a.group;
  const int p0 = seq.length - seq.rows;  // position of row 0
  int from = seq.base + chunk * a.chunk, to = min(from + a.chunk, min(p0 + t1, seq.length - 1) + 1);
  if (a.window) from = max(from, max(p0 + t0 - a.window + 1, 0) & ~(kStep - 1));
  if (left <= 0) to = from;

  i32x4 q[QP][NT][N];
  int last[NT];  // the newest token that the lane's row sees
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + n * 16 + r16, t = r / a.group, h = kv * a.group + r - t * a.group;
    last[n] = p0 + t;
    const T* row = static_cast<const T*>(a.q) + (int64_t)(seq.begin + t) * a.ldq + (int64_t)h * D + quad * (D / 4);
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
      for (int p = 0; p < QP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned low = leading(v[2 * i]);
          q[p][n][w][i] = (int)(low | leading(v[2 * i + 1]) << 16);
        }
    }
  }

  f32x4 o[NT][S];
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -__builtin_inff();
    l[n] = 0.f;
#pragma unroll
    for (int j = 0; j < S; ++j) o[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int* table = a.table + s * a.ldt;
  const uint8_t* head = a.data + (int64_t)kv * a.granules * (17 * D);
  for (int at = from + (SHARED ? wave * kStep : 0); at < to; at += SHARED ? W * kStep : kStep) {
    Granule<D> g[2];
    int upto[2];  // tokens of the granule that are there
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int token = at + 16 * u, there = min(seq.length - token, 16);
      int page = -1;
      if (there > 0) page = table[token / a.page];
      const bool good = (unsigned)page < (unsigned)a.pages;
      upto[u] = good ? there : 0;
      g[u].load(head + (good ? page : 0) * a.page_bytes + (token % a.page / 16) * (17 * D), lane);
    }
    // whether every row of the block sees all 32
    const bool plain = upto[0] == 16 && upto[1] == 16 && at + kStep - 1 <= p0 + t0 && (!a.window || at > p0 + t1 - a.window);
    unsigned nan = 0;  // bit 16 u + i: value of token 4 quad + i of granule u is NaN for the lane; (any block's, where the lane has several)
    if (!plain) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < Granule<D>::VS; ++c) {
            const unsigned byte = g[u].vs[c] >> (8 * i) & 255u;
            const bool there = 4 * quad + i < upto[u];
            if (byte == 255u && there) nan |= 1u << (16 * u + i);
            if (byte >= 253u && !there) g[u].vs[c] = (g[u].vs[c] & ~(255u << (8 * i))) | 127u << (8 * i);
          }
    }

    i32x4 p[PP][NT], seen[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 x[2] = {};
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < N; ++w) {
          const i32x4 key = g[u].key(w);
#pragma unroll
          for (int i = QP - 1; i >= 0; --i) x[u] = product(key, q[i][n][w], x[u]);
        }
      // Scaled here, before any branch: where a branch comes between a matrix instruction and the first use of its result, the compiler has
      // left out the wait that the instruction needs (tests/test_matrix_waits.py looks for that in the built library).
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float scaled = x[u][i] * a.scale;
          asm volatile("" : "+v"(scaled));
          x[u][i] = scaled;
        }
      float top = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!plain) {
            const int place = 16 * u + 4 * quad + i, j = at + place;
            const bool see = place - 16 * u < upto[u] && j <= last[n] && (!a.window || j > last[n] - a.window);
            x[u][i] = see ? x[u][i] : -__builtin_inff();
            const unsigned one = see ? 0x3f80u : 0u;
            const int k = 2 * u + i / 2;
            seen[n][k] = i & 1 ? seen[n][k] | (int)(one << 16) : (int)one;
          }
          top = fmaxf(top, x[u][i]);
        }
      if (__ballot(top > m[n] + kRoom)) {
        const float best = max_of_row(top), higher = best > m[n] + kRoom ? best : m[n];  // (a row's own matter, whatever its neighbours do)
        const float by = m[n] == higher ? 1.f : exp2f(m[n] - higher);
        m[n] = higher;
        l[n] *= by;
#pragma unroll
        for (int j = 0; j < S; ++j) o[n][j] *= by;
      }
      const float base = m[n] == -__builtin_inff() ? 0.f : m[n];
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[u][i] = exp2f(x[u][i] - base);
          sum += x[u][i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          unsigned parts[PP];
          split_pair<PP>(x[u][2 * i], x[u][2 * i + 1], parts);
#pragma unroll
          for (int k = 0; k < PP; ++k) p[k][n][2 * u + i] = (int)parts[k];
        }
      }
      l[n] += sum;
    }

    if (!plain && __ballot(nan != 0)) {
      // A NaN that some rows see and others do not: rows that see it get it by a product of their own (a one for each
      // NaN value by a one for each token that is seen), and the value counts as zero below.
#pragma unroll
      for (int c = 0; c < N; ++c) {
        i32x4 is_nan{};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool is = (g[u].vs[neighbours(D) ? 0 : c] >> (8 * i) & 255u) == 255u;
            is_nan[2 * u + i / 2] |= is ? 0x3f80 << (16 * (i & 1)) : 0;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const f32x4 hit = product(is_nan, seen[n], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0.f) o[n][2 * c][i] = o[n][2 * c + 1][i] = __builtin_nanf("");
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < Granule<D>::VS; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((g[u].vs[c] >> (8 * i) & 255u) == 255u) g[u].vs[c] = (g[u].vs[c] & ~(255u << (8 * i))) | 127u << (8 * i);
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

#pragma unroll
  for (int n = 0; n < NT; ++n) l[n] = sum_of_row(l[n]);

  // outputs of row r of the block: of this workgroup's chunk or, if that is all, finished
  auto finish = [&](int r, int element, float v, float top, float sum) {
    const int t = (r0 + r) / a.group, h = kv * a.group + r0 + r - t * a.group;
    const int64_t row = (int64_t)(seq.begin + t) * a.heads + h;
    if (a.part) {
      const int64_t at = (int64_t)chunk * a.rows * a.heads + row;
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
      if (quad == 0) tops[wave][n * 16 + r16] = m[n], sums[wave][n * 16 + r16] = l[n];
#pragma unroll
      for (int j = 0; j < S; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) out[wave][n * 16 + r16][element_of<D>(j, 4 * quad + i)] = o[n][j][i];
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
        const float by = tops[w][r] == top ? 1.f : exp2f(tops[w][r] - top);
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
          for (int i = 0; i < 4; ++i) finish(n * 16 + r16, element_of<D>(j, 4 * quad + i), o[n][j][i], m[n], l[n]);
      }
  }
}

// Chunks' outputs joined: a wave has a row and head.
template <int TYPE>
__global__ __launch_bounds__(256) void join_kernel(Attend a, int head) {
  using T = typename Elem<TYPE>::type;
  const int lane = threadIdx.x & 63;
  int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t each = (int64_t)a.most_rows * a.heads;
  if (id >= each * a.sequences) return;
  const int s = (int)(id / each), t = (int)(id - s * each) / a.heads, h = (int)(id - s * each) - t * a.heads;
  const Sequence seq = sequence_of(a, s);
  if (t >= seq.rows) return;
  const int64_t row = (int64_t)(seq.begin + t) * a.heads + h, rows = (int64_t)a.rows * a.heads;
  // (chunks past the sequence's newest token are not written)
  const int chunks = min(a.chunks, (max(seq.length - seq.base, 0) + a.chunk - 1) / a.chunk);
  float top = -__builtin_inff();
  for (int c = 0; c < chunks; ++c) top = fmaxf(top, a.part[2 * (c * rows + row)]);
  float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < chunks; ++c) {
    const float m = a.part[2 * (c * rows + row)], by = m == top ? 1.f : exp2f(m - top);
    sum += a.part[2 * (c * rows + row) + 1] * by;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < head) v[i] += a.part[2 * a.chunks * rows + (c * rows + row) * head + lane + 64 * i] * by;
  }
  T* y = static_cast<T*>(a.y) + (int64_t)(seq.begin + t) * a.ldy + (int64_t)h * head;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < head) y[lane + 64 * i] = (T)(sum == 0.f ? 0.f : v[i] / sum);
}

// How a call is cut: by its sizes alone, so that its workspace can be made ahead.
struct Cut { int tiles; bool shared; int blocks, chunk, chunks; size_t space; };
Cut cut_of(const tetris_cache* c, const tetris_attention* a, int type) {
  Cut k{};
  const int group = a->heads / c->kv_heads;
  const int64_t rows = (int64_t)std::min(a->most_rows, a->rows) * group;
  k.tiles = rows <= 16 ? 1 : 2;
  k.shared = true;
  k.blocks = (int)((rows + 16 * k.tiles - 1) / (16 * k.tiles));
  const int window = a->window ? a->window : a->most_length;
  const int64_t span = std::min<int64_t>(a->most_length, (int64_t)window + a->most_rows + kStep);
  const int64_t units = (int64_t)a->sequences * c->kv_heads * k.blocks;
  // about 2048 workgroups, of at least two steps a wave
  int64_t chunks = std::max<int64_t>(1, std::min<int64_t>(2048 / std::max<int64_t>(units, 1), (span + 8 * kStep - 1) / (8 * kStep)));
  k.chunk = (int)(((span + chunks - 1) / chunks + 4 * kStep - 1) / (4 * kStep) * (4 * kStep));
  k.chunks = (int)std::max<int64_t>(1, (span + k.chunk - 1) / k.chunk);
  if (k.chunks > 1) k.space = (size_t)k.chunks * a->rows * a->heads * (c->head + 2) * sizeof(float);
  return k;
}

template <int TYPE, int D>
int launch(Attend a, const Cut& k, hipStream_t s) {
  const int64_t groups = (int64_t)k.chunks * a.kv_heads * a.sequences * (k.shared ? k.blocks : ceil_div(k.blocks, 4));
  if (groups > 0x7fffffff) return fail(TETRIS_EUNSUPPORTED, "%lld workgroups are more than a launch has", (long long)groups);
  const dim3 grid((unsigned)groups), block(256);
  if (k.tiles == 1) hipLaunchKernelGGL((attend_kernel<TYPE, D, 1, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((attend_kernel<TYPE, D, 2, true>), grid, block, 0, s, a);
  TETRIS_HIP(hipGetLastError());
  if (k.chunks > 1) {
    const int64_t waves = (int64_t)a.sequences * a.most_rows * a.heads;
    hipLaunchKernelGGL((join_kernel<TYPE>), dim3((unsigned)((waves + 3) / 4)), block, 0, s, a, D);
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
  if (a->most_length > 0x40000000 || a->rows > 0x40000000 / a->heads) return fail(TETRIS_EINVAL, "%d rows of %d heads, %d tokens (up to 2^30)", a->rows, a->heads, a->most_length);
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
  t.scale = a->scale * 1.44269504088896340736f;
  if (type == TETRIS_F32) return by_head<TETRIS_F32>(c->head, t, k, s);
  if (type == TETRIS_F16) return by_head<TETRIS_F16>(c->head, t, k, s);
  return by_head<TETRIS_BF16>(c->head, t, k, s);
}

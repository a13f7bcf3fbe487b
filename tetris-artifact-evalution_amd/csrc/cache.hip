// The cache of keys and values in MX4: keys and values rounded into their slots, and read back.  One pass over memory, bound by HBM and by stores of
// 4 bytes that are spread over a granule: 16384 tokens of 8 heads of 128 bf16 written and read take 45 us together (170 MB, 3.8 TB/s; 41 where the last-level cache
// has some of it); a token of each of 64 sequences is two launches, 5.4 us.  A lane's eight elements of a value are one word only in heads of 128 and 256, which take 1.13 to
// 1.17 times what the bytes do at a copy's rate; heads of 64 go by two bytes and those of 96, 160, 192 and 224 by one, 1.31 to 1.41 times (23 us at 64, 69 at 192), and those of
// 32 by one at 1.75 (15 us).
#include <new>

#include "cache.h"
#include "rows.h"

namespace tetris {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

struct Slots {
  const int64_t* slot;
  uint8_t* pages;
  int64_t page_bytes;
  int tokens, kv_heads, page, slots;
  int64_t ld[2];  // of keys, of values
};

// Pieces of eight elements are numbered through head by head, token by token: the lanes of a wave have a few tokens of one head, whose bytes lie together in
// their granule where the slots follow one another (one token's alone lie 16 bytes apart: prompts of 16384 tokens of 8 x 128 written and read took 52 us).
struct Spot { uint8_t* granule; int64_t token; int head, place, piece; bool there, in; };  // there: a token; in: its slot is one of the cache's
template <int D>
__device__ inline Spot spot_of(const Slots& a, Place p) {
  Spot s{};
  s.token = p.piece / (D / 8);
  s.piece = p.piece % (D / 8);
  s.head = (int)p.row;
  s.there = p.row < a.kv_heads;
  if (!s.there) return s;
  const int64_t slot = a.slot[s.token];
  s.in = slot >= 0 && slot < a.slots;
  const unsigned at = s.in ? (unsigned)slot : 0u, page = at / (unsigned)a.page, place = at - page * a.page;
  s.granule = a.pages + page * a.page_bytes + (int64_t)(s.head * (a.page / kGranule) + (int)(place / kGranule)) * (17 * D);
  s.place = place % kGranule;
  return s;
}
// where the word of eight of a key's codes lies in its granule
template <int D>
__device__ inline int key_word(int token, int piece) {
  constexpr int N = D / 32;
  return ((piece / N * 16 + token) * N + piece % N) * 4;
}
// where byte c of lane 16 (token / 4) + m of a value's codes lies in those of its granule
template <int D>
__device__ inline int value_byte(int token, int m, int c) {
  return ((token / 4 * 16 + m) * 4 + token % 4) * (D / 32) + c;
}

constexpr int kAtOnce = 2;  // pieces that a lane has under way

// A lane has eight elements, four lanes a block.  blockIdx.y: keys, values.
template <int TYPE, int D, bool VEC>
__global__ __launch_bounds__(256) void append_kernel(Slots a, const typename Elem<TYPE>::type* __restrict__ k,
                                                     const typename Elem<TYPE>::type* __restrict__ v, unsigned per_row) {
  constexpr int N = D / 32;
  const bool value = blockIdx.y;
  const auto* x = value ? v : k;
  const int64_t waves = ((int64_t)a.kv_heads * per_row + 63) / 64, stride = (int64_t)gridDim.x * (blockDim.x >> 6);
  for (int64_t w = wave_of(); w < waves; w += kAtOnce * stride) {
    float es[kAtOnce][8];
    Spot spots[kAtOnce];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {  // (all loads first)
      const Spot s = spots[n] = spot_of<D>(a, place_of(w + n * stride, per_row));
      if (s.there) load8<typename Elem<TYPE>::type, VEC>(x + s.token * a.ld[blockIdx.y] + s.head * D, s.piece * 8, D, es[n]);
    }
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const Spot& s = spots[n];
      float(&e)[8] = es[n];
      if (!s.in) continue;  // (the lanes of a block are in or out together)
      unsigned top = 0;
  #pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(e[i]) & 0x7fffffffu);
      top = quad_max(top);
      const bool fine = top < 0x7f800000u;
      const int scale = max((int)(top >> 23) - 2, 0);
      const float by = __uint_as_float((unsigned)scale << 23);
      unsigned c = 0;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e[0], e[1], by, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e[2], e[3], by, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e[4], e[5], by, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e[6], e[7], by, 3);
      if (!fine) c = 0;
      const uint8_t byte = fine ? (uint8_t)scale : 255;
      const int block = s.piece / 4, q = s.piece & 3;
      if (!value) {
        *reinterpret_cast<unsigned*>(s.granule + key_word<D>(s.place, s.piece)) = c;
        if (q == 0) s.granule[16 * D + s.place * N + block] = byte;
        continue;
      }
      uint8_t* to = s.granule + 8 * D;
      if constexpr (!neighbours(D)) {
        // lanes q and q ^ 2 have the low and the high halves of bytes; each writes four of the eight
        const unsigned other = (unsigned)__builtin_amdgcn_mov_dpp((int)c, 0x4e, 0xf, 0xf, true);
        const unsigned low = q < 2 ? c : other >> 16, high = q < 2 ? other : c >> 16;
  #pragma unroll
        for (int i = 0; i < 4; ++i)
          to[value_byte<D>(s.place, 8 * (q & 1) + (q & 2) * 2 + i, block)] = (uint8_t)((low >> (4 * i) & 15) | (high >> (4 * i) & 15) << 4);
      } else if constexpr (D >= 128) {
        *reinterpret_cast<unsigned*>(to + value_byte<D>(s.place, s.piece * 8 / (D / 16), s.piece * 8 % (D / 16) / 2)) = c;
      } else {
        constexpr int M = 128 / D;  // lanes that the eight go to
  #pragma unroll
        for (int i = 0; i < M; ++i) {
          uint8_t* at = to + value_byte<D>(s.place, s.piece * M + i, 0);
          if constexpr (M == 2) *reinterpret_cast<unsigned short*>(at) = (unsigned short)(c >> (16 * i));
          else *at = (uint8_t)(c >> (8 * i));
        }
      }
      if (q == 0) s.granule[16 * D + D / 2 + (s.place / 4 * N + block) * 4 + s.place % 4] = byte;
    }
  }
}

template <int TYPE, int D, bool VEC>
__global__ __launch_bounds__(256) void read_kernel(Slots a, typename Elem<TYPE>::type* __restrict__ k, typename Elem<TYPE>::type* __restrict__ v,
                                                   unsigned per_row) {
  using T = typename Elem<TYPE>::type;
  constexpr int N = D / 32;
  const bool value = blockIdx.y;
  const int64_t waves = ((int64_t)a.kv_heads * per_row + 63) / 64, stride = (int64_t)gridDim.x * (blockDim.x >> 6);
  for (int64_t w = wave_of(); w < waves; w += kAtOnce * stride) {
    unsigned codes[kAtOnce], scales[kAtOnce];
    Spot spots[kAtOnce];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) spots[n] = spot_of<D>(a, place_of(w + n * stride, per_row));
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const Spot& s = spots[n];
      unsigned c = 0, byte = 127;
      const int block = s.piece / 4;
      if (s.in && !value) {
        c = *reinterpret_cast<const unsigned*>(s.granule + key_word<D>(s.place, s.piece));
        byte = s.granule[16 * D + s.place * N + block];
      } else if (s.in) {
        const uint8_t* from = s.granule + 8 * D;
        if constexpr (!neighbours(D)) {
          const int q = s.piece & 3;
  #pragma unroll
          for (int i = 0; i < 8; ++i) c |= ((unsigned)from[value_byte<D>(s.place, 8 * (q & 1) + i, block)] >> (q & 2) * 2 & 15u) << (4 * i);
        } else if constexpr (D >= 128) {
          c = *reinterpret_cast<const unsigned*>(from + value_byte<D>(s.place, s.piece * 8 / (D / 16), s.piece * 8 % (D / 16) / 2));
        } else {
          constexpr int M = 128 / D;
  #pragma unroll
          for (int i = 0; i < M; ++i) {
            const uint8_t* at = from + value_byte<D>(s.place, s.piece * M + i, 0);
            if constexpr (M == 2) c |= (unsigned)*reinterpret_cast<const unsigned short*>(at) << (16 * i);
            else c |= (unsigned)*at << (8 * i);
          }
        }
        byte = s.granule[16 * D + D / 2 + (s.place / 4 * N + block) * 4 + s.place % 4];
      }
      codes[n] = c;
      scales[n] = byte;
    }
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      const Spot& s = spots[n];
      const unsigned c = codes[n], byte = scales[n];
      if (!s.there) continue;
      const float by = __uint_as_float(byte << 23);
      T t[8];
      if (TYPE == TETRIS_BF16) {
        int* o = reinterpret_cast<int*>(t);
        o[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, by, 0));
        o[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, by, 1));
        o[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, by, 2));
        o[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, by, 3));
      } else {
        const f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, by, 0), f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, by, 1);
        const f32x2 g = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, by, 2), h = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, by, 3);
        t[0] = (T)e.x; t[1] = (T)e.y; t[2] = (T)f.x; t[3] = (T)f.y;
        t[4] = (T)g.x; t[5] = (T)g.y; t[6] = (T)h.x; t[7] = (T)h.y;
      }
      T* out = (value ? v : k) + s.token * a.ld[blockIdx.y] + s.head * D + s.piece * 8;
      if (VEC) {
  #pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<int4*>(out)[i] = reinterpret_cast<const int4*>(t)[i];
      } else {
  #pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = t[i];
      }
    }
  }
}

template <int TYPE, bool APPEND, int D, bool VEC>
void launch(const Slots& a, void* k, void* v, hipStream_t s) {
  using T = typename Elem<TYPE>::type;
  const unsigned per_row = (unsigned)(a.tokens * (D / 8));  // pieces of a head
  const int64_t pieces = (int64_t)a.kv_heads * per_row;
  const int few = pieces > 256 * 1024 ? kAtOnce : 1;  // pieces of a lane: one where that does not fill the chip
  const dim3 grid((unsigned)std::min<int64_t>((pieces + 256 * few - 1) / (256 * few), 256 * 64), 2), block(256);
  if constexpr (APPEND)
    hipLaunchKernelGGL((append_kernel<TYPE, D, VEC>), grid, block, 0, s, a, static_cast<const T*>(k), static_cast<const T*>(v), per_row);
  else
    hipLaunchKernelGGL((read_kernel<TYPE, D, VEC>), grid, block, 0, s, a, static_cast<T*>(k), static_cast<T*>(v), per_row);
}
template <int TYPE, bool APPEND, bool VEC>
void by_head(int head, const Slots& a, void* k, void* v, hipStream_t s) {
  switch (head) {
    case 32: return launch<TYPE, APPEND, 32, VEC>(a, k, v, s);
    case 64: return launch<TYPE, APPEND, 64, VEC>(a, k, v, s);
    case 96: return launch<TYPE, APPEND, 96, VEC>(a, k, v, s);
    case 128: return launch<TYPE, APPEND, 128, VEC>(a, k, v, s);
    case 160: return launch<TYPE, APPEND, 160, VEC>(a, k, v, s);
    case 192: return launch<TYPE, APPEND, 192, VEC>(a, k, v, s);
    case 224: return launch<TYPE, APPEND, 224, VEC>(a, k, v, s);
    default: return launch<TYPE, APPEND, 256, VEC>(a, k, v, s);
  }
}
template <bool APPEND>
int move(const tetris_cache* c, void* k, int64_t ldk, void* v, int64_t ldv, int type, int tokens, const int64_t* slot, hipStream_t s) {
  if (!c) return fail(TETRIS_EINVAL, "null argument");
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (tokens < 0) return fail(TETRIS_EINVAL, "%d tokens", tokens);
  const int64_t width = (int64_t)c->kv_heads * c->head;
  if (ldk < width || ldv < width)
    return fail(TETRIS_EINVAL, "leading dimension %lld below the %lld elements of a token", (long long)std::min(ldk, ldv), (long long)width);
  if (tokens == 0) return TETRIS_OK;
  if (!k || !v || !slot) return fail(TETRIS_EINVAL, "null argument");
  if ((reinterpret_cast<size_t>(k) | reinterpret_cast<size_t>(v)) % elem_size(type)) return fail(TETRIS_EINVAL, "rows not aligned to their elements");
  if (reinterpret_cast<size_t>(slot) & 7) return fail(TETRIS_EINVAL, "slots not aligned to their elements");
  int rc = check_cache(c);
  if (rc) return rc;
  constexpr int kMost = 1 << 25;  // tokens of a launch: so that a head's pieces are numbered in 31 bits
  if (tokens > kMost) {
    for (int from = 0; from < tokens; from += kMost) {
      const int n = std::min(kMost, tokens - from);
      auto at = [&](void* p, int64_t ld) { return static_cast<char*>(p) + from * ld * elem_size(type); };
      if ((rc = move<APPEND>(c, at(k, ldk), ldk, at(v, ldv), ldv, type, n, slot + from, s))) return rc;
      if (from > tokens - kMost) break;
    }
    return TETRIS_OK;
  }
  const Slots a{slot, c->data, c->page_bytes, tokens, c->kv_heads, c->page, c->pages * c->page, {ldk, ldv}};
  const int size = elem_size(type);
  const bool vec = ((reinterpret_cast<size_t>(k) | reinterpret_cast<size_t>(v)) & 15) == 0 && ldk * size % 16 == 0 && ldv * size % 16 == 0;
  if (type == TETRIS_F32) vec ? by_head<TETRIS_F32, APPEND, true>(c->head, a, k, v, s) : by_head<TETRIS_F32, APPEND, false>(c->head, a, k, v, s);
  else if (type == TETRIS_F16) vec ? by_head<TETRIS_F16, APPEND, true>(c->head, a, k, v, s) : by_head<TETRIS_F16, APPEND, false>(c->head, a, k, v, s);
  else vec ? by_head<TETRIS_BF16, APPEND, true>(c->head, a, k, v, s) : by_head<TETRIS_BF16, APPEND, false>(c->head, a, k, v, s);
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

bool good_shape(int kv_heads, int head, int page) {
  return kv_heads > 0 && kv_heads <= kCacheHeads && head > 0 && head <= kCacheHead && head % 32 == 0 && page > 0 && page <= kCachePage && page % kGranule == 0;
}

}  // namespace

int check_cache(const tetris_cache* c) {
  int device = 0;
  TETRIS_HIP(hipGetDevice(&device));
  if (device != c->device) return fail(TETRIS_EINVAL, "the cache belongs to device %d, the current one is %d", c->device, device);
  return TETRIS_OK;
}

}  // namespace tetris

using namespace tetris;

extern "C" size_t tetris_cache_page_bytes(int kv_heads, int head, int page) {
  return good_shape(kv_heads, head, page) ? (size_t)kv_heads * (page / kGranule) * (17 * head) : 0;
}

extern "C" int tetris_cache_create(int kv_heads, int head, int page, int64_t pages, void* d_pages, tetris_cache** out) {
  if (!out) return fail(TETRIS_EINVAL, "null argument");
  *out = nullptr;
  if (!good_shape(kv_heads, head, page))
    return fail(TETRIS_EINVAL, "a cache of %d heads of %d elements in pages of %d tokens (1 to %d heads, multiples of 32 up to %d, of %d up to %d)", kv_heads,
                head, page, kCacheHeads, kCacheHead, kGranule, kCachePage);
  if (pages <= 0 || pages > 0x7fffffff / page) return fail(TETRIS_EINVAL, "%lld pages of %d tokens (fewer than 2^31 slots)", (long long)pages, page);
  if (!d_pages) return fail(TETRIS_EINVAL, "null argument");
  if (reinterpret_cast<size_t>(d_pages) & 15) return fail(TETRIS_EINVAL, "pages must lie on 16 bytes");
  std::unique_ptr<tetris_cache, void (*)(tetris_cache*)> c(new (std::nothrow) tetris_cache, tetris_cache_destroy);
  if (!c) return fail(TETRIS_EINVAL, "no host memory for a handle");
  if (hipGetDevice(&c->device) != hipSuccess) {
    (void)hipGetLastError();
    c->device = -1;  // there is none, and nothing will be launched
  }
  c->kv_heads = kv_heads; c->head = head; c->page = page; c->pages = (int)pages;
  c->page_bytes = (int64_t)tetris_cache_page_bytes(kv_heads, head, page);
  c->data = static_cast<uint8_t*>(d_pages);
  *out = c.release();
  return TETRIS_OK;
}

extern "C" void tetris_cache_destroy(tetris_cache* c) {
  if (!c) return;
  c->space.release();
  delete c;
}

extern "C" int tetris_cache_append(tetris_cache* c, const void* d_k, int64_t ldk, const void* d_v, int64_t ldv, int type, int tokens,
                                   const int64_t* d_slot, void* stream) {
  return move<true>(c, const_cast<void*>(d_k), ldk, const_cast<void*>(d_v), ldv, type, tokens, d_slot, static_cast<hipStream_t>(stream));
}

extern "C" int tetris_cache_read(tetris_cache* c, const int64_t* d_slot, int tokens, void* d_k, int64_t ldk, void* d_v, int64_t ldv, int type,
                                 void* stream) {
  return move<false>(c, d_k, ldk, d_v, ldv, type, tokens, d_slot, static_cast<hipStream_t>(stream));
}

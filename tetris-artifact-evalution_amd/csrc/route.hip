// Routing of tokens to experts: scores, groups, choice and weights, and the gradient of the weights.  L lanes of a wave have a token (sixteen up
// to 256 experts, else the whole wave); the logits are read once and stay in registers, expert e with lane e / V of them.  Bound by the instructions of the
// choice -- `top` rounds of a maximum over a token's lanes -- and, for few tokens, by the launch: 16384 tokens of 256 experts, eight groups of which
// four stay, eight chosen, 14.4 us; a wave a token, logits loaded one by one, 25.2 us.
#include <algorithm>
#include <type_traits>

#include "mx4.h"

namespace tetris {
namespace {

constexpr int kMostExperts = 1024, kMostTop = 32, kMostGroups = 64;

struct Route {
  const void* logits;
  int64_t ld;
  int tokens, experts, top, score, groups, top_groups, group_by, renorm;
  float scale;
  const float* bias;
  int whole; // rows and bias lie on 16 bytes, and every lane has V experts
  int span;  // lanes that a group fills, of sixteen; 0: groups begin or end inside a lane's experts
};

// Numbers to integers of the same order; NaN as -inf.  Zero is below all of them.
__device__ inline unsigned key_of(float v) {
  const unsigned u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0x007fffffu;
  const unsigned w = u == 0x80000000u ? 0u : u;  // -0 ranks as 0
  return (w & 0x80000000u) ? ~w : w | 0x80000000u;
}

template <int CTRL>
__device__ inline unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
// f over the values of a token's L lanes, in all of them.  Sixteen lanes: rotations by 8, 4, 2 and 1 of a row.
template <int L, typename F>
__device__ inline unsigned lanes(unsigned v, F f) {
  v = f(v, dpp<0x128>(v));
  v = f(v, dpp<0x124>(v));
  v = f(v, dpp<0x122>(v));
  v = f(v, dpp<0x121>(v));
  if constexpr (L == 64) {
    v = f(v, (unsigned)__shfl_xor((int)v, 16));
    v = f(v, (unsigned)__shfl_xor((int)v, 32));
  }
  return v;
}
template <int L>
__device__ inline unsigned lanes_max(unsigned v) { return lanes<L>(v, [](unsigned a, unsigned b) { return max(a, b); }); }
template <int L>
__device__ inline unsigned lanes_min(unsigned v) { return lanes<L>(v, [](unsigned a, unsigned b) { return min(a, b); }); }
template <int L>
__device__ inline float lanes_sum(float v) {
  return __uint_as_float(lanes<L>(__float_as_uint(v), [](unsigned a, unsigned b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

// V numbers from p on, which lie on 16 bytes
template <typename T, int V>
__device__ inline void load_whole(const T* p, float (&x)[V]) {
  constexpr int N = V * (int)sizeof(T) / 16;
  int4 raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) raw[i] = reinterpret_cast<const int4*>(p)[i];
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = (float)reinterpret_cast<const T*>(raw)[v];
}

// the lane's V logits; those past the last expert -inf
template <int TYPE, int V>
__device__ inline void load_logits(const Route& a, int token, int lane, float (&x)[V]) {
  using T = typename Elem<TYPE>::type;
  const T* row = static_cast<const T*>(a.logits) + token * a.ld;
  if constexpr (V * sizeof(T) >= 16) {
    if (a.whole) return load_whole<T, V>(row + lane * V, x);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    x[v] = e < a.experts ? (float)row[e] : -__builtin_inff();
  }
}

// What a token's scores need besides the logit: softmax's largest logit and the sum of the exponentials.
struct Norm { float top, sum; };
__device__ inline float exponential(float x, float top) {
  return top == -__builtin_inff() && !(x != x) ? 0.f : x == top ? 1.f : expf(x - top);
}
__device__ inline float score_of(const Route& a, float x, Norm n) {
  if (a.score == TETRIS_SCORE_SIGMOID) return 1.f / (1.f + expf(-x));
  return n.sum == 0.f ? 0.f : exponential(x, n.top) / n.sum;
}

// x to scores
template <int L, int V>
__device__ inline Norm scores(const Route& a, const float (&x)[V], float (&s)[V]) {
  if (a.score == TETRIS_SCORE_SIGMOID) {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = score_of(a, x[v], Norm{});
    return {};
  }
  unsigned key = 0x007fffffu;
#pragma unroll
  for (int v = 0; v < V; ++v) key = max(key, key_of(x[v]));
  key = lanes_max<L>(key);
  Norm n{__uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key), 0.f};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s[v] = exponential(x[v], n.top);
    n.sum += s[v];
  }
  n.sum = lanes_sum<L>(n.sum);
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = n.sum == 0.f ? 0.f : s[v] / n.sum;
  return n;
}

// Keys of the experts that may be chosen, zero for the others.  `by_expert`: LDS of the token, a float for each expert; `lane`: among the token's.
template <int L, int V>
__device__ inline void keys_of(const Route& a, int lane, float* by_expert, const float (&rank)[V], const float (&two)[V], unsigned (&key)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) key[v] = lane * V + v < a.experts ? key_of(rank[v]) : 0u;
  if (a.top_groups == a.groups) return;
  const float inf = __builtin_inff();
  const int size = a.experts / a.groups;
  if (L == 16 && a.span) {  // a group is the experts of 1, 2, 4, 8 or 16 neighbouring lanes
    float first = -inf, second = -inf;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float u = a.group_by == TETRIS_GROUP_TWO ? two[v] : rank[v];
      u = u != u || lane * V + v >= a.experts ? -inf : u;
      second = fmaxf(second, fminf(first, u));
      first = fmaxf(first, u);
    }
    auto join = [&](float f, float o) {
      second = fmaxf(fmaxf(second, o), fminf(first, f));
      first = fmaxf(first, f);
    };
    auto of = [](float v, auto ctrl) { return __uint_as_float(dpp<decltype(ctrl)::value>(__float_as_uint(v))); };
#define TETRIS_JOIN(CTRL) join(of(first, std::integral_constant<int, CTRL>{}), of(second, std::integral_constant<int, CTRL>{}))
    if (a.span > 1) TETRIS_JOIN(0xb1);   // lane ^ 1
    if (a.span > 2) TETRIS_JOIN(0x4e);   // lane ^ 2
    if (a.span > 4) TETRIS_JOIN(0x141);  // the other four of eight
    if (a.span > 8) TETRIS_JOIN(0x140);  // the other eight of sixteen
#undef TETRIS_JOIN
    const int shift = 31 - __builtin_clz(a.span), g = lane >> shift;
    const unsigned mine = g < a.groups ? key_of(a.group_by == TETRIS_GROUP_TWO ? first + second : first) : 0u;
    unsigned other = mine;
    int before = 0;  // lanes of groups that come first, a.span of each
#pragma unroll
    for (int k = 1; k < 16; ++k) {
      other = dpp<0x121>(other);  // that of lane - k
      before += other > mine || (other == mine && (((lane - k) & 15) >> shift) < g);
    }
    const bool stays = before < a.top_groups * a.span;
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = stays ? key[v] : 0u;
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (lane * V + v < a.experts) by_expert[lane * V + v] = a.group_by == TETRIS_GROUP_TWO ? two[v] : rank[v];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  // lane l has groups l, l + L, ...; it begins with the l-th of a group's experts, so that lanes read different banks
  unsigned mine[64 / L];
#pragma unroll
  for (int t = 0; t < 64 / L; ++t) {
    const int g = lane + t * L;
    float first = -inf, second = -inf;
    if (g < a.groups) {
      int i = g % size;
      for (int n = 0; n < size; ++n) {
        float v = by_expert[g * size + i];
        v = v != v ? -inf : v;
        second = fmaxf(second, fminf(first, v));
        first = fmaxf(first, v);
        if (++i == size) i = 0;
      }
    }
    mine[t] = g < a.groups ? key_of(a.group_by == TETRIS_GROUP_TWO ? first + second : first) : 0u;
  }
  unsigned long long stay = 0;
  const int shift = (threadIdx.x & 63) & ~(L - 1);
#pragma unroll
  for (int t = 0; t < 64 / L; ++t) {
    if (t * L >= a.groups) break;
    int before = 0;
    for (int g = 0; g < a.groups; ++g) {
      unsigned other = 0;
#pragma unroll
      for (int q = 0; q < 64 / L; ++q) {
        const unsigned o = (unsigned)__shfl((int)mine[q], g % L, L);
        if (g / L == q) other = o;
        if ((q + 1) * L >= a.groups) break;
      }
      before += other > mine[t] || (other == mine[t] && g < lane + t * L);
    }
    const unsigned long long in = __ballot(lane + t * L < a.groups && before < a.top_groups) >> shift;
    stay |= (L == 64 ? in : in & 0xffff) << (t * L % 64);
  }
  int g = lane * V / size, i = lane * V - g * size;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (!((stay >> (g & 63)) & 1)) key[v] = 0;
    if (++i == size) i = 0, ++g;
  }
}

template <int TYPE, int L, int V>
__global__ __launch_bounds__(256) void route_kernel(Route a, int* __restrict__ index, float* __restrict__ weight) {
  __shared__ float shared[256 / L][L * V];
  const int lane = threadIdx.x & (L - 1), mine = threadIdx.x / L;
  const int token = blockIdx.x * (256 / L) + mine, read = min(token, a.tokens - 1);  // (lanes without a token follow the last one's)
  float x[V], s[V], rank[V], two[V];
  unsigned key[V];
  load_logits<TYPE, V>(a, read, lane, x);
  const Norm norm = scores<L, V>(a, x, s);
  float bias[V];
  bool read_whole = false;
  if constexpr (V >= 4) {
    read_whole = a.bias && a.whole;
    if (read_whole) load_whole<float, V>(a.bias + lane * V, bias);
  }
  if (!read_whole) {
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = a.bias && lane * V + v < a.experts ? a.bias[lane * V + v] : 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    two[v] = s[v] + bias[v];
    rank[v] = a.bias ? two[v] : x[v];
  }
  keys_of<L, V>(a, lane, shared[mine], rank, two, key);

  // the best that is left, `top` times, the lowest index of equal ones; lane r keeps the r-th
  unsigned my_index = 0;
  for (int r = 0; r < a.top; ++r) {
    unsigned best = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) best = max(best, key[v]);
    best = lanes_max<L>(best);
    unsigned e = ~0u;
#pragma unroll
    for (int v = V - 1; v >= 0; --v) e = key[v] == best ? (unsigned)(lane * V + v) : e;
    e = lanes_min<L>(e);
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = e == (unsigned)(lane * V + v) ? 0u : key[v];
    if (lane == r) my_index = e;
  }
  // its score from its logit again, rather than from the lane that has it
  const auto* row = static_cast<const typename Elem<TYPE>::type*>(a.logits) + read * a.ld;
  const float score = lane < a.top ? score_of(a, (float)row[my_index], norm) : 0.f;
  const float sum = a.renorm ? lanes_sum<L>(score) : 1.f;
  if (lane < a.top && token < a.tokens) {
    index[(int64_t)token * a.top + lane] = (int)my_index;
    weight[(int64_t)token * a.top + lane] = sum == 0.f ? 0.f : (a.renorm ? score / sum : score) * a.scale;
  }
}

// With s the scores, c the chosen, S the sum of theirs, p = s and d_j = scale dweight_j (renorm: p = s / S and d_j less sum_l d_l p_l):
//   sigmoid  dlogit_i = p_i (1 - s_i) d_i for the chosen, else 0
//   softmax  dlogit_i = p_i (d_i - sum_j s_j d_j), with d_i = 0 for those not chosen; with renorm that sum is zero
// A wave a token.  8192 tokens of 128 experts in bf16: 6.2 us (4.7 MB); the launch and one wave's chain of instructions, not memory.
template <int TYPE, int V>
__global__ __launch_bounds__(256) void route_backward_kernel(Route a, const int* __restrict__ index, const float* __restrict__ dweight,
                                                             typename Elem<TYPE>::type* __restrict__ out, int64_t ld_out) {
  __shared__ float shared[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = blockIdx.x * 4 + wave;
  if (token >= a.tokens) return;
  float x[V], s[V], d[V];
  load_logits<TYPE, V>(a, token, lane, x);
  scores<64, V>(a, x, s);
  float* mine = shared[wave];
#pragma unroll
  for (int v = 0; v < V; ++v) mine[lane * V + v] = s[v], d[v] = 0.f;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  int e = -1;
  float dw = 0.f, score = 0.f;
  if (lane < a.top) {
    e = index[(int64_t)token * a.top + lane];
    if (e < 0 || e >= a.experts) e = -1;
    if (e >= 0) dw = a.scale * dweight[(int64_t)token * a.top + lane], score = mine[e];
  }
  float sum = 1.f;  // what scores are divided by: they, not d, so that nothing overflows where all of them are small
  if (a.renorm) {
    sum = lanes_sum<64>(score);
    const float mean = sum == 0.f ? 0.f : lanes_sum<64>(dw * (score / sum));
    dw = sum == 0.f || e < 0 ? 0.f : dw - mean;
  }
  const float all = a.score == TETRIS_SCORE_SOFTMAX && !a.renorm ? lanes_sum<64>(dw * score) : 0.f;
  for (int j = 0; j < a.top; ++j) {
    const int ej = __builtin_amdgcn_readlane(e, j);
    const float dj = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(dw), j));
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (ej == lane * V + v) d[v] = dj;
  }
  auto* row = out + token * ld_out;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    // (1 - s from the logit: from s, which is 1 to 32 bits beyond a logit of 17, nothing would be left)
    // (those not chosen may be any times `sum`, but not infinitely: they are multiplied by zero)
    const float share = sum == 0.f ? 0.f : a.renorm ? fminf(s[v], sum) / sum : s[v];
    const float g = a.score == TETRIS_SCORE_SIGMOID ? share * (1.f / (1.f + expf(x[v]))) * d[v] : share * (d[v] - all);
    if (lane * V + v < a.experts) row[lane * V + v] = (typename Elem<TYPE>::type)g;
  }
}

template <int TYPE, int L, int V>
void launch_route(Route a, int* index, float* weight, hipStream_t s) {
  const int size = a.experts / a.groups, lanes_each = size / V;
  a.whole = a.experts == L * V && (reinterpret_cast<size_t>(a.logits) & 15) == 0 && a.ld * elem_size(TYPE) % 16 == 0 && (reinterpret_cast<size_t>(a.bias) & 15) == 0;
  a.span = L == 16 && size % V == 0 && (lanes_each & (lanes_each - 1)) == 0 ? lanes_each : 0;
  hipLaunchKernelGGL((route_kernel<TYPE, L, V>), dim3(ceil_div(a.tokens, 256 / L)), dim3(256), 0, s, a, index, weight);
}
template <int TYPE>
void route_any(const Route& a, int* index, float* weight, hipStream_t s) {
  if (a.experts <= 256 && a.top <= 16) {
    if (a.experts <= 16) launch_route<TYPE, 16, 1>(a, index, weight, s);
    else if (a.experts <= 64) launch_route<TYPE, 16, 4>(a, index, weight, s);
    else if (a.experts <= 128) launch_route<TYPE, 16, 8>(a, index, weight, s);
    else launch_route<TYPE, 16, 16>(a, index, weight, s);
  } else if (a.experts <= 256) launch_route<TYPE, 64, 4>(a, index, weight, s);
  else if (a.experts <= 512) launch_route<TYPE, 64, 8>(a, index, weight, s);
  else launch_route<TYPE, 64, 16>(a, index, weight, s);
}
template <int TYPE, int V>
void launch_backward(const Route& a, const int* index, const float* dweight, void* out, int64_t ld, hipStream_t s) {
  hipLaunchKernelGGL((route_backward_kernel<TYPE, V>), dim3((a.tokens + 3) / 4), dim3(256), 0, s, a, index, dweight,
                     static_cast<typename Elem<TYPE>::type*>(out), ld);
}

template <int TYPE, typename F>
void by_width(int experts, F f) {
  if (experts <= 64) f(std::integral_constant<int, 1>{});
  else if (experts <= 128) f(std::integral_constant<int, 2>{});
  else if (experts <= 256) f(std::integral_constant<int, 4>{});
  else if (experts <= 512) f(std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 16>{});
}
template <typename F>
void by_type(int type, F f) {
  if (type == TETRIS_F32) f(std::integral_constant<int, TETRIS_F32>{});
  else if (type == TETRIS_F16) f(std::integral_constant<int, TETRIS_F16>{});
  else f(std::integral_constant<int, TETRIS_BF16>{});
}

int check(const tetris_router* r, int type, int tokens, int64_t ld) {
  if (!r) return fail(TETRIS_EINVAL, "null argument");
  if (bad_type(type)) return fail(TETRIS_EINVAL, "type %d is not TETRIS_F32, TETRIS_F16 or TETRIS_BF16", type);
  if (r->experts <= 0 || r->experts > kMostExperts) return fail(TETRIS_EINVAL, "%d experts (1 to %d)", r->experts, kMostExperts);
  if (r->score != TETRIS_SCORE_SOFTMAX && r->score != TETRIS_SCORE_SIGMOID) return fail(TETRIS_EINVAL, "score %d", r->score);
  if (r->groups <= 0 || r->groups > kMostGroups || r->experts % r->groups)
    return fail(TETRIS_EINVAL, "%d groups of %d experts (1 to %d, dividing them)", r->groups, r->experts, kMostGroups);
  if (r->top_groups <= 0 || r->top_groups > r->groups) return fail(TETRIS_EINVAL, "%d of %d groups", r->top_groups, r->groups);
  if (r->group_by != TETRIS_GROUP_MAX && r->group_by != TETRIS_GROUP_TWO) return fail(TETRIS_EINVAL, "group_by %d", r->group_by);
  if (r->group_by == TETRIS_GROUP_TWO && r->groups > 1 && r->experts / r->groups < 2)
    return fail(TETRIS_EINVAL, "groups of one expert have no second best");
  if (r->top <= 0 || r->top > kMostTop || r->top > r->experts / r->groups * r->top_groups)
    return fail(TETRIS_EINVAL, "top %d of the %d experts that stay (at most %d)", r->top, r->experts / r->groups * r->top_groups, kMostTop);
  if (tokens < 0) return fail(TETRIS_EINVAL, "%d tokens", tokens);
  if (ld < r->experts) return fail(TETRIS_EINVAL, "leading dimension %lld below the %d experts", (long long)ld, r->experts);
  return TETRIS_OK;
}

Route route_of(const tetris_router* r, const void* logits, int tokens, int64_t ld, const float* bias) {
  return {logits, ld, tokens, r->experts, r->top, r->score, r->groups, r->top_groups, r->group_by, r->renorm, r->scale, bias, 0, 0};
}

}  // namespace
}  // namespace tetris

using namespace tetris;

extern "C" int tetris_route(const tetris_router* r, const void* d_logits, int type, int tokens, int64_t ld, const float* d_bias,
                            int32_t* d_index, float* d_weight, void* stream) {
  const int rc = check(r, type, tokens, ld);
  if (rc || tokens == 0) return rc;
  if (!d_logits || !d_index || !d_weight) return fail(TETRIS_EINVAL, "null argument");
  if (reinterpret_cast<size_t>(d_logits) % elem_size(type)) return fail(TETRIS_EINVAL, "logits not aligned to their elements");
  const Route a = route_of(r, d_logits, tokens, ld, d_bias);
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_type(type, [&](auto t) { route_any<decltype(t)::value>(a, d_index, d_weight, s); });
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

extern "C" int tetris_route_backward(const tetris_router* r, const void* d_logits, int type, int tokens, int64_t ld,
                                     const int32_t* d_index, const float* d_dweight, void* d_dlogits, int64_t ld_out, void* stream) {
  int rc = check(r, type, tokens, ld);
  if (!rc) rc = check(r, type, tokens, ld_out);
  if (rc || tokens == 0) return rc;
  if (!d_logits || !d_index || !d_dweight || !d_dlogits) return fail(TETRIS_EINVAL, "null argument");
  if ((reinterpret_cast<size_t>(d_logits) | reinterpret_cast<size_t>(d_dlogits)) % elem_size(type))
    return fail(TETRIS_EINVAL, "logits not aligned to their elements");
  const Route a = route_of(r, d_logits, tokens, ld, nullptr);
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_type(type, [&](auto t) {
    by_width<decltype(t)::value>(r->experts, [&](auto v) {
      launch_backward<decltype(t)::value, decltype(v)::value>(a, d_index, d_dweight, d_dlogits, ld_out, s);
    });
  });
  TETRIS_HIP(hipGetLastError());
  return TETRIS_OK;
}

// Routing of tokens to experts: scores, groups, choice and weights, and the gradient of the weights.  One wave a token; the
// logits are read once and stay in registers, expert e with lane e / V, place e % V of the lane's V.  Bound by the instructions of
// the choice -- `top` rounds of a maximum over the wave -- and, for few tokens, by the launch.
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
// the largest of the wave's values, in every lane
__device__ inline unsigned wave_max(unsigned v) {
  v = max(v, dpp<0x111>(v));  // row_shr 1, 2, 4, 8: lane 15 of a row of sixteen has the row's
  v = max(v, dpp<0x112>(v));
  v = max(v, dpp<0x114>(v));
  v = max(v, dpp<0x118>(v));
  v = max(v, dpp<0x142>(v));  // row_bcast 15, 31: lane 63 has the wave's
  v = max(v, dpp<0x143>(v));
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// the lane's V logits; those past the last expert -inf
template <int TYPE, int V>
__device__ inline void load_logits(const Route& a, int token, int lane, float (&x)[V]) {
  const auto* row = static_cast<const typename Elem<TYPE>::type*>(a.logits) + token * a.ld;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    x[v] = e < a.experts ? (float)row[e] : -__builtin_inff();
  }
}

// x to scores
template <int V>
__device__ inline void scores(const Route& a, const float (&x)[V], float (&s)[V]) {
  const float inf = __builtin_inff();
  if (a.score == TETRIS_SCORE_SIGMOID) {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = 1.f / (1.f + expf(-x[v]));
    return;
  }
  unsigned key = 0x007fffffu;
#pragma unroll
  for (int v = 0; v < V; ++v) key = max(key, key_of(x[v]));
  key = wave_max(key);
  const float top = __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
  float sum = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s[v] = top == -inf && !(x[v] != x[v]) ? 0.f : x[v] == top ? 1.f : expf(x[v] - top);
    sum += s[v];
  }
  sum = wave_sum(sum);
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = sum == 0.f ? 0.f : s[v] / sum;
}

// ranks -> keys of the experts that may be chosen, zero for the others
template <int V>
__device__ inline void keys_of(const Route& a, int lane, float* shared, const float (&rank)[V], const float (&two)[V], unsigned (&key)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) key[v] = lane * V + v < a.experts ? key_of(rank[v]) : 0u;
  if (a.groups == 1 || a.top_groups == a.groups) return;
  const float inf = __builtin_inff();
  const int size = a.experts / a.groups;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (lane * V + v < a.experts) shared[lane * V + v] = a.group_by == TETRIS_GROUP_TWO ? two[v] : rank[v];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  unsigned mine = 0;
  if (lane < a.groups) {
    float first = -inf, second = -inf;
    for (int i = 0; i < size; ++i) {
      float v = shared[lane * size + i];
      v = v != v ? -inf : v;
      second = fmaxf(second, fminf(first, v));
      first = fmaxf(first, v);
    }
    mine = key_of(a.group_by == TETRIS_GROUP_TWO ? first + second : first);
  }
  int before = 0;
  for (int g = 0; g < a.groups; ++g) {
    const unsigned other = (unsigned)__builtin_amdgcn_readlane((int)mine, g);
    before += other > mine || (other == mine && g < lane);
  }
  const unsigned long long stay = __ballot(lane < a.groups && before < a.top_groups);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    if (e < a.experts && !((stay >> (e / size)) & 1)) key[v] = 0;
  }
}

template <int TYPE, int V>
__global__ __launch_bounds__(256) void route_kernel(Route a, int* __restrict__ index, float* __restrict__ weight) {
  __shared__ float shared[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = blockIdx.x * 4 + wave;
  if (token >= a.tokens) return;
  float x[V], s[V], rank[V], two[V];
  unsigned key[V];
  load_logits<TYPE, V>(a, token, lane, x);
  scores<V>(a, x, s);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float b = a.bias && lane * V + v < a.experts ? a.bias[lane * V + v] : 0.f;
    two[v] = s[v] + b;
    rank[v] = a.bias ? two[v] : x[v];
  }
  keys_of<V>(a, lane, shared[wave], rank, two, key);

  // the best that is left, `top` times; lane r keeps the r-th
  int my_index = 0;
  float my_score = 0.f, sum = 0.f;
  for (int r = 0; r < a.top; ++r) {
    unsigned best = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) best = max(best, key[v]);
    const unsigned all = wave_max(best);
    const int owner = __builtin_ctzll(__ballot(best == all));
    int place = 0;
    float score = 0.f;
    bool found = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool this_one = !found && key[v] == all;
      if (this_one) place = v, score = s[v];
      found |= this_one;
      if (this_one && lane == owner) key[v] = 0;
    }
    place = __builtin_amdgcn_readlane(place, owner);
    score = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(score), owner));
    sum += score;
    if (lane == r) my_index = owner * V + place, my_score = score;
  }
  if (lane < a.top) {
    const float w = !a.renorm ? my_score : sum == 0.f ? 0.f : my_score / sum;
    index[(int64_t)token * a.top + lane] = my_index;
    weight[(int64_t)token * a.top + lane] = w * a.scale;
  }
}

// With s the scores, c the chosen, S the sum of theirs and d_j = scale dweight_j (renorm: (d_j - sum_l d_l s_l / S) / S):
//   sigmoid  dlogit_i = s_i (1 - s_i) d_i for the chosen, else 0
//   softmax  dlogit_i = s_i (d_i - sum_j s_j d_j), with d_i = 0 for those not chosen; with renorm that sum is zero
template <int TYPE, int V>
__global__ __launch_bounds__(256) void route_backward_kernel(Route a, const int* __restrict__ index, const float* __restrict__ dweight,
                                                             typename Elem<TYPE>::type* __restrict__ out, int64_t ld_out) {
  __shared__ float shared[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = blockIdx.x * 4 + wave;
  if (token >= a.tokens) return;
  float x[V], s[V], d[V];
  load_logits<TYPE, V>(a, token, lane, x);
  scores<V>(a, x, s);
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
  if (a.renorm) {
    const float sum = wave_sum(score);
    const float mean = sum == 0.f ? 0.f : wave_sum(dw * score) / sum;
    dw = sum == 0.f || e < 0 ? 0.f : (dw - mean) / sum;
  }
  const float all = a.score == TETRIS_SCORE_SOFTMAX && !a.renorm ? wave_sum(dw * score) : 0.f;
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
    const float g = a.score == TETRIS_SCORE_SIGMOID ? s[v] * (1.f - s[v]) * d[v] : s[v] * (d[v] - all);
    if (lane * V + v < a.experts) row[lane * V + v] = (typename Elem<TYPE>::type)g;
  }
}

template <int TYPE, int V>
void launch_route(const Route& a, int* index, float* weight, hipStream_t s) {
  hipLaunchKernelGGL((route_kernel<TYPE, V>), dim3((a.tokens + 3) / 4), dim3(256), 0, s, a, index, weight);
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
  return {logits, ld, tokens, r->experts, r->top, r->score, r->groups, r->top_groups, r->group_by, r->renorm, r->scale, bias};
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
  by_type(type, [&](auto t) {
    by_width<decltype(t)::value>(r->experts, [&](auto v) { launch_route<decltype(t)::value, decltype(v)::value>(a, d_index, d_weight, s); });
  });
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

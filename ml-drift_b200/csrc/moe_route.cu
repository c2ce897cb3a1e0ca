// Routing of tokens to experts: scores, a bias for balance, groups, the k best, their weights.
//
// A warp takes a token, a lane every 32nd expert.  Values (score + bias) become integers that are ordered as they are, so that the
// largest of a warp's is two reductions of 32 bits and the lowest number among equals one more.  Without a bias and with groups
// that go by one expert the order is that of the logits, whatever the score: nothing is computed but the chosen ones' scores
// (and, without renormalising, the softmax's sum).  With them values are compared in 64 bits: in 32 some token of a long prompt
// has two within a rounding of one another.
#include <cuda_fp16.h>

#include <cfloat>

#include "common.cuh"
#include "kernels.h"

namespace mld {
namespace {

constexpr uint32_t kAll = 0xffffffffu;
constexpr int kRouteWarps = 4;

struct RouteArgs {
  const void* logits;
  int64_t stride;
  const float* bias;
  int32_t* ids;
  float* weights;
  int tokens, experts, top_k, sigmoid, groups, per_group, top_groups, group_best, renormalise, f16;
  float factor;
};

// Numbers in the order of the values; every value that is one (not NaN) has a number above 0.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ ((u >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
  return u ^ ((u >> 63) != 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
  const uint32_t hi = static_cast<uint32_t>(k >> 32), top = warp_max(hi);
  const uint32_t lo = warp_max(hi == top ? static_cast<uint32_t>(k) : 0u);
  return static_cast<uint64_t>(top) << 32 | lo;
}
__device__ __forceinline__ double value_of(uint64_t key) {
  return __longlong_as_double(static_cast<long long>(key ^ ((key >> 63) != 0 ? 1ull << 63 : ~0ull)));
}

// VALUES: the order goes by values in 64 bits, else by logits.  N: experts of a lane.
template <bool VALUES, int N>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_kernel(RouteArgs a) {
  using Key = typename std::conditional<VALUES, uint64_t, uint32_t>::type;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, token = static_cast<int>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
  if (token >= a.tokens) return;
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = 32 * i + lane;
    x[i] = -INFINITY;
    if (e < a.experts) {
      const int64_t at = token * a.stride + e;
      x[i] = a.f16 ? __half2float(static_cast<const __half*>(a.logits)[at]) : static_cast<const float*>(a.logits)[at];
      x[i] = x[i] == x[i] ? fminf(x[i], FLT_MAX) + 0.0f : -INFINITY;  // (+ 0: -0 is ordered as 0)
    }
  }
  float top = -INFINITY;  // the largest logit
#pragma unroll
  for (int i = 0; i < N; ++i) top = fmaxf(top, x[i]);
  {
    const uint32_t k = warp_max(ordered(top));
    top = __uint_as_float(k ^ ((k >> 31) != 0 ? 0x80000000u : 0xffffffffu));
  }
  // keys: 0 for an expert that is not to be had
  Key key[N];
  if constexpr (VALUES) {
    double v[N], sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0;
      if (x[i] > -INFINITY) {
        v[i] = a.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x[i]))) : exp(static_cast<double>(x[i]) - static_cast<double>(top));
        sum += v[i];
      }
    }
    if (!a.sigmoid) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kAll, sum, off);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!a.sigmoid) v[i] /= sum;
      if (a.bias != nullptr && 32 * i + lane < a.experts) v[i] += static_cast<double>(a.bias[32 * i + lane]);
      key[i] = x[i] > -INFINITY && v[i] > -INFINITY ? ordered(v[i]) : 0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = x[i] > -INFINITY ? ordered(x[i]) : 0;
  }
  if (a.groups > 1 && a.top_groups < a.groups) {
    // lane g gets the key of group g
    Key mine = 0;
    for (int g = 0; g < a.groups; ++g) {
      const int from = g * a.per_group, to = from + a.per_group;
      Key first = 0, second = 0;  // of this lane's experts in the group
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = 32 * i + lane;
        const Key k = e >= from && e < to ? key[i] : 0;
        second = k > first ? first : k > second ? k : second;
        first = k > first ? k : first;
      }
      Key best = warp_max(first);
      if constexpr (VALUES) {
        if (a.group_best == 2) {
          // the largest once out of the way, of the one lane that holds it
          const int holder = __ffs(__ballot_sync(kAll, first == best)) - 1;
          const Key next = warp_max(lane == holder ? second : first);
          const double s = (best == 0 ? -INFINITY : value_of(best)) + (next == 0 ? -INFINITY : value_of(next));
          best = s > -INFINITY ? ordered(s) : 0;
        }
      }
      if (lane == g) mine = best;
    }
    uint32_t kept = 0;
    for (int n = 0; n < a.top_groups; ++n) {
      const bool open = lane < a.groups && (kept >> lane & 1u) == 0;
      const Key best = warp_max(open ? mine : static_cast<Key>(0));
      kept |= 1u << (__ffs(__ballot_sync(kAll, open && mine == best)) - 1);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = 32 * i + lane;
      if (e >= a.experts || (kept >> (e / a.per_group) & 1u) == 0) key[i] = 0;
    }
  }
  // the k best: each time the largest of the lanes' largest, which its lane then gives up
  float chosen = -INFINITY;  // lane j: the logit of the j-th
  int id = -1;
  for (int j = 0; j < a.top_k; ++j) {
    Key best = 0;
    float best_x = -INFINITY;
    int best_e = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool more = VALUES ? key[i] > best || (key[i] == best && x[i] > best_x) : key[i] > best;
      if (more) {
        best = key[i];
        best_x = x[i];
        best_e = 32 * i + lane;
      }
    }
    const Key top_key = warp_max(best);
    if (top_key == 0) break;  // none left
    bool here = best == top_key;
    if constexpr (VALUES) {
      const uint32_t k = here ? ordered(best_x) : 0u, top_x = warp_max(k);
      here = here && k == top_x;
    }
    const int e = static_cast<int>(__reduce_min_sync(kAll, here ? static_cast<uint32_t>(best_e) : 0xffffffffu));
    const float its_x = __shfl_sync(kAll, best_x, e & 31);
    if (lane == j) {
      id = e;
      chosen = its_x;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (32 * i + lane == e) key[i] = 0;
  }
  // Their weights.  Renormalised, a softmax's sum cancels, and what is common to the chosen, too: they are taken against the largest
  // of them (of a sigmoid when all are so small that it is the exponential), so that they never vanish together.
  const float chosen_top = [&] {
    const uint32_t k = warp_max(id >= 0 ? ordered(chosen) : 0u);
    return __uint_as_float(k ^ ((k >> 31) != 0 ? 0x80000000u : 0xffffffffu));
  }();
  float score = 0.0f, by = 1.0f;
  if (id >= 0) {
    if (a.sigmoid && !(a.renormalise && chosen_top < -30.0f))
      score = 1.0f / (1.0f + expf(-chosen));
    else
      score = expf(chosen - (a.renormalise ? chosen_top : top));
  }
  if (a.renormalise || !a.sigmoid) {
    by = score;
    if (!a.renormalise) {
      by = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) by += x[i] > -INFINITY ? expf(x[i] - top) : 0.0f;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) by += __shfl_xor_sync(kAll, by, off);
  }
  if (lane < a.top_k) {
    a.ids[static_cast<int64_t>(token) * a.top_k + lane] = id;
    a.weights[static_cast<int64_t>(token) * a.top_k + lane] = id >= 0 ? a.factor * (score / by) : 0.0f;
  }
}

template <bool VALUES>
int launch(const RouteArgs& a, cudaStream_t stream) {
  const int n = div_up(a.experts, 32);
  void (*kern)(RouteArgs) = n <= 2    ? moe_route_kernel<VALUES, 2>
                            : n <= 4  ? moe_route_kernel<VALUES, 4>
                            : n <= 8  ? moe_route_kernel<VALUES, 8>
                            : n <= 16 ? moe_route_kernel<VALUES, 16>
                                      : moe_route_kernel<VALUES, 32>;
  MLD_CUDA_CHECK(launch_overlapped(kern, dim3(div_up(a.tokens, kRouteWarps)), dim3(kRouteWarps * 32), 0, stream, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

}  // namespace
}  // namespace mld

using namespace mld;

extern "C" int mld_moe_route(const mld_moe_route_desc* d, const void* logits, int64_t stride, const float* bias, int32_t* ids,
                             float* weights, int32_t tokens, void* stream) {
  MLD_REQUIRE(d != nullptr, "null argument");
  MLD_REQUIRE(d->experts >= 1 && d->experts <= 1024, "experts must be 1 to 1024");
  MLD_REQUIRE(d->score == MLD_MOE_SOFTMAX || d->score == MLD_MOE_SIGMOID, "bad score");
  MLD_REQUIRE(d->groups >= 1 && d->groups <= 32 && d->experts % d->groups == 0, "groups must be 1 to 32 and divide experts");
  MLD_REQUIRE(d->top_groups >= 1 && d->top_groups <= d->groups, "top_groups must be 1 to groups");
  MLD_REQUIRE(d->top_k >= 1 && d->top_k <= 32 && d->top_k <= d->top_groups * (d->experts / d->groups),
              "top_k must be 1 to 32 and at most the experts of the groups that are kept");
  MLD_REQUIRE(d->group_best == 1 || (d->group_best == 2 && d->experts / d->groups >= 2),
              "group_best must be 1, or 2 with groups of two experts or more");
  MLD_REQUIRE(d->factor > -INFINITY && d->factor < INFINITY, "factor must be finite");
  MLD_REQUIRE(tokens >= 0, "negative number of tokens");
  if (tokens == 0) return MLD_OK;
  MLD_REQUIRE(logits != nullptr && ids != nullptr && weights != nullptr, "null tensor");
  MLD_REQUIRE(stride >= 0, "negative stride");
  const uintptr_t esz = d->f16 ? 2 : 4;
  MLD_REQUIRE(reinterpret_cast<uintptr_t>(logits) % esz == 0 &&
                  ((reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights)) & 3) == 0,
              "a tensor that is not aligned to its type");
  RouteArgs a = {};
  a.logits = logits;
  a.stride = stride;
  a.bias = bias;
  a.ids = ids;
  a.weights = weights;
  a.tokens = tokens;
  a.experts = d->experts;
  a.top_k = d->top_k;
  a.sigmoid = d->score == MLD_MOE_SIGMOID;
  a.groups = d->groups;
  a.per_group = d->experts / d->groups;
  a.top_groups = d->top_groups;
  a.group_best = d->group_best;
  a.renormalise = d->renormalise != 0;
  a.f16 = d->f16 != 0;
  a.factor = d->factor;
  const bool values = bias != nullptr || (d->groups > d->top_groups && d->group_best == 2);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return values ? launch<true>(a, s) : launch<false>(a, s);
}

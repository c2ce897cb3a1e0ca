// Routing of tokens to experts: scores, a bias for balance, groups, the k best, their weights.
//
// A warp takes a token, a lane a run of neighbouring experts.  Without a bias and with groups that go by one expert the order is that
// of the logits, whatever the score: nothing is computed but the chosen ones' scores (and, without renormalising, the softmax's
// sum).  Else experts are compared by values in 32 bits first; where two that the choice hangs on lie closer to one another
// than the error of those (some token of a long prompt always has such), the token is gone through again in 64.  So it is where the
// choice hangs on two groups whose logits differ and whose values in 64 bits might not: of equal groups the first counts, not
// the one with the larger logit.
// Bound by instructions: k rounds of the largest of each lane's, the warp's largest (one instruction), its lane and place.
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
  int wide;  // rows may be read in pieces
  float factor;
};

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_min(float v) {
  float r;
  asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// (as integers in the order of the values, the upper halves first)
__device__ __forceinline__ double warp_max(double v) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v)), k = u ^ ((u >> 63) != 0 ? ~0ull : 1ull << 63);
  const uint32_t hi = static_cast<uint32_t>(k >> 32), top = __reduce_max_sync(kAll, hi);
  const uint32_t low = __reduce_max_sync(kAll, hi == top ? static_cast<uint32_t>(k) : 0u);
  const uint64_t m = static_cast<uint64_t>(top) << 32 | low;
  return __longlong_as_double(static_cast<long long>(m ^ ((m >> 63) != 0 ? 1ull << 63 : ~0ull)));
}
__device__ __forceinline__ double warp_min(double v) { return -warp_max(-v); }

// Whether two logits, of which the upper is the larger, surely have different values in 64 bits: apart by more than 2^-16, where
// neither a sigmoid rounds to 1 (below 16, such differ by 1e-12) nor an exponential vanishes.
__device__ __forceinline__ bool apart_in_64(const RouteArgs& a, float upper, float lower, float top) {
  return upper - lower > 0x1p-16f && (a.sigmoid ? lower < 16.0f && lower > -600.0f : lower - top > -600.0f);
}

// The k best of keys (-infinity: not to be had), into lane j the j-th: its expert (-1: none) and its logit.  Of equal keys (64 bits)
// the larger logit, then the lower number.  False: something that the choice hangs on is closer than `tolerance` (0: never), or
// is not surely the same by values, of keys that are logits (the largest is `top`).
template <bool LOGITS, typename Key, int N>
__device__ __forceinline__ bool choose(const RouteArgs& a, Key (&key)[N], const float (&x)[N], int lane, float tolerance, float top, int& id,
                                       float& logit) {
  constexpr bool kWide = sizeof(Key) == 8;
  constexpr Key kNone = static_cast<Key>(-INFINITY);
  bool clear = true;
  const auto close = [&](Key upper, Key lower, float tol) {  // (an infinite value is close to nothing but its like)
    return !(upper - lower > static_cast<Key>(tol) * (1 + (upper < 0 ? -upper : upper)));
  };
  if (a.top_groups < a.groups) {
    const auto better = [](Key p, Key q) { return p > q ? p : q; };
    const auto worse = [](Key p, Key q) { return p < q ? p : q; };
    const int run = a.per_group / N;  // lanes of a group, if it is whole lanes
    const bool whole = a.per_group % N == 0 && (run & (run - 1)) == 0;
    Key sum = kNone, size = 0;  // of this lane's group (whole), or of group `lane`; the sum of its terms without their signs
    int group = lane;
    const auto no_sign = [](Key v) { return v < 0 ? -v : v; };
    if (whole) {
      Key first = kNone, second = kNone;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        second = better(second, worse(first, key[i]));
        first = better(first, key[i]);
      }
      for (int off = 1; off < run; off <<= 1) {
        const Key f = __shfl_xor_sync(kAll, first, off), s = __shfl_xor_sync(kAll, second, off);
        second = better(better(second, s), worse(first, f));
        first = better(first, f);
      }
      sum = a.group_best == 2 ? first + second : first;
      size = a.group_best == 2 ? no_sign(first) + no_sign(second) : no_sign(first);
      group = lane / run;
    } else {
      for (int g = 0; g < a.groups; ++g) {
        const int from = g * a.per_group - lane * N, to = from + a.per_group;
        Key first = kNone, second = kNone;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const Key k = i >= from && i < to ? key[i] : kNone;
          second = better(second, worse(first, k));
          first = better(first, k);
        }
        const Key best = warp_max(first);
        Key s = best, z = no_sign(best);
        if (a.group_best == 2) {
          // the largest once out of the way, of the first lane that has it
          const int holder = __ffs(__ballot_sync(kAll, first == best)) - 1;
          const Key next = warp_max(lane == holder ? second : first);
          s += next;
          z += no_sign(next);
        }
        if (lane == g) {
          sum = s;
          size = z;
        }
      }
    }
    if (!(sum > kNone)) sum = kNone;  // (a NaN, too)
    int ahead = 0;  // groups before this one in the order
    for (int g = 0; g < a.groups; ++g) {
      const Key s = __shfl_sync(kAll, sum, whole ? g * run : g);
      ahead += s > sum || (s == sum && g < group) ? 1 : 0;
    }
    const bool exists = group < a.groups, kept = exists && ahead < a.top_groups;
    if (tolerance > 0) {
      // A sum is as exact as its terms, not as itself: of two sigmoids with their biases within 2^-24 (10 + 2 size), below the
      // tolerance of 16.7 2^-24 (1 + size); a softmax's likewise.
      const Key error = static_cast<Key>(tolerance) * (1 + size), kMost = static_cast<Key>(INFINITY);
      const bool known = error < kMost;
      const Key least = warp_min(!kept ? kMost : sum > kNone && !known ? kNone : sum - error);
      const Key most = warp_max(!exists || kept || !(sum > kNone) ? kNone : known ? sum + error : kMost);
      clear = !(most > kNone && !(least > most));
    }
    if constexpr (LOGITS) {
      // the best one that is not kept: those above it have to be apart from it, and, where one of its like is kept, those below it
      const float most = warp_max(exists && !kept ? sum : kNone);
      const bool like = __any_sync(kAll, kept && sum == most);
      const bool counts = exists && sum > kNone && sum != most && (kept || like);
      clear = !__any_sync(kAll, most > kNone && counts && !apart_in_64(a, fmaxf(sum, most), fminf(sum, most), top));
    }
    if (whole) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (!kept) key[i] = kNone;
    } else {
      const uint32_t mask = __ballot_sync(kAll, kept);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = lane * N + i;
        if (e >= a.experts || (mask >> (e / a.per_group) & 1u) == 0) key[i] = kNone;
      }
    }
  }
  Key before = static_cast<Key>(INFINITY);
  for (int j = 0; j < a.top_k + (tolerance > 0 ? 1 : 0); ++j) {
    Key best[N];
#pragma unroll
    for (int i = 0; i < N; ++i) best[i] = key[i];
#pragma unroll
    for (int s = N / 2; s > 0; s /= 2)
#pragma unroll
      for (int i = 0; i < s; ++i) best[i] = best[i + s] > best[i] ? best[i + s] : best[i];
    const Key most = warp_max(best[0]);
    if (!(most > kNone)) break;  // none left
    if (tolerance > 0) {
      if (j > 0 && close(before, most, tolerance)) clear = false;
      before = most;
      if (j == a.top_k) break;
    }
    // the lane's first place with it; of equal values, the one with the larger logit
    int place = -1;
    float its = -INFINITY;
#pragma unroll
    for (int i = N - 1; i >= 0; --i)
      if (key[i] == most && (!kWide || x[i] >= its)) {
        place = i;
        its = x[i];
      }
    bool here = place >= 0;
    if constexpr (kWide) {
      const float larger = warp_max(its);
      here = here && its == larger;
    }
    const int holder = __ffs(__ballot_sync(kAll, here)) - 1;
    const int e = __shfl_sync(kAll, lane * N + place, holder);
    const float l = __shfl_sync(kAll, its, holder);
    if (lane == j) {
      id = e;
      logit = l;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane == holder && i == place) key[i] = kNone;
  }
  return clear;
}

// A logit as it counts: NaN as -infinity, +infinity as the largest number, -0 as 0.
__device__ __forceinline__ float counted(float x) { return x == x ? fminf(x, FLT_MAX) + 0.0f : -INFINITY; }

// The same by values in 64 bits, from the logits on (which then need not lie in memory for it while it is not needed).  The expert
// in the upper half, the logit in the lower.
template <int N>
__device__ __noinline__ uint64_t choose_in_64(RouteArgs a, int token, float top) {
  const int lane = threadIdx.x & 31;
  float x[N];
  double v[N], sum = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t at = token * a.stride + lane * N + i;
    x[i] = -INFINITY;
    if (lane * N + i < a.experts)
      x[i] = counted(a.f16 ? __half2float(static_cast<const __half*>(a.logits)[at]) : static_cast<const float*>(a.logits)[at]);
    v[i] = 0.0;
    if (x[i] > -INFINITY) {
      if (a.sigmoid) {
        v[i] = 1.0 / (1.0 + exp(-static_cast<double>(x[i])));
      } else {
        // (below the normal numbers as the square of one, which is rounded once: there exp's error may be all of a value)
        const double y = static_cast<double>(x[i]) - static_cast<double>(top);
        const double e = exp(y < -700.0 ? 0.5 * y : y);
        v[i] = y < -700.0 ? e * e : e;
      }
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
    if (a.bias != nullptr && lane * N + i < a.experts) v[i] += static_cast<double>(a.bias[lane * N + i]);
    if (!(x[i] > -INFINITY && v[i] > -INFINITY)) v[i] = -INFINITY;
  }
  int id = -1;
  float logit = -INFINITY;
  choose<false, double, N>(a, v, x, lane, 0.0f, top, id, logit);
  return static_cast<uint64_t>(static_cast<uint32_t>(id)) << 32 | __float_as_uint(logit);
}

// VALUES: the order goes by values, else by logits.  N: experts of a lane.
template <bool VALUES, int N>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_kernel(RouteArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, token = static_cast<int>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
  if (token >= a.tokens) return;
  float x[N];
  {
    const int64_t at = token * a.stride + lane * N;
    if (a.wide) {  // (whole lanes, 16-byte pieces of 32-bit logits, 2 N bytes of halves)
      if (lane * N < a.experts) {
        if (a.f16) {
          __half h[N];
          constexpr int kPiece = N * 2 < 16 ? N * 2 : 16;
#pragma unroll
          for (int i = 0; i < N * 2 / kPiece; ++i) {
            const __half* p = static_cast<const __half*>(a.logits) + at + i * (kPiece / 2);
            if constexpr (kPiece == 16)
              reinterpret_cast<uint4*>(h)[i] = *reinterpret_cast<const uint4*>(p);
            else if constexpr (kPiece == 8)
              reinterpret_cast<uint2*>(h)[i] = *reinterpret_cast<const uint2*>(p);
            else
              reinterpret_cast<uint32_t*>(h)[i] = *reinterpret_cast<const uint32_t*>(p);
          }
#pragma unroll
          for (int i = 0; i < N; ++i) x[i] = __half2float(h[i]);
        } else {
          constexpr int kPiece = N < 4 ? N : 4;
#pragma unroll
          for (int i = 0; i < N / kPiece; ++i) {
            const float* p = static_cast<const float*>(a.logits) + at + i * kPiece;
            if constexpr (kPiece == 4)
              reinterpret_cast<float4*>(x)[i] = *reinterpret_cast<const float4*>(p);
            else
              reinterpret_cast<float2*>(x)[i] = *reinterpret_cast<const float2*>(p);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (lane * N + i < a.experts)
          x[i] = a.f16 ? __half2float(static_cast<const __half*>(a.logits)[at + i]) : static_cast<const float*>(a.logits)[at + i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = lane * N + i < a.experts ? counted(x[i]) : -INFINITY;
  }
  float top = x[0];  // the largest logit
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  top = warp_max(top);
  int id = -1;
  float chosen = -INFINITY;  // lane j: the logit of the j-th
  bool clear;
  if constexpr (VALUES) {
    float v[N], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = x[i] > -INFINITY ? (a.sigmoid ? 1.0f / (1.0f + expf(-x[i])) : expf(x[i] - top)) : 0.0f;
      sum += v[i];
    }
    if (!a.sigmoid) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kAll, sum, off);
      sum = 1.0f / sum;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!a.sigmoid) v[i] *= sum;
      if (a.bias != nullptr && lane * N + i < a.experts) v[i] += a.bias[lane * N + i];
      if (!(x[i] > -INFINITY && v[i] > -INFINITY)) v[i] = -INFINITY;
    }
    // Errors of two values: 2^-24 times 6 each of a sigmoid's score (exp 2, a sum, a quotient, the bias); N + 5 more of a softmax's
    // sum, which has 37 at most.
    const float tolerance = a.sigmoid ? 1.0e-6f : 6.0e-6f;
    clear = choose<false, float, N>(a, v, x, lane, tolerance, top, id, chosen);
  } else {
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = x[i];
    clear = choose<true, float, N>(a, v, x, lane, 0.0f, top, id, chosen);
  }
  if (!clear) {
    const uint64_t again = choose_in_64<N>(a, token, top);
    id = static_cast<int>(again >> 32);
    chosen = __uint_as_float(static_cast<uint32_t>(again));
  }
  // Their weights.  Renormalised, a softmax's sum cancels, and what is common to the chosen, too: they are taken against the largest
  // of them (of a sigmoid when all are so small that it is the exponential), so that they never vanish together.
  const float chosen_top = warp_max(chosen);
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

template <bool VALUES, int N>
int launch_of(RouteArgs a, cudaStream_t stream) {
  const int piece = a.f16 ? (N * 2 < 16 ? N * 2 : 16) : (N < 4 ? N * 4 : 16);
  a.wide = a.experts % N == 0 && reinterpret_cast<uintptr_t>(a.logits) % piece == 0 && (a.tokens == 1 || a.stride * (a.f16 ? 2 : 4) % piece == 0);
  MLD_CUDA_CHECK(launch_overlapped(moe_route_kernel<VALUES, N>, dim3(div_up(a.tokens, kRouteWarps)), dim3(kRouteWarps * 32), 0, stream, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}
template <bool VALUES>
int launch(const RouteArgs& a, cudaStream_t stream) {
  const int n = div_up(a.experts, 32);
  return n <= 2    ? launch_of<VALUES, 2>(a, stream)
         : n <= 4  ? launch_of<VALUES, 4>(a, stream)
         : n <= 8  ? launch_of<VALUES, 8>(a, stream)
         : n <= 16 ? launch_of<VALUES, 16>(a, stream)
                   : launch_of<VALUES, 32>(a, stream);
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
  MLD_REQUIRE(tokens >= 0 && tokens <= 1 << 30, "tokens must be 0 to 2^30");
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

// Norms of queries and keys for each head and the position rotation in one pass; with a 4-bit cache the keys, and the values
// beside them, are quantised into its pages in the same pass.
//
// The reference assembles this from an RMS norm per head, a rotation (ml_drift/common/kernels/rope.cc:70-89) and, behind them,
// the write into the cache (samples/llm/qwen3_model_builder.cc:426-508, 543-846): three passes over q and k.
//   y = x * w / sqrt(mean(x^2) + eps);   pair i of a head: (a, b) -> (a cos - b sin, b cos + a sin),
//   angle = position[axis of i] / (min_timescale * (max_timescale / min_timescale)^(2 i / rotary_dim))
// The angle is taken in turns, as a product of 32 x 64-bit integers modulo one turn (2^64), since a 32-bit float loses the
// decimals of position * frequency for long contexts (position 131071: 0.008 rad); what is left is exact to 2^-31 turns.
//
// D / 8 lanes hold a head, eight neighbouring values each (one 16-byte load); a block takes 2048 values of one token.
// Cosines and sines of a token are worked out once per block.
#include <cuda_fp16.h>
#include <math.h>
#include <string.h>

#include <new>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace mld {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;

struct RopeArgs {
  const void *q, *k, *v;
  void *q_out, *k_out;
  const void *q_weight, *k_weight;
  long long q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements from token to token
  const int32_t* positions;                                            // [axes][tokens]
  uint8_t* pool;
  const int32_t* slots;  // [tokens]
  int slots_end;         // slots of the pool
  int page_tokens, kv_heads_pool;
  int tokens, q_heads, k_heads, v_heads;
  int half_pairs;        // pairs of a head that are turned
  int neighbours;
  float eps;
  int section_end[4];
  unsigned long long steps[kMaxPairs];  // 2^-64 turns per position
};

template <typename T>
struct Eight;
template <>
struct Eight<__half> {
  static __device__ __forceinline__ void load(const __half* p, float (&x)[8]) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__half* p, const float (&x)[8]) {
    __align__(16) __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  }
};
template <>
struct Eight<float> {
  static __device__ __forceinline__ void load(const float* p, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 f = reinterpret_cast<const float4*>(p)[i];
      x[4 * i] = f.x;
      x[4 * i + 1] = f.y;
      x[4 * i + 2] = f.z;
      x[4 * i + 3] = f.w;
    }
  }
  static __device__ __forceinline__ void store(float* p, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  }
};

// Quantises the eight values of a lane (its place in the head: l) into the tile at `tile`; the four lanes of a group of 32
// call it together.  A group that holds an infinity or a NaN gets a NaN scale.
template <int D>
__device__ __forceinline__ void put_eight(uint8_t* tile, bool is_v, int tau, int l, const float (&x)[8], unsigned mask, bool store) {
  float r[8], top = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r[i] = __half2float(__float2half_rn(x[i]));
    top = fmaxf(top, fabsf(r[i]));
    finite = finite && fabsf(r[i]) <= 65504.0f;
  }
  if (!finite) top = INFINITY;
  top = fmaxf(top, __shfl_xor_sync(mask, top, 1));
  top = fmaxf(top, __shfl_xor_sync(mask, top, 2));
  // eight significant bits (round to nearest even), then fp16, which rounds only what is below its normal range
  uint32_t bits = __float_as_uint(__fdiv_rn(top, 7.0f));
  bits = (bits + 0x7FFFu + ((bits >> 16) & 1u)) & 0xFFFF0000u;
  const __half scale = top == INFINITY ? __ushort_as_half(0x7E00) : __float2half_rn(__uint_as_float(bits));
  const float s = __half2float(scale);
  uint32_t code[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = s > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(r[i], s)), -7.0f), 7.0f) : 0.0f;
    code[i] = static_cast<uint32_t>(static_cast<int>(c) + 8);
  }
  if (!store) return;
  const int j = l >> 2, t = l & 3;
  if (!is_v) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= code[i] << (4 * (4 * (i & 1) + (i >> 1)));
    *reinterpret_cast<uint32_t*>(tile + kv4::k_word<D>(tau, j, t)) = w;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<uint16_t*>(tile + kv4::v_half<D>(tau, j, 2 * t + h)) =
          static_cast<uint16_t>(code[4 * h] | code[4 * h + 1] << 4 | code[4 * h + 2] << 8 | code[4 * h + 3] << 12);
  }
  if (t == 0) *reinterpret_cast<__half*>(tile + kv4::scale_at<D>(is_v, tau, j)) = scale;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) qk_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int kLanes = D / 8;
  constexpr int kHeads = kThreads / kLanes;
  __shared__ float cosines[kMaxPairs], sines[kMaxPairs];
  pdl_wait();
  const int token = blockIdx.x;
  const int l = threadIdx.x % kLanes;
  const int head = blockIdx.y * kHeads + threadIdx.x / kLanes;
  const bool is_q = head < a.q_heads;
  const bool is_k = !is_q && head < a.q_heads + a.k_heads;
  const bool is_v = !is_q && !is_k && head < a.q_heads + a.k_heads + a.v_heads;
  const int h = is_q ? head : is_k ? head - a.q_heads : head - a.q_heads - a.k_heads;
  float x[8] = {};
  if (is_q || is_k || is_v) {
    const T* src = is_q   ? static_cast<const T*>(a.q) + token * a.q_stride
                   : is_k ? static_cast<const T*>(a.k) + token * a.k_stride
                          : static_cast<const T*>(a.v) + token * a.v_stride;
    Eight<T>::load(src + h * D + 8 * l, x);
  }
  for (int i = threadIdx.x; i < a.half_pairs; i += kThreads) {
    int axis = 0;
#pragma unroll
    for (int s = 0; s < 3; ++s) axis += i >= a.section_end[s] ? 1 : 0;
    const long long pos = a.positions[static_cast<long long>(axis) * a.tokens + token];
    const unsigned long long turn = static_cast<unsigned long long>(pos) * a.steps[i];
    sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 4.656612873077393e-10f, &sines[i], &cosines[i]);
  }
  __syncthreads();
  // the lanes of a head stay together in what follows
  const unsigned mask = kLanes == 32 ? 0xFFFFFFFFu : ((1u << kLanes) - 1u) << ((threadIdx.x & 31) / kLanes * kLanes);
  if (is_q || is_k) {
    const T* w = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
    if (w != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
      const float r = rsqrtf(fmaf(sum, 1.0f / D, a.eps));
      float wf[8];
      Eight<T>::load(w + 8 * l, wf);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wf[i];
    }
    const int rot = 2 * a.half_pairs;
    if (a.neighbours) {
      if (8 * l < rot) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float c = cosines[4 * l + i], s = sines[4 * l + i], p = x[2 * i], n = x[2 * i + 1];
          x[2 * i] = p * c - n * s;
          x[2 * i + 1] = n * c + p * s;
        }
      }
    } else {
      const int far = a.half_pairs / 8;  // lanes between the halves of a pair
      const bool second = l >= far;
      const int other = l < far ? l + far : l < 2 * far ? l - far : l;
      const int from = ((threadIdx.x & 31) - l) + other;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(mask, x[i], from);
      if (l < 2 * far) {
        const int at = 8 * (second ? other : l);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = cosines[at + i], s = sines[at + i];
          x[i] = second ? x[i] * c + y[i] * s : x[i] * c - y[i] * s;
        }
      }
    }
    if (is_q) {
      Eight<T>::store(static_cast<T*>(a.q_out) + token * a.q_out_stride + h * D + 8 * l, x);
    } else if (a.k_out != nullptr) {
      Eight<T>::store(static_cast<T*>(a.k_out) + token * a.k_out_stride + h * D + 8 * l, x);
    }
  }
  if ((is_k || is_v) && a.pool != nullptr) {
    const int slot = a.slots[token];
    const bool store = slot >= 0 && slot < a.slots_end;
    const int page = store ? slot / a.page_tokens : 0, in_page = store ? slot - page * a.page_tokens : 0;
    uint8_t* tile = a.pool + ((static_cast<long long>(page) * a.kv_heads_pool + h) * (a.page_tokens / kv4::kTile) +
                              in_page / kv4::kTile) * kv4::tile_bytes(D);
    put_eight<D>(tile, is_v, in_page % kv4::kTile, l, x, mask, store);
  }
}

struct ReadArgs {
  const uint8_t* pool;
  const int32_t* slots;
  __half *k, *v;
  long long k_stride, v_stride;
  int slots_end, page_tokens, kv_heads, tokens;
};

// One lane gives eight neighbouring values of a token's key or value.  A slot outside the pool gives zeros.
template <int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8;
  pdl_wait();
  const int unit = blockIdx.y * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (unit >= 2 * a.kv_heads) return;
  const int token = blockIdx.x, l = threadIdx.x % kLanes, j = l >> 2, t = l & 3;
  const bool is_v = unit >= a.kv_heads;
  const int h = is_v ? unit - a.kv_heads : unit;
  const int slot = a.slots[token];
  __align__(16) __half2 y[4] = {};
  if (slot >= 0 && slot < a.slots_end) {
    const int page = slot / a.page_tokens, in_page = slot - page * a.page_tokens, tau = in_page % kv4::kTile;
    const uint8_t* tile = a.pool + ((static_cast<long long>(page) * a.kv_heads + h) * (a.page_tokens / kv4::kTile) +
                                    in_page / kv4::kTile) * kv4::tile_bytes(D);
    const float s = __half2float(*reinterpret_cast<const __half*>(tile + kv4::scale_at<D>(is_v, tau, j)));
    float c[8];
    if (!is_v) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + kv4::k_word<D>(tau, j, t));
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = static_cast<float>(static_cast<int>(w >> (4 * (4 * (i & 1) + (i >> 1))) & 15u) - 8);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w = *reinterpret_cast<const uint16_t*>(tile + kv4::v_half<D>(tau, j, 2 * t + i));
#pragma unroll
        for (int e = 0; e < 4; ++e) c[4 * i + e] = static_cast<float>(static_cast<int>(w >> (4 * e) & 15u) - 8);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __floats2half2_rn(c[2 * i] * s, c[2 * i + 1] * s);
  }
  __half* dst = is_v ? a.v + token * a.v_stride : a.k + token * a.k_stride;
  *reinterpret_cast<uint4*>(dst + h * D + 8 * l) = *reinterpret_cast<const uint4*>(y);
}

template <typename T, int D>
int launch_rope_t(const RopeArgs& a, cudaStream_t stream) {
  const dim3 grid(a.tokens, div_up(a.q_heads + a.k_heads + a.v_heads, kThreads / (D / 8)));
  MLD_CUDA_CHECK(launch_overlapped(qk_rope_kernel<T, D>, grid, dim3(kThreads), 0, stream, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}
int launch_rope(const RopeArgs& a, int head_dim, bool f16, cudaStream_t stream) {
  if (f16)
    return head_dim == 64    ? launch_rope_t<__half, 64>(a, stream)
           : head_dim == 128 ? launch_rope_t<__half, 128>(a, stream)
                             : launch_rope_t<__half, 256>(a, stream);
  return head_dim == 64    ? launch_rope_t<float, 64>(a, stream)
         : head_dim == 128 ? launch_rope_t<float, 128>(a, stream)
                           : launch_rope_t<float, 256>(a, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int check_kv4_desc(const mld_kv4_desc* d) {
  MLD_REQUIRE(d != nullptr, "null cache descriptor");
  MLD_REQUIRE(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, "head_dim must be 64, 128 or 256");
  MLD_REQUIRE(d->kv_heads >= 1 && d->kv_heads <= 1024, "kv_heads must be 1 to 1024");
  MLD_REQUIRE(d->page_tokens >= 16 && d->page_tokens % 16 == 0 && d->page_tokens <= 65536,
              "page_tokens must be a multiple of 16, 16 to 65536");
  MLD_REQUIRE(d->pages >= 1 && static_cast<int64_t>(d->pages) * d->page_tokens <= 0x7FFFFFFF,
              "a pool holds 1 to 2^31 - 1 tokens in whole pages");
  return MLD_OK;
}

}  // namespace mld

using namespace mld;

struct mld_qk_rope_plan {
  mld_qk_rope_desc d;
  unsigned long long steps[kMaxPairs];
  int section_end[4];
};

extern "C" {

size_t mld_kv4_page_bytes(const mld_kv4_desc* d) {
  if (check_kv4_desc(d) != MLD_OK) return 0;
  return static_cast<size_t>(d->kv_heads) * (d->page_tokens / kv4::kTile) * kv4::tile_bytes(d->head_dim);
}
size_t mld_kv4_pool_bytes(const mld_kv4_desc* d) { return mld_kv4_page_bytes(d) * (d != nullptr ? d->pages : 0); }

int mld_qk_rope_plan_create(const mld_qk_rope_desc* d, mld_qk_rope_plan** out) {
  MLD_REQUIRE(d != nullptr && out != nullptr, "null argument");
  MLD_REQUIRE(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, "head_dim must be 64, 128 or 256");
  MLD_REQUIRE(d->heads >= 0 && d->heads <= 4096 && d->kv_heads >= 0 && d->kv_heads <= 1024 && d->heads + d->kv_heads > 0,
              "heads must be 0 to 4096 and kv_heads 0 to 1024");
  MLD_REQUIRE(d->rotary_dim >= 0 && d->rotary_dim <= d->head_dim && d->rotary_dim % 16 == 0,
              "rotary_dim must be a multiple of 16 up to head_dim");
  MLD_REQUIRE(d->pairing == MLD_ROPE_HALVES || d->pairing == MLD_ROPE_NEIGHBOURS, "bad pairing");
  MLD_REQUIRE(d->axes >= 1 && d->axes <= 4, "positions have 1 to 4 axes");
  int64_t pairs = 0;
  for (int i = 0; i < d->axes; ++i) {
    MLD_REQUIRE(d->sections[i] >= 0, "negative section");
    pairs += d->sections[i];
  }
  MLD_REQUIRE(pairs == d->rotary_dim / 2, "the sections must add up to rotary_dim / 2 pairs");
  MLD_REQUIRE(d->min_timescale > 0.0f && d->max_timescale > 0.0f && isfinite(d->min_timescale) && isfinite(d->max_timescale),
              "timescales must be positive");
  MLD_REQUIRE(d->rms_eps >= 0.0f, "rms_eps must not be negative");
  mld_qk_rope_plan* p = new (std::nothrow) mld_qk_rope_plan();
  MLD_REQUIRE(p != nullptr, "out of host memory");
  p->d = *d;
  int end = 0;
  for (int i = 0; i < 4; ++i) p->section_end[i] = i < d->axes ? (end += d->sections[i]) : 0x7FFFFFFF;
  p->section_end[d->axes - 1] = 0x7FFFFFFF;
  const double ratio = static_cast<double>(d->max_timescale) / d->min_timescale;
  for (int i = 0; i < d->rotary_dim / 2; ++i) {
    const double timescale = d->min_timescale * pow(ratio, 2.0 * i / d->rotary_dim);
    const double turns = 1.0 / (timescale * 6.283185307179586476925);
    // whole turns per position change nothing
    const double part = turns - floor(turns);
    const double scaled = rint(part * 18446744073709551616.0);
    p->steps[i] = scaled >= 18446744073709551616.0 ? 0ull : static_cast<unsigned long long>(scaled);
  }
  *out = p;
  return MLD_OK;
}

int mld_qk_rope_plan_destroy(mld_qk_rope_plan* plan) {
  delete plan;
  return MLD_OK;
}

int mld_qk_rope_run(mld_qk_rope_plan* plan, const mld_qk_rope_io* io, int32_t tokens, void* stream) {
  MLD_REQUIRE(plan != nullptr && io != nullptr, "null argument");
  const mld_qk_rope_desc& d = plan->d;
  MLD_REQUIRE(tokens >= 0, "bad token count");
  const bool cached = io->pool != nullptr;
  if (cached) {
    if (const int rc = check_kv4_desc(io->cache); rc != MLD_OK) return rc;
    MLD_REQUIRE(io->cache->head_dim == d.head_dim && io->cache->kv_heads == d.kv_heads,
                "the cache's heads differ from the plan's");
    MLD_REQUIRE(aligned16(io->pool), "the pool must be 16-byte aligned");
  }
  if (tokens == 0) return MLD_OK;
  MLD_REQUIRE(d.heads == 0 || (io->q != nullptr && io->q_out != nullptr), "null query tensor");
  MLD_REQUIRE(d.kv_heads == 0 || (io->k != nullptr && (io->k_out != nullptr || cached)), "null key tensor");
  MLD_REQUIRE(d.rotary_dim == 0 || io->positions != nullptr, "null positions");
  MLD_REQUIRE(!cached || (io->v != nullptr && io->slots != nullptr), "a cache needs values and slots");
  const int per16 = d.f16 ? 8 : 4;
  const void* const tensors[] = {io->q, io->k, io->v, io->q_out, io->k_out, io->q_weight, io->k_weight};
  for (const void* p : tensors) MLD_REQUIRE(aligned16(p), "tensors must be 16-byte aligned");
  const int64_t strides[] = {d.heads ? io->q_stride : 0, d.kv_heads ? io->k_stride : 0, cached ? io->v_stride : 0,
                             d.heads ? io->q_out_stride : 0, io->k_out != nullptr ? io->k_out_stride : 0};
  const int64_t widths[] = {d.heads, d.kv_heads, d.kv_heads, d.heads, d.kv_heads};
  for (int i = 0; i < 5; ++i) {
    MLD_REQUIRE(strides[i] % per16 == 0, "token strides must be multiples of 16 bytes");
    MLD_REQUIRE(strides[i] == 0 || strides[i] >= widths[i] * d.head_dim || tokens == 1, "token strides must not be shorter than a token");
  }
  RopeArgs a = {};
  a.q = io->q;
  a.k = io->k;
  a.v = cached ? io->v : nullptr;
  a.q_out = io->q_out;
  a.k_out = io->k_out;
  a.q_weight = io->q_weight;
  a.k_weight = io->k_weight;
  a.q_stride = io->q_stride;
  a.k_stride = io->k_stride;
  a.v_stride = io->v_stride;
  a.q_out_stride = io->q_out_stride;
  a.k_out_stride = io->k_out_stride;
  a.positions = io->positions;
  a.tokens = tokens;
  a.q_heads = d.heads;
  a.k_heads = d.kv_heads;
  a.v_heads = cached ? d.kv_heads : 0;
  a.half_pairs = d.rotary_dim / 2;
  a.neighbours = d.pairing == MLD_ROPE_NEIGHBOURS;
  a.eps = d.rms_eps;
  if (cached) {
    a.pool = static_cast<uint8_t*>(io->pool);
    a.slots = io->slots;
    a.slots_end = io->cache->pages * io->cache->page_tokens;
    a.page_tokens = io->cache->page_tokens;
    a.kv_heads_pool = io->cache->kv_heads;
  }
  for (int i = 0; i < 4; ++i) a.section_end[i] = plan->section_end[i];
  memcpy(a.steps, plan->steps, sizeof(a.steps[0]) * a.half_pairs);
  return launch_rope(a, d.head_dim, d.f16 != 0, static_cast<cudaStream_t>(stream));
}

int mld_kv4_write(const mld_kv4_desc* d, void* pool, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                  int32_t f16, const int32_t* slots, int32_t tokens, void* stream) {
  if (const int rc = check_kv4_desc(d); rc != MLD_OK) return rc;
  MLD_REQUIRE(pool != nullptr, "null pool");
  mld_qk_rope_plan plan = {};
  plan.d.kv_heads = d->kv_heads;
  plan.d.head_dim = d->head_dim;
  plan.d.f16 = f16;
  mld_qk_rope_io io = {};
  io.k = k;
  io.k_stride = k_stride;
  io.v = v;
  io.v_stride = v_stride;
  io.cache = d;
  io.pool = pool;
  io.slots = slots;
  return mld_qk_rope_run(&plan, &io, tokens, stream);
}

int mld_kv4_read(const mld_kv4_desc* d, const void* pool, const int32_t* slots, int32_t tokens, void* k, int64_t k_stride,
                 void* v, int64_t v_stride, void* stream) {
  if (const int rc = check_kv4_desc(d); rc != MLD_OK) return rc;
  MLD_REQUIRE(tokens >= 0, "bad token count");
  if (tokens == 0) return MLD_OK;
  MLD_REQUIRE(pool != nullptr && slots != nullptr && k != nullptr && v != nullptr, "null tensor");
  MLD_REQUIRE(aligned16(pool) && aligned16(k) && aligned16(v), "tensors must be 16-byte aligned");
  MLD_REQUIRE(k_stride % 8 == 0 && v_stride % 8 == 0, "token strides must be multiples of 16 bytes");
  const int64_t width = static_cast<int64_t>(d->kv_heads) * d->head_dim;
  MLD_REQUIRE(tokens == 1 || (k_stride >= width && v_stride >= width), "token strides must not be shorter than a token");
  ReadArgs a = {static_cast<const uint8_t*>(pool), slots, static_cast<__half*>(k), static_cast<__half*>(v), k_stride, v_stride,
                d->pages * d->page_tokens, d->page_tokens, d->kv_heads, tokens};
  const dim3 grid(tokens, div_up(2 * d->kv_heads, kThreads / (d->head_dim / 8)));
  auto kern = d->head_dim == 64 ? kv4_read_kernel<64> : d->head_dim == 128 ? kv4_read_kernel<128> : kv4_read_kernel<256>;
  MLD_CUDA_CHECK(launch_overlapped(kern, grid, dim3(kThreads), 0, static_cast<cudaStream_t>(stream), a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

}  // extern "C"

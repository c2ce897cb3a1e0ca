// Norms of queries and keys for each head and the position rotation in one pass; with a 4-bit cache the keys, and the values
// beside them, are quantised into its pages in the same pass.
//
// The reference assembles this from an RMS norm per head, a rotation (ml_drift/common/kernels/rope.cc:70-89) and, behind them,
// the write into the cache (samples/llm/qwen3_model_builder.cc:426-508, 543-846): three passes over q and k.
//   y = x * w / sqrt(mean(x^2) + eps);   pair i of a head: (a, b) -> (a cos - b sin, b cos + a sin),
//   angle = position[axis of i] / (min_timescale * (max_timescale / min_timescale)^(2 i / rotary_dim))
// The angle is taken in turns, as a product of 32 x 64-bit integers modulo one turn (2^64), since a 32-bit float loses the
// decimals of position * frequency for long contexts (position 131071: 0.008 rad).  What is left is off by 2^-26 turns at most, when
// half a turn becomes a 32-bit float; a table of 64-bit floats adds 2^-31 turns at position 2^24 and 2^-24.4 at 2^31.
//
// D / 8 lanes hold a head, eight neighbouring values each (16 bytes of fp16), and go through heads of one token.  With x' a value's
// partner in its pair, a turned value is r (x A + x' B), r = 1 / sqrt(...): A = w cos and B = -+ w' sin are worked out once per token
// and lane, so that a head costs an exchange of the raw values and three operations per value.  Blocks of two warps, 16 to an SM (64
// registers: 8 to 28 bytes of a lane's lie in local memory): 8192 tokens of 32 + 8 + 8 heads of 128 into the cache take 67 us with the
// read behind it (71 with 12 blocks of more registers to an SM, 73 to 81 in blocks of four warps), 56 without, 2.6 TB/s.  Three
// quarters of the issue slots are taken (225 instructions to a warp's two heads, of which rounding K and V to codes, 26 us for them
// alone, is about half and sines and cosines a twentieth); behind a full scheduler ("not selected") warps wait for their own results,
// then for loads.
#include <cuda_fp16.h>
#include <math.h>
#include <string.h>

#include <new>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace mld {
namespace {

constexpr int kThreads = 64;  // few lanes to a token: each works out its cosines and weights once for all its heads
constexpr int kBlocksPerSm = 16;
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

// Two 32-bit operations in one.
__device__ __forceinline__ float2 pair(const float (&x)[8], int i) { return make_float2(x[i], x[i + 1]); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}

// Eight neighbouring values as they lie in memory.
template <typename T>
struct Eight;
template <>
struct Eight<__half> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const __half* p) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    w[0] = r.x;
    w[1] = r.y;
    w[2] = r.z;
    w[3] = r.w;
  }
  __device__ __forceinline__ void store(__half* p) const { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  __device__ __forceinline__ void put(const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  __device__ __forceinline__ Eight from(unsigned mask, int lane) const {
    Eight r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __shfl_sync(mask, w[i], lane);
    return r;
  }
  __device__ __forceinline__ Eight<__half> halves() const { return *this; }
};
template <>
struct Eight<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 f = reinterpret_cast<const float4*>(p)[i];
      v[4 * i] = f.x;
      v[4 * i + 1] = f.y;
      v[4 * i + 2] = f.z;
      v[4 * i + 3] = f.w;
    }
  }
  __device__ __forceinline__ void store(float* p) const {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[i];
  }
  __device__ __forceinline__ void put(const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i];
  }
  __device__ __forceinline__ Eight from(unsigned mask, int lane) const {
    Eight r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = __shfl_sync(mask, v[i], lane);
    return r;
  }
  __device__ __forceinline__ Eight<__half> halves() const {
    Eight<__half> h;
    h.put(v);
    return h;
  }
};

// Quantises the eight values of a lane (its place in the head: l) into the tile at `tile`; the four lanes of a group of 32
// call it together.  A group that holds an infinity or a NaN gets a NaN scale.
template <int D>
__device__ __forceinline__ void put_eight(uint8_t* tile, bool is_v, int tau, int l, const Eight<__half>& h, unsigned mask, bool store) {
  uint32_t top2 = 0;  // of magnitudes, as bits: infinities and NaN are above all numbers
#pragma unroll
  for (int i = 0; i < 4; ++i) top2 = __vmaxu2(top2, h.w[i] & 0x7FFF7FFFu);
  top2 = __vmaxu2(top2, __shfl_xor_sync(mask, top2, 1));
  top2 = __vmaxu2(top2, __shfl_xor_sync(mask, top2, 2));
  const uint32_t top = max(top2 & 0xFFFFu, top2 >> 16);
  // eight significant bits (round to nearest even), then fp16, which rounds only what is below its normal range
  uint32_t bits = __float_as_uint(__fdiv_rn(__half2float(__ushort_as_half(static_cast<unsigned short>(top))), 7.0f));
  bits = (bits + 0x7FFFu + ((bits >> 16) & 1u)) & 0xFFFF0000u;
  const __half scale = top >= 0x7C00u ? __ushort_as_half(0x7E00) : __float2half_rn(__uint_as_float(bits));
  const float s = __half2float(scale);
  float r[8];
  h.get(r);
  // The product with the reciprocal decides, unless it is within 10^-5 of a halfway point (it is off by less than 2 10^-6), or
  // the scale is one of fp16's subnormal numbers, whose rounding may leave more than 7.
  constexpr float kMagic = 12582920.0f;  // 1.5 2^23 + 8: a sum's low bits are the code
  const float inv = __frcp_rn(s);
  uint32_t code[8];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = r[i] * inv, y = t + kMagic;
    off = fmaxf(off, fabsf(t - (y - kMagic)));
    code[i] = __float_as_uint(y);
  }
  if (!(off < 0.49999f) || !(s >= 6.103515625e-05f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = s > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(r[i], s)), -7.0f), 7.0f) : 0.0f;
      code[i] = static_cast<uint32_t>(static_cast<int>(c) + 8);
    }
  }
  if (!store) return;
  const int j = l >> 2, t = l & 3;
  // nibble p of the low half and of the high half: values 2 p and 2 p + 1 of K, p and 4 + p of V
  uint32_t w = 0;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t two = is_v ? __byte_perm(code[p], code[4 + p], 0x5410) : __byte_perm(code[2 * p], code[2 * p + 1], 0x5410);
    w |= (two << (4 * p)) & (0x000F000Fu << (4 * p));
  }
  if (!is_v) {
    *reinterpret_cast<uint32_t*>(tile + kv4::k_word<D>(tau, j, t)) = w;
  } else {
    uint8_t* const at = tile + kv4::v_half<D>(tau, j, 2 * t);
    *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(w);
    *reinterpret_cast<uint16_t*>(at + D / 16) = static_cast<uint16_t>(w >> 16);
  }
  if (t == 0) *reinterpret_cast<__half*>(tile + kv4::scale_at<D>(is_v, tau, j)) = scale;
}

// Blocks: tokens along x; along y, parts of a token's heads (each takes every gridDim.y-th of the groups of kHeads heads).
template <typename T, int D, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) qk_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int kLanes = D / 8;
  constexpr int kHeads = kThreads / kLanes;
  __shared__ float2 turned[8][kMaxPairs / 8];  // cosine, sine of pair 8 j + i at [i][j]
  pdl_wait();
  const int token = blockIdx.x;
  const int l = threadIdx.x % kLanes;
  const int step = kHeads * gridDim.y, head0 = blockIdx.y * kHeads + threadIdx.x / kLanes;
  Eight<T> ahead;  // the next head
  const T* src = static_cast<const T*>(a.q) + token * a.q_stride + 8 * l;
  if (head0 < a.q_heads) ahead.load(src + head0 * D);
  for (int i = threadIdx.x; i < a.half_pairs; i += kThreads) {
    int axis = 0;
#pragma unroll
    for (int s = 0; s < 3; ++s) axis += i >= a.section_end[s] ? 1 : 0;
    const long long pos = a.positions[static_cast<long long>(axis) * a.tokens + token];
    const unsigned long long turn = static_cast<unsigned long long>(pos) * a.steps[i];
    float sine, cosine;
    sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 4.656612873077393e-10f, &sine, &cosine);
    turned[i & 7][i >> 3] = make_float2(cosine, sine);
  }
  int slot = -1, in_page = 0;
  uint8_t* tile0 = a.pool;
  const int page_tiles = a.page_tokens / kv4::kTile;
  if (a.pool != nullptr) {
    slot = a.slots[token];
    if (slot < 0 || slot >= a.slots_end) slot = -1;
    const int page = max(slot, 0) / a.page_tokens;
    in_page = max(slot, 0) - page * a.page_tokens;
    tile0 += (static_cast<long long>(page) * a.kv_heads_pool * page_tiles + in_page / kv4::kTile) * kv4::tile_bytes(D);
  }
  __syncthreads();
  // the lanes of a head stay together in what follows
  const unsigned mask = kLanes == 32 ? 0xFFFFFFFFu : ((1u << kLanes) - 1u) << ((threadIdx.x & 31) / kLanes * kLanes);
  const int far = a.half_pairs / 8;  // lanes between the halves of a pair
  const bool turns = 8 * l < 2 * a.half_pairs, second = l >= far;
  const int partner = NEIGHBOURS || !turns ? l : second ? l - far : l + far;
  const int from = ((threadIdx.x & 31) - l) + partner;
#pragma unroll 1
  for (int kind = 0; kind < 2; ++kind) {
    const int count = kind ? a.k_heads : a.q_heads;
    const T* const w = static_cast<const T*>(kind ? a.k_weight : a.q_weight);
    // what multiplies a value and its partner
    float mine[8], other[8];
    {
      float wm[8], wo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) wm[i] = wo[i] = 1.0f;
      if (w != nullptr) {
        Eight<T> e;
        e.load(w + 8 * l);
        e.get(wm);
        e.load(w + 8 * partner);
        e.get(wo);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float2 cs = make_float2(1.0f, 0.0f);
        if (turns) cs = NEIGHBOURS ? turned[4 * (l & 1) + i / 2][l >> 1] : turned[i][second ? partner : l];
        mine[i] = wm[i] * cs.x;
        other[i] = (NEIGHBOURS ? wo[i ^ 1] : wo[i]) * ((NEIGHBOURS ? (i & 1) == 0 : !second) ? -cs.y : cs.y);
      }
    }
    if (kind) {
      src = static_cast<const T*>(a.k) + token * a.k_stride + 8 * l;
      if (head0 < count) ahead.load(src + head0 * D);
    }
    T* const out = kind ? static_cast<T*>(a.k_out) : static_cast<T*>(a.q_out);
    T* const dst = out == nullptr ? nullptr : out + token * (kind ? a.k_out_stride : a.q_out_stride) + 8 * l;
#pragma unroll 1
    for (int h = head0; h < count; h += step) {
      Eight<T> e = ahead;
      if (h + step < count) ahead.load(src + (h + step) * D);
      float x[8], y[8];
      e.get(x);
      float r = 1.0f;
      if (w != nullptr) {
        float2 two = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int c = 0; c < 8; c += 2) two = fma2(pair(x, c), pair(x, c), two);
        float sum = two.x + two.y;
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
        r = rsqrtf(fmaf(sum, 1.0f / D, a.eps));
      }
      if (NEIGHBOURS) {
#pragma unroll
        for (int c = 0; c < 8; ++c) y[c] = x[c ^ 1];
      } else {
        e.from(mask, from).get(y);
      }
#pragma unroll
      for (int c = 0; c < 8; c += 2) {
        // a value that is not turned has no partner: an infinity there, times zero, would be a NaN
        const float2 z = mul2(make_float2(r, r), turns ? fma2(pair(x, c), pair(mine, c), mul2(pair(y, c), pair(other, c)))
                                                       : mul2(pair(x, c), pair(mine, c)));
        x[c] = z.x;
        x[c + 1] = z.y;
      }
      e.put(x);
      if (dst != nullptr) e.store(dst + h * D);
      if (kind && a.pool != nullptr)
        put_eight<D>(tile0 + static_cast<long long>(h) * page_tiles * kv4::tile_bytes(D), false, in_page % kv4::kTile, l, e.halves(), mask, slot >= 0);
    }
  }
  src = static_cast<const T*>(a.v) + token * a.v_stride + 8 * l;
#pragma unroll 1
  for (int h = head0; h < a.v_heads; h += step) {
    Eight<T> e;
    e.load(src + h * D);
    put_eight<D>(tile0 + static_cast<long long>(h) * page_tiles * kv4::tile_bytes(D), true, in_page % kv4::kTile, l, e.halves(), mask, slot >= 0);
  }
}

struct ReadArgs {
  const uint8_t* pool;
  const int32_t* slots;
  __half *k, *v;
  long long k_stride, v_stride;
  int slots_end, page_tokens, kv_heads, tokens;
};

// One lane gives eight neighbouring values of a token's key or value at a time.  A slot outside the pool gives zeros.
template <int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8;
  constexpr int kHeads = kThreads / kLanes;
  pdl_wait();
  const int token = blockIdx.x, l = threadIdx.x % kLanes, j = l >> 2, t = l & 3;
  const int slot = a.slots[token];
  const bool there = slot >= 0 && slot < a.slots_end;
  const int page = there ? slot / a.page_tokens : 0, in_page = there ? slot - page * a.page_tokens : 0, tau = in_page % kv4::kTile;
  const long long head_bytes = static_cast<long long>(a.page_tokens / kv4::kTile) * kv4::tile_bytes(D);
  const uint8_t* const tile0 = a.pool + static_cast<long long>(page) * a.kv_heads * head_bytes + in_page / kv4::kTile * kv4::tile_bytes(D);
  const int at_k = kv4::k_word<D>(tau, j, t), at_v = kv4::v_half<D>(tau, j, 2 * t);
  __half* const k = a.k + token * a.k_stride + 8 * l;
  __half* const v = a.v + token * a.v_stride + 8 * l;
#pragma unroll 2
  for (int unit = blockIdx.y * kHeads + threadIdx.x / kLanes; unit < 2 * a.kv_heads; unit += kHeads * gridDim.y) {
    const bool is_v = unit >= a.kv_heads;
    const int h = is_v ? unit - a.kv_heads : unit;
    uint4 y = make_uint4(0, 0, 0, 0);
    if (there) {
      const uint8_t* const tile = tile0 + h * head_bytes;
      const __half2 s = __half2half2(*reinterpret_cast<const __half*>(tile + kv4::scale_at<D>(is_v, tau, j)));
      uint32_t w;
      if (!is_v)
        w = *reinterpret_cast<const uint32_t*>(tile + at_k);
      else
        w = *reinterpret_cast<const uint16_t*>(tile + at_v) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(tile + at_v + D / 16)) << 16;
      uint32_t p[4];  // values 2 i and 2 i + 1 of K, i and 4 + i of V
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = (w >> (4 * i) & 0x000F000Fu) | 0x64006400u;  // 1024 + u
        const __half2 x = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(1032.0f)), s);
        p[i] = *reinterpret_cast<const uint32_t*>(&x);
      }
      y = is_v ? make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[0], p[1], 0x7632),
                            __byte_perm(p[2], p[3], 0x7632))
               : make_uint4(p[0], p[1], p[2], p[3]);
    }
    *reinterpret_cast<uint4*>((is_v ? v : k) + h * D) = y;
  }
}

// Blocks of a token: as many as it has groups of heads while the GPU has room for them at once, else one, which works a token's cosines
// and weights out once.  One / a group each, us, 32 + 8 + 8 heads of 128 into the cache: 74 tokens 8.8 / 5.1, 148 9.3 / 5.5, 296 (2368
// blocks) 9.3 / 6.6, 600 (4800) 10.1 / 11; 8 + 1 heads of 256 in fp32: 148 tokens 5.7 / 5.3, 296 5.9 / 6.2, 600 (2400) 6.7 / 8.4.
// (148 SMs: asking the runtime for them takes 0.3 us of a call's 4.)
int parts_of_token(int tokens, int groups) {
  return groups > 1 && static_cast<int64_t>(tokens) * groups <= kBlocksPerSm * 148 ? groups : 1;
}

template <typename T, int D>
int launch_rope_t(const RopeArgs& a, cudaStream_t stream) {
  const int most = a.q_heads > a.k_heads ? a.q_heads : a.k_heads;
  const dim3 grid(a.tokens, parts_of_token(a.tokens, div_up(most, kThreads / (D / 8))));
  MLD_CUDA_CHECK(launch_overlapped(a.neighbours ? qk_rope_kernel<T, D, true> : qk_rope_kernel<T, D, false>, grid, dim3(kThreads), 0, stream, a));
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
  const bool keys = d.kv_heads > 0, keys_out = keys && io->k_out != nullptr;
  const struct {
    bool there, out;
    int64_t stride, heads;
  } rows[] = {{d.heads > 0, false, io->q_stride, d.heads},
              {keys, false, io->k_stride, d.kv_heads},
              {cached, false, io->v_stride, d.kv_heads},
              {d.heads > 0, true, io->q_out_stride, d.heads},
              {keys_out, true, io->k_out_stride, d.kv_heads}};
  for (const auto& r : rows) {
    if (!r.there) continue;
    MLD_REQUIRE(r.stride % per16 == 0, "token strides must be multiples of 16 bytes");
    // all tokens may read one row, but not write it
    MLD_REQUIRE(tokens == 1 || r.stride >= r.heads * d.head_dim || (r.stride == 0 && !r.out), "token strides must not be shorter than a token");
  }
  MLD_REQUIRE(tokens == 1 || d.heads == 0 || io->q_out != io->q || io->q_out_stride == io->q_stride, "in place, queries go out with the stride that they come with");
  MLD_REQUIRE(tokens == 1 || !keys_out || io->k_out != io->k || io->k_out_stride == io->k_stride, "in place, keys go out with the stride that they come with");
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
  const dim3 grid(tokens, parts_of_token(tokens, div_up(2 * d->kv_heads, kThreads / (d->head_dim / 8))));
  auto kern = d->head_dim == 64 ? kv4_read_kernel<64> : d->head_dim == 128 ? kv4_read_kernel<128> : kv4_read_kernel<256>;
  MLD_CUDA_CHECK(launch_overlapped(kern, grid, dim3(kThreads), 0, static_cast<cudaStream_t>(stream), a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

}  // extern "C"

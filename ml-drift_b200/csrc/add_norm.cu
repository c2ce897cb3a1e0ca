// The residual's addition and the RMS norm behind it, with an output in the tensors' type, in 8-bit codes with a scale for
// each token, or both:
//   h = x + residual                       rounded to the tensors' type, as it is written
//   y = h (offset + w) / sqrt(mean(h^2) + eps)
// and for codes, of v = h (offset + w), which a row's norm does not change:
//   symmetric    scale = max|y| / 127,             zero = 0,                    code = floor(127 v / max|v| + 1/2)
//   asymmetric   scale = (max y - min y) / 255,    zero = min y + 128 scale,    code = floor(255 (v - min v) / (max v - min v) + 1/2) - 128
// (the rules of quantize_act_kernel, ml_drift/common/kernels/quantize_and_dequantize.cc:355-441, ahead of the rounding to fp16).
//
// Bound by HBM: x and the residual in, the sum, y and the codes out, each once.  A row stays in the registers of the warp or the
// block that owns it, together with its part of the weights, which serve all of its rows; the sum of squares and the extremes of
// v go through one exchange.  Sums and products are held in 32 bits.  A code whose value in 32 bits lies near a border between two
// codes is worked out again in 64, with its seven neighbours, so that codes are those of the formula, whoever works it out.  Near is
// 2^-13, above six roundings of 2^-24 at a value of 255 at most: of the span, its reciprocal and a value's distance from the row's
// smallest, and, with an offset or 32-bit tensors, of offset + w, v and that smallest.  The last three are relative to v, so for
// them near grows with max|v| / span where that is above 1; where it passes a quarter, the whole row is worked out in 64.  (Of rows
// about zero one chunk in 500 is worked out again: 2048 rows of 4096 in fp32, asymmetric, take 33 us; of a mean of 10 deviations 35,
// of 1000 44.)
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace mld {
namespace {

struct NormArgs {
  const void *x, *residual, *weight;
  void *sum, *out;
  int8_t* codes;
  float* params;
  int64_t x_stride, residual_stride, sum_stride, out_stride, codes_stride;
  int tokens, width;
  int codes_width;  // columns of codes that are written: width rounded up to 16, zeros behind the row
  float eps, offset;
  int symmetric;
  int ahead;  // rows that a block fetches ahead, 0 to 3
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

constexpr int kChunk = 8;
template <typename T>
struct alignas(16) Chunk {
  T v[kChunk];
};

// The values `at` .. of a row; one by one where rows may begin anywhere and end inside a chunk (zeros behind the end).
template <typename T, bool WIDE>
__device__ __forceinline__ Chunk<T> load_chunk(const void* row, int at, int width) {
  const T* p = static_cast<const T*>(row) + at;
  if constexpr (WIDE) {
    return *reinterpret_cast<const Chunk<T>*>(p);
  } else {
    Chunk<T> c;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) c.v[i] = at + i < width ? p[i] : from_float<T>(0.0f);
    return c;
  }
}
template <typename T, bool WIDE>
__device__ __forceinline__ void store_chunk(void* row, int at, int width, const Chunk<T>& c) {
  T* p = static_cast<T*>(row) + at;
  if constexpr (WIDE) {
    *reinterpret_cast<Chunk<T>*>(p) = c;
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (at + i < width) p[i] = c.v[i];
  }
}

// A chunk's arithmetic, halves two at a time.  (Their sum in halves is the sum in 32 bits rounded once: that is exact to 24 bits.)
__device__ __forceinline__ Chunk<__half> operator+(Chunk<__half> a, const Chunk<__half>& b) {
#pragma unroll
  for (int i = 0; i < kChunk / 2; ++i)
    reinterpret_cast<__half2*>(a.v)[i] = __hadd2_rn(reinterpret_cast<const __half2*>(a.v)[i], reinterpret_cast<const __half2*>(b.v)[i]);
  return a;
}
__device__ __forceinline__ Chunk<float> operator+(Chunk<float> a, const Chunk<float>& b) {
#pragma unroll
  for (int i = 0; i < kChunk; ++i) a.v[i] += b.v[i];
  return a;
}
__device__ __forceinline__ Chunk<float> widen(const Chunk<__half>& c) {
  Chunk<float> f;
#pragma unroll
  for (int i = 0; i < kChunk / 2; ++i) reinterpret_cast<float2*>(f.v)[i] = __half22float2(reinterpret_cast<const __half2*>(c.v)[i]);
  return f;
}
__device__ __forceinline__ Chunk<float> widen(const Chunk<float>& c) { return c; }
template <typename T>
__device__ __forceinline__ Chunk<T> narrow(const Chunk<float>& f) {
  if constexpr (sizeof(T) == 2) {
    Chunk<T> c;
#pragma unroll
    for (int i = 0; i < kChunk / 2; ++i) reinterpret_cast<__half2*>(c.v)[i] = __floats2half2_rn(f.v[2 * i], f.v[2 * i + 1]);
    return c;
  } else {
    return f;
  }
}
// The lowest bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <int BYTES>
__device__ __forceinline__ void fetch_chunk(void* to, const void* from) {
#pragma unroll
  for (int i = 0; i < BYTES / 16; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to) + 16 * i), "l"(static_cast<const uint8_t*>(from) + 16 * i)
                 : "memory");
}
// Until all but the last n groups of this thread's copies have landed.
__device__ __forceinline__ void wait_fetched(int n) {
  if (n >= 2)
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (n == 1)
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  else
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// What a row's threads know together: the sum of squares and the extremes of v.
struct RowStats {
  float sum, low, high;
};
__device__ __forceinline__ float warp_low(float v) {
  float r;
  asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_high(float v) {  // (NaN if any is)
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <bool CODED>
__device__ __forceinline__ RowStats over_warp(RowStats s) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, off);
  if constexpr (CODED) {
    s.low = warp_low(s.low);
    s.high = warp_high(s.high);
  }
  return s;
}
// Doubles as numbers in their order, for the maximum in shared memory.
__device__ __forceinline__ unsigned long long ordered(double v) {
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v));
  return u ^ ((u >> 63) != 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double in_order(unsigned long long u) {
  return __longlong_as_double(static_cast<long long>(u ^ ((u >> 63) != 0 ? 1ull << 63 : ~0ull)));
}

// T: the tensors' type.  WIDE: 16-byte accesses, else any width, stride and alignment.  NV: chunks of a thread.  WARP: a row per
// warp, else per block.  CODED: with codes.  EXACT: halves and no offset, whose products with weights 32 bits hold (22 of them).
template <typename T, bool WIDE, int NV, bool WARP, bool CODED, bool EXACT>
__global__ void __launch_bounds__(WARP ? 128 : 1024) add_norm_kernel(NormArgs a) {
  pdl_wait();
  pdl_launch_dependents();  // (after the wait: whoever begins now may rely on what this launch waited for)
  __shared__ RowStats part[2][32];
  __shared__ unsigned long long ends[2][2];  // the largest of v and of -v in 64 bits
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lanes = WARP ? 32 : static_cast<int>(blockDim.x), me = WARP ? lane : static_cast<int>(threadIdx.x);
  const int rows_at_once = WARP ? static_cast<int>(blockDim.x >> 5) : 1;
  const int chunks = (a.width + kChunk - 1) / kChunk;
  const auto at_of = [&](int j) { return (me + j * lanes) * kChunk; };
  const auto there = [&](int j, int i) { return WIDE || at_of(j) + i < a.width; };  // whether a chunk has its i-th value
  const float offset = EXACT || a.weight == nullptr ? 0.0f : a.offset;
  const auto weights_of = [&](int j) {  // (from the SM's own cache from the second row on)
    Chunk<T> c;
    if (a.weight != nullptr) {
      c = load_chunk<T, WIDE>(a.weight, at_of(j), a.width);
    } else {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) c.v[i] = from_float<T>(1.0f);
    }
    return c;
  };
  const auto weighted = [&](const Chunk<T>& h, int j) {
    Chunk<float> f = widen(h);
    const Chunk<float> w = widen(weights_of(j));
#pragma unroll
    for (int i = 0; i < kChunk; ++i) f.v[i] *= EXACT ? w.v[i] : offset + w.v[i];
    return f;
  };
  const auto in64 = [&](T h, T w) {
    return static_cast<double>(to_float(h)) * (static_cast<double>(offset) + static_cast<double>(to_float(w)));
  };
  if (CODED && !EXACT && !WARP && threadIdx.x < 4) ends[threadIdx.x >> 1][threadIdx.x & 1] = 0;  // (seen after the first row's exchange)
  // Rows ahead of the one that is worked on: every thread fetches its own values into shared memory.
  constexpr bool kPipe = WIDE && !WARP;
  extern __shared__ uint4 ring[];
  const int row_step = static_cast<int>(gridDim.x) * rows_at_once;
  const auto slot = [&](int s, int j, int which) {
    return reinterpret_cast<Chunk<T>*>(ring) + static_cast<unsigned>((s * NV + j) * 2 + which) * blockDim.x + threadIdx.x;
  };
  const auto fetch = [&](int row, int s) {
    if (row < a.tokens) {
      const T* const x = static_cast<const T*>(a.x) + row * a.x_stride;
      const T* const r = static_cast<const T*>(a.residual) + row * a.residual_stride;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (me + j * lanes < chunks) {
          fetch_chunk<sizeof(Chunk<T>)>(slot(s, j, 0), x + at_of(j));
          if (a.residual != nullptr) fetch_chunk<sizeof(Chunk<T>)>(slot(s, j, 1), r + at_of(j));
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // (an empty one behind the last row keeps the count)
  };
  int stage = 0;
  if (kPipe)
    for (int s = 0; s < a.ahead; ++s) fetch(static_cast<int>(blockIdx.x) + s * row_step, s);
  int turn = 0;
  for (int row = static_cast<int>(blockIdx.x) * rows_at_once + (WARP ? warp : 0); row < a.tokens; row += row_step, turn ^= 1) {
    Chunk<T> h[NV];
    {
      Chunk<T> r[NV];
      if (kPipe && a.ahead > 0) {
        // (a thread reads what it fetched itself: there is nothing to meet for)
        wait_fetched(a.ahead - 1);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          h[j] = *slot(stage, j, 0);
          if (a.residual != nullptr) r[j] = *slot(stage, j, 1);
        }
        fetch(row + a.ahead * row_step, stage);
        stage = stage + 1 == a.ahead ? 0 : stage + 1;
      } else {
        const T* const xs = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* const rs = static_cast<const T*>(a.residual) + row * a.residual_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (me + j * lanes < chunks) {
            h[j] = load_chunk<T, WIDE>(xs, at_of(j), a.width);
            if (a.residual != nullptr) r[j] = load_chunk<T, WIDE>(rs, at_of(j), a.width);
          }
      }
      if (a.residual != nullptr) {
        T* const to = static_cast<T*>(a.sum) + row * a.sum_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (me + j * lanes < chunks) {
            h[j] = h[j] + r[j];
            if (a.sum != nullptr) store_chunk<T, WIDE>(to, at_of(j), a.width, h[j]);
          }
      }
    }
    RowStats st = {0.0f, INFINITY, -INFINITY};
    Chunk<float> held[EXACT ? NV : 1];  // v, where it need not be worked out again
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (me + j * lanes < chunks) {
        const Chunk<float> f = widen(h[j]);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) st.sum += f.v[i] * f.v[i];
        if constexpr (EXACT) held[j] = weighted(h[j], j);
        if constexpr (CODED) {
          const Chunk<float> v = EXACT ? held[EXACT ? j : 0] : weighted(h[j], j);
#pragma unroll
          for (int i = 0; i < kChunk; ++i)
            if (there(j, i)) {
              st.low = fminf(st.low, v.v[i]);
              st.high = max_or_nan(st.high, v.v[i]);
            }
        }
      }
    const float my_low = st.low, my_high = st.high;
    st = over_warp<CODED>(st);
    if constexpr (!WARP) {
      if (lane == 0) part[turn][warp] = st;
      __syncthreads();  // (one a row: the next row's parts go to the other place)
      st = over_warp<CODED>(lane < lanes / 32 ? part[turn][lane] : RowStats{0.0f, INFINITY, -INFINITY});
    }
    const float rstd = 1.0f / sqrtf(st.sum / static_cast<float>(a.width) + a.eps);
    const auto v_of = [&](int j) {
      if constexpr (EXACT)
        return held[j];
      else
        return weighted(h[j], j);
    };
    if (a.out != nullptr) {
      T* const to = static_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (me + j * lanes < chunks) {
          Chunk<float> y = v_of(j);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) y.v[i] *= rstd;
          store_chunk<T, WIDE>(to, at_of(j), a.width, narrow<T>(y));
        }
    }
    if constexpr (CODED) {
      // (a row with an infinity or a NaN, or whose squares leave 32 bits, gets NaN parameters, so that whatever is computed from
      // it is NaN; its codes are zeros)
      const bool fine = st.sum < INFINITY && fabsf(st.low) < INFINITY && fabsf(st.high) < INFINITY;
      double low = st.low, high = st.high;
      if constexpr (!EXACT) {
        // the extremes in 64 bits: of the threads whose own come near them in 32
        const float near = 1.0e-6f * fmaxf(fabsf(st.low), fabsf(st.high)) + 0x1p-147f;  // (of subnormal v: a few of their steps)
        double lo = INFINITY, hi = -INFINITY;
        if (fine && (my_low <= st.low + near || my_high >= st.high - near)) {
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (me + j * lanes < chunks) {
              const Chunk<T> w = weights_of(j);
#pragma unroll
              for (int i = 0; i < kChunk; ++i) {
                const double v = in64(h[j].v[i], w.v[i]);
                if (!there(j, i)) continue;
                lo = fmin(lo, v);
                hi = fmax(hi, v);
              }
            }
          if constexpr (!WARP) {
            atomicMax(&ends[turn][0], ordered(hi));
            atomicMax(&ends[turn][1], ordered(-lo));
          }
        }
        if constexpr (WARP) {
          for (int off = 16; off > 0; off >>= 1) {
            lo = fmin(lo, __shfl_xor_sync(0xffffffffu, lo, off));
            hi = fmax(hi, __shfl_xor_sync(0xffffffffu, hi, off));
          }
        } else {
          if (threadIdx.x < 2) ends[turn ^ 1][threadIdx.x] = 0;  // the next row's: all have read the last row's, ahead of the exchange
          __syncthreads();
          hi = in_order(ends[turn][0]);
          lo = -in_order(ends[turn][1]);
        }
        low = lo;
        high = hi;
      }
      const double span = a.symmetric ? fmax(high, -low) : high - low, from64 = a.symmetric ? 0.0 : low;
      const float top = a.symmetric ? 127.0f : 255.0f, from = static_cast<float>(from64);
      const bool live = fine && span > 0.0;
      const float per = live ? top / static_cast<float>(span) : 0.0f;
      constexpr float kBorder = 0x1p-13f;
      const float error = EXACT ? kBorder : fmaxf(kBorder, fmaxf(fabsf(st.low), fabsf(st.high)) * per * (kBorder / 255.0f));
      // a span whose factor leaves 32 bits, or that leaves them itself, or is small against v: everything in 64
      const bool wide = !(per > 0.0f && per < 1.0e36f && error <= 0.25f);
      int8_t* const codes = a.codes + row * a.codes_stride;
      // Rounded by the addition of 1.5 2^23, whose last byte then is the code (of 0 .. 255 less 128: with its top bit turned).
      // A value near the middle between two codes, or on it, is compared with it in 64 bits, and goes up from there.
      constexpr float kRound = 12582912.0f;
      const float clear = 0.5f - error;
      const uint32_t turned = a.symmetric ? 0u : 0x80808080u;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (me + j * lanes < chunks) {
          const Chunk<float> v = v_of(j);
          uint32_t q[kChunk];
          float off = 0.0f;  // the furthest of the chunk's values from their codes
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            const float d = v.v[i] - from, r = fmaf(d, per, kRound);
            off = fmaxf(off, fabsf(fmaf(d, per, kRound - r)));
            q[i] = __float_as_uint(r);
          }
          if (!(off < clear) || wide || !live) {
            Chunk<T> w;
            if constexpr (!EXACT) w = weights_of(j);
#pragma unroll
            for (int i = 0; i < kChunk; ++i) {
              const double d = (EXACT ? static_cast<double>(v.v[i]) : in64(h[j].v[i], EXACT ? h[j].v[i] : w.v[i])) - from64;
              // the code by 32 bits (or, where that fails, below it) and whether the middles on both sides of it move it
              double at = wide ? floor(d * (top / span)) : static_cast<double>(static_cast<int>(q[i] - 0x4B400000u));
              at = fmin(fmax(at, -128.0), 255.0);
              const double twice = d * (2.0f * top);
              at += twice >= (2.0 * at + 1.0) * span ? 1.0 : twice < (2.0 * at - 1.0) * span ? -1.0 : 0.0;
              q[i] = live ? static_cast<uint32_t>(static_cast<int>(at)) : turned;
            }
          }
          if constexpr (!WIDE) {
#pragma unroll
            for (int i = 0; i < kChunk; ++i)
              if (!there(j, i)) q[i] = turned;
          }
          *reinterpret_cast<uint2*>(codes + at_of(j)) =
              make_uint2(low_bytes(q[0], q[1], q[2], q[3]) ^ turned, low_bytes(q[4], q[5], q[6], q[7]) ^ turned);
        }
      if (me == 0 && chunks * kChunk < a.codes_width) *reinterpret_cast<uint2*>(codes + chunks * kChunk) = make_uint2(0u, 0u);
      if (me < 3) {
        // (a row of equal values has scale 0, and each is the zero point)
        const double by = rstd;
        const float value = me == 0 ? static_cast<float>(span * by * (a.symmetric ? 1.0 / 127.0 : 1.0 / 255.0))
                            : me == 2 || a.symmetric ? 0.0f : static_cast<float>((low + span * (128.0 / 255.0)) * by);
        a.params[static_cast<int64_t>(row) * 3 + me] = fine || me == 2 ? value : NAN;
      }
    }
  }
}

template <typename T, bool WIDE, int NV, bool WARP, bool CODED, bool EXACT>
int launch_as(NormArgs a, int threads, int sms, cudaStream_t stream) {
  const auto kern = add_norm_kernel<T, WIDE, NV, WARP, CODED, EXACT>;
  // Rows ahead: three of halves, one of 32-bit values, as 1024 threads' take 192 and 128 KB.
  constexpr int kAhead = !WIDE || WARP ? 0 : sizeof(T) == 2 ? 3 : 1;
  size_t smem = static_cast<size_t>(kAhead) * NV * 2 * sizeof(Chunk<T>) * threads;
  static bool done[kMaxDevices];
  int dev;
  if (kAhead > 0 && needs_configure(done, &dev)) {
    MLD_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    if (dev >= 0) done[dev] = true;
  }
  static std::atomic<int> resident[33];  // blocks to an SM, by warps of a block
  int at_once = resident[threads / 32].load(std::memory_order_relaxed);
  if (at_once == 0) {
    MLD_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&at_once, kern, threads, smem));
    at_once = at_once > 0 ? at_once : 1;
    resident[threads / 32].store(at_once, std::memory_order_relaxed);
  }
  const int rows = WARP ? threads / 32 : 1;
  const int grid = div_up(a.tokens, rows) < sms * at_once ? div_up(a.tokens, rows) : sms * at_once;
  a.ahead = a.tokens > grid ? kAhead : 0;
  if (a.ahead == 0) smem = 0;
  MLD_CUDA_CHECK(launch_overlapped(kern, dim3(grid), dim3(threads), smem, stream, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}
template <typename T, bool WIDE, int NV, bool WARP>
int launch(const NormArgs& a, int threads, int sms, cudaStream_t stream) {
  constexpr bool kHalf = sizeof(T) == 2;
  if (kHalf && a.offset == 0.0f)
    return a.codes != nullptr ? launch_as<T, WIDE, NV, WARP, true, kHalf>(a, threads, sms, stream)
                              : launch_as<T, WIDE, NV, WARP, false, kHalf>(a, threads, sms, stream);
  return a.codes != nullptr ? launch_as<T, WIDE, NV, WARP, true, false>(a, threads, sms, stream)
                            : launch_as<T, WIDE, NV, WARP, false, false>(a, threads, sms, stream);
}

template <typename T, bool WIDE>
int launch_of(const NormArgs& a, int sms, cudaStream_t stream) {
  // A thread holds 8 or 16 values (with 32 they no longer fit 64 registers, and 1024 threads an SM are what it takes); few rows are
  // spread over as many threads as have 8.
  const int chunks = div_up(a.width, kChunk);
  if (a.width <= 512) {
    if (chunks <= 32) return launch<T, WIDE, 1, true>(a, 128, sms, stream);
    return launch<T, WIDE, 2, true>(a, 128, sms, stream);
  }
  int threads = div_up(a.width, a.tokens <= sms ? 8 * 32 : 16 * 32) * 32;
  threads = threads < 64 ? 64 : threads > 1024 ? 1024 : threads;
  if (div_up(chunks, threads) <= 1) return launch<T, WIDE, 1, false>(a, threads, sms, stream);
  return launch<T, WIDE, 2, false>(a, threads, sms, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace mld

using namespace mld;

extern "C" int mld_add_rms_norm(const mld_add_norm_desc* d, const mld_add_norm_io* io, int32_t tokens, void* stream) {
  MLD_REQUIRE(d != nullptr && io != nullptr, "null argument");
  MLD_REQUIRE(d->width >= 1 && d->width <= 16384, "width must be 1 to 16384");
  MLD_REQUIRE(d->eps >= 0.0f && d->eps < INFINITY && d->weight_offset > -INFINITY && d->weight_offset < INFINITY,
              "eps must be finite and not negative, weight_offset finite");
  MLD_REQUIRE(tokens >= 0 && tokens <= 1 << 30, "tokens must be 0 to 2^30");
  if (tokens == 0) return MLD_OK;  // (whose tensors may have no address)
  MLD_REQUIRE(io->out != nullptr || io->codes != nullptr, "neither out nor codes");
  MLD_REQUIRE((io->codes == nullptr) == (io->params == nullptr), "codes and params go together");
  MLD_REQUIRE(io->sum_out == nullptr || io->residual != nullptr, "sum_out needs a residual");
  MLD_REQUIRE(io->x != nullptr, "null tensor");
  const uintptr_t esz = d->f16 ? 2 : 4;
  const uintptr_t all = reinterpret_cast<uintptr_t>(io->x) | reinterpret_cast<uintptr_t>(io->residual) |
                        reinterpret_cast<uintptr_t>(io->weight) | reinterpret_cast<uintptr_t>(io->sum_out) |
                        reinterpret_cast<uintptr_t>(io->out);
  MLD_REQUIRE(all % esz == 0, "a tensor that is not aligned to its type");
  MLD_REQUIRE(io->x_stride >= 0 && (io->residual == nullptr || io->residual_stride >= 0), "negative stride");
  if (tokens > 1) {
    MLD_REQUIRE((io->sum_out == nullptr || io->sum_stride >= d->width) && (io->out == nullptr || io->out_stride >= d->width),
                "an output's stride is less than its width");
    const auto apart = [&](const void* in, int64_t in_stride, const void* out, int64_t out_stride) {
      return in == nullptr || out == nullptr || in != out || in_stride == out_stride;
    };
    MLD_REQUIRE(apart(io->x, io->x_stride, io->sum_out, io->sum_stride) && apart(io->x, io->x_stride, io->out, io->out_stride) &&
                    apart(io->residual, io->residual_stride, io->sum_out, io->sum_stride) &&
                    apart(io->residual, io->residual_stride, io->out, io->out_stride),
                "an output in the place of an input needs the input's stride");
  }
  MLD_REQUIRE(io->sum_out == nullptr || io->sum_out != io->out, "sum_out and out are the same tensor");
  const int codes_width = align_n(d->width, 16);
  if (io->codes != nullptr)
    MLD_REQUIRE(aligned16(io->codes) && io->codes_stride >= codes_width && io->codes_stride % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(io->params) % 4 == 0,
                "codes need 16-byte aligned rows of the width rounded up to 16");
  NormArgs a = {};
  a.x = io->x;
  a.residual = io->residual;
  a.weight = io->weight;
  a.sum = io->sum_out;
  a.out = io->out;
  a.codes = io->codes;
  a.params = io->params;
  a.x_stride = io->x_stride;
  a.residual_stride = io->residual_stride;
  a.sum_stride = io->sum_stride;
  a.out_stride = io->out_stride;
  a.codes_stride = io->codes_stride;
  a.tokens = tokens;
  a.width = d->width;
  a.codes_width = codes_width;
  a.eps = d->eps;
  a.offset = d->weight_offset;
  a.symmetric = d->asymmetric == 0;
  int dev = 0;
  MLD_CUDA_CHECK(cudaGetDevice(&dev));
  const int sms = sm_count(dev);
  MLD_REQUIRE(sms > 0, "no device");
  const int per16 = d->f16 ? 8 : 4;  // values of 16 bytes
  const auto wide = [&](const void* p, int64_t stride) { return p == nullptr || (aligned16(p) && (tokens == 1 || stride % per16 == 0)); };
  const bool v8 = d->width % 8 == 0 && wide(io->x, io->x_stride) && wide(io->residual, io->residual_stride) && aligned16(io->weight) &&
                  wide(io->sum_out, io->sum_stride) && wide(io->out, io->out_stride);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->f16) return v8 ? launch_of<__half, true>(a, sms, s) : launch_of<__half, false>(a, sms, s);
  return v8 ? launch_of<float, true>(a, sms, s) : launch_of<float, false>(a, sms, s);
}

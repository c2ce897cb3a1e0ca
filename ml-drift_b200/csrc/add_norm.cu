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
// v go through one exchange.  Sums and products are held in 32 bits.  A code whose value in 32 bits lies within 2^-13 of a border
// between two codes (the error is below 2^-14: four roundings of 2^-24 at a value of 255 at most) is worked out again in 64, so
// that codes are those of the formula, whoever works it out.  (One in 4000 is.)
#include <cuda_fp16.h>

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

template <typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Chunk {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Chunk<T, V> load_chunk(const void* base, int64_t at) {
  return *reinterpret_cast<const Chunk<T, V>*>(static_cast<const T*>(base) + at);
}

// What a row's threads know together: the sum of squares and the extremes of v.
struct RowStats {
  float sum, low, high;
};
__device__ __forceinline__ RowStats fold(RowStats a, RowStats b) {
  return {a.sum + b.sum, fminf(a.low, b.low), fmaxf(a.high, b.high)};
}

// T: the tensors' type.  V: values of a chunk (8: 16-byte accesses; 1: any width, stride and alignment).  NV: chunks of a thread.
// WARP: a row per warp, else per block.
template <typename T, int V, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512) add_norm_kernel(NormArgs a) {
  pdl_wait();
  pdl_launch_dependents();  // (after the wait: whoever begins now may rely on what this launch waited for)
  __shared__ RowStats part[2][32];
  __shared__ double part64[2][32][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lanes = WARP ? 32 : static_cast<int>(blockDim.x), me = WARP ? lane : static_cast<int>(threadIdx.x);
  const int rows_at_once = WARP ? static_cast<int>(blockDim.x >> 5) : 1;
  const int chunks = a.width / V;
  const bool coded = a.codes != nullptr;
  Chunk<T, V> w[NV];
  if (a.weight != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (me + j * lanes < chunks) w[j] = load_chunk<T, V>(a.weight, static_cast<int64_t>(me + j * lanes) * V);
  }
  // The weight's product is exact in 32 bits for halves with no offset: 22 bits.
  const bool inexact = sizeof(T) == 4 || a.offset != 0.0f;
  const auto factor = [&](int j, int i) { return a.weight != nullptr ? a.offset + to_float(w[j].v[i]) : 1.0f; };
  int turn = 0;
  for (int row = static_cast<int>(blockIdx.x) * rows_at_once + (WARP ? warp : 0); row < a.tokens;
       row += static_cast<int>(gridDim.x) * rows_at_once, turn ^= 1) {
    Chunk<T, V> h[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (me + j * lanes < chunks) h[j] = load_chunk<T, V>(a.x, row * a.x_stride + static_cast<int64_t>(me + j * lanes) * V);
    if (a.residual != nullptr) {
      Chunk<T, V> r[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (me + j * lanes < chunks)
          r[j] = load_chunk<T, V>(a.residual, row * a.residual_stride + static_cast<int64_t>(me + j * lanes) * V);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (me + j * lanes < chunks) {
#pragma unroll
          for (int i = 0; i < V; ++i) h[j].v[i] = from_float<T>(to_float(h[j].v[i]) + to_float(r[j].v[i]));
          if (a.sum != nullptr)
            *reinterpret_cast<Chunk<T, V>*>(static_cast<T*>(a.sum) + row * a.sum_stride + static_cast<int64_t>(me + j * lanes) * V) = h[j];
        }
    }
    RowStats st = {0.0f, INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (me + j * lanes < chunks) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float f = to_float(h[j].v[i]);
          st.sum += f * f;
          if (coded) {
            const float v = f * factor(j, i);
            st.low = fminf(st.low, v);
            st.high = fmaxf(st.high, v == v ? v : INFINITY);  // (a NaN is not lost)
          }
        }
      }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
      st = fold(st, {__shfl_xor_sync(0xffffffffu, st.sum, off), __shfl_xor_sync(0xffffffffu, st.low, off),
                     __shfl_xor_sync(0xffffffffu, st.high, off)});
    if constexpr (!WARP) {
      if (lane == 0) part[turn][warp] = st;
      __syncthreads();  // (one a row: the next row's parts go to the other place)
      st = lane < lanes / 32 ? part[turn][lane] : RowStats{0.0f, INFINITY, -INFINITY};
#pragma unroll
      for (int off = 16; off > 0; off >>= 1)
        st = fold(st, {__shfl_xor_sync(0xffffffffu, st.sum, off), __shfl_xor_sync(0xffffffffu, st.low, off),
                       __shfl_xor_sync(0xffffffffu, st.high, off)});
    }
    const float rstd = 1.0f / sqrtf(st.sum / static_cast<float>(a.width) + a.eps);
    if (coded) {
      // (a row with an infinity or a NaN, or whose squares leave 32 bits, gets NaN parameters, so that whatever is computed from
      // it is NaN; its codes are zeros)
      const bool fine = st.sum < INFINITY && fabsf(st.low) < INFINITY && fabsf(st.high) < INFINITY;
      // v of one value in 64 bits, fetched again: rare, and what is in registers cannot be indexed
      const auto exactly = [&](int e) {
        float f;
        if (a.residual == nullptr)
          f = to_float(static_cast<const T*>(a.x)[row * a.x_stride + e]);
        else if (a.sum != nullptr)
          f = to_float(static_cast<const T*>(a.sum)[row * a.sum_stride + e]);
        else
          f = to_float(from_float<T>(to_float(static_cast<const T*>(a.x)[row * a.x_stride + e]) +
                                     to_float(static_cast<const T*>(a.residual)[row * a.residual_stride + e])));
        if (a.weight == nullptr) return static_cast<double>(f);
        return static_cast<double>(f) * (static_cast<double>(a.offset) + static_cast<double>(to_float(static_cast<const T*>(a.weight)[e])));
      };
      const auto place = [&](int bit) { return (me + bit / V * lanes) * V + bit % V; };  // of a thread's bit-th value
      double low = st.low, high = st.high;
      if (inexact && fine) {
        // the extremes in 64 bits: of the values that come near them in 32
        const float near = 1.0e-6f * fmaxf(fabsf(st.low), fabsf(st.high));
        uint32_t ends = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (me + j * lanes < chunks) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float v = to_float(h[j].v[i]) * factor(j, i);
              ends |= static_cast<uint32_t>(v <= st.low + near || v >= st.high - near) << (j * V + i);
            }
          }
        low = INFINITY;
        high = -INFINITY;
#pragma unroll 1
        for (; ends != 0; ends &= ends - 1) {
          const double v = exactly(place(__ffs(ends) - 1));
          low = fmin(low, v);
          high = fmax(high, v);
        }
        for (int off = 16; off > 0; off >>= 1) {
          low = fmin(low, __shfl_xor_sync(0xffffffffu, low, off));
          high = fmax(high, __shfl_xor_sync(0xffffffffu, high, off));
        }
        if constexpr (!WARP) {
          if (lane == 0) {
            part64[turn][warp][0] = low;
            part64[turn][warp][1] = high;
          }
          __syncthreads();
          low = lane < lanes / 32 ? part64[turn][lane][0] : INFINITY;
          high = lane < lanes / 32 ? part64[turn][lane][1] : -INFINITY;
          for (int off = 16; off > 0; off >>= 1) {
            low = fmin(low, __shfl_xor_sync(0xffffffffu, low, off));
            high = fmax(high, __shfl_xor_sync(0xffffffffu, high, off));
          }
        }
      }
      const double span = a.symmetric ? fmax(high, -low) : high - low, from64 = a.symmetric ? 0.0 : low;
      const double top = a.symmetric ? 127.0 : 255.0;
      const float from = static_cast<float>(from64);
      const float per = span > 0.0 ? static_cast<float>(top / span) : 0.0f;
      const int zero_code = a.symmetric ? 0 : 128, most = a.symmetric ? 127 : 255;
      const bool tiny = !(per < 1.0e36f);  // a span so small that its factor leaves 32 bits: everything in 64
      const bool live = fine && span > 0.0;
      int8_t* const codes = a.codes + row * a.codes_stride;
      uint32_t again = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (me + j * lanes < chunks) {
          Chunk<int8_t, V> q;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float u = (to_float(h[j].v[i]) * factor(j, i) - from) * per + 0.5f, down = floorf(u);
            q.v[i] = static_cast<int8_t>(live ? min(most, static_cast<int>(down)) - zero_code : 0);
            again |= static_cast<uint32_t>(u - down < 0x1p-13f || u - down > 1.0f - 0x1p-13f || tiny) << (j * V + i);
          }
          *reinterpret_cast<Chunk<int8_t, V>*>(codes + static_cast<int64_t>(me + j * lanes) * V) = q;
        }
      if (!live) again = 0;
#pragma unroll 1
      for (; again != 0; again &= again - 1) {
        const int e = place(__ffs(again) - 1);
        const int code = static_cast<int>(floor((exactly(e) - from64) * top / span + 0.5));
        codes[e] = static_cast<int8_t>(min(most, code) - zero_code);
      }
      if (me < a.codes_width - a.width) codes[a.width + me] = 0;
      if (me < 3) {
        // (a row of equal values has scale 0, and each is the zero point)
        const float value = me == 0 ? static_cast<float>(span / top * rstd)
                            : me == 2 || a.symmetric ? 0.0f : static_cast<float>((low + span * (128.0 / 255.0)) * rstd);
        a.params[static_cast<int64_t>(row) * 3 + me] = fine || me == 2 ? value : NAN;
      }
    }
    if (a.out != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (me + j * lanes < chunks) {
          Chunk<T, V> y;
#pragma unroll
          for (int i = 0; i < V; ++i) y.v[i] = from_float<T>(to_float(h[j].v[i]) * rstd * factor(j, i));
          *reinterpret_cast<Chunk<T, V>*>(static_cast<T*>(a.out) + row * a.out_stride + static_cast<int64_t>(me + j * lanes) * V) = y;
        }
    }
  }
}

template <typename T, int V, int NV, bool WARP>
int launch(const NormArgs& a, int threads, int sms, cudaStream_t stream) {
  const int rows = WARP ? threads / 32 : 1;
  const int at_once = WARP ? 12 : threads <= 256 ? 4 : 2;  // blocks to an SM
  const int grid = a.tokens < sms * at_once * rows ? div_up(a.tokens, rows) : sms * at_once;
  MLD_CUDA_CHECK(launch_overlapped(add_norm_kernel<T, V, NV, WARP>, dim3(grid), dim3(threads), 0, stream, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

template <typename T, int V>
int launch_of(const NormArgs& a, int sms, cudaStream_t stream) {
  const int chunks = div_up(a.width, V);
  constexpr int kMost = V == 8 ? 4 : 32;  // chunks of a thread: 32 values
  if (a.width <= 1024) {
    if (chunks <= 32 * kMost / 4) return launch<T, V, kMost / 4, true>(a, 128, sms, stream);
    return launch<T, V, kMost, true>(a, 128, sms, stream);
  }
  // few rows: as many threads as there are chunks of 8 values; many: a block of 256 as long as it holds the row
  const bool few = a.tokens <= sms;
  int threads = few ? div_up(div_up(a.width, 8), 32) * 32 : div_up(div_up(a.width, 32), 32) * 32;
  threads = threads < 256 ? 256 : threads > 512 ? 512 : threads;
  const int each = div_up(chunks, threads);
  if (each <= kMost / 4) return launch<T, V, kMost / 4, false>(a, threads, sms, stream);
  if (each <= kMost / 2) return launch<T, V, kMost / 2, false>(a, threads, sms, stream);
  return launch<T, V, kMost, false>(a, threads, sms, stream);
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
  MLD_REQUIRE(tokens >= 0, "negative number of tokens");
  MLD_REQUIRE(io->out != nullptr || io->codes != nullptr, "neither out nor codes");
  MLD_REQUIRE((io->codes == nullptr) == (io->params == nullptr), "codes and params go together");
  MLD_REQUIRE(io->sum_out == nullptr || io->residual != nullptr, "sum_out needs a residual");
  if (tokens == 0) return MLD_OK;
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
  if (d->f16) return v8 ? launch_of<__half, 8>(a, sms, s) : launch_of<__half, 1>(a, sms, s);
  return v8 ? launch_of<float, 8>(a, sms, s) : launch_of<float, 1>(a, sms, s);
}

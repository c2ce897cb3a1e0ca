// Experts' gated feed-forward networks over INT4 / INT8 FullyConnected weights: the plan, the order of rows by experts, the
// weighted sum.  (Products: moe_few.cu, moe_gemm.cu.)
#include <cuda_fp16.h>

#include <cstring>
#include <new>

#include "common.cuh"
#include "kernels.h"
#include "moe.cuh"

namespace mld {
namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortCtas = 8;            // of a cluster, where one block would take long
constexpr int kSortAlone = 8192;        // pairs that one block sorts
constexpr int kMaxExperts = 1024;
constexpr int kFewShare = 8;            // rows to an expert, on average, that the products for few rows are for
constexpr int kTileSizes = kMoeTileRows / 64 + 1;  // of tiles, in steps of 64 rows
constexpr size_t kControlBytes = 256;   // of a plan's memory: the error, numbers of tiles and rows

// ------------------------------------------------------------------------------------------------ order by experts
// Pairs (token, place) counted by expert, the counts summed up, and every pair put behind those of its expert that came before
// it.  The blocks of a cluster take a part of the pairs each and read one another's counts.  (Rows of an expert come in any
// order; no row's results depend on where it stands.)
__global__ void __launch_bounds__(kSortThreads) moe_sort_kernel(const int32_t* __restrict__ ids, int pairs, int experts, int tile_rows,
                                                                 bool even, MoeBuffers b) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ int count[kMaxExperts], next[kMaxExperts];
  __shared__ int sums[2][32];
  __shared__ int of_size[kTileSizes];  // tiles by size, the largest first
  const int me = threadIdx.x, lane = me & 31, warp = me >> 5;
  const int ctas = static_cast<int>(gridDim.x), rank = static_cast<int>(blockIdx.x);  // (one cluster)
  count[me] = 0;
  if (me < kTileSizes) of_size[me] = 0;
  __syncthreads();
  const int per = (pairs + ctas - 1) / ctas, from = min(pairs, rank * per), to = min(pairs, from + per);
  for (int p = from + me; p < to; p += kSortThreads) {
    const unsigned e = static_cast<unsigned>(ids[p]);
    if (e < static_cast<unsigned>(experts)) atomicAdd(&count[e], 1);
  }
  if (ctas > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
  // expert `me`: how many rows in all, and in the blocks before
  int all = 0, before = 0;
  for (int r = 0; r < ctas; ++r) {
    int c = count[me];
    if (r != rank) {
      uint32_t there;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(&count[me])), "r"(r));
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c) : "r"(there) : "memory");
    }
    all += c;
    before += r < rank ? c : 0;
  }
  // running sums of rows and of tiles over the experts
  const int tiles = (all + tile_rows - 1) / tile_rows;
  int row_sum = all, tile_sum = tiles;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int r = __shfl_up_sync(0xffffffffu, row_sum, off), t = __shfl_up_sync(0xffffffffu, tile_sum, off);
    if (lane >= off) {
      row_sum += r;
      tile_sum += t;
    }
  }
  if (lane == 31) {
    sums[0][warp] = row_sum;
    sums[1][warp] = tile_sum;
  }
  __syncthreads();
  int row0 = row_sum - all, tile0 = tile_sum - tiles;
  for (int w = 0; w < warp; ++w) {
    row0 += sums[0][w];
    tile0 += sums[1][w];
  }
  const int all_tiles = tile0 + tiles;  // (the last expert's)
  next[me] = row0 + before;
  // (even: an expert's tiles alike, in steps of 64 rows, since a tile costs its dequantised weights, however few its rows; and
  // large tiles first, so that what is left for the end is small)
  const int rows = even && tiles > 0 ? ((all + tiles - 1) / tiles + 63) / 64 * 64 : tile_rows;
  const int size = kTileSizes - 1 - min(kTileSizes - 1, rows / 64);
  if (even && rank == 0) {
    if (tiles > 0) atomicAdd(&of_size[size], tiles);
    __syncthreads();
    if (me == 0) {
      int at = 0;
      for (int i = 0; i < kTileSizes; ++i) {
        const int n = of_size[i];
        of_size[i] = at;
        at += n;
      }
    }
    __syncthreads();
    if (tiles > 0) tile0 = atomicAdd(&of_size[size], tiles);
  }
  if (rank == 0) {
    for (int i = 0; i < tiles; ++i) b.tiles[tile0 + i] = {me, row0 + i * rows, min(rows, all - i * rows), 0};
    if (me == kSortThreads - 1) {
      b.n_tiles[0] = all_tiles;
      b.n_tiles[1] = row0 + all;
    }
  }
  __syncthreads();
  for (int p = from + me; p < to; p += kSortThreads) {
    const unsigned e = static_cast<unsigned>(ids[p]);
    int at = -1;
    if (e < static_cast<unsigned>(experts)) {
      at = atomicAdd(&next[e], 1);
      b.order[at] = p;
    }
    b.position[p] = at;
  }
  // (nobody leaves while another may still read its counts)
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Rows of x and their weights in the order of positions, a warp to a row.
__global__ void __launch_bounds__(256) moe_gather_kernel(const __half* __restrict__ x, int64_t x_stride, const float* __restrict__ weights,
                                                          int top_k, int width, MoeBuffers b) {
  pdl_wait();
  pdl_launch_dependents();
  const int at = static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (at >= b.n_tiles[1]) return;
  const int pair = b.order[at];
  if (lane == 0 && b.gates != nullptr) b.gates[at] = weights[pair];
  const uint4* from = reinterpret_cast<const uint4*>(x + pair / top_k * x_stride);
  uint4* to = reinterpret_cast<uint4*>(static_cast<__half*>(b.sorted) + static_cast<int64_t>(at) * width);
#pragma unroll 4
  for (int c = lane; c < width / 8; c += 32) to[c] = from[c];
}

// ------------------------------------------------------------------------------------------------- weighted sum
struct SumArgs {
  MoeBuffers b;
  const int32_t* ids;  // one token: its experts, no order was made
  const float* weights;
  const __half* residual;
  __half* out;
  int64_t residual_stride, out_stride;
  int experts, top_k, width;
};

// out = residual + sum_j weight_j part_j, in the order of j (fp16 parts come weighted).  A block takes a token, a thread eight
// neighbours.
template <typename P>
__global__ void __launch_bounds__(256) moe_sum_kernel(SumArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int token = blockIdx.x;
  for (int c = 8 * threadIdx.x; c < a.width; c += 8 * 256) {
    float v[8] = {};
    if (a.residual != nullptr) {
      const uint4 r = *reinterpret_cast<const uint4*>(a.residual + token * a.residual_stride + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(reinterpret_cast<const __half2*>(&r)[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
#pragma unroll 4
    for (int j = 0; j < a.top_k; ++j) {
      const int pair = token * a.top_k + j;
      const int at = a.ids == nullptr ? a.b.position[pair] : static_cast<unsigned>(a.ids[j]) < static_cast<unsigned>(a.experts) ? j : -1;
      if (at < 0) continue;
      const float w = sizeof(P) == 4 ? a.weights[pair] : 1.0f;
      const P* p = static_cast<const P*>(a.b.part) + static_cast<int64_t>(at) * a.width + c;
      if constexpr (sizeof(P) == 4) {
        const float4 lo = *reinterpret_cast<const float4*>(p), hi = *reinterpret_cast<const float4*>(p + 4);
        v[0] += w * lo.x, v[1] += w * lo.y, v[2] += w * lo.z, v[3] += w * lo.w;
        v[4] += w * hi.x, v[5] += w * hi.y, v[6] += w * hi.z, v[7] += w * hi.w;
      } else {
        const uint4 h = *reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(reinterpret_cast<const __half2*>(&h)[i]);
          v[2 * i] += f.x;
          v[2 * i + 1] += f.y;
        }
      }
    }
    uint4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<__half2*>(&o)[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(a.out + token * a.out_stride + c) = o;
  }
}

int launch_sort(const int32_t* ids, int pairs, int experts, int tile_rows, bool even, const MoeBuffers& b, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const int ctas = pairs <= kSortAlone ? 1 : kSortCtas;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MLD_CUDA_CHECK(cudaLaunchKernelEx(&cfg, moe_sort_kernel, ids, pairs, experts, tile_rows, even, b));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

}  // namespace
}  // namespace mld

using namespace mld;

struct mld_moe_plan {
  mld_moe_desc d;
  int device, sms;
  size_t bytes;
  uint8_t* memory;
  MoeBuffers b;
};

namespace {

int most_tiles(int pairs, int experts, int rows) { return pairs < experts + pairs / rows ? pairs : experts + pairs / rows; }

bool takes_many(const mld_moe_desc& d, int tokens) {
  if (d.force_path != MLD_MOE_PATH_AUTO) return d.force_path == MLD_MOE_PATH_MANY_ROWS;
  // By the rows of an expert, were all alike.  us, few / many, at 6, 8 and 10: 64 experts of 2048 x 1024 in 4 bits 86 / 105, 101 / 106,
  // 115 / 105; 8 of 4096 x 4096 76 / 108, 89 / 109, 113 / 109, in 8 bits 91 / 124, 107 / 124, 134 / 124; 128 of 2048 x 768
  // 121 / 130, 144 / 141, 166 / 141.  (Measured with rows spread evenly.  The host does not see the ids: a batch of up to this many rows
  // that goes to a few of many experts takes tiles of eight, each of which streams its expert's weights; force_path is for callers
  // who know.)
  return static_cast<int64_t>(tokens) * d.top_k > kFewShare * static_cast<int64_t>(d.experts);
}

}  // namespace

extern "C" {

int mld_moe_plan_create(const mld_moe_desc* d, mld_moe_plan** out) {
  MLD_REQUIRE(d != nullptr && out != nullptr, "null argument");
  *out = nullptr;
  MLD_REQUIRE(d->experts >= 1 && d->experts <= kMaxExperts, "experts must be 1 to 1024");
  MLD_REQUIRE(d->top_k >= 1 && d->top_k <= 32, "top_k must be 1 to 32");
  MLD_REQUIRE(d->d_model >= 32 && d->d_model <= 32768 && d->d_model % 32 == 0 && d->ffn >= 32 && d->ffn <= 32768 && d->ffn % 32 == 0,
              "d_model and ffn must be multiples of 32, 32 to 32768");
  MLD_REQUIRE(d->weight_bits == 4 || d->weight_bits == 8, "Unsupported WeightsDescription type.");
  MLD_REQUIRE(d->block == 0 || d->block == 32 || d->block == 64 || d->block == 128 || d->block == 256, "block must be 0, 32, 64, 128 or 256");
  MLD_REQUIRE(d->block == 0 || (d->d_model % d->block == 0 && d->ffn % d->block == 0), "d_model and ffn must be multiples of the block");
  MLD_REQUIRE(d->activation == MLD_MOE_SILU || d->activation == MLD_MOE_GELU_TANH, "bad activation");
  MLD_REQUIRE(d->max_tokens >= 1 && d->max_tokens <= 65536, "max_tokens must be 1 to 65536");
  MLD_REQUIRE(d->force_path >= MLD_MOE_PATH_AUTO && d->force_path <= MLD_MOE_PATH_MANY_ROWS, "bad force_path");
  int device = d->device;
  if (device < 0) MLD_CUDA_CHECK(cudaGetDevice(&device));
  mld_moe_plan* p = new (std::nothrow) mld_moe_plan();
  if (p == nullptr) {
    set_last_error_text("out of host memory");
    return MLD_OUT_OF_RANGE;
  }
  p->d = *d;
  p->device = device;
  p->sms = sm_count(device);
  // The most pairs that either path may get.  The rows of x in order and the experts' outputs share their place: those are read by the
  // first product, these written by the second.
  const size_t pairs = static_cast<size_t>(d->max_tokens) * d->top_k;
  const bool may_many = takes_many(*d, d->max_tokens);
  const size_t few = d->force_path == MLD_MOE_PATH_FEW_ROWS || !may_many ? pairs : d->force_path == MLD_MOE_PATH_AUTO ? kFewShare * static_cast<size_t>(d->experts) : 0;
  const size_t width = static_cast<size_t>(d->d_model), most = may_many ? pairs * width * (moe_weighted_parts(d->block) ? 2 : 4) : 0, shared = most > few * width * 4 ? most : few * width * 4;
  const bool weighted = may_many && moe_weighted_parts(d->block);
  size_t at = 0;
  const auto room = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t control = room(kControlBytes), order = room(pairs * 4), position = room(pairs * 4),
               tiles = room(most_tiles(static_cast<int>(pairs), d->experts, kMoeFewRows) * sizeof(MoeTile)), hidden = room(pairs * d->ffn * 2), rows = room(shared),
               gates = room(weighted ? pairs * 4 : 0);
  int before = -1;
  cudaError_t e = cudaGetDevice(&before);
  if (e == cudaSuccess && before != device) e = cudaSetDevice(device);
  if (e == cudaSuccess) e = cudaMalloc(reinterpret_cast<void**>(&p->memory), at);
  if (e == cudaSuccess) e = zero_now(p->memory, kControlBytes);
  if (before >= 0 && before != device) cudaSetDevice(before);
  if (e != cudaSuccess) {
    set_last_error("experts' workspace", e);
    if (p->memory != nullptr) cudaFree(p->memory);
    delete p;
    return MLD_CUDA_ERROR;
  }
  p->bytes = at;
  p->b.error = reinterpret_cast<int*>(p->memory + control);
  p->b.n_tiles = p->b.error + 1;
  p->b.order = reinterpret_cast<int*>(p->memory + order);
  p->b.position = reinterpret_cast<int*>(p->memory + position);
  p->b.tiles = reinterpret_cast<MoeTile*>(p->memory + tiles);
  p->b.hidden = p->memory + hidden;
  p->b.gates = weighted ? reinterpret_cast<float*>(p->memory + gates) : nullptr;
  p->b.part = p->b.sorted = p->memory + rows;
  *out = p;
  return MLD_OK;
}

int mld_moe_plan_destroy(mld_moe_plan* plan) {
  if (plan == nullptr) return MLD_OK;
  if (plan->memory != nullptr) cudaFree(plan->memory);
  delete plan;
  return MLD_OK;
}

size_t mld_moe_plan_workspace_bytes(const mld_moe_plan* plan) { return plan != nullptr ? plan->bytes : 0; }

int mld_moe_plan_device_status(mld_moe_plan* plan, int32_t* code) {
  MLD_REQUIRE(plan != nullptr && code != nullptr, "null argument");
  int before = -1, c = 0;
  MLD_CUDA_CHECK(cudaGetDevice(&before));
  if (before != plan->device) MLD_CUDA_CHECK(cudaSetDevice(plan->device));
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(&c, plan->b.error, sizeof c, cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && c != 0) e = zero_now(plan->memory, kControlBytes);
  if (before != plan->device) cudaSetDevice(before);
  MLD_CUDA_CHECK(e);
  *code = c != 0 ? MLD_TIMEOUT : 0;
  if (c != 0) {
    set_last_error_text("a bounded device-side wait of the experts' products gave up");
    return MLD_TIMEOUT;
  }
  return MLD_OK;
}

int mld_moe_run(mld_moe_plan* plan, const mld_moe_io* io, int32_t tokens, void* stream_v) {
  MLD_REQUIRE(plan != nullptr && io != nullptr, "null argument");
  const mld_moe_desc& d = plan->d;
  MLD_REQUIRE(tokens >= 0 && tokens <= d.max_tokens, "tokens exceeds the plan's max_tokens");
  if (tokens == 0) return MLD_OK;
  MLD_REQUIRE(io->x != nullptr && io->ids != nullptr && io->weights != nullptr && io->gate_up != nullptr && io->gate_up_scale != nullptr &&
                  io->down != nullptr && io->down_scale != nullptr && io->out != nullptr,
              "null tensor");
  const uintptr_t wide = reinterpret_cast<uintptr_t>(io->x) | reinterpret_cast<uintptr_t>(io->gate_up) |
                         reinterpret_cast<uintptr_t>(io->gate_up_scale) | reinterpret_cast<uintptr_t>(io->down) |
                         reinterpret_cast<uintptr_t>(io->down_scale) | reinterpret_cast<uintptr_t>(io->residual) |
                         reinterpret_cast<uintptr_t>(io->out);
  MLD_REQUIRE((wide & 15) == 0, "tensors must be 16-byte aligned");
  MLD_REQUIRE(((reinterpret_cast<uintptr_t>(io->ids) | reinterpret_cast<uintptr_t>(io->weights)) & 3) == 0,
              "ids and weights must be aligned to their type");
  if (tokens > 1) {
    MLD_REQUIRE(io->x_stride >= 0 && io->x_stride % 8 == 0 && io->out_stride >= d.d_model && io->out_stride % 8 == 0 &&
                    (io->residual == nullptr || (io->residual_stride >= 0 && io->residual_stride % 8 == 0)),
                "strides must be multiples of 8, an output's at least d_model");
    MLD_REQUIRE(io->residual != io->out || io->residual_stride == io->out_stride, "an output in the place of the residual needs its stride");
  }
  int current = -1;
  MLD_CUDA_CHECK(cudaGetDevice(&current));
  MLD_REQUIRE(current == plan->device, "the plan belongs to another device than the current one");
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const int pairs = tokens * d.top_k;
  const bool one = tokens == 1, many = takes_many(d, tokens);
  int rc = MLD_OK;
  const MoeShape shape = {d.experts, d.top_k, d.d_model, d.ffn, d.weight_bits, d.block, d.activation};
  SumArgs s = {};
  s.b = plan->b;
  s.ids = one && !many ? io->ids : nullptr;
  s.weights = io->weights;
  s.residual = static_cast<const __half*>(io->residual);
  s.out = static_cast<__half*>(io->out);
  s.residual_stride = io->residual_stride;
  s.out_stride = io->out_stride;
  s.experts = d.experts;
  s.top_k = d.top_k;
  s.width = d.d_model;
  if (many) {
    const int rows = kMoeTileRows;
    rc = launch_sort(io->ids, pairs, d.experts, rows, true, plan->b, stream);
    if (rc != MLD_OK) return rc;
    MLD_CUDA_CHECK(launch_overlapped(moe_gather_kernel, dim3(div_up(pairs, 8)), dim3(256), 0, stream, static_cast<const __half*>(io->x),
                                     io->x_stride, io->weights, d.top_k, d.d_model, plan->b));
    MLD_LAUNCH_CHECK();
    rc = launch_moe_gemm(true, shape, plan->b, io->gate_up, io->gate_up_scale, pairs, plan->sms, stream);
    if (rc == MLD_OK) rc = launch_moe_gemm(false, shape, plan->b, io->down, io->down_scale, pairs, plan->sms, stream);
    if (rc != MLD_OK) return rc;
    MLD_CUDA_CHECK(launch_overlapped(moe_weighted_parts(d.block) ? moe_sum_kernel<__half> : moe_sum_kernel<float>, dim3(tokens), dim3(256), 0,
                                     stream, s));
    MLD_LAUNCH_CHECK();
    return MLD_OK;
  }
  int tiles = pairs;
  if (!one) {
    rc = launch_sort(io->ids, pairs, d.experts, kMoeFewRows, false, plan->b, stream);
    if (rc != MLD_OK) return rc;
    tiles = most_tiles(pairs, d.experts, kMoeFewRows);
  }
  rc = launch_moe_few(true, shape, plan->b, s.ids, io->x, io->x_stride, io->gate_up, io->gate_up_scale, tiles, plan->sms, stream);
  if (rc == MLD_OK)
    rc = launch_moe_few(false, shape, plan->b, s.ids, nullptr, 0, io->down, io->down_scale, tiles, plan->sms, stream);
  if (rc != MLD_OK) return rc;
  MLD_CUDA_CHECK(launch_overlapped(moe_sum_kernel<float>, dim3(tokens), dim3(256), 0, stream, s));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

}  // extern "C"

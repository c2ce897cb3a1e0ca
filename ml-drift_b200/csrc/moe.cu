// Experts' gated feed-forward networks over INT4 / INT8 FullyConnected weights: the plan, the order of rows by experts, the
// products for few rows, the weighted sum.  (Products for many rows: moe_gemm.cu.)
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
constexpr int kFewWarps = 8;
constexpr int kFewOutputs = 64;         // outputs of a block with few rows
constexpr int kMaxExperts = 1024;

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
  const int me = threadIdx.x, lane = me & 31, warp = me >> 5;
  const int ctas = static_cast<int>(gridDim.x), rank = static_cast<int>(blockIdx.x);  // (one cluster)
  count[me] = 0;
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
  next[me] = row0 + before;
  if (rank == 0) {
    // (even: an expert's tiles alike, in steps of 64 rows: one costs its dequantised weights, however few its rows)
    const int rows = even && tiles > 0 ? ((all + tiles - 1) / tiles + 63) / 64 * 64 : tile_rows;
    for (int i = 0; i < tiles; ++i) b.tiles[tile0 + i] = {me, row0 + i * rows, min(rows, all - i * rows), 0};
    if (me == kSortThreads - 1) {
      b.n_tiles[0] = tile0 + tiles;
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

// Rows of x in the order of positions, a warp to a row.
__global__ void __launch_bounds__(256) moe_gather_kernel(const __half* __restrict__ x, int64_t x_stride, int top_k, int width, MoeBuffers b) {
  pdl_wait();
  pdl_launch_dependents();
  const int at = static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (at >= b.n_tiles[1]) return;
  const uint4* from = reinterpret_cast<const uint4*>(x + b.order[at] / top_k * x_stride);
  uint4* to = reinterpret_cast<uint4*>(static_cast<__half*>(b.sorted) + static_cast<int64_t>(at) * width);
#pragma unroll 4
  for (int c = lane; c < width / 8; c += 32) to[c] = from[c];
}

// ---------------------------------------------------------------------------------------------------- few rows
struct FewArgs {
  MoeBuffers b;
  const int32_t* ids;      // one token: its experts, no order was made
  const __half* x;         // the first product: rows by token
  int64_t x_stride;
  const uint8_t* weights;
  const __half* scale;
  int64_t expert_bytes, expert_scales;
  int experts, top_k, n, k, groups, block_shift;  // block_shift: log2 of the inputs of a scale
  int activation;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t less(uint32_t biased, __half2 zero) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&biased), zero);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// 32 inputs x 64 outputs as a lane (g = lane / 4, t = lane % 4) holds them: the 4x4 blocks of output slices 2 g and 2 g + 1, input
// slices t and t + 4, and the scales of its eight outputs.
template <int BITS>
struct FewGroup {
  uint4 w[BITS == 4 ? 2 : 4];
  uint4 s;
};

// FIRST: x -> hidden, else hidden -> part.  NT: eights of rows.
template <int BITS, int NT, bool FIRST>
__global__ void __launch_bounds__(kFewWarps * 32) moe_few_kernel(FewArgs a) {
  constexpr int kAhead = BITS == 4 ? 4 : 3;  // groups of a lane under way
  constexpr int kBlk = BITS == 4 ? 8 : 16;
  constexpr int kCols = 8 * NT;
  extern __shared__ float red[];  // [warps][kCols][kFewOutputs + 4]
  constexpr int kPitch = kFewOutputs + 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  if constexpr (FIRST) pdl_wait();
  // (The second product's tiles and weights were complete before the launch ahead let this one begin; its rows were not.)
  const int nth = static_cast<int>(blockIdx.z * gridDim.y + blockIdx.y);
  MoeTile tile = {0, nth, 1, 0};
  if (a.ids != nullptr) {
    tile.expert = a.ids[nth];
    if (static_cast<unsigned>(tile.expert) >= static_cast<unsigned>(a.experts)) return;
  } else {
    if (nth >= *a.b.n_tiles) return;
    tile = a.b.tiles[nth];
  }
  const int n0 = static_cast<int>(blockIdx.x) * kFewOutputs;
  const bool has_n = n0 + 8 * g < a.n;
  const int64_t pitch = static_cast<int64_t>(a.n >> 2) * kBlk;  // bytes of an input slice
  const uint8_t* const wp = a.weights + tile.expert * a.expert_bytes + t * pitch + ((n0 >> 2) + 2 * g) * kBlk;
  const __half* const sp = a.scale + tile.expert * a.expert_scales + n0 + 8 * g;
  const int groups = a.k >> 5;
  FewGroup<BITS> ring[kAhead];
  const auto fetch = [&](FewGroup<BITS>& r, int group) {
    if (has_n && group < groups) {
      const uint8_t* p = wp + static_cast<int64_t>(group) * 8 * pitch;
      r.w[0] = load_stream(p);
      if constexpr (BITS == 4) {
        r.w[1] = load_stream(p + 4 * pitch);
      } else {
        r.w[1] = load_stream(p + 16);
        r.w[2] = load_stream(p + 4 * pitch);
        r.w[3] = load_stream(p + 4 * pitch + 16);
      }
      r.s = *reinterpret_cast<const uint4*>(sp + static_cast<int64_t>(min((group << 5) >> a.block_shift, a.groups - 1)) * a.n);
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    ring[i] = {};
    fetch(ring[i], warp + i * kFewWarps);
  }
  if constexpr (!FIRST) pdl_wait();
  pdl_launch_dependents();
  const uint2* row[NT];  // this lane's row of every eight: its input slices t, t + 4, ...
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    row[nt] = nullptr;
    if (8 * nt + g < tile.rows) {
      const int at = tile.row0 + 8 * nt + g;
      if constexpr (FIRST) {
        const int token = a.ids != nullptr ? 0 : a.b.order[at] / a.top_k;
        row[nt] = reinterpret_cast<const uint2*>(a.x + token * a.x_stride) + t;
      } else {
        row[nt] = reinterpret_cast<const uint2*>(static_cast<const __half*>(a.b.hidden) + static_cast<int64_t>(at) * a.k) + t;
      }
    }
  }
  float acc[2][2][NT][4];  // [output slice of the pair][outputs 0, 1 / 2, 3][eight of rows]
#pragma unroll
  for (int i = 0; i < 2 * 2 * NT * 4; ++i) (&acc[0][0][0][0])[i] = 0.0f;
  const __half2 zero = __float2half2_rn(BITS == 4 ? 1032.0f : 1152.0f);
  for (int base = warp; base < groups; base += kAhead * kFewWarps) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int group = base + i * kFewWarps;
      if (group < groups) {
        uint2 xb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) xb[nt][h] = row[nt] != nullptr ? row[nt][group * 8 + 4 * h] : make_uint2(0u, 0u);
        const FewGroup<BITS> cur = ring[i];
        fetch(ring[i], group + kAhead * kFewWarps);
        const __half2* const s2 = reinterpret_cast<const __half2*>(&cur.s);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float sum[NT][4];
#pragma unroll
            for (int i4 = 0; i4 < NT * 4; ++i4) (&sum[0][0])[i4] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t a0, a1, a2, a3;
              if constexpr (BITS == 4) {
                const uint32_t lo = b == 0 ? cur.w[h].x : cur.w[h].z, hi = b == 0 ? cur.w[h].y : cur.w[h].w;
                a0 = less(((lo >> (8 * r)) & 0x000F000Fu) | 0x64006400u, zero);
                a1 = less(((lo >> (8 * r + 4)) & 0x000F000Fu) | 0x64006400u, zero);
                a2 = less(((hi >> (8 * r)) & 0x000F000Fu) | 0x64006400u, zero);
                a3 = less(((hi >> (8 * r + 4)) & 0x000F000Fu) | 0x64006400u, zero);
              } else {
                // a word per input channel, a byte per output
                const uint4 v = cur.w[2 * h + b];
                a0 = less((__byte_perm(v.x, v.y, 0x0400u + (2 * r) * 0x0101u) & 0x00FF00FFu) | 0x64006400u, zero);
                a1 = less((__byte_perm(v.x, v.y, 0x0400u + (2 * r + 1) * 0x0101u) & 0x00FF00FFu) | 0x64006400u, zero);
                a2 = less((__byte_perm(v.z, v.w, 0x0400u + (2 * r) * 0x0101u) & 0x00FF00FFu) | 0x64006400u, zero);
                a3 = less((__byte_perm(v.z, v.w, 0x0400u + (2 * r + 1) * 0x0101u) & 0x00FF00FFu) | 0x64006400u, zero);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16(sum[nt], a0, a1, a2, a3, xb[nt][h].x, xb[nt][h].y);
            }
            const float2 s = __half22float2(s2[2 * b + r]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              acc[b][r][nt][0] += sum[nt][0] * s.x;
              acc[b][r][nt][1] += sum[nt][1] * s.x;
              acc[b][r][nt][2] += sum[nt][2] * s.y;
              acc[b][r][nt][3] += sum[nt][3] * s.y;
            }
          }
      }
    }
  }
  // the warps' sums meet in shared memory
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<float2*>(&red[(warp * kCols + 8 * nt + 2 * t + c) * kPitch + 8 * g + 4 * b + 2 * r]) =
              make_float2(acc[b][r][nt][c], acc[b][r][nt][2 + c]);
  __syncthreads();
  for (int i = threadIdx.x; i < kCols * (kFewOutputs / 2); i += kFewWarps * 32) {
    const int col = i / (kFewOutputs / 2), pair = i % (kFewOutputs / 2);
    if (col >= tile.rows || n0 + 2 * pair >= a.n) continue;
    float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float2 p = *reinterpret_cast<const float2*>(&red[(w * kCols + col) * kPitch + 2 * pair]);
      v.x += p.x;
      v.y += p.y;
    }
    const int64_t at = tile.row0 + col;
    if constexpr (FIRST)
      static_cast<__half*>(a.b.hidden)[at * (a.n >> 1) + (n0 >> 1) + pair] = __float2half_rn(moe_gated(v.x, v.y, a.activation));
    else
      *reinterpret_cast<float2*>(static_cast<float*>(a.b.part) + at * a.n + n0 + 2 * pair) = v;
  }
}

// ------------------------------------------------------------------------------------------------- weighted sum
struct SumArgs {
  MoeBuffers b;
  const int32_t* ids;  // one token: as FewArgs
  const float* weights;
  const __half* residual;
  __half* out;
  int64_t residual_stride, out_stride;
  int experts, top_k, width;
};

// out = residual + sum_j weight_j part_j, in the order of j.  A block takes a token, a thread eight neighbours.
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
      int at;
      if (a.ids != nullptr)
        at = static_cast<unsigned>(a.ids[j]) < static_cast<unsigned>(a.experts) ? j : -1;
      else
        at = a.b.position[pair];
      if (at < 0) continue;
      const float w = a.weights[pair];
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
          v[2 * i] += w * f.x;
          v[2 * i + 1] += w * f.y;
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

template <int BITS, int NT, bool FIRST>
int launch_few_of(const FewArgs& a, int tiles, cudaStream_t stream) {
  constexpr size_t smem = static_cast<size_t>(kFewWarps) * 8 * NT * (kFewOutputs + 4) * sizeof(float);
  auto kern = moe_few_kernel<BITS, NT, FIRST>;
  static bool done[kMaxDevices];
  int dev;
  if (needs_configure(done, &dev)) {
    MLD_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    if (dev >= 0) done[dev] = true;
  }
  MLD_CUDA_CHECK(launch_overlapped(kern, dim3(div_up(a.n, kFewOutputs), tiles < 32768 ? tiles : 32768, div_up(tiles, 32768)),
                                   dim3(kFewWarps * 32), smem, stream, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}
template <bool FIRST>
int launch_few(const FewArgs& a, int bits, int eights, int tiles, cudaStream_t stream) {
  if (bits == 4)
    return eights == 1   ? launch_few_of<4, 1, FIRST>(a, tiles, stream)
           : eights == 2 ? launch_few_of<4, 2, FIRST>(a, tiles, stream)
                         : launch_few_of<4, 4, FIRST>(a, tiles, stream);
  return eights == 1   ? launch_few_of<8, 1, FIRST>(a, tiles, stream)
         : eights == 2 ? launch_few_of<8, 2, FIRST>(a, tiles, stream)
                       : launch_few_of<8, 4, FIRST>(a, tiles, stream);
}

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
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

// With many rows, tiles of up to 256 (two SMs) or 128; with few, of 8 to 32: enough for a usual expert's share.
int few_eights(int pairs, int experts) { return pairs <= 6 * experts ? 1 : pairs <= 12 * experts ? 2 : 4; }
int most_tiles(int pairs, int experts, int rows) { return pairs < experts + pairs / rows ? pairs : experts + pairs / rows; }

bool takes_many(const mld_moe_desc& d, int tokens) {
  if (d.force_path != MLD_MOE_PATH_AUTO) return d.force_path == MLD_MOE_PATH_MANY_ROWS;
  return static_cast<int64_t>(tokens) * d.top_k >= 24ll * d.experts;
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
  const size_t pairs = static_cast<size_t>(d->max_tokens) * d->top_k;
  size_t at = 0;
  const auto room = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t error = room(256), order = room(pairs * 4), position = room(pairs * 4),
               tiles = room(most_tiles(static_cast<int>(pairs), d->experts, 8) * sizeof(MoeTile)), hidden = room(pairs * d->ffn * 2),
               part = room(pairs * d->d_model * 4), sorted = room(pairs * d->d_model * 2);
  int before = -1;
  cudaError_t e = cudaGetDevice(&before);
  if (e == cudaSuccess && before != device) e = cudaSetDevice(device);
  if (e == cudaSuccess) e = cudaMalloc(reinterpret_cast<void**>(&p->memory), at);
  if (e == cudaSuccess) e = zero_now(p->memory, 256);
  if (before >= 0 && before != device) cudaSetDevice(before);
  if (e != cudaSuccess) {
    set_last_error("experts' workspace", e);
    if (p->memory != nullptr) cudaFree(p->memory);
    delete p;
    return MLD_CUDA_ERROR;
  }
  p->bytes = at;
  p->b.error = reinterpret_cast<int*>(p->memory + error);
  p->b.n_tiles = reinterpret_cast<int*>(p->memory + error) + 1;
  p->b.order = reinterpret_cast<int*>(p->memory + order);
  p->b.position = reinterpret_cast<int*>(p->memory + position);
  p->b.tiles = reinterpret_cast<MoeTile*>(p->memory + tiles);
  p->b.hidden = p->memory + hidden;
  p->b.part = p->memory + part;
  p->b.sorted = p->memory + sorted;
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
  if (e == cudaSuccess && c != 0) e = zero_now(plan->b.error, sizeof c);
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
  const int eights = one ? 1 : few_eights(pairs, d.experts);
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
    const int rows = pairs > 64 * d.experts ? 256 : 128;
    rc = launch_sort(io->ids, pairs, d.experts, rows, true, plan->b, stream);
    if (rc != MLD_OK) return rc;
    MLD_CUDA_CHECK(launch_overlapped(moe_gather_kernel, dim3(div_up(pairs, 8)), dim3(256), 0, stream, static_cast<const __half*>(io->x),
                                     io->x_stride, d.top_k, d.d_model, plan->b));
    MLD_LAUNCH_CHECK();
    rc = launch_moe_gemm(true, shape, plan->b, io->gate_up, io->gate_up_scale, pairs, rows, plan->sms, stream);
    if (rc == MLD_OK) rc = launch_moe_gemm(false, shape, plan->b, io->down, io->down_scale, pairs, rows, plan->sms, stream);
    if (rc != MLD_OK) return rc;
    MLD_CUDA_CHECK(launch_overlapped(moe_sum_kernel<__half>, dim3(tokens), dim3(256), 0, stream, s));
    MLD_LAUNCH_CHECK();
    return MLD_OK;
  }
  int tiles = pairs;
  if (!one) {
    rc = launch_sort(io->ids, pairs, d.experts, 8 * eights, false, plan->b, stream);
    if (rc != MLD_OK) return rc;
    tiles = most_tiles(pairs, d.experts, 8 * eights);
  }
  FewArgs f = {};
  f.b = plan->b;
  f.ids = one ? io->ids : nullptr;
  f.x = static_cast<const __half*>(io->x);
  f.x_stride = io->x_stride;
  f.experts = d.experts;
  f.top_k = d.top_k;
  f.activation = d.activation;
  const auto matrix = [&](const void* w, const void* s, int n, int k) {
    f.weights = static_cast<const uint8_t*>(w);
    f.scale = static_cast<const __half*>(s);
    f.n = n;
    f.k = k;
    f.groups = d.block != 0 ? k / d.block : 1;
    f.block_shift = d.block != 0 ? log2_of(d.block) : 30;
    f.expert_bytes = static_cast<int64_t>(n) * k * d.weight_bits / 8;
    f.expert_scales = static_cast<int64_t>(f.groups) * n;
  };
  matrix(io->gate_up, io->gate_up_scale, 2 * d.ffn, d.d_model);
  rc = launch_few<true>(f, d.weight_bits, eights, tiles, stream);
  if (rc != MLD_OK) return rc;
  matrix(io->down, io->down_scale, d.d_model, d.ffn);
  rc = launch_few<false>(f, d.weight_bits, eights, tiles, stream);
  if (rc != MLD_OK) return rc;
  MLD_CUDA_CHECK(launch_overlapped(moe_sum_kernel<float>, dim3(tokens), dim3(256), 0, stream, s));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

}  // extern "C"

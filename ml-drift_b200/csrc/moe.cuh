// What the kernels of the experts' networks share.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace mld {

// Rows of one expert that are worked on together: positions row0 .. row0 + rows - 1 of the order by experts.
struct MoeTile {
  int expert, row0, rows, unused;
};

// Device memory of a plan.
struct MoeBuffers {
  int* order;        // [pairs]: position -> pair (token * top_k + place)
  int* position;     // [pairs]: pair -> position, -1: no expert
  MoeTile* tiles;    // [most tiles]
  int* n_tiles;
  void* hidden;      // fp16 [pairs][ffn], by position
  float* gates;      // [pairs]: the pairs' weights by position (where parts are weighted, else null)
  void* part;        // [pairs][d_model], by position: fp32; with many rows and scales to groups fp16, times the weights
  void* sorted;      // fp16 [pairs][d_model]: x by position (many rows); in the place of `part`, which is written later
  int* error;
};

struct MoeShape {
  int experts, top_k, d_model, ffn, bits, block, activation;
};

#ifdef __CUDACC__
// act(gate) * up
__device__ __forceinline__ float moe_gated(float gate, float up, int activation) {
  const float u = activation == MLD_MOE_SILU ? gate : 1.5957691216057308f * (gate + 0.044715f * gate * gate * gate);
  // (GELU's (1 + tanh(u / 2)) / 2 is 1 / (1 + exp(-u)).  A quotient good to 2 ulp: the exact one took the products' results longer
  // than their sums, and what is rounded to fp16 next does not show the difference.)
  return __fdividef(gate, 1.0f + __expf(-u)) * up;
}
#endif

// The products of tiles of up to kMoeTileRows rows on the tensor cores.  first: x by position -> hidden; else hidden -> part (fp32, or
// moe_weighted_parts: in fp16, times the pairs' weights, so that a part is finite where their sum is).
inline bool moe_weighted_parts(int block) { return block != 0; }
constexpr int kMoeTileRows = 256;
int launch_moe_gemm(bool first, const MoeShape& s, const MoeBuffers& b, const void* weights, const void* scale, int pairs, int sms,
                    cudaStream_t stream);

// The products of tiles of up to kMoeFewRows rows, bound by the weights.  first: x (rows by token) -> hidden; else hidden -> part (fp32).
// ids: one token's experts, without an order, or null; tiles: how many there may be.
constexpr int kMoeFewRows = 8;
int launch_moe_few(bool first, const MoeShape& s, const MoeBuffers& b, const int32_t* ids, const void* x, int64_t x_stride,
                   const void* weights, const void* scale, int tiles, int sms, cudaStream_t stream);

}  // namespace mld

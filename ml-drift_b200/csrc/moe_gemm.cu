// The experts' products for many rows: tiles of one expert's rows on pairs of SMs, the dequantised weights in tensor memory.
//
// The form is gemm_wtmem_kernel's (Y^T = W X^T, tcgen05 cta_group::2, weights as the A operand in tensor memory, rows as the B
// operand in shared memory), with what a grouped product needs in place of what a single one does:
//   - a tile is 256 outputs of one expert x up to 256 of its rows; which expert and which rows stands in a list that the
//     ordering kernel left in device memory.  Every role reads the list for itself and goes through the same tiles.
//   - rows of an expert follow one another, so a tile's rows are one box after another of 32; as many are fetched as the tile has
//     rows, and the MMAs' N is that many, too (in steps of 64).  Columns behind the tile's rows belong to other experts, or are
//     zeros, and are not written.
//   - the epilogue writes rows (not slices): of the first product act(gate) * up, for which neighbouring lanes, which hold a gate
//     and an up channel, exchange half of their tokens; of the second the expert's output times the row's weight.
// Weights with a scale to an output (CHANNEL) are multiplied as the integers that they are, which halves hold, and the sums are scaled;
// the second product's go out in 32 bits then.  So nothing is rounded but x, the gated values and the result, as with few rows.  Weights
// with scales to groups of inputs have to be scaled, and rounded to halves, ahead of the product; there outputs are halves, too (in
// 32 bits 2048 tokens through 8 of 64 experts of 2048 x 1024 took 323 us in place of 301, and were 1.1 times as exact).
// Per CTA: warps 0 and 23 fetch rows, every other stage each, warp 22 packed weights, warp 1 issues the MMAs (of the pair's first
// CTA), warps 6..21 dequantise (four to a stage of 128 inputs), warps 2..5 write the results.  Tensor memory: four stages of weights
// and two halves of 128 columns of accumulators.  A tile of up to 128 rows takes the half that is free, and the next tile goes on
// while it is written; a larger one takes both, so the sixteen help writing.
// With few rows bound by what a stage costs each role, whatever is in it (the warps that fetch and the one that issues MMAs 300 to
// 500 cycles, the dequantisation about 1700 for a quarter of the stages): hence 128 inputs to a stage, where 64 took 122 us against
// 107 (128 tokens through 8 of 64 experts, 2048 x 1024) and 139 against 127 (512 tokens), at a cost of 1 to 2 % at 1531 and 2048.  With
// many rows by the MMAs, 4 cycles a row and stage, and by the clock that the power limit leaves: 1501 tokens through 2 of 8 experts of
// 4096 x 14336 take 1051 us, 1.01 PFLOP/s.
// Every wait is bounded.
#include <cuda_fp16.h>

#include <cstring>

#include "common.cuh"
#include "moe.cuh"
#include "pair_common.cuh"
#include "wtmem.cuh"

namespace mld {
namespace {

constexpr int kStages = 4;              // rows in shared memory + weights in tensor memory
constexpr int kWStages = 4;             // packed weights
constexpr int kChannels = 128;          // outputs per CTA
constexpr int kBoxRows = 32;
constexpr int kBoxBytes = kBoxRows * kKBytes;
constexpr int kInputs = 128;            // of a stage
constexpr int kSlices = kInputs / 4;    // packed rows of a stage
constexpr int kAtom = 128 * kKBytes;    // shared memory of 64 inputs of a CTA's rows
constexpr int kHalf = 128;               // columns of one of two halves of accumulators
constexpr int kColumns = 2 * kHalf;      // the weights' follow
static_assert(kColumns == kMoeTileRows, "a tile's rows");
constexpr int kThreads = 24 * 32;
constexpr int kReaders = 5;             // warps that can read a lane quarter's accumulators
constexpr int kErrMoeBase = 70;

struct GemmArgs {
  const MoeTile* tiles;
  const int* n_tiles;
  int n_channel_tiles, k_blocks;
  int n, k;                             // outputs, inputs
  const __half* scale;
  int64_t expert_scales;
  int groups, group_shift;              // log2 of a group's input slices
  void* out;                            // rows by position: fp16 act(gate) * up [n / 2]; fp32 outputs [n], or fp16 times the row's weight
  const float* gates;                   // the rows' weights (not with a scale to an output)
  int activation;
  int* error;
};

struct Work {
  int t, total, step, n_channel_tiles;
  const MoeTile* tiles;
  __device__ __forceinline__ bool next(MoeTile& tile, int& n0) {
    if (t >= total) return false;
    const int4 v = *reinterpret_cast<const int4*>(tiles + t / n_channel_tiles);
    tile.expert = v.x;
    tile.row0 = v.y;
    tile.rows = v.z;
    n0 = t % n_channel_tiles * (2 * kChannels);
    t += step;
    return true;
  }
  __device__ __forceinline__ bool done() const { return t >= total; }
};
__device__ __forceinline__ int columns_of(const MoeTile& t) { return (t.rows + 63) & ~63; }

// Which accumulators a tile has, and which barriers: worked out alike by every role that goes through the tiles.
struct Turns {
  uint32_t half = 0;              // the next small tile's
  uint32_t uses = 0;              // of each half so far, odd or even, a bit each
  uint32_t read = 0;              // tiles so far, odd or even: read by the writing warps alone in each half (bits 0, 1), by all (bit 2)
  uint32_t at = 0;                // the tile's half (its first, of a large one)
  bool large = false, all = false;
  __device__ __forceinline__ void take(const MoeTile& t, bool last) {
    large = t.rows > kHalf;
    all = large || last;
    at = large ? 0 : half;
  }
  // barrier of the finished MMAs: [0], [1] of halves that the writing warps read alone, [2] of what all read.  (A wait tells one use
  // of a barrier from the one before and no more, so nobody may miss a use of one that it waits on.)
  __device__ __forceinline__ uint32_t full() const { return all ? 2 : at; }
  __device__ __forceinline__ uint32_t full_phase() const { return read >> full() & 1u; }
  __device__ __forceinline__ uint32_t uses_of(uint32_t h) const { return uses >> h & 1u; }
  __device__ __forceinline__ void next() {
    read ^= 1u << full();
    uses ^= large ? 3u : 1u << at;
    half ^= large ? 0u : 1u;
  }
};

// x0..x3: a lane's four pairs of tokens -> pair q of the tokens of four lanes' channels.  A: lane bits that number the four.
template <int LOW>
__device__ __forceinline__ void turn_pairs(uint32_t& x0, uint32_t& x1, uint32_t& x2, uint32_t& x3, int q) {
  {
    const bool up = (q & 2) != 0;
    const uint32_t s0 = up ? x0 : x2, s1 = up ? x1 : x3;
    const uint32_t r0 = __shfl_xor_sync(0xffffffffu, s0, 2 * LOW), r1 = __shfl_xor_sync(0xffffffffu, s1, 2 * LOW);
    if (up) {
      x0 = r0;
      x1 = r1;
    } else {
      x2 = r0;
      x3 = r1;
    }
  }
  {
    const bool up = (q & 1) != 0;
    const uint32_t s0 = up ? x0 : x1, s1 = up ? x2 : x3;
    const uint32_t r0 = __shfl_xor_sync(0xffffffffu, s0, LOW), r1 = __shfl_xor_sync(0xffffffffu, s1, LOW);
    if (up) {
      x0 = r0;
      x2 = r1;
    } else {
      x1 = r0;
      x3 = r1;
    }
  }
}
// The four channels of a token pair, after turn_pairs, to two rows of the output.
__device__ __forceinline__ void store_pair(__half* first, int64_t pitch, bool one, bool two, uint32_t x0, uint32_t x1, uint32_t x2,
                                           uint32_t x3) {
  if (one) *reinterpret_cast<uint2*>(first) = make_uint2(__byte_perm(x0, x1, 0x5410), __byte_perm(x2, x3, 0x5410));
  if (two) *reinterpret_cast<uint2*>(first + pitch) = make_uint2(__byte_perm(x0, x1, 0x7632), __byte_perm(x2, x3, 0x7632));
}

template <int BITS, bool CHANNEL, bool FIRST>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    moe_gemm_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, GemmArgs a) {
  constexpr int kBlk = BITS == 4 ? 8 : 16;
  constexpr int kPitch = kChannels / 4 * kBlk;        // bytes of a packed row of the box
  constexpr int kWBytes = kSlices * kPitch;
  constexpr int kXBytes = 2 * kAtom;                  // a CTA's rows of a stage
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = smem;
  uint8_t* sW = sX + kStages * kXBytes;
  uint64_t* full_w = reinterpret_cast<uint64_t*>(sW + kWStages * kWBytes);
  uint64_t* w_empty = full_w + kWStages;       // the dequantising warps have read the box
  uint64_t* full_ab = w_empty + kWStages;      // first CTA: rows and weights of both CTAs are there
  uint64_t* empty = full_ab + kStages;         // the stage's MMAs are done (arrives in both CTAs)
  uint64_t* tmem_full = empty + kStages;       // [3], see Turns
  uint64_t* tmem_empty = tmem_full + 3;        // [2], first CTA: a half has been read (by a quarter's five warps, or by one for all)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kWStages; ++s) {
      mbar_init(&full_w[s], 1);
      mbar_init(&w_empty[s], 4);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_ab[s], 1 + 2 * 4);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 3; ++b) mbar_init(&tmem_full[b], 1);
    for (int b = 0; b < 2; ++b) mbar_init(&tmem_empty[b], 2 * 4 * kReaders);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc_all<true>(tmem_slot);
  tc_before();
  __syncthreads();
  cluster_sync_all();
  tc_after();
  // (the ordering kernel's list, and for the first product its rows, come from launches ahead; for the second the list is older
  // than the launch ahead, which began only when it was complete)
  if constexpr (FIRST) {
    pdl_wait();
  }
  pdl_launch_dependents();
  Work work0;
  work0.n_channel_tiles = a.n_channel_tiles;
  work0.t = static_cast<int>(blockIdx.x) / 2;
  work0.step = static_cast<int>(gridDim.x) / 2;
  work0.total = *a.n_tiles * a.n_channel_tiles;
  work0.tiles = a.tiles;
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t full_ab_lead = map_shared(smem_u32(full_ab), 0), tmem_empty_lead = map_shared(smem_u32(tmem_empty), 0);

  // The weights of the rows that a warp is going to write, of two pieces of 16 rows to a register: eight pieces at most of a tile that
  // it writes alone, else four.  Asked for ahead of the wait for the products.  (A load to a piece took 2048 tokens through 8 of 64
  // experts 2 us longer.)
  constexpr bool kWeighted = !FIRST && !CHANNEL;
  const auto weights_of = [&](const MoeTile& tile, int part, int parts, auto& w) {
    if constexpr (kWeighted) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof w / 4); ++i) {
        const int m = 16 * (part + parts * (2 * i + (lane >> 4))) + (lane & 15);
        w[i] = m < tile.rows ? a.gates[tile.row0 + m] : 0.0f;
      }
    }
  };
  static_assert(kHalf <= 8 * 16 && kMoeTileRows <= 4 * 16 * kReaders, "rows of a warp");
  // The scale of a lane's channel.
  const auto scale_of = [&](const MoeTile& tile, int n0) {
    const int n = n0 + static_cast<int>(rank) * kChannels + (warp & 3) * 32 + lane;
    return CHANNEL && n < a.n ? __half2float(a.scale[tile.expert * a.expert_scales + n]) : 0.0f;
  };
  const auto drain = [&](const MoeTile& tile, int n0, int part, const Turns& turn, auto& weights, float scale) {
    const int parts = turn.all ? kReaders : 1;
    const int quad = warp & 3;
    const uint32_t base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(turn.at * kHalf);
    const int n = n0 + static_cast<int>(rank) * kChannels + quad * 32;  // the warp's first channel
    const bool has_n = n < a.n;                                         // (a.n is a multiple of 32)
    const int pieces = (tile.rows + 15) >> 4;
    [[maybe_unused]] int from = 0;  // the lane with the weight of the piece's first row
    for (int pc = part; pc < pieces; pc += parts) {
      uint32_t r[16];
      tmem_ld16(base + static_cast<uint32_t>(16 * pc), r);
      tmem_ld_wait();
      if constexpr (CHANNEL) {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * scale);
      }
      if constexpr (FIRST) {
        const bool odd = (lane & 1) != 0;
        uint32_t x[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          float v[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int j = 2 * p + i;
            const float got = __uint_as_float(__shfl_xor_sync(0xffffffffu, odd ? r[j] : r[8 + j], 1));
            const float gate = odd ? got : __uint_as_float(r[j]), up = odd ? __uint_as_float(r[8 + j]) : got;
            v[i] = moe_gated(gate, up, a.activation);
          }
          const __half2 h = __floats2half2_rn(v[0], v[1]);
          x[p] = *reinterpret_cast<const uint32_t*>(&h);
        }
        const int q = (lane >> 1) & 3;
        turn_pairs<2>(x[0], x[1], x[2], x[3], q);
        const int m = 16 * pc + (odd ? 8 : 0) + 2 * q;
        __half* to = static_cast<__half*>(a.out) + static_cast<int64_t>(tile.row0 + m) * (a.n >> 1) + (n >> 1) + (lane >> 3) * 4;
        store_pair(to, a.n >> 1, has_n && m < tile.rows, has_n && m + 1 < tile.rows, x[0], x[1], x[2], x[3]);
      } else if constexpr (CHANNEL) {
        // (a warp's 32 channels of a row are 128 bytes)
        float* const to = static_cast<float*>(a.out) + static_cast<int64_t>(tile.row0 + 16 * pc) * a.n + n + lane;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (has_n && 16 * pc + j < tile.rows) to[j * static_cast<int64_t>(a.n)] = __uint_as_float(r[j]);
      } else {
        uint32_t x[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const float w0 = __shfl_sync(0xffffffffu, weights[0], from + 2 * p), w1 = __shfl_sync(0xffffffffu, weights[0], from + 2 * p + 1);
          const __half2 h = __floats2half2_rn(__uint_as_float(r[2 * p]) * w0, __uint_as_float(r[2 * p + 1]) * w1);
          x[p] = *reinterpret_cast<const uint32_t*>(&h);
        }
        const int q = lane & 3;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          turn_pairs<1>(x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3], q);
          const int m = 16 * pc + 8 * h + 2 * q;
          __half* to = static_cast<__half*>(a.out) + static_cast<int64_t>(tile.row0 + m) * a.n + n + (lane >> 2) * 4;
          store_pair(to, a.n, has_n && m < tile.rows, has_n && m + 1 < tile.rows, x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]);
        }
        from ^= 16;
        if (from == 0) {
#pragma unroll
          for (int i = 0; i + 1 < static_cast<int>(sizeof weights / 4); ++i) weights[i] = weights[i + 1];
        }
      }
    }
    tc_before();
    __syncwarp();
    if (lane == 0) {
      arrive_in_pair(tmem_empty_lead + turn.at * 8, kReaders / parts);
      if (turn.large) arrive_in_pair(tmem_empty_lead + 8, kReaders / parts);
    }
  };

  if (warp == 0 || warp == 23) {
    // ------------------------------------------------------------------ rows
    if (lane == 0) prefetch_tmap(&tmap_x);
    if constexpr (!FIRST) pdl_wait();
    const int mine = warp == 0 ? 0 : 1;  // every other stage
    int before = 0;                      // stages before the tile
    bool ok = true;
    Work work = work0;
    MoeTile tile;
    int n0;
    while (ok && work.next(tile, n0)) {
      const int cols = columns_of(tile), row = tile.row0 + static_cast<int>(rank) * (cols >> 1);
      for (int kb = (mine ^ before) & 1; kb < a.k_blocks; kb += 2) {
        const int iter = before + kb, stage = iter % kStages;
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], (static_cast<uint32_t>(iter / kStages) & 1u) ^ 1u))) {
          if (lane == 0) atomicExch(a.error, kErrMoeBase + 1);
          ok = false;
          break;
        }
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&full_ab[stage], static_cast<uint32_t>(cols) * (2 * kKBytes));
          uint8_t* const to = sX + stage * kXBytes;
          for (int i = 0; i < cols >> 6; ++i) {
            tma_load_2d_pair(to + i * kBoxBytes, &tmap_x, full_ab_lead + stage * 8, kb * kInputs, row + i * kBoxRows);
            tma_load_2d_pair(to + kAtom + i * kBoxBytes, &tmap_x, full_ab_lead + stage * 8, kb * kInputs + 64, row + i * kBoxRows);
          }
        }
        __syncwarp();
      }
      before += a.k_blocks;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------- MMAs
    if (rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      Work work = work0;
      MoeTile tile;
      int n0;
      for (Turns turn; ok && work.next(tile, n0); turn.next()) {
        turn.take(tile, work.done());
        const uint32_t idesc = 1u << 4 | static_cast<uint32_t>(columns_of(tile) >> 3) << 17 | 16u << 24;
        const uint32_t d = tmem_base + static_cast<uint32_t>(turn.at * kHalf);
        bool free = mbar_wait(&tmem_empty[turn.at], turn.uses_of(turn.at) ^ 1u);
        if (turn.large) free = mbar_wait(&tmem_empty[1], turn.uses_of(1) ^ 1u) && free;
        if (!__all_sync(0xffffffffu, free)) {
          if (lane == 0) atomicExch(a.error, kErrMoeBase + 2);
          break;
        }
        tc_after();
        for (int kb = 0; kb < a.k_blocks; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&full_ab[stage], phase))) {
            if (lane == 0) atomicExch(a.error, kErrMoeBase + 3);
            ok = false;
            break;
          }
          tc_after();
          const uint64_t db = make_desc(smem_u32(sX + stage * kXBytes));
          const uint32_t ta = tmem_base + kColumns + static_cast<uint32_t>(stage * (kInputs / 2));
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kInputs / 16; ++i)
              umma_ts<true, false>(d, ta + 8u * i, db + static_cast<uint64_t>(((i >> 2) * kAtom + (i & 3) * 32) >> 4), idesc,
                                   (kb > 0 || i > 0) ? 1u : 0u);
            commit<true>(&empty[stage]);
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok && elect_one()) commit<true>(&tmem_full[turn.full()]);
        __syncwarp();
      }
    }
  } else if (warp < 6) {
    // ---------------------------------------------------------------- results
    if constexpr (!FIRST) pdl_wait();  // (what is written here may still be read by launches ahead of the one ahead)
    Work work = work0;
    MoeTile tile;
    int n0;
    for (Turns turn; work.next(tile, n0); turn.next()) {
      turn.take(tile, work.done());
      float weights[4];
      weights_of(tile, 0, turn.all ? kReaders : 1, weights);
      const float scale = scale_of(tile, n0);
      if (!mbar_wait(&tmem_full[turn.full()], turn.full_phase())) {
        atomicExch(a.error, kErrMoeBase + 4);
        break;
      }
      tc_after();
      drain(tile, n0, 0, turn, weights, scale);
    }
  } else if (warp == 22) {
    // --------------------------------------------------------- packed weights
    if (lane == 0) prefetch_tmap(&tmap_w);
    int ws = 0;
    uint32_t phase = 0;
    bool ok = true;
    Work work = work0;
    MoeTile tile;
    int n0;
    while (ok && work.next(tile, n0)) {
      const int column = (n0 + static_cast<int>(rank) * kChannels) / 4 * kBlk / 4;  // in 32-bit elements
      const int row = tile.expert * (a.k >> 2);
      for (int kb = 0; kb < a.k_blocks; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait(&w_empty[ws], phase ^ 1))) {
          if (lane == 0) atomicExch(a.error, kErrMoeBase + 5);
          ok = false;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(&full_w[ws], kWBytes);
          tma_load_2d(sW + ws * kWBytes, &tmap_w, &full_w[ws], column, row + kb * kSlices);
        }
        __syncwarp();
        if (++ws == kWStages) {
          ws = 0;
          phase ^= 1;
        }
      }
    }
  } else {
    // -------------------------------------------------------- dequantisation
    const int group = (warp - 6) >> 2;  // this group of four warps takes every fourth stage
    const int quad = warp & 3;
    const int row = quad * 32 + lane;   // output channel of the CTA's 128 = tensor-memory lane
    const int col4 = row & 3;
    const uint32_t turn6 = (6u - 4u * static_cast<uint32_t>(col4)) & 31u;
    const uint32_t sel8 = static_cast<uint32_t>(col4) | static_cast<uint32_t>(4 + col4) << 8;
    const __half2 offset = __float2half2_rn(BITS == 4 ? 1032.0f : 1152.0f);
    bool ok = true;
    int before = 0;  // stages before the tile
    if constexpr (!FIRST) pdl_wait();  // (it writes results, too)
    Work work = work0;
    MoeTile tile;
    int n0;
    for (Turns turn; ok && work.next(tile, n0); turn.next()) {
      turn.take(tile, work.done());
      const int n = n0 + static_cast<int>(rank) * kChannels + row;
      const bool has_n = n < a.n;
      const __half* const scales = a.scale + tile.expert * a.expert_scales + n;
      // the scale of 32 inputs, asked for four stages ahead (by hand, so that nothing looks at it before)
      const auto ask = [&](unsigned short& v, int slice) {
        const int g = min(slice >> a.group_shift, a.groups - 1);
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p ld.global.nc.u16 %0, [%1];\n\t}"
                     : "+h"(v)
                     : "l"(scales + static_cast<int64_t>(g) * a.n), "r"(has_n ? 1u : 0u));
      };
      int kb = (group - before) & 3;
      unsigned short next[4] = {0, 0, 0, 0};
      if (!CHANNEL && kb < a.k_blocks) {
#pragma unroll
        for (int i = 0; i < 4; ++i) ask(next[i], kb * kSlices + 8 * i);
      }
      for (; kb < a.k_blocks; kb += 4) {
        const int iter = before + kb, stage = iter & (kStages - 1), ws = iter & (kWStages - 1);
        unsigned short cur[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) cur[i] = next[i];
        if (!CHANNEL && kb + 4 < a.k_blocks) {
#pragma unroll
          for (int i = 0; i < 4; ++i) ask(next[i], (kb + 4) * kSlices + 8 * i);
        }
        if (!mbar_wait(&full_w[ws], static_cast<uint32_t>(iter / kWStages) & 1u)) {
          atomicExch(a.error, kErrMoeBase + 6);
          ok = false;
          break;
        }
        const uint8_t* wp = sW + ws * kWBytes + (row >> 2) * kBlk;
        const uint32_t columns = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + kColumns + static_cast<uint32_t>(stage * (kInputs / 2));
        using Block = typename std::conditional<BITS == 4, uint2, uint4>::type;
#pragma unroll
        for (int sixty_four = 0; sixty_four < 2; ++sixty_four) {
          uint32_t o[32];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            Block blk[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) blk[i] = *reinterpret_cast<const Block*>(wp + (16 * sixty_four + 8 * half + i) * kPitch);
            const __half s = __ushort_as_half(cur[2 * sixty_four + half]);
            const __half2 s2 = __half2half2(s);
            if constexpr (CHANNEL) {
              const auto exact = [&](uint32_t codes) {  // (1024 + u less 1024 and the zero)
                const uint32_t biased = codes | 0x64006400u;
                const __half2 w = __hsub2(*reinterpret_cast<const __half2*>(&biased), offset);
                return *reinterpret_cast<const uint32_t*>(&w);
              };
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if constexpr (BITS == 4) {
                  o[16 * half + 2 * i] = exact((blk[i].x >> (4 * col4)) & 0x000F000Fu);
                  o[16 * half + 2 * i + 1] = exact((blk[i].y >> (4 * col4)) & 0x000F000Fu);
                } else {
                  o[16 * half + 2 * i] = exact(__byte_perm(blk[i].x, blk[i].y, sel8) & 0x00FF00FFu);
                  o[16 * half + 2 * i + 1] = exact(__byte_perm(blk[i].z, blk[i].w, sel8) & 0x00FF00FFu);
                }
              }
            } else if constexpr (BITS == 4) {
              // A nibble at bits 6..9 is the subnormal half u 2^-18: u 2^-18 (2^18 s) - 8 s is (u - 8) s rounded once, in one
              // instruction.  2^18 s has to be a half; else from 1024 + u, the zero off exactly first.
              if (__all_sync(0xffffffffu, __habs(s) < __float2half_rn(0.249f))) {
                const __half2 up = __hmul2(s2, __float2half2_rn(512.0f)), large = __hmul2(up, __float2half2_rn(512.0f));
                const __half2 zero = __hmul2(s2, __float2half2_rn(-8.0f));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const uint32_t lo = __funnelshift_l(blk[i].x, blk[i].x, turn6) & 0x03C003C0u;
                  const uint32_t hi = __funnelshift_l(blk[i].y, blk[i].y, turn6) & 0x03C003C0u;
                  const __half2 r0 = __hfma2(*reinterpret_cast<const __half2*>(&lo), large, zero);
                  const __half2 r1 = __hfma2(*reinterpret_cast<const __half2*>(&hi), large, zero);
                  o[16 * half + 2 * i] = *reinterpret_cast<const uint32_t*>(&r0);
                  o[16 * half + 2 * i + 1] = *reinterpret_cast<const uint32_t*>(&r1);
                }
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  o[16 * half + 2 * i] = dq_once(((blk[i].x >> (4 * col4)) & 0x000F000Fu) | 0x64006400u, offset, s2);
                  o[16 * half + 2 * i + 1] = dq_once(((blk[i].y >> (4 * col4)) & 0x000F000Fu) | 0x64006400u, offset, s2);
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                o[16 * half + 2 * i] = dq_once((__byte_perm(blk[i].x, blk[i].y, sel8) & 0x00FF00FFu) | 0x64006400u, offset, s2);
                o[16 * half + 2 * i + 1] = dq_once((__byte_perm(blk[i].z, blk[i].w, sel8) & 0x00FF00FFu) | 0x64006400u, offset, s2);
              }
            }
          }
          if (sixty_four == 1) {
            fence_proxy_async();  // (what has been asked for is here before a copy may overwrite it)
            __syncwarp();
            if (lane == 0) mbar_arrive(&w_empty[ws]);
          } else if (!mbar_wait(&empty[stage], (static_cast<uint32_t>(iter / kStages) & 1u) ^ 1u)) {
            // (the first weights are ready in registers when the stage's last MMAs are done with its columns)
            atomicExch(a.error, kErrMoeBase + 6);
            ok = false;
            break;
          } else {
            tc_after();
          }
          tmem_st32(columns + static_cast<uint32_t>(32 * sixty_four), o);
        }
        if (!ok) break;
        tmem_st_wait();
        tc_before();
        __syncwarp();
        if (lane == 0) arrive_in_pair(full_ab_lead + stage * 8);
      }
      before += a.k_blocks;
      if (!ok) break;
      if (!turn.all) continue;
      float weights[2];
      weights_of(tile, 1 + group, kReaders, weights);
      const float scale = scale_of(tile, n0);
      if (!mbar_wait(&tmem_full[2], turn.full_phase())) {
        atomicExch(a.error, kErrMoeBase + 7);
        break;
      }
      tc_after();
      drain(tile, n0, 1 + group, turn, weights, scale);
    }
  }
  // Nobody leaves while the partner may still arrive on this CTA's barriers or the pair's MMAs write its tensor memory.
  tc_before();
  __syncthreads();
  cluster_sync_all();
  if (*reinterpret_cast<volatile int*>(a.error) != 0) {
    // a wait ran out somewhere: copies may still be in flight towards this CTA's shared memory
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  if (warp == 1) {
    tc_after();
    tmem_dealloc_all<true>(tmem_base);
  }
}

template <int BITS, bool CHANNEL, bool FIRST>
int launch_of(const CUtensorMap& tx, const CUtensorMap& tw, const GemmArgs& a, int grid, cudaStream_t stream) {
  constexpr size_t smem = 1024 + kStages * 2 * kAtom + kWStages * kSlices * (kChannels / 4) * (BITS == 4 ? 8 : 16) +
                          (2 * kWStages + 2 * kStages + 5) * 8 + 64;
  static_assert(smem <= 227 * 1024, "shared memory");
  auto kern = moe_gemm_kernel<BITS, CHANNEL, FIRST>;
  static bool done[kMaxDevices];
  int dev;
  if (needs_configure(done, &dev)) {
    MLD_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    if (dev >= 0) done[dev] = true;
  }
  MLD_CUDA_CHECK(launch_overlapped(kern, dim3(grid), dim3(kThreads), smem, stream, tx, tw, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

}  // namespace

int launch_moe_gemm(bool first, const MoeShape& s, const MoeBuffers& b, const void* weights, const void* scale, int pairs, int sms,
                    cudaStream_t stream) {
  const int n = first ? 2 * s.ffn : s.d_model, k = first ? s.d_model : s.ffn, blk = s.bits == 4 ? 8 : 16;
  CUtensorMap tx, tw;
  int rc = make_tmap_2d(&tx, first ? b.sorted : b.hidden, static_cast<uint64_t>(k) * 2, pairs, static_cast<uint64_t>(k) * 2, kKBytes,
                        kBoxRows, 2, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, true);
  if (rc != MLD_OK) return rc;
  rc = make_tmap_2d(&tw, weights, static_cast<uint64_t>(n / 4) * blk, static_cast<uint64_t>(s.experts) * (k / 4),
                    static_cast<uint64_t>(n / 4) * blk, kChannels / 4 * blk, kSlices, 4, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc != MLD_OK) return rc;
  GemmArgs a = {};
  a.tiles = b.tiles;
  a.n_tiles = b.n_tiles;
  a.n_channel_tiles = div_up(n, 2 * kChannels);
  a.k_blocks = div_up(k, kInputs);
  a.n = n;
  a.k = k;
  a.scale = static_cast<const __half*>(scale);
  a.groups = s.block != 0 ? k / s.block : 1;
  a.group_shift = 30;
  if (s.block != 0)
    for (a.group_shift = 3; (4 << a.group_shift) < s.block;) ++a.group_shift;
  a.expert_scales = static_cast<int64_t>(a.groups) * n;
  a.out = first ? b.hidden : b.part;
  a.gates = b.gates;
  a.activation = s.activation;
  a.error = b.error;
  const int grid = sms / 2 * 2;
  const auto launch = s.bits == 4 ? (s.block == 0 ? (first ? launch_of<4, true, true> : launch_of<4, true, false>)
                                                  : (first ? launch_of<4, false, true> : launch_of<4, false, false>))
                                  : (s.block == 0 ? (first ? launch_of<8, true, true> : launch_of<8, true, false>)
                                                  : (first ? launch_of<8, false, true> : launch_of<8, false, false>));
  return launch(tx, tw, a, grid, stream);
}

}  // namespace mld

// The experts' products for few rows: weights streamed once past tiles of up to eight rows.
//
// Bound by HBM: a weight is read once for all rows of a tile, and there are too few of those to fill the tensor cores.  An item is 64
// outputs of one tile over all inputs; a persistent block takes every grid-th item.
//   four warps   fetch: boxes of 128 inputs x 64 outputs, packed as they lie, and their scales, of the block's items, one after
//                another, into a ring of shared memory.  They wait for nothing but free places, so the next item's weights
//                are under way while this one's are multiplied.  (One warp, among those that multiply, took 400 cycles to a box:
//                33 tokens 110 us against 85.)  One of them also looks up where an item's rows are, two items ahead, and leaves
//                that for the others.  (Warps that looked for themselves spent half of the time on it; rows copied into the
//                ring, 256 bytes each, took the copying warp longer than the weights.)
//   then warps that take a box each in turn and multiply it: m16n8k16, the weights as A straight from the packed blocks (a lane's
//                4x4 block is its part of two fragments, if the rows of a fragment are outputs 4 g + c and the k of a lane are
//                the block's four inputs), the rows of x as B.  A weight enters as the subnormal half that its bits are, u 2^-24
//                (or u 2^-20 for every second nibble, which then need not be shifted): exact, and an instruction a pair.  The
//                zero, 8 or 128, comes off through the accumulator's start, - zero sum(x), for which a row of ones is
//                multiplied.  The sums of 32 inputs are scaled in 32 bits.  Lane t of four takes the input slices 2 t and 2 t + 1,
//                whose 16-byte pieces the copies' swizzle puts on different banks for the eight lanes that read together.
//   and four warps that add up the warps' parts of an item, in the order of the inputs, and write act(gate) * up or the expert's
//                output.
// Columns behind a tile's rows hold whatever was there: no column sees another, and they are not written.
// Each side waits for the other through barriers in shared memory, every wait bounded.  Parts have two places per warp, so that
// multiplying goes on meanwhile.
#include <cuda_fp16.h>

#include <cstring>

#include "common.cuh"
#include "few_ring.h"
#include "moe.cuh"

namespace mld {
namespace {

constexpr int kOutputs = kFewOutputs, kRows = kFewRows, kInputs = kFewInputs, kCopyWarps = kFewCopyWarps, kSumWarps = kFewSumWarps;
constexpr int kItemBars = kFewItemBars, kBoxBytes = kFewBoxBytes;
constexpr int kErrFewBase = 90;
static_assert(kRows == kMoeFewRows, "rows of a tile");
template <int BITS>
using Shape = FewShape<BITS>;

struct FewArgs {
  MoeBuffers b;
  const int32_t* ids;      // one token: its experts, no order was made
  const __half* x;         // the first product: rows by token
  int64_t x_stride;
  int experts, top_k, n, k, n_items;  // n_items: items of a tile
  int groups;              // scales of an output
  int scale_rows;          // rows of scales of a box
  int scale_shift;         // log2 of the inputs of a scale (0 inputs: 30)
  int activation;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b, const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Bounded wait that leaves the warp asleep between looks: sixteen warps that poll take the issue slots of those that work.
__device__ __forceinline__ bool wait_asleep(uint64_t* bar, uint32_t parity) {
  unsigned long long t0 = 0;
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)  // (nanoseconds)
        : "memory");
    if (done != 0) return true;
    if (t0 == 0)
      t0 = globaltimer_ns();
    else if (globaltimer_ns() - t0 > kWaitLimitNs)
      return false;
  }
}

// A block's items in order: every grid-th of (tile, 64 outputs).
struct Items {
  int tile, part, tiles, parts, tile_step, part_step;
  __device__ __forceinline__ Items(int count, int n_items) : tiles(count), parts(n_items) {
    tile = static_cast<int>(blockIdx.x) / parts;
    part = static_cast<int>(blockIdx.x) - tile * parts;
    tile_step = static_cast<int>(gridDim.x) / parts;
    part_step = static_cast<int>(gridDim.x) - tile_step * parts;
  }
  __device__ __forceinline__ bool there() const { return tile < tiles; }
  __device__ __forceinline__ void next() {
    tile += tile_step;
    part += part_step;
    if (part >= parts) {
      part -= parts;
      ++tile;
    }
  }
};
// A tile of the ordering kernel's list, or one of one token's experts (without rows where the id is none).
__device__ __forceinline__ MoeTile tile_of(const FewArgs& a, int i) {
  if (a.ids != nullptr) {
    const int e = a.ids[i];
    return static_cast<unsigned>(e) < static_cast<unsigned>(a.experts) ? MoeTile{e, i, 1, 0} : MoeTile{0, i, 0, 0};
  }
  const int4 v = *reinterpret_cast<const int4*>(a.b.tiles + i);
  return {v.x, v.y, v.z, 0};
}

// FIRST: x -> hidden, else hidden -> part.
template <int BITS, bool FIRST>
__global__ void __launch_bounds__(Shape<BITS>::kThreads, 1)
    moe_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_s, FewArgs a) {
  using S = Shape<BITS>;
  constexpr int kWarps = S::kWarps, kStages = S::kStages, kPlaces = S::kPlaces, kPart = S::kPart;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const scale_ring = ring + kStages * S::kWBytes;
  float2* const parts = reinterpret_cast<float2*>(scale_ring + kStages * S::kScaleBytes);  // [warp][place][kPart]
  const uint4** const rows = reinterpret_cast<const uint4**>(parts + kWarps * kPlaces * kPart);  // [item % kItemBars][kRows]
  uint64_t* const full = reinterpret_cast<uint64_t*>(rows + kItemBars * kRows);
  uint64_t* const empty = full + kStages;
  uint64_t* const item_full = empty + kStages;          // [kItemBars]: all parts of an item are there
  uint64_t* const item_rows = item_full + kItemBars;    // [kItemBars]: it is known where an item's rows are
  uint64_t* const part_free = item_rows + kItemBars;    // [warp][place]: the part has been read

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int boxes = (a.k + kInputs - 1) / kInputs;      // of an item
  const int sharing = min(boxes, kWarps);               // warps that have a part of an item
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_s);
  }
  for (int i = threadIdx.x; i < kItemBars; i += S::kThreads) {  // (one thread alone would take a microsecond)
    mbar_init(&item_full[i], sharing);
    mbar_init(&item_rows[i], 1);
    if (i < kStages) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    if (i < kWarps * kPlaces) mbar_init(&part_free[i], kSumWarps);
    fence_barrier_init();
  }
  static_assert(kStages <= kItemBars && kWarps * kPlaces <= kItemBars, "barriers");
  __syncthreads();
  if constexpr (FIRST) pdl_wait();
  // (The second product's tiles, ids and weights were complete before the launch ahead let this one begin; its rows were not.)
  pdl_launch_dependents();
  const int count = a.ids != nullptr ? a.top_k : *a.b.n_tiles;
  Items items(count, a.n_items);

  if (warp < kCopyWarps) {
    // ------------------------------------------------------------------ copies
    // A warp takes every kCopyWarps-th box.  The first one's lane r looks row r of a tile up: two items ahead the tile is asked for,
    // one ahead its rows' tokens.
    const auto tile_at = [&](const Items& it) { return it.there() ? tile_of(a, it.tile) : MoeTile{0, 0, 0, 0}; };
    const auto token_of = [&](const MoeTile& t) {  // of lane r's row, as the number of its pair or position
      if (lane >= t.rows) return t.row0;
      if (!FIRST || a.ids != nullptr) return t.row0 + lane;
      return a.b.order[t.row0 + lane];
    };
    Items ahead = items;
    MoeTile tile = tile_at(ahead);
    int token = warp == 0 ? token_of(tile) : 0;
    ahead.next();
    MoeTile next_tile = tile_at(ahead);
    int s = warp, c0 = warp, nth = 0;  // the place and, in its item, the number of this warp's next box
    uint32_t phase = 0;
    bool ok = true;
    for (; ok && items.there(); items.next(), ++nth) {
      ahead.next();
      const MoeTile after = tile_at(ahead);
      int next_token = 0;
      if (warp == 0) {
        next_token = token_of(next_tile);
        // (places behind the tile's rows get one that exists; a slot's last readers are done with it, see kFewItemBars)
        if (lane < kRows) {
          const __half* p;
          if constexpr (FIRST)
            p = a.x + (a.ids != nullptr ? 0 : (lane < tile.rows ? token / a.top_k : 0) * a.x_stride);
          else
            p = static_cast<const __half*>(a.b.hidden) + static_cast<int64_t>(token) * a.k;
          rows[nth % kItemBars * kRows + lane] = reinterpret_cast<const uint4*>(p);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_rows[nth % kItemBars]);
      }
      const int n0 = items.part * kOutputs, row0 = tile.expert * (a.k >> 2), group0 = tile.expert * a.groups;
      for (; c0 < boxes; c0 += kCopyWarps) {
        if (!__all_sync(0xffffffffu, wait_asleep(&empty[s], phase ^ 1))) {
          if (lane == 0) atomicExch(a.b.error, kErrFewBase + 1);
          ok = false;
          break;
        }
        if (elect_one()) {
          uint8_t* const to = ring + s * S::kWBytes;
          mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>(S::kWBytes + a.scale_rows * kOutputs * 2));
          const int row = row0 + c0 * (kInputs / 4);
          if constexpr (BITS == 4) {
            tma_load_2d(to, &tmap_w, &full[s], n0 / 2, row);  // (in 32-bit elements)
          } else {
            tma_load_2d(to, &tmap_w, &full[s], n0, row);
            tma_load_2d(to + kBoxBytes, &tmap_w, &full[s], n0 + kOutputs / 2, row);
          }
          tma_load_2d(scale_ring + s * S::kScaleBytes, &tmap_s, &full[s], n0, group0 + min(c0 * kInputs >> a.scale_shift, a.groups - 1));
        }
        __syncwarp();
        s += kCopyWarps;
        if (s >= kStages) {
          s -= kStages;
          phase ^= 1;
        }
      }
      c0 -= boxes;
      tile = next_tile;
      token = next_token;
      next_tile = after;
    }
  } else if (warp < kCopyWarps + kWarps) {
    // ----------------------------------------------------------------- products
    const int me = warp - kCopyWarps, g = lane >> 2, t = lane & 3;
    int first = me;                  // this warp's first box of the item: every kWarps-th from there
    int s = me, nth = 0, mine = 0;   // the place of its next box, the item's number, parts handed over
    uint32_t phase = 0;
    bool ok = true;
    if constexpr (!FIRST) pdl_wait();
    for (; ok && items.there(); items.next(), ++nth) {
      if (first < boxes) {
        float acc[2][2][4];  // [block of the pair][outputs 0, 1 / 2, 3 of it]
#pragma unroll
        for (int i = 0; i < 16; ++i) (&acc[0][0][0])[i] = 0.0f;
        if (!wait_asleep(&item_rows[nth % kItemBars], static_cast<uint32_t>(nth / kItemBars) & 1u)) {
          atomicExch(a.b.error, kErrFewBase + 5);
          break;
        }
        int c = first;
        for (; c < boxes; c += kWarps) {
          if (!wait_asleep(&full[s], phase)) {
            atomicExch(a.b.error, kErrFewBase + 2);
            ok = false;
            break;
          }
          const uint8_t* const box = ring + s * S::kWBytes;
          const uint8_t* const scale_box = scale_ring + s * S::kScaleBytes + (BITS == 4 ? 16 : 8) * g;
          uint4 held[4];  // input slices 2 t (.x, .y) and 2 t + 1 of this lane's row, of the box's four groups of 32
          const uint4* const row = rows[nth % kItemBars * kRows + g] + c * (kInputs / 8) + t;
#pragma unroll
          for (int i = 0; i < 4; ++i) held[i] = c * kInputs + 32 * i < a.k ? row[4 * i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (c * kInputs + 32 * i >= a.k) break;  // (what lies behind the last input is another expert's)
            const uint2 x0 = make_uint2(held[i].x, held[i].y), x1 = make_uint2(held[i].z, held[i].w);
            uint4 w[2][BITS == 4 ? 1 : 2];
            uint4 scales;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int slice = 8 * i + 2 * t + h, at = slice * 128 + ((g ^ (2 * t + h)) << 4);  // (128-byte swizzle)
              w[h][0] = *reinterpret_cast<const uint4*>(box + at);
              if constexpr (BITS == 8) w[h][1] = *reinterpret_cast<const uint4*>(box + kBoxBytes + at);
            }
            const uint8_t* const sp = scale_box + (32 * i >> a.scale_shift) * (kOutputs * 2);
            if constexpr (BITS == 4) {
              scales = *reinterpret_cast<const uint4*>(sp);  // of output slices 2 g, 2 g + 1
            } else {
              const uint2 lo = *reinterpret_cast<const uint2*>(sp), hi = *reinterpret_cast<const uint2*>(sp + 64);  // g, g + 8
              scales = make_uint4(lo.x, lo.y, hi.x, hi.y);
            }
            const __half2* const s2 = reinterpret_cast<const __half2*>(&scales);
            constexpr uint32_t kOnes = 0x3C003C00u;
            constexpr float kZero = BITS == 4 ? -8.0f * 0x1p-24f : -128.0f * 0x1p-24f, kZeroOdd = BITS == 4 ? -8.0f * 0x1p-20f : kZero;
            float start[4];
            {
              const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              float half[4], sum[4];
              mma_f16(half, kOnes, kOnes, kOnes, kOnes, x0, none);
              mma_f16(sum, kOnes, kOnes, kOnes, kOnes, x1, half);
              start[0] = kZero * sum[0];
              start[1] = kZero * sum[1];
              start[2] = kZeroOdd * sum[0];
              start[3] = kZeroOdd * sum[1];
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                uint32_t m[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  if constexpr (BITS == 4) {
                    const uint32_t lo = (b == 0 ? w[h][0].x : w[h][0].z) >> (8 * r), hi = (b == 0 ? w[h][0].y : w[h][0].w) >> (8 * r);
                    m[h][0] = lo & 0x000F000Fu;
                    m[h][1] = lo & 0x00F000F0u;  // (16 times as large)
                    m[h][2] = hi & 0x000F000Fu;
                    m[h][3] = hi & 0x00F000F0u;
                  } else {
                    // a word per input channel, a byte per output
                    const uint4 v = w[h][BITS == 8 ? b : 0];
                    m[h][0] = __byte_perm(v.x, v.y, 0x0400u + (2 * r) * 0x0101u) & 0x00FF00FFu;
                    m[h][1] = __byte_perm(v.x, v.y, 0x0400u + (2 * r + 1) * 0x0101u) & 0x00FF00FFu;
                    m[h][2] = __byte_perm(v.z, v.w, 0x0400u + (2 * r) * 0x0101u) & 0x00FF00FFu;
                    m[h][3] = __byte_perm(v.z, v.w, 0x0400u + (2 * r + 1) * 0x0101u) & 0x00FF00FFu;
                  }
                }
                const float2 sc = __half22float2(s2[2 * b + r]);
                float half[4], sum[4];
                mma_f16(half, m[0][0], m[0][1], m[0][2], m[0][3], x0, start);
                mma_f16(sum, m[1][0], m[1][1], m[1][2], m[1][3], x1, half);
                acc[b][r][0] += sum[0] * sc.x;
                acc[b][r][1] += sum[1] * sc.x;
                acc[b][r][2] += sum[2] * sc.y;
                acc[b][r][3] += sum[3] * sc.y;
              }
          }
          fence_proxy_async();  // (what has been asked for is here before a copy may overwrite it)
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[s]);
          s += kWarps;
          if (s >= kStages) {
            s -= kStages;
            phase ^= 1;
          }
        }
        if (!ok) break;
        first = c;
        // the part: pairs of neighbouring outputs, for the lane's two rows
        const int place = mine % kPlaces;
        if (!wait_asleep(&part_free[me * kPlaces + place], (static_cast<uint32_t>(mine / kPlaces) & 1u) ^ 1u)) {
          atomicExch(a.b.error, kErrFewBase + 3);
          ok = false;
          break;
        }
        float2* const to = parts + (me * kPlaces + place) * kPart + lane;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) to[((b * 2 + r) * 2 + e) * 32] = make_float2(acc[b][r][e], acc[b][r][2 + e]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_full[nth % kItemBars]);
        ++mine;
      }
      first -= boxes;
    }
  } else {
    // --------------------------------------------------------------------- sums
    constexpr int kShare = kPart / (32 * kSumWarps);  // float2s of a thread
    const int me = threadIdx.x - 32 * (kCopyWarps + kWarps);
    int w0 = 0, nth = 0;  // the warp that has the item's first box, the item's number
    uint32_t odd = 0;     // which place a warp's next part is in, a bit each
    MoeTile tile = items.there() ? tile_of(a, items.tile) : MoeTile{0, 0, 0, 0};
    if constexpr (!FIRST) pdl_wait();  // (what is written here may still be read by launches ahead of the one ahead)
    while (items.there()) {
      const int n0 = items.part * kOutputs;
      items.next();
      const MoeTile next_tile = items.there() ? tile_of(a, items.tile) : MoeTile{0, 0, 0, 0};
      if (!wait_asleep(&item_full[nth % kItemBars], static_cast<uint32_t>(nth / kItemBars) & 1u)) {
        atomicExch(a.b.error, kErrFewBase + 4);
        break;
      }
      float2 v[kShare];
#pragma unroll
      for (int i = 0; i < kShare; ++i) v[i] = make_float2(0.0f, 0.0f);
      uint32_t turned = 0;
#pragma unroll
      for (int p = 0; p < kWarps; ++p) {
        const int w = (w0 + p) % kWarps;
        if (p < sharing) {
          const float2* const from = parts + (w * kPlaces + (odd >> w) % kPlaces) * kPart + me;
          turned |= 1u << w;
#pragma unroll
          for (int i = 0; i < kShare; ++i) {
            const float2 f = from[i * 32 * kSumWarps];
            v[i].x += f.x;
            v[i].y += f.y;
          }
        }
      }
      __syncwarp();
      if ((turned >> lane & 1u) != 0) mbar_arrive(&part_free[lane * kPlaces + (odd >> lane) % kPlaces]);
      odd ^= turned;
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        // float2 number `at` of a part: [block][outputs][row of two][lane]
        const int at = me + 32 * kSumWarps * i, l = at & 31, e = at >> 5 & 1, r = at >> 6 & 1, b = at >> 7;
        const int n = n0 + (BITS == 4 ? 8 * (l >> 2) + 4 * b : 4 * (l >> 2) + 32 * b) + 2 * r, col = 2 * (l & 3) + e;
        if (col >= tile.rows || n >= a.n) continue;
        const float x = v[i].x * 0x1p24f, y = v[i].y * (BITS == 4 ? 0x1p20f : 0x1p24f);
        const int64_t pos = tile.row0 + col;
        if constexpr (FIRST)
          static_cast<__half*>(a.b.hidden)[pos * (a.n >> 1) + (n >> 1)] = __float2half_rn(moe_gated(x, y, a.activation));
        else
          *reinterpret_cast<float2*>(static_cast<float*>(a.b.part) + pos * a.n + n) = make_float2(x, y);
      }
      w0 = (w0 + boxes) % kWarps;
      ++nth;
      tile = next_tile;
    }
  }
  if constexpr (!FIRST) pdl_wait();  // (a block without items waits, too: whoever comes next relies on the launch ahead being done)
  __syncthreads();
  if (*reinterpret_cast<volatile int*>(a.b.error) != 0) {
    // a wait ran out somewhere: copies may still be in flight towards this block's shared memory
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
}

template <int BITS, bool FIRST>
int launch_of(const CUtensorMap& tw, const CUtensorMap& ts, const FewArgs& a, int grid, cudaStream_t stream) {
  using S = Shape<BITS>;
  auto kern = moe_few_kernel<BITS, FIRST>;
  static bool done[kMaxDevices];
  int dev;
  if (needs_configure(done, &dev)) {
    MLD_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem)));
    if (dev >= 0) done[dev] = true;
  }
  MLD_CUDA_CHECK(launch_overlapped(kern, dim3(grid), dim3(S::kThreads), S::kSmem, stream, tw, ts, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

}  // namespace

int launch_moe_few(bool first, const MoeShape& s, const MoeBuffers& b, const int32_t* ids, const void* x, int64_t x_stride,
                   const void* weights, const void* scale, int tiles, int sms, cudaStream_t stream) {
  const int n = first ? 2 * s.ffn : s.d_model, k = first ? s.d_model : s.ffn, blk = s.bits == 4 ? 8 : 16;
  FewArgs a = {};
  a.b = b;
  a.ids = ids;
  a.x = static_cast<const __half*>(x);
  a.x_stride = x_stride;
  a.experts = s.experts;
  a.top_k = s.top_k;
  a.n = n;
  a.k = k;
  a.n_items = div_up(n, kOutputs);
  a.groups = s.block != 0 ? k / s.block : 1;
  a.scale_rows = s.block != 0 && s.block < kInputs ? kInputs / s.block : 1;
  a.scale_shift = 30;
  if (s.block != 0)
    for (a.scale_shift = 5; (1 << a.scale_shift) < s.block;) ++a.scale_shift;
  a.activation = s.activation;
  CUtensorMap tw, ts;
  int rc = make_tmap_2d(&tw, weights, static_cast<uint64_t>(n / 4) * blk, static_cast<uint64_t>(s.experts) * (k / 4),
                        static_cast<uint64_t>(n / 4) * blk, 128, kInputs / 4, 4, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != MLD_OK) return rc;
  rc = make_tmap_2d(&ts, scale, static_cast<uint64_t>(n) * 2, static_cast<uint64_t>(s.experts) * a.groups, static_cast<uint64_t>(n) * 2,
                    kOutputs * 2, a.scale_rows, 2, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc != MLD_OK) return rc;
  const int64_t items = static_cast<int64_t>(tiles) * a.n_items;
  const int grid = items < sms ? static_cast<int>(items) : sms;
  if (s.bits == 4) return first ? launch_of<4, true>(tw, ts, a, grid, stream) : launch_of<4, false>(tw, ts, a, grid, stream);
  return first ? launch_of<8, true>(tw, ts, a, grid, stream) : launch_of<8, false>(tw, ts, a, grid, stream);
}

}  // namespace mld

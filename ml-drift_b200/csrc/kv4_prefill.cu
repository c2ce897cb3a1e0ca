// Attention over the 4-bit cache for many query rows per key/value head (prompts, chunks of prompts), on tcgen05.
//
// The rows of a block are the queries of 256 / group tokens for all heads that share a key/value head: two tiles of 128 rows (one
// for heads of 256 values).  A block walks the cached tokens in steps of 64:
//   S = Q K^T        both operands fp16 from shared memory, 128 x 64 fp32 in tensor memory, two of them per tile
//   P = 2^(S - ref)  a thread per row; written over S as fp16, where the next product takes it from
//   O += P V         V from shared memory, 128 x D fp32 in tensor memory
// The next step's S is asked for ahead of this step's O, so that the threads that make P find it ready: steps of 128 tokens, of
// which tensor memory holds one S per tile beside O, had every thread wait for its own products (ragged chunks 938 us against
// 902, whole blocks).  A step of a pair of tiles takes about 2200 cycles where its products take 1024.  No one pipe is full (tensor 29 %,
// exponentials 31 %, 1.7 of 4 issue slots), and forms of an earlier stage without the exponentials, the maxima or the unpacking took
// as long as the whole.  A score product of 128 x 64 x 16 reads 6 KB of shared memory, 48 cycles at 128 bytes, for 32 of tensor work:
// the likeliest bound, beside the chain from scores to weights.
// Blocks of long sequences are cut along the tokens where that fills the SMs (kv4_prefill_pieces_kernel): a piece leaves its sums
// and their reference in the plan's workspace, and the last one of a block joins them in the pieces' order.  Whole / cut, us, 8
// heads of 128: 2048 rows, 16384 tokens 303 / 187; 4 times that 583 / 454; 256 rows, 65536 tokens 1210 / 126.
// Measured (32 heads of 128 over 8): 588 TFLOP/s for a prompt of 2048 tokens, 802 for ragged chunks behind up to 16384; a prompt of
// 2048 with heads of 64 45 us, with heads of 256 136, 386 and 504 TFLOP/s.
// The cache's values are fp16 numbers exactly, so unpacking rounds nothing; V's rows lie with the head's values contiguous, as the
// cache has them (the product takes them transposed), four of eight neighbours interleaved, which the output undoes for nothing.
// ref is a row's running maximum, which moves only when a step exceeds it by 2^5: then the row's sums in tensor memory are scaled
// by its thread itself, after the last product.  Weights are 2^10 at ref, so that fp16 holds 2^-24 of it as a normal number.
//
// Roles of the twenty warps: 0-7 make P and write the rows out (a warpgroup to a tile), 8-15 unpack, 16 asks for packed tiles, 17
// and 18 issue the products, a tile each (one warp for both took as long to issue as the products take).
#include <cuda_fp16.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "kv4_attn.cuh"
#include "pair_common.cuh"

namespace mld {
namespace {

constexpr int kPrefillThreads = 20 * 32;
constexpr int kRowWarps = 8, kUnpackWarps = 8, kLoadWarp = 16, kMmaWarp = 17;  // and the one behind it for a second tile
// Registers a thread: 640 x 96 at launch, dealt out anew as 256 x 136 + 256 x 72 + 128 x 64.
constexpr int kRegsRows = 136, kRegsUnpack = 72, kRegsRest = 64;
constexpr int kRowsPerTile = 128;
constexpr float kPrefillHeadroom = 5.0f, kPrefillLift = 10.0f, kPrefillFloor = -1e30f;
// What a block of rows takes beside its steps, a piece of one that is cut, and joining one piece to others, in steps; chosen by
// sweeps over 9, 14, 20 and 28 for a piece (8 heads of 128: 2048 rows, 16384 tokens 227 / 187 / 187 / 225 us; 4 times that 453 / 454 /
// 474 / 584; 1024 rows, 32768 tokens 202 / 197 / 233 / 266).
constexpr float kBlockCost = 4.0f, kCutCost = 14.0f, kJoinCost = 1.5f;
constexpr int kMaskedBlocks = 24;  // blocks of tokens that only some rows of a block of rows see, at most

template <int D>
struct Prefill {
  static constexpr int kTilesM = D == 256 ? 1 : 2;
  static constexpr int kRows = kTilesM * kRowsPerTile;
  static constexpr int kN = 64;                              // tokens of a step
  static constexpr int kQBytes = kRowsPerTile * D * 2;       // of a tile
  static constexpr int kKvBytes = kN * D * 2;                // of K or V of a step
  static constexpr int kBuffers = D == 256 ? 2 : 4;          // of K and of V
  static constexpr int kTileBytes = kv4::tile_bytes(D);
  static constexpr int kPackTiles = kN / 16;                 // packed tiles of a step
  static constexpr int kPackBytes = kPackTiles * kTileBytes;
  static constexpr int kRing = D == 256 ? 1 : 3;             // steps that are in flight packed
  static constexpr int kO = 256;                             // tensor-memory column of the first O
  static constexpr size_t kSmem = 1024 + kTilesM * kQBytes + 2 * kBuffers * kKvBytes + kRing * kPackBytes + kMaskedBlocks * kN;
};

struct PrefillBars {
  // What is numbered by steps has as many barriers as there are buffers of K and V: a step's products are also what its buffers
  // become free by.
  uint64_t pack_full[3], pack_empty[3], k_full[4], v_full[4], s_full[2][4], p_full[2][4], pv_done[2][4];
  uint64_t gave_up[2];  // all products of a tile, when the block gives up
};

// mbar_wait that looks at the clock only now and then: a waiting warp's polls take issue slots from the others.
__device__ __forceinline__ bool wait_quietly(uint64_t* bar, uint32_t parity) {
  unsigned long long t0 = 0;
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i) {
      uint32_t done;
      asm volatile(
          "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.b32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
          : "memory");
      if (done) return true;
    }
    const unsigned long long t = globaltimer_ns();
    if (t0 == 0) t0 = t;
    if (t - t0 > kWaitLimitNs) return false;
  }
}
// The same for a warp, which gives up together: what follows needs all of its lanes.
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, wait_quietly(bar, parity)) != 0; }
// Products are issued by one elected lane, predicated inside a block without branches: the warp stays together, so that the
// operands can live in uniform registers, which the instruction takes them from.  Descriptors come as their low words, the high
// word is the same for all operands here (1024 bytes from eight rows to the next, 128-byte swizzle).
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t elected() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
__device__ __forceinline__ void umma_ss(uint32_t issue, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %6, 0;\n\tmov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void umma_tmem_a(uint32_t issue, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %6, 0;\n\tmov.b64 db, {%2, %5};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t issue, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar)), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Low word of an operand's descriptor: its address, and for V, whose 128-byte rows hold 64 of a head's values (along N, a row per
// step of K), the bytes between neighbouring 64 values.
__device__ __forceinline__ uint32_t desc_low(const uint8_t* p, uint32_t columns) { return smem_u32(p) >> 4 | columns >> 4 << 16; }

__device__ __forceinline__ uint32_t lop3_and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}
// s (u - 8), exactly, of the codes in bits 0..3 (lo), 4..7 (hi) of both halves.
__device__ __forceinline__ uint32_t value_lo(uint32_t x, __half2 s) {
  const uint32_t b = lop3_and_or(x, 0x000F000Fu, 0x64006400u);  // 1024 + u
  const __half2 h = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(1032.0f)), s);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t value_hi(uint32_t x, __half2 s) {
  const uint32_t b = lop3_and_or(x, 0x00F000F0u, 0x64006400u);  // 1024 + 16 u
  const __half2 h = __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f)), s);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 values8(uint32_t x, __half2 s) {
  const uint32_t y = x >> 8;
  return make_uint4(value_lo(x, s), value_hi(x, s), value_lo(y, s), value_hi(y, s));
}

// Two weights at once: 2^(s * scale - ref).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm volatile("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float exp2_hw(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Barrier `id` of 256 threads.  One warp of them waits for a transaction barrier and the others for it here, without polls.
__device__ __forceinline__ void sync_256(int id) { asm volatile("barrier.cta.sync.aligned %0, 256;" ::"r"(id) : "memory"); }

// The same for the N threads that have rows.
template <int N>
__device__ __forceinline__ void sync_rows() {
  __syncwarp();
  asm volatile("barrier.cta.sync 4, %0;" ::"n"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// The steps that a block of rows walks.
struct BlockSteps {
  int at_lo, at_hi, first_step, steps;  // what the first and the last row see ends at at_lo and at_hi
};
template <int D>
__device__ __forceinline__ BlockSteps block_steps(const Kv4AttnArgs& a, const Kv4Sequence& q, int block) {
  using S = Prefill<D>;
  const int row0 = block * S::kRows, row_end = min(q.m * a.group, row0 + S::kRows);
  BlockSteps s;
  s.at_lo = q.n - q.m + row0 / a.group;
  s.at_hi = q.n - q.m + (row_end - 1) / a.group;
  s.first_step = (a.window > 0 ? max(0, s.at_lo - a.window + 1) : 0) / S::kN;
  s.steps = s.at_hi < 0 ? 0 : s.at_hi / S::kN + 1 - s.first_step;
  return s;
}

// Blocks of rows that a sequence has.
template <int D>
__device__ __forceinline__ int blocks_of(const Kv4AttnArgs& a, const Kv4Sequence& q) {
  return static_cast<int>((static_cast<long long>(q.m) * a.group + Prefill<D>::kRows - 1) / Prefill<D>::kRows);
}

// Cuts long blocks of rows along the cached tokens where all SMs are done sooner for it.  One block of 1024 threads; an entry is a
// block of rows of a sequence, those with the most blocks of their sequence ahead of them first (every sequence's last block, if it has
// as many as the one with the most, and so on).  Warp w weighs cutting everything longer than
// 1 / pieces_of(w) of the longest entry into pieces no longer than that: the time is an SM's share of all pieces and half of the
// longest one's (or that, if longer), and what the last of a block's pieces takes to join them.  A piece is (sequence, block,
// piece | pieces << 16, slot of the block's first); one for each key/value head.
__device__ __forceinline__ int pieces_of(int w) { return w < 16 ? w + 1 : 16 + (w - 15) * 8; }

// Ahead of the thread in the block of 1024, and in all; every thread calls it.
__device__ __forceinline__ int sum_before(int mine, int (&warps)[32], int& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warps[warp] = incl;
  __syncthreads();
  int before = incl - mine;
  all = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) before += warps[w];
    all += warps[w];
  }
  return before;
}

template <int D>
__global__ void __launch_bounds__(1024, 1) kv4_prefill_pieces_kernel(const __grid_constant__ Kv4AttnArgs a, int entries, int sms) {
  constexpr int kPer = kKv4MaxEntries / 1024;
  // sequences in the order of their blocks, most first: key, number; end[c]: entries of the blocks that more than c sequences have
  __shared__ __align__(16) int s_place[kKv4MaxEntries];  // of the entries: number of the block, sequence
  int* const s_key = s_place;                            // ahead of that
  __shared__ int s_blocks[kKv4MaxBatch + 1], s_sequence[kKv4MaxBatch], s_end[kKv4MaxBatch];
  __shared__ int s_steps[kKv4MaxEntries], s_scan[2][32], s_longest;
  __shared__ float s_time[32];
  static_assert(kKv4MaxBatch == 1024, "a thread to a sequence");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int own = threadIdx.x;  // a sequence, then a place in their order
  if (threadIdx.x == 0) s_longest = 1;
  pdl_wait();
  int blocks = 0;
  if (own < a.batch) blocks = min(blocks_of<D>(a, kv4_sequence(a, own)), entries);
  const int key = own < a.batch ? blocks << 10 | (1023 - own) : -1;
  s_key[own] = key;
  __syncthreads();
  if (own < a.batch) {
    int place = 0;
    for (int i = 0; i < a.batch; i += 4) {
      const int4 others = *reinterpret_cast<const int4*>(s_key + i);
      place += (others.x > key ? 1 : 0) + (others.y > key ? 1 : 0) + (others.z > key ? 1 : 0) + (others.w > key ? 1 : 0);
    }
    s_blocks[place] = blocks;
    s_sequence[place] = own;
  }
  if (own == 0) s_blocks[a.batch] = 0;
  __syncthreads();
  {
    int all;
    blocks = own < a.batch ? s_blocks[own] : 0;
    const int before = sum_before(blocks, s_scan[0], all);
    // the first own + 1 sequences' blocks from the number on that the next sequence has
    if (own < a.batch) s_end[own] = before + blocks - (own + 1) * s_blocks[own + 1];
  }
  __syncthreads();
  const int there = min(s_end[a.batch - 1], entries);
  int longest = 1;
  for (int e = threadIdx.x; e < entries; e += 1024) {
    int steps = -1;  // no rows
    if (e < there) {
      int lo = 0, hi = a.batch - 1;
      while (lo < hi) {  // the first group of blocks that ends behind the entry
        const int mid = (lo + hi) >> 1;
        if (s_end[mid] > e) hi = mid; else lo = mid + 1;
      }
      const int in = lo > 0 ? e - s_end[lo - 1] : e, row = in / (lo + 1);
      const int b = s_sequence[in - row * (lo + 1)], block = s_blocks[lo] - 1 - row;
      s_place[e] = block << 10 | b;
      steps = block_steps<D>(a, kv4_sequence(a, b), block).steps;
    }
    s_steps[e] = steps;
    longest = max(longest, steps);
  }
  longest = __reduce_max_sync(0xFFFFFFFFu, longest);
  if (lane == 0) atomicMax(&s_longest, longest);
  __syncthreads();
  longest = s_longest;
  const int room = a.slots / a.kv_heads;
  {
    const int most = (longest + pieces_of(warp) - 1) / pieces_of(warp);
    const float inv = 1.0f / static_cast<float>(most);
    float work = 0.0f;
    int cut = 0, joined = 1;
    for (int e = lane; e < entries; e += 32) {
      const int steps = s_steps[e];
      if (steps < 0) continue;
      const int k = steps > most ? static_cast<int>(ceilf(static_cast<float>(steps) * inv)) : 1;
      work += static_cast<float>(steps) + static_cast<float>(k) * (k > 1 ? kCutCost : kBlockCost);
      cut += k > 1 ? k + 1 : 0;  // one more than there may be after rounding
      joined = max(joined, k);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xFFFFFFFFu, work, o);
    cut = __reduce_add_sync(0xFFFFFFFFu, cut);
    joined = __reduce_max_sync(0xFFFFFFFFu, joined);
    const float piece = static_cast<float>(most) + (joined > 1 ? kCutCost : kBlockCost);
    const float time = fmaxf(piece, work * static_cast<float>(a.kv_heads) / static_cast<float>(sms) + 0.5f * piece) +
                       (joined > 1 ? kJoinCost * static_cast<float>(joined) : 0.0f);
    if (lane == 0) s_time[warp] = cut <= room ? time : INFINITY;
  }
  __syncthreads();
  int best = 0;
  for (int w = 1; w < 32; ++w)
    if (s_time[w] < s_time[best]) best = w;
  const int most = (longest + pieces_of(best) - 1) / pieces_of(best);
  int count = 0, slots = 0;  // of the entries before the thread's, after the scan
  int pieces[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = threadIdx.x * kPer + i, steps = e < entries ? s_steps[e] : -1;
    pieces[i] = steps < 0 ? 0 : max(1, (steps + most - 1) / most);
    count += pieces[i];
    slots += pieces[i] > 1 ? pieces[i] : 0;
  }
  // both sums in one number: fewer than 2^13 pieces in all, fewer than 2^12 slots
  static_assert(kKv4MaxEntries + 256 * kKv4Slots < 1 << 13, "a list's pieces");
  int both;
  const int before = sum_before(count << 12 | slots, s_scan[1], both), end = both >> 12;
  count = before >> 12;
  slots = before & 0xFFF;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (pieces[i] == 0) continue;
    const int at = s_place[threadIdx.x * kPer + i], b = at & 1023, block = at >> 10;
    for (int k = 0; k < pieces[i]; ++k) a.pieces[count + k] = make_int4(b, block, k | pieces[i] << 16, slots);
    count += pieces[i];
    slots += pieces[i] > 1 ? pieces[i] : 0;
  }
  for (int i = end + threadIdx.x; i < entries + room; i += 1024) a.pieces[i] = make_int4(-1, 0, 0, 0);
}

// The item-th block of rows of a call without a list, in the list's order; a warp together, which gets the same as any other.  `counts`:
// blocks of each sequence, none more than `most`.  False: there are not so many.
__device__ __forceinline__ bool find_block(const int* counts, int batch, int most, int item, int& b, int& block) {
  const int lane = threadIdx.x & 31, first = lane < batch ? counts[lane] : 0;
  const auto from = [&](int k) {  // blocks of all sequences from number k on
    unsigned sum = max(0, first - k);
    for (int i = lane + 32; i < batch; i += 32) sum += max(0, counts[i] - k);
    return __reduce_add_sync(0xFFFFFFFFu, min(sum, 1u << 26));  // no 32 bits overflow, whatever row ranges a call has
  };
  if (from(0) <= static_cast<unsigned>(item)) return false;
  int lo = 0, hi = most;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (from(mid) > static_cast<unsigned>(item)) lo = mid; else hi = mid;
  }
  block = lo;
  int left = item - static_cast<int>(from(lo + 1));
  for (int i = 0; i < batch; i += 32) {
    const bool mine = i + lane < batch && counts[i + lane] > lo;
    const unsigned has = __ballot_sync(0xFFFFFFFFu, mine);
    if (left < __popc(has)) {
      b = i + __ffs(__ballot_sync(0xFFFFFFFFu, mine && __popc(has & ((1u << lane) - 1u)) == left)) - 1;
      return true;
    }
    left -= __popc(has);
  }
  return false;
}

// kCut: blocks may be cut, and are listed.  Calls whose sequences are too short for that take the form without the joining, which
// costs the loop registers (a prompt of 2048 tokens 60 us in its own form, 62 to 65 in the other).
template <int D, bool kCut>
__global__ void __launch_bounds__(kPrefillThreads, 1) kv4_prefill_kernel(const __grid_constant__ Kv4AttnArgs a, int row_blocks, bool alike) {
  using S = Prefill<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const s_q = smem;                                  // [kTilesM][D / 64][128 rows][128 bytes]
  uint8_t* const s_k = s_q + S::kTilesM * S::kQBytes;         // [kBuffers][D / 64][kN rows][128 bytes]
  uint8_t* const s_v = s_k + S::kBuffers * S::kKvBytes;       // [kBuffers][D / 64][kN rows][128 bytes]
  uint8_t* const s_pack = s_v + S::kBuffers * S::kKvBytes;    // [kRing][kPackBytes]
  uint8_t* const s_bad = s_pack + S::kRing * S::kPackBytes;   // [kMaskedBlocks][kN]: groups of V that are not finite
  __shared__ PrefillBars bars;
  __shared__ uint32_t tmem_base;
  __shared__ int any_bad;
  __shared__ bool is_last;
  __shared__ int2 last_asked;  // stage and phase of the packed tiles that would be asked for next
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kRing; ++i) {
      mbar_init(&bars.pack_full[i], 1);
      mbar_init(&bars.pack_empty[i], kUnpackWarps);
    }
    for (int t = 0; t < S::kTilesM; ++t) mbar_init(&bars.gave_up[t], 1);
    for (int i = 0; i < S::kBuffers; ++i) {
      mbar_init(&bars.k_full[i], kUnpackWarps);
      mbar_init(&bars.v_full[i], kUnpackWarps);
      for (int t = 0; t < S::kTilesM; ++t) {
        mbar_init(&bars.s_full[t][i], 1);
        mbar_init(&bars.p_full[t][i], 4);
        mbar_init(&bars.pv_done[t][i], 1);
      }
    }
    fence_barrier_init();
    any_bad = 0;
  }
  pdl_wait();
  // ---- which rows: the blocks with the most tokens ahead of them first
  const int item = blockIdx.x / a.kv_heads, h = blockIdx.x - item * a.kv_heads;
  int b, block, piece = 0, pieces = 1, slot = 0;
  if constexpr (kCut) {
    const int4 p = __ldcg(a.pieces + item);
    b = p.x;
    block = p.y;
    piece = p.z & 0xFFFF;
    pieces = p.z >> 16;
    slot = p.w * a.kv_heads + h;
  } else if (alike) {
    const int rank = item / a.batch;
    b = item - rank * a.batch;
    block = row_blocks - 1 - rank;
  } else {
    int* const counts = reinterpret_cast<int*>(s_pack);
    static_assert(kKv4MaxBatch * sizeof(int) <= S::kRing * S::kPackBytes, "a count for each sequence");
    for (int i = threadIdx.x; i < a.batch; i += kPrefillThreads) counts[i] = blocks_of<D>(a, kv4_sequence(a, i));
    __syncthreads();
    if (!find_block(counts, a.batch, row_blocks, item, b, block)) b = -1;
  }
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < a.batch; i += kPrefillThreads)
      if (!kv4_fits(a, i, kv4_sequence(a, i))) atomicExch(a.error, kErrLength);
  }
  if (b < 0) return;
  const Kv4Sequence q = kv4_sequence(a, b);
  const int rows = q.m * a.group, row0 = block * S::kRows;
  if (row0 >= rows) return;
  const BlockSteps all_steps = block_steps<D>(a, q, block);
  const int at_lo = all_steps.at_lo, at_hi = all_steps.at_hi;
  const int step_from = static_cast<int>(static_cast<long long>(all_steps.steps) * piece / pieces);
  const int step0 = all_steps.first_step + step_from;
  const int steps = static_cast<int>(static_cast<long long>(all_steps.steps) * (piece + 1) / pieces) - step_from;
  // whether all rows see all of a step's tokens
  const auto whole = [&](int t0, int lo, int hi) { return t0 + S::kN - 1 <= lo && (a.window == 0 || t0 >= hi - a.window + 1); };

  if (warp == kMmaWarp) tmem_alloc_512(&tmem_base);
  for (int i = threadIdx.x; i < S::kTilesM * kRowsPerTile * (D / 8); i += kPrefillThreads) {
    const int r = i / (D / 8), c = i - r * (D / 8);
    const int row = row0 + r, token = row / a.group, head = h * a.group + row - token * a.group;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows) v = __ldg(reinterpret_cast<const uint4*>(a.q + (q.first_token + token) * a.q_stride + static_cast<long long>(head) * D) + c);
    *reinterpret_cast<uint4*>(s_q + (r / kRowsPerTile) * S::kQBytes + (c >> 3) * (kRowsPerTile * 128) + (r % kRowsPerTile) * 128 +
                              (((c & 7) ^ (r & 7)) << 4)) = v;
  }
  for (int i = threadIdx.x; i < kMaskedBlocks * S::kN / 4; i += kPrefillThreads) reinterpret_cast<uint32_t*>(s_bad)[i] = 0;
  fence_proxy_async();
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = 0;  // all columns are this block's: they begin at 0
  constexpr int kB = S::kBuffers;
  bool ok = true;

  if (warp < kRowWarps) {
    more_registers<kRegsRows>();
    // ------------------------------------------------------------------ weights, rows
    const int tile = warp >> 2;
    if (tile < S::kTilesM) {
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t t_s0 = tmem + lanes + tile * 2 * S::kN, t_o = tmem + lanes + S::kO + tile * D;
      const int row = row0 + tile * kRowsPerTile + (warp & 3) * 32 + lane;
      const int at = q.n - q.m + min(row, rows - 1) / a.group;
      const int tile_lo = q.n - q.m + min(row0 + tile * kRowsPerTile, rows - 1) / a.group;
      const int tile_hi = q.n - q.m + min(row0 + tile * kRowsPerTile + kRowsPerTile - 1, rows - 1) / a.group;
      float top = kPrefillFloor, minus_ref = -kPrefillFloor;
      float2 sums[2] = {};
      const float2 scale2 = make_float2(a.scale_log2, a.scale_log2);
      const float inv_scale = 1.0f / a.scale_log2;
      float limit = kPrefillFloor * inv_scale;  // scores that may not be exceeded
#pragma unroll 1
      for (int j = 0; j < steps; ++j) {
        // who gives up goes on without waiting: the warp's lanes are needed together
        ok = ok && wait_quietly(&bars.s_full[tile][j % kB], j / kB & 1);
        __syncwarp();
        tc_after();
        const uint32_t t_s = t_s0 + (j & 1) * S::kN;
        const int t0 = (step0 + j) * S::kN;
        uint32_t s[2][32];
        tmem_ld32(t_s, s[0]);
        tmem_ld32(t_s + 32, s[1]);
        tmem_ld_wait();
        if (!whole(t0, tile_lo, tile_hi)) {
          const int hi = at - t0, lo = a.window > 0 ? hi - a.window + 1 : 0;  // what the row sees of the step
#pragma unroll
          for (int e = 0; e < S::kN; ++e)
            if (e > hi || e < lo) s[e / 32][e % 32] = 0xFF800000u;
        }
        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < S::kN; e += 2)
          most[e / 2 % 4] = max3(most[e / 2 % 4], __uint_as_float(s[e / 32][e % 32]), __uint_as_float(s[e / 32][e % 32 + 1]));
        const float m = fmaxf(max3(most[0], most[1], most[2]), most[3]);
        if (__any_sync(0xFFFFFFFFu, m > limit)) {
          const float new_top = m > limit ? m * a.scale_log2 : top;
          const float ref = new_top > kPrefillFloor ? new_top - kPrefillLift : kPrefillFloor;
          const float f = exp2_hw(-minus_ref - ref);
          top = new_top;
          minus_ref = -ref;
          limit = new_top > kPrefillFloor ? (new_top + kPrefillHeadroom) * inv_scale : kPrefillFloor * inv_scale;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            sums[i].x *= f;
            sums[i].y *= f;
          }
          if (j > 0) {
            ok = ok && wait_quietly(&bars.pv_done[tile][(j - 1) % kB], (j - 1) / kB & 1);
            __syncwarp();
            tc_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld16(t_o + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(t_o + c, o);
            }
          }
        }
        const float2 ref2 = make_float2(minus_ref, minus_ref);
        // Three pairs are in the works at a time, so that the exponentials' unit, which takes an instruction in eight cycles, has
        // the next one while the pair before is added up and packed.
        const auto pair = [&](int e) { return make_float2(__uint_as_float(s[e / 32][e % 32]), __uint_as_float(s[e / 32][e % 32 + 1])); };
        uint32_t p[2][16];
        float2 x0 = fma2(pair(0), scale2, ref2), x1 = fma2(pair(2), scale2, ref2), y;
        x0.x = exp2_hw(x0.x);
        x0.y = exp2_hw(x0.y);
#pragma unroll
        for (int e = 0; e < S::kN; e += 2) {
          if (e + 2 < S::kN) {
            y = x1;
            y.x = exp2_hw(y.x);
          }
          if (e + 4 < S::kN) x1 = fma2(pair(e + 4), scale2, ref2);
          sums[e / 2 & 1] = add2(sums[e / 2 & 1], x0);
          if (e + 2 < S::kN) y.y = exp2_hw(y.y);
          p[e / 32][e % 32 / 2] = half2_bits(x0.x, x0.y);
          x0 = y;
          if (e == 30) tmem_st16(t_s, p[0]);  // over the thread's own scores
        }
        tmem_st16(t_s + 16, p[1]);
        tmem_st_wait();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[tile][j % kB]);
      }
      // ---- out
      const float l = (sums[0].x + sums[1].x) + (sums[0].y + sums[1].y);
      if (steps > 0) ok = ok && wait_quietly(&bars.pv_done[tile][(steps - 1) % kB], (steps - 1) / kB & 1);
      tc_after();
      uint32_t bad = 0;  // groups of the row's values that are not finite
      if (any_bad) {
        int k = 0;
        for (int j = 0; j < steps; ++j) {
          const int t0 = (step0 + j) * S::kN;
          if (whole(t0, at_lo, at_hi)) continue;
          for (int t = 0; t < S::kN; ++t)
            if (t0 + t <= at && (a.window == 0 || t0 + t > at - a.window)) bad |= s_bad[min(k, kMaskedBlocks - 1) * S::kN + t];
          ++k;
        }
      }
      const int token = row / a.group, head = h * a.group + row - token * a.group;
      __half* dst = a.out + (q.first_token + token) * a.out_stride + static_cast<long long>(head) * D;
      const auto put = [&](int c, const float* o, uint32_t bad_groups, float inv) {  // 16 columns
        const float f = (bad_groups >> (c / 32)) & 1 ? __int_as_float(0x7FFFFFFF) : inv;
        if (row < rows) {
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            // value k of eight lies in column 2 k, value 4 + k in column 2 k + 1
            const auto x = [&](int k) { return o[e + (k < 4 ? 2 * k : 2 * k - 7)] * f; };
            *reinterpret_cast<uint4*>(dst + c + e) =
                make_uint4(half2_bits(x(0), x(1)), half2_bits(x(2), x(3)), half2_bits(x(4), x(5)), half2_bits(x(6), x(7)));
          }
        }
      };
      const auto inverse = [](float sum) { return sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f; };
      constexpr int kSlot = (D / 4 + 1) * S::kRows;
      float4* const parts = reinterpret_cast<float4*>(a.part) + static_cast<long long>(slot) * kSlot + tile * kRowsPerTile + (warp & 3) * 32 + lane;
      const long long next = static_cast<long long>(a.kv_heads) * kSlot;  // the block's next piece
      float4* const mine = parts + piece * next;
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        if (steps > 0) {
          tmem_ld16(t_o + c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0;
        }
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(o[e]);
        if (!kCut || pieces == 1) {
          put(c, x, bad, inverse(l));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) __stcg(mine + (c / 4 + e) * S::kRows, make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]));
        }
      }
      if (kCut && pieces > 1) {
        // ---- the last of the block's pieces joins them, in their order
        __stcg(mine + D / 4 * S::kRows, make_float4(-minus_ref, l, __uint_as_float(bad), 0.0f));
        __threadfence();
        sync_rows<S::kTilesM * kRowsPerTile>();
        if (threadIdx.x == 0) {
          const bool last = atomicAdd(a.tickets + slot, 1) == pieces - 1;
          if (last) a.tickets[slot] = 0;
          is_last = last;
          __threadfence();
        }
        sync_rows<S::kTilesM * kRowsPerTile>();
        if (is_last) {
          __threadfence();
          float ref = kPrefillFloor, sum = 0.0f;
          bad = 0;
          const float4* const states = parts + D / 4 * S::kRows;
          for (int p = 0; p < pieces; ++p) ref = fmaxf(ref, __ldcg(states + p * next).x);
          for (int p = 0; p < pieces; ++p) {
            const float4 state = __ldcg(states + p * next);
            sum += exp2_hw(state.x - ref) * state.y;
            bad |= __float_as_uint(state.z);
          }
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float x[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = 0.0f;
#pragma unroll 2
            for (int p = 0; p < pieces; ++p) {
              const float f = exp2_hw(__ldcg(states + p * next).x - ref);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 y = __ldcg(parts + p * next + (c / 4 + e) * S::kRows);
                x[4 * e] = fmaf(f, y.x, x[4 * e]);
                x[4 * e + 1] = fmaf(f, y.y, x[4 * e + 1]);
                x[4 * e + 2] = fmaf(f, y.z, x[4 * e + 2]);
                x[4 * e + 3] = fmaf(f, y.w, x[4 * e + 3]);
              }
            }
            put(c, x, bad, inverse(sum));
            put(c + 16, x + 16, bad, inverse(sum));
          }
        }
      }
      tc_before();
    }
  } else if (warp < kLoadWarp) {
    fewer_registers<kRegsUnpack>();
    // ------------------------------------------------------------------ unpacking
    const int w = warp - kRowWarps;
    // lanes of one 128-byte access lie four rows apart, so that the swizzle spreads them over all banks
    const int g = lane >> 2, t = lane & 3, in8 = (g >> 1) | (g & 1) << 2;
    constexpr int kG = D / 32, kWords = kG < 4 ? kG : 4;
    const int tau = (w & 1) * 8 + in8, row = (w >> 1) * 16 + tau;  // a warp takes eight tokens of a step
    uint8_t* const dst = s_k + row * 128;
    int stage = 0, phase = 0, masked = -1, buf = 0, use = 0;
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      const int t0 = (step0 + j) * S::kN;
      const bool all = whole(t0, at_lo, at_hi);
      if (!all) masked = min(masked + 1, kMaskedBlocks - 1);
      if (w == 0) {
        ok = ok && wait_all(&bars.pack_full[stage], phase);
        for (int i = 0; i < S::kTilesM; ++i) ok = ok && wait_all(&bars.pv_done[i][buf], use ^ 1);  // then K is free as well
      }
      sync_256(3);
      // all of the lane's words of K and V are asked for before the first is turned into values
      const uint8_t* const tile = s_pack + stage * S::kPackBytes + (w >> 1) * S::kTileBytes;
      uint32_t x[2][kG], sc[2][kG / 2];
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) kv4_lds(tile + kv4::scale_at<D>(kind, tau, 0), sc[kind]);
#pragma unroll
      for (int q4 = 0; q4 < kG / kWords; ++q4)
        kv4_lds(tile + kv4::k_word<D>(tau, q4 * kWords, t), reinterpret_cast<uint32_t(&)[kWords]>(x[0][q4 * kWords]));
      {
        // pieces 2 t and 2 t + 1 lie side by side; two bytes of each make a word of eight neighbours
        const int vr = kv4::v_row(tau);
        const uint8_t* piece = tile + 8 * D + vr * (D / 2) + kv4::v_piece<D>(vr, 2 * t) * (D / 16);
        uint32_t y[kG / 2], z[kG / 2];
        kv4_lds(piece, y);
        kv4_lds(piece + D / 16, z);
#pragma unroll
        for (int e = 0; e < kG; ++e) x[1][e] = __byte_perm(y[e >> 1], z[e >> 1], e & 1 ? 0x7632 : 0x5410);
      }
      if (!all) {
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
          for (int e = 0; e < kG; ++e) {
            const uint32_t bits = 0x7C00u << (16 * (e & 1));
            const bool there = t0 + row <= at_hi;  // behind lies anything
            if (there && (kind == 0 || (sc[kind][e >> 1] & bits) != bits)) continue;
            // A NaN scale of V: its product with a zero weight would not be zero; noted, and told to the rows that see the token.
            sc[kind][e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
            if (there) {
              any_bad = 1;
              atomicOr(reinterpret_cast<uint32_t*>(s_bad + masked * S::kN + (row & ~3)), 1u << (e + 8 * (row & 3)));
            }
          }
        }
      }
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        uint8_t* const to = dst + (kind * S::kBuffers + buf) * S::kKvBytes;  // V's buffers follow K's
#pragma unroll
        for (int e = 0; e < kG; ++e) {
          const int c = e * 4 + t;
          const uint32_t s2 = __byte_perm(sc[kind][e >> 1], 0, e & 1 ? 0x3232 : 0x1010);
          *reinterpret_cast<uint4*>(to + (c >> 3) * (S::kN * 128) + (((c & 7) ^ (row & 7)) << 4)) =
              values8(x[kind][e], *reinterpret_cast<const __half2*>(&s2));
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(kind ? &bars.v_full[buf] : &bars.k_full[buf]);
          // Behind the fence, which orders the reads ahead of the next copy's writes: an arrival right after them let copies
          // overtake them.
          if (kind == 1) mbar_arrive(&bars.pack_empty[stage]);
        }
      }
      if (++stage == S::kRing) {
        stage = 0;
        phase ^= 1;
      }
      if (++buf == S::kBuffers) {
        buf = 0;
        use ^= 1;
      }
    }
  } else {
    fewer_registers<kRegsRest>();
  }
  if (warp == kLoadWarp) {
    // ------------------------------------------------------------------ packed tiles
    // Lane l looks up every 32nd tile and brings it when its stage's turn comes, with the tiles behind it that lie in the same page.
    int asked = 0, asked_phase = 0;
    const int tiles = (min(at_hi, q.n - 1) >> 4) + 1, tile0 = step0 * (S::kN / 16);
#pragma unroll 1
    for (int from = tile0; from < tile0 + steps * (S::kN / 16) && ok; from += 32) {
      const int tile = from + lane, page = tile / a.page_tiles, in_page = tile - page * a.page_tiles;
      int run = 0;
      const uint8_t* src = nullptr;
      if (tile < tiles && (in_page == 0 || lane % S::kPackTiles == 0)) {
        int pid = __ldg(a.table + static_cast<long long>(b) * a.max_pages + page);
        if (pid < 0 || pid >= a.pages) {
          atomicExch(a.error, kErrPage);
          pid = 0;
        }
        run = min(min(a.page_tiles - in_page, S::kPackTiles - lane % S::kPackTiles), tiles - tile);
        src = a.pool + ((static_cast<long long>(pid) * a.kv_heads + h) * a.page_tiles + in_page) * S::kTileBytes;
      }
#pragma unroll 1
      for (int l = 0; l < 32 && from + l < tile0 + steps * (S::kN / 16); l += S::kPackTiles) {
        ok = wait_all(&bars.pack_empty[asked], asked_phase ^ 1);
        if (!ok) break;
        const int there = min(S::kPackTiles, max(0, tiles - from - l));
        if (lane == 0) mbar_arrive_expect_tx(&bars.pack_full[asked], there * S::kTileBytes);
        __syncwarp();
        if (run > 0 && lane >= l && lane < l + S::kPackTiles)
          bulk_load_1d(s_pack + asked * S::kPackBytes + (lane - l) * S::kTileBytes, src, run * S::kTileBytes, &bars.pack_full[asked]);
        if (++asked == S::kRing) {
          asked = 0;
          asked_phase ^= 1;
        }
      }
    }
    if (lane == 0) last_asked = make_int2(asked, asked_phase);
  } else if (warp >= kMmaWarp && warp < kMmaWarp + S::kTilesM) {
    // ------------------------------------------------------------------ products of a tile
    const int tile = warp - kMmaWarp;
    const uint32_t idesc_s = 1u << 4 | static_cast<uint32_t>(S::kN >> 3) << 17 | 8u << 24;
    const uint32_t idesc_o = 1u << 4 | 1u << 16 | static_cast<uint32_t>(D >> 3) << 17 | 8u << 24;
    const uint32_t q_low = desc_low(s_q + tile * S::kQBytes, 16), k_low = desc_low(s_k, 16), v_low = desc_low(s_v, S::kN * 128);
    const uint32_t t_s = tmem + tile * 2 * S::kN, t_o = tmem + S::kO + tile * D, me = elected();
    const auto scores = [&](int j) {  // of step j, into the tile's j % 2nd place
      ok = wait_all(&bars.k_full[j % kB], j / kB & 1);
      if (j > 1) ok = ok && wait_all(&bars.pv_done[tile][(j - 2) % kB], (j - 2) / kB & 1);  // whose weights lie there
      if (!ok) return;
      tc_after();
      const uint32_t dk = k_low + j % kB * (S::kKvBytes >> 4);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        umma_ss(me, t_s + (j & 1) * S::kN, q_low + (((k >> 2) * (kRowsPerTile * 128) + (k & 3) * 32) >> 4),
                dk + (((k >> 2) * (S::kN * 128) + (k & 3) * 32) >> 4), idesc_s, k > 0);
      umma_commit(me, &bars.s_full[tile][j % kB]);
    };
    if (steps > 0) scores(0);
#pragma unroll 1
    for (int j = 0; j < steps && ok; ++j) {
      if (j + 1 < steps) scores(j + 1);
      ok = ok && wait_all(&bars.v_full[j % kB], j / kB & 1) && wait_all(&bars.p_full[tile][j % kB], j / kB & 1);
      if (!ok) break;
      tc_after();
      const uint32_t dv = v_low + j % kB * (S::kKvBytes >> 4), p = t_s + (j & 1) * S::kN;
#pragma unroll
      for (int k = 0; k < S::kN / 16; ++k)
        umma_tmem_a(me, t_o, p + 8 * k, dv + (k * 2048 >> 4), idesc_o, k > 0 ? 1u : static_cast<uint32_t>(j));
      umma_commit(me, &bars.pv_done[tile][j % kB]);
    }
  }
  tc_before();
  if (__syncthreads_or(!ok)) {
    // Some role gave up: the copies and products that others have in flight end before the memory that they use does.
    if (threadIdx.x == 0) atomicExch(a.error, kErrWait);
    if (warp == kLoadWarp) {
      for (int i = 0; i < S::kRing; ++i) wait_all(&bars.pack_full[i], ring_last_phase(i, last_asked.x, last_asked.y));
    } else if (warp >= kMmaWarp && warp < kMmaWarp + S::kTilesM) {
      umma_commit(elected(), &bars.gave_up[warp - kMmaWarp]);
      wait_all(&bars.gave_up[warp - kMmaWarp], 0);
    }
    __syncthreads();
  }
  tc_after();
  if (warp == kMmaWarp) tmem_dealloc_512(tmem_base);
}

template <int D, bool kCut>
int launch_prefill_t(const Kv4AttnArgs& a, int sms, cudaStream_t stream) {
  using S = Prefill<D>;
  static bool configured[kMaxDevices];
  int dev;
  if (needs_configure(configured, &dev)) {
    MLD_CUDA_CHECK(cudaFuncSetAttribute(kv4_prefill_kernel<D, kCut>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem)));
    if (dev >= 0) configured[dev] = true;
  }
  const int64_t row_blocks = div_up64(static_cast<int64_t>(a.max_queries) * a.group, S::kRows);
  const int64_t blocks = kv4_blocks(a.batch, a.max_queries, a.q_tokens, a.group, S::kRows);
  const int64_t grid = (blocks + (kCut ? a.slots / a.kv_heads : 0)) * a.kv_heads;
  if (grid > 0x7FFFFFFF) {
    set_last_error_text("more work than one call can count: fewer sequences or queries");
    return MLD_OUT_OF_RANGE;
  }
  if constexpr (kCut) {
    MLD_CUDA_CHECK(launch_overlapped(kv4_prefill_pieces_kernel<D>, dim3(1), dim3(1024), 0, stream, a, static_cast<int>(blocks), sms));
    MLD_LAUNCH_CHECK();
  }
  MLD_CUDA_CHECK(launch_overlapped(kv4_prefill_kernel<D, kCut>, dim3(static_cast<unsigned>(grid)), dim3(kPrefillThreads), S::kSmem, stream, a,
                                   static_cast<int>(row_blocks), blocks == row_blocks * a.batch));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

template <int D>
int launch_prefill_d(const Kv4AttnArgs& a, int sms, cudaStream_t stream) {
  return a.pieces != nullptr ? launch_prefill_t<D, true>(a, sms, stream) : launch_prefill_t<D, false>(a, sms, stream);
}

template <int D>
constexpr size_t kSlotBytes = static_cast<size_t>(Prefill<D>::kRows) * (D + 4) * sizeof(float);

}  // namespace

size_t kv4_slot_bytes(int head_dim) { return head_dim == 64 ? kSlotBytes<64> : head_dim == 128 ? kSlotBytes<128> : kSlotBytes<256>; }

// Up to 4096 tokens the pieces are hardly worth what they cost (8 heads of 128, 2048 rows, 4096 tokens: 85 us whole, 86 cut), and
// the list takes a launch more (a prompt of 2048 tokens 60 us without, 63 with it).
bool kv4_can_cut(int64_t tokens) { return tokens > 4096; }

bool kv4_cuts(const Kv4AttnArgs& a, int head_dim) {
  const int rows = head_dim == 256 ? Prefill<256>::kRows : Prefill<128>::kRows;
  return kv4_blocks(a.batch, a.max_queries, a.q_tokens, a.group, rows) <= kKv4MaxEntries && (a.window == 0 || kv4_can_cut(a.window));
}

int launch_kv4_prefill(const Kv4AttnArgs& a, int head_dim, int sms, cudaStream_t stream) {
  return head_dim == 64 ? launch_prefill_d<64>(a, sms, stream)
                        : head_dim == 128 ? launch_prefill_d<128>(a, sms, stream) : launch_prefill_d<256>(a, sms, stream);
}

}  // namespace mld

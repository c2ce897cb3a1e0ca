// Attention over the 4-bit cache for few query rows per key/value head: decoding, a few drafted tokens.
//
//   o_i = sum_t softmax_t(scale q_i.k_t) v_t over the tokens t that row i sees; nothing seen gives zeros.
//
// What it cannot do without is reading the cache once: 18 D / 16 bytes per token and head (144 for D = 128, 3.6 times fewer than
// fp16).  One token over 131071 of 8 heads of 128 takes 48 us, 3.1 TB/s, where copies into the same rings without the arithmetic take
// 22; 64 ragged sequences of up to 8191 tokens 97 us, 2.9 TB/s; 300 tokens 8 us, all latencies.  What bounds the long ones is a warp's
// chain of instructions (scores, vote, exponentials, transposition, values), of which three to a scheduler fill 2.2 of 4 issue slots:
// 390 for a tile of 16 tokens, 120 of them unpacking; then about 8 us of joining.
// The queries of all heads that share a key/value head, and of all new tokens of a sequence, are the columns of the products,
// so a code is unpacked once for all of them:
//   S^T[token][row] = K q:  A = codes of K as they lie, masked into fp16 subnormals u 2^-24 (and 16 u 2^-24 for the odd nibbles,
//     whose q is divided by 16), a 32-value group at a time, so that the group's scale multiplies an fp32 sum; -8 sum(q) is added
//     to it.  A row of q is scaled by a power of two that leaves its largest value near 2^10, so that a sixteenth of any value
//     that counts is a normal number.
//   O^T[value][row] = V^T P: A = codes of V made (u - 8) 2^-9 by a mask and a multiply-add, exactly (sums of P u minus 8 sums of P
//     would lose what a token of great weight leaves to the others where its own value is zero); the scales of V, which belong to
//     tokens and groups, go into P before it is rounded to fp16, a P per group.  S^T's accumulator layout becomes P's operand
//     layout by an 8x8 transposition in registers (movmatrix).
// P's range: 2^top is a row's reference weight and 2^e no smaller than any scale of V so far; weights are taken as
// 2^(s - top - e + 13), so that weight times scale stays below 2^15 and is a normal number down to 2^-27 of the largest, whatever
// the values' magnitude.  top and e move only when a step exceeds them (top by 2^2); sums are kept per lane until the end.
//
// Work is cut without regard to sequences: all chunks (of 4.5 KB: 64, 32 or 16 tokens of a head) of all sequences, heads and
// blocks of rows in a row, dealt out evenly over CTAs and their warps, which keep rings of bulk copies of their own (no producer,
// no block-wide barrier while streaming).  A sequence that several warps share is joined in shared memory, one that
// several CTAs share through the plan's workspace by whichever CTA comes last, in the order of the tokens: results do not depend
// on who that is.
#include <cuda_fp16.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "kv4_attn.cuh"

namespace mld {
namespace {

constexpr int kMaxGrid = 256, kTickets = kMaxGrid * kKv4Slots;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }

// (u - 8) 2^-9 of the codes in bits 0..3 (lo), 4..7 (hi) of both halves: what the mask leaves is an fp16 subnormal, u 2^-24 or
// u 2^-20, which one fused multiply-add turns into that, exactly.  Masks, shifts and these multiply-adds share a pipe that takes one
// in two cycles: 64 masks, 24 shifts and permutations and 32 multiply-adds to 16 tokens of 128 values, 13.5 us for 131071 tokens of
// 8 heads.
constexpr float kCodeUnit = 512.0f;
__device__ __forceinline__ uint32_t fma_half2(uint32_t x, float scale, float offset) {
  const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(scale), __float2half2_rn(offset));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t code_lo(uint32_t x) { return fma_half2(x & 0x000F000Fu, 32768.0f, -0.015625f); }
__device__ __forceinline__ uint32_t code_hi(uint32_t x) { return fma_half2(x & 0x00F000F0u, 2048.0f, -0.015625f); }

// Two halves, each zero where it is an infinity or a NaN.
__device__ __forceinline__ uint32_t finite_halves(uint32_t x) {
  return ((x & 0x7C00u) == 0x7C00u ? 0u : x & 0xFFFFu) | ((x & 0x7C000000u) == 0x7C000000u ? 0u : x & 0xFFFF0000u);
}

constexpr float kFloor = -1e30f;   // reference of a row that has seen nothing
constexpr float kHeadroom = 2.0f;  // how far weights may exceed the reference, as a power of two
constexpr float kLift = 13.0f;

template <int D, int NT>
struct Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kGroups = D / 32;
  static constexpr int kTileBytes = kv4::tile_bytes(D);
  static constexpr int kTiles = D == 64 ? 4 : D == 128 ? 2 : 1;  // of a chunk
  static constexpr int kStep = D == 256 ? 1 : 2;                 // tiles that are worked on together
  static constexpr int kChunk = kTiles * kv4::kTile;
  static constexpr int kStageBytes = kTiles * kTileBytes;
  static constexpr int kStages = 3;
  static constexpr int kRecord = D + 4;                          // floats: values, reference, sum
  static constexpr int kSlotBytes = kRows * kRecord * 4;
};

// A sequence's share of the work list.
struct Span {
  int n, m, first_row_token, c0, chunks, blocks;
};

template <int D, int NT>
__device__ __forceinline__ Span span_of(const Kv4AttnArgs& a, int b) {
  using S = Shape<D, NT>;
  const Kv4Sequence q = kv4_sequence(a, b);
  Span s;
  s.n = q.n;
  s.m = q.m;
  s.first_row_token = q.first_token;
  const int first = a.window > 0 ? max(0, s.n - s.m + 1 - a.window) : 0;
  s.c0 = first / S::kChunk;
  s.chunks = max(1, (s.n - 1) / S::kChunk + 1 - s.c0);  // no sum here may pass 2^31 - 1, which n comes close to
  s.blocks = (s.m * a.group + S::kRows - 1) / S::kRows;
  return s;
}

// Where an item of the work list lies: sequence, key/value head, block of rows, chunk.
struct Place {
  Span s;
  int b, h, r, c;   // c counts from the segment's first chunk
  int start, end;   // the segment, all chunks of a block of rows, as items
};

template <int D, int NT>
__device__ __forceinline__ Place locate(const Kv4AttnArgs& a, const int* prefix, int item) {
  int lo = 0, hi = a.batch - 1;
  while (lo < hi) {  // the last sequence that begins at or before the item
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= item) lo = mid; else hi = mid - 1;
  }
  Place p;
  p.b = lo;
  p.s = span_of<D, NT>(a, lo);
  const int in = item - prefix[lo], seg = in / p.s.chunks;
  p.c = in - seg * p.s.chunks;
  p.h = seg / p.s.blocks;
  p.r = seg - p.h * p.s.blocks;
  p.start = item - p.c;
  p.end = p.start + p.s.chunks;
  return p;
}

// Where a lane (g, t) reads in a tile; everything else is these plus constants.
template <int D>
struct LaneAt {
  int g, t, k, k2, ks, v, vs;
  __device__ __forceinline__ explicit LaneAt(int lane) : g(lane >> 2), t(lane & 3) {
    k = kv4::k_word<D>(g, 0, t);
    k2 = D == 256 ? kv4::k_word<D>(g, 4, t) : 0;
    ks = kv4::scale_at<D>(false, g, 0);
    vs = kv4::scale_at<D>(true, g, 0);
    const int row = kv4::v_row(2 * t);
    v = 8 * D + row * (D / 2) + kv4::v_piece<D>(row, g) * (D / 16);
  }
};

// The state of a segment in a warp.  Lane (g, t) holds the rows (columns of the products) 8 i + 2 t and + 1.
template <int D, int NT>
struct Rows {
  using S = Shape<D, NT>;
  float o[S::kGroups][2][NT][4];
  float top[NT][2], sum[NT][2];
  float minus_ref[NT][2];  // -(top + e - kLift)
  float limit[NT][2];      // scores that may not be exceeded: (top + kHeadroom) / cs
  float cs[NT][2];         // log2(e) times the scale of the scores, as the products give them
  float q8[S::kGroups][NT][2];  // -8 sum(q) of a group, in the codes' units
  uint32_t scale_limit;    // largest scale of V, as the bits of fp16, that e covers
  float e;
  uint32_t q[S::kGroups][NT][4];

  __device__ __forceinline__ void clear() {
    scale_limit = 0;
    e = -14.0f;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < S::kGroups; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[j][0][i][k] = o[j][1][i][k] = 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[i][c] = kFloor;
        minus_ref[i][c] = -kFloor;
        limit[i][c] = kFloor / cs[i][c];
        sum[i][c] = 0.0f;
      }
    }
  }
};

// Query rows of a block as the MMAs' B operand: lane (g, t) holds values 8 t.. of row 8 i + g.
template <int D, int NT>
__device__ __forceinline__ void load_q(const Kv4AttnArgs& a, const Place& p, const LaneAt<D>& at, Rows<D, NT>& w) {
  using S = Shape<D, NT>;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int row = p.r * S::kRows + 8 * i + at.g;
    const bool there = row < p.s.m * a.group;
    const int token = row / a.group, head = p.h * a.group + row - token * a.group;
    const __half* src = a.q + (p.s.first_row_token + token) * a.q_stride + static_cast<long long>(head) * D + 8 * at.t;
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < S::kGroups; ++j) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (there) v = *reinterpret_cast<const uint4*>(src + 32 * j);
      w.q[j][i][0] = v.x;
      w.q[j][i][1] = v.y;
      w.q[j][i][2] = v.z;
      w.q[j][i][3] = v.w;
#pragma unroll
      for (int e = 0; e < 4; ++e) most = __vmaxu2(most, w.q[j][i][e] & 0x7FFF7FFFu);
    }
    most = max(most & 0xFFFFu, most >> 16);
    most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
    most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
    const int exponent = static_cast<int>(most >> 10);              // 31: an infinity or a NaN, which stays what it is
    const int up = exponent == 31 ? 0 : 25 - exponent;              // 2^10 for the largest
    const float by = __int_as_float((127 + up) << 23);
#pragma unroll
    for (int j = 0; j < S::kGroups; ++j) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 f = unpack_half2(w.q[j][i][e]);
        f.x *= by;
        f.y *= by;
        sum += f.x + f.y;
        const float odd = e & 1 ? 0.0625f : 1.0f;
        w.q[j][i][e] = pack_half2(f.x * odd, f.y * odd);
      }
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      // this lane's columns of the accumulators are rows 2 t and 2 t + 1
      const float unit = -8.0f / 16777216.0f;
      w.q8[j][i][0] = unit * __shfl_sync(0xFFFFFFFFu, sum, 8 * at.t);
      w.q8[j][i][1] = unit * __shfl_sync(0xFFFFFFFFu, sum, 8 * at.t + 4);
    }
    const float cs = a.scale_log2 * 16777216.0f * __int_as_float((127 - up) << 23);
    w.cs[i][0] = __shfl_sync(0xFFFFFFFFu, cs, 8 * at.t);
    w.cs[i][1] = __shfl_sync(0xFFFFFFFFu, cs, 8 * at.t + 4);
  }
}

// Scores of 16 tokens.
template <int D, int NT>
__device__ __forceinline__ void tile_scores(const uint8_t* tile, const LaneAt<D>& at, const Rows<D, NT>& w, float (&s)[NT][4]) {
  constexpr int kG = D / 32;
  constexpr int kW = kG < 4 ? kG : 4;
#pragma unroll
  for (int u = 0; u < kG / kW; ++u) {
    uint32_t k0[kW], k1[kW], sc0[kW / 2], sc1[kW / 2];
    const uint8_t* row = tile + (u == 0 ? at.k : at.k2);
    kv4_lds(row, k0);
    kv4_lds(row + 8 * (D / 2), k1);
    kv4_lds(tile + at.ks + 8 * u, sc0);
    kv4_lds(tile + at.ks + 8 * u + 8 * (D / 16), sc1);
#pragma unroll
    for (int v = 0; v < kW; ++v) {
      const int j = u * kW + v;
      const float2 f0 = unpack_half2(sc0[v >> 1]), f1 = unpack_half2(sc1[v >> 1]);
      const float s0 = v & 1 ? f0.y : f0.x, s1 = v & 1 ? f1.y : f1.x;
      const uint32_t x0 = k0[v], x1 = k1[v], y0 = x0 >> 8, y1 = x1 >> 8;
      const uint32_t a0 = x0 & 0x000F000Fu, a1 = x1 & 0x000F000Fu, a2 = x0 & 0x00F000F0u, a3 = x1 & 0x00F000F0u;
      const uint32_t b0 = y0 & 0x000F000Fu, b1 = y1 & 0x000F000Fu, b2 = y0 & 0x00F000F0u, b3 = y1 & 0x00F000F0u;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma16816(c, a0, a1, a2, a3, w.q[j][i][0], w.q[j][i][1]);
        mma16816(c, b0, b1, b2, b3, w.q[j][i][2], w.q[j][i][3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] += w.q8[j][i][e & 1];
        if (j == 0) {
          s[i][0] = s0 * c[0];
          s[i][1] = s0 * c[1];
          s[i][2] = s1 * c[2];
          s[i][3] = s1 * c[3];
        } else {
          s[i][0] = fmaf(s0, c[0], s[i][0]);
          s[i][1] = fmaf(s0, c[1], s[i][1]);
          s[i][2] = fmaf(s1, c[2], s[i][2]);
          s[i][3] = fmaf(s1, c[3], s[i][3]);
        }
      }
    }
  }
}

// Adds P V of 16 tokens; p: weights in the layout of the scores, v0, v1: scales of V of the tokens g and g + 8.
template <int D, int NT>
__device__ __forceinline__ void tile_values(const uint8_t* tile, const LaneAt<D>& at, Rows<D, NT>& w, const float (&p)[NT][4],
                                            const uint32_t (&v0)[D / 64], const uint32_t (&v1)[D / 64], bool wild) {
  constexpr int kG = D / 32;
  uint32_t va[kG / 2], vb[kG / 2], vc[kG / 2], vd[kG / 2];  // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
  kv4_lds(tile + at.v, va);
  kv4_lds(tile + at.v + 4 * (D / 2), vb);
  kv4_lds(tile + at.v + 8 * (D / 2), vc);
  kv4_lds(tile + at.v + 12 * (D / 2), vd);
#pragma unroll
  for (int j = 0; j < kG; ++j) {
    const float2 f0 = unpack_half2(v0[j >> 1]), f1 = unpack_half2(v1[j >> 1]);
    const float s0 = j & 1 ? f0.y : f0.x, s1 = j & 1 ? f1.y : f1.x;
    const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
    const uint32_t x = __byte_perm(va[j >> 1], vb[j >> 1], sel), y = __byte_perm(vc[j >> 1], vd[j >> 1], sel);
    const uint32_t x8 = x >> 8, y8 = y >> 8;
    const uint32_t a0 = code_lo(x), a1 = code_hi(x), a2 = code_lo(y), a3 = code_hi(y);
    const uint32_t b0 = code_lo(x8), b1 = code_hi(x8), b2 = code_lo(y8), b3 = code_hi(y8);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float z[4] = {p[i][0] * s0, p[i][1] * s0, p[i][2] * s1, p[i][3] * s1};
      if (wild) {  // a scale is NaN: the rows that do not see it keep out of it
#pragma unroll
        for (int c = 0; c < 4; ++c) z[c] = p[i][c] == 0.0f ? 0.0f : z[c];
      }
      const uint32_t p0 = transpose8x8(pack_half2(z[0], z[1])), p1 = transpose8x8(pack_half2(z[2], z[3]));
      mma16816(w.o[j][0][i], a0, a1, a2, a3, p0, p1);
      mma16816(w.o[j][1][i], b0, b1, b2, b3, p0, p1);
    }
  }
}

// 16 * TILES tokens, the first of them `from`.  sees[i][c]: the last token that the lane's row sees; MASKED: some token is hidden
// from some row or does not exist.
template <int D, int NT, int TILES, bool MASKED>
__device__ __forceinline__ void step(const uint8_t* tiles, const LaneAt<D>& at, Rows<D, NT>& w, const int (&sees)[NT][2], int window,
                                     int from, int n) {
  using S = Shape<D, NT>;
  constexpr int kG = S::kGroups;
  float s[TILES][NT][4];
  uint32_t v0[TILES][kG / 2], v1[TILES][kG / 2];
#pragma unroll
  for (int k = 0; k < TILES; ++k) {
    tile_scores<D, NT>(tiles + k * S::kTileBytes, at, w, s[k]);
    kv4_lds(tiles + k * S::kTileBytes + at.vs, v0[k]);
    kv4_lds(tiles + k * S::kTileBytes + at.vs + 8 * (D / 16), v1[k]);
  }
  if (MASKED) {
#pragma unroll
    for (int k = 0; k < TILES; ++k) {
      const int token = from + 16 * k + at.g;
#pragma unroll
      for (int e = 0; e < kG / 2; ++e) {  // what lies behind the last token is anything
        if (token >= n) v0[k][e] = 0;
        if (token + 8 >= n) v1[k][e] = 0;
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = token + (e < 2 ? 0 : 8), last = sees[i][e & 1];
          if (t > last || (window > 0 && t <= last - window)) s[k][i][e] = -INFINITY;
        }
    }
  }
  uint32_t most = 0;  // two halves
  float high[NT][2];
  bool over = false;
#pragma unroll
  for (int k = 0; k < TILES; ++k)
#pragma unroll
    for (int e = 0; e < kG / 2; ++e) most = __vmaxu2(most, __vmaxu2(v0[k][e], v1[k][e]));
  most = max(most & 0xFFFFu, most >> 16);
  bool wild = false;
  over = most > w.scale_limit || most >= 0x7C00u;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float m = fmaxf(s[0][i][c], s[0][i][c + 2]);
      if (TILES == 2) m = fmaxf(m, fmaxf(s[TILES - 1][i][c], s[TILES - 1][i][c + 2]));
      high[i][c] = m;
      over = over || m > w.limit[i][c];
    }
  if (__any_sync(0xFFFFFFFFu, over)) {
    wild = __any_sync(0xFFFFFFFFu, most >= 0x7C00u);
    if (wild) {
      // What is not finite stays that whatever it is multiplied by; rows that do not see it keep their weights' decimals.
      most = 0;
#pragma unroll
      for (int k = 0; k < TILES; ++k)
#pragma unroll
        for (int e = 0; e < kG / 2; ++e) most = __vmaxu2(most, __vmaxu2(finite_halves(v0[k][e]), finite_halves(v1[k][e])));
      most = max(most & 0xFFFFu, most >> 16);
    }
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (most > w.scale_limit) {
      w.scale_limit = most | 0x3FFu;  // the end of its binade
      w.e = static_cast<float>(static_cast<int>(most >> 10) - 14);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = high[i][c];
        m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 16));
        w.top[i][c] = fmaxf(w.top[i][c], m * w.cs[i][c]);
        const float ref = w.top[i][c] > kFloor ? w.top[i][c] + w.e - kLift : kFloor;
        const float f = exp2_fast(-w.minus_ref[i][c] - ref);
        w.minus_ref[i][c] = -ref;
        w.limit[i][c] = (w.top[i][c] > kFloor ? w.top[i][c] + kHeadroom : kFloor) / w.cs[i][c];
        w.sum[i][c] *= f;
#pragma unroll
        for (int j = 0; j < kG; ++j) {
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            w.o[j][0][i][c + e] *= f;
            w.o[j][1][i][c + e] *= f;
          }
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < TILES; ++k) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[k][i][e] = exp2_fast(fmaf(s[k][i][e], w.cs[i][e & 1], w.minus_ref[i][e & 1]));
        w.sum[i][e & 1] += s[k][i][e];
      }
    tile_values<D, NT>(tiles + k * S::kTileBytes, at, w, s[k], v0[k], v1[k], wild);
  }
}

// Writes four neighbouring values of a row.
__device__ __forceinline__ void put4(__half* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_half2(a, b), pack_half2(c, d));
}

// What joining the parts of a segment has to know of it.
struct Segment {
  int start, end;               // as items; start < 0: no part here
  int h, r, rows, first_token;  // key/value head, block of rows, rows of the sequence, its first row in q
};
template <int D, int NT>
__device__ __forceinline__ Segment segment_of(const Kv4AttnArgs& a, const Place& p) {
  return {p.start, p.end, p.h, p.r, p.s.m * a.group, p.s.first_row_token};
}
// Row `row` of a block in the output tensor; null beyond the sequence's rows.
template <int D, int NT>
__device__ __forceinline__ __half* out_row(const Kv4AttnArgs& a, const Segment& p, int row) {
  row += p.r * Shape<D, NT>::kRows;
  if (row >= p.rows) return nullptr;
  const int token = row / a.group, head = p.h * a.group + row - token * a.group;
  return a.out + (p.first_token + token) * a.out_stride + static_cast<long long>(head) * D;
}

// Ends a warp's part of a segment: `slot` null: it is the whole segment, the rows are written out; else the values as they
// are, the references and the sums go to the slot.
template <int D, int NT>
__device__ __forceinline__ void finish(const Kv4AttnArgs& a, const Segment& p, const LaneAt<D>& at, Rows<D, NT>& w, float* slot) {
  using S = Shape<D, NT>;
  const int g = at.g, t = at.t;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = w.sum[i][c];
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 4);
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
      const int row = 8 * i + 2 * t + c;
      float inv = kCodeUnit;
      __half* dst = nullptr;
      if (slot == nullptr) {
        dst = out_row<D, NT>(a, p, row);
        inv = l > 0.0f || l != l ? kCodeUnit / l : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < S::kGroups; ++j) {
        const float x0 = w.o[j][0][i][c] * inv, x1 = w.o[j][0][i][c + 2] * inv;
        const float x2 = w.o[j][1][i][c] * inv, x3 = w.o[j][1][i][c + 2] * inv;
        if (slot != nullptr)
          *reinterpret_cast<float4*>(slot + row * S::kRecord + 32 * j + 4 * g) = make_float4(x0, x1, x2, x3);
        else if (dst != nullptr)
          put4(dst + 32 * j + 4 * g, x0, x1, x2, x3);
      }
      if (slot != nullptr && g == 0) {
        slot[row * S::kRecord + D] = -w.minus_ref[i][c];
        slot[row * S::kRecord + D + 1] = l;
      }
    }
}

// Adds `count` records of one row in shared memory (at `first`, then at `rest` and every `step` floats behind it), a warp together:
// lane l has values l VALUES.. of the row, not yet divided by `sum`.
template <int D>
struct Joined {
  static constexpr int kValues = D / 32;
  float x[kValues];
  float top, sum;
};
template <int D>
__device__ __forceinline__ void join(Joined<D>& r, const float* first, const float* rest, int step, int count, int lane) {
  constexpr int kV = Joined<D>::kValues;
#pragma unroll 2
  for (int i = 0; i < count; ++i) {
    const float* p = i == 0 ? first : rest + (i - 1) * step;
    const float2 m = *reinterpret_cast<const float2*>(p + D);
    float x[kV];
    if constexpr (kV == 2) {
      const float2 v = reinterpret_cast<const float2*>(p)[lane];
      x[0] = v.x;
      x[1] = v.y;
    } else {
#pragma unroll
      for (int e = 0; e < kV; e += 4) {
        const float4 v = reinterpret_cast<const float4*>(p)[lane * (kV / 4) + e / 4];
        x[e] = v.x;
        x[e + 1] = v.y;
        x[e + 2] = v.z;
        x[e + 3] = v.w;
      }
    }
    const float top = fmaxf(r.top, m.x), f = exp2_fast(r.top - top), g = exp2_fast(m.x - top);
    r.top = top;
    r.sum = fmaf(m.y, g, r.sum * f);
#pragma unroll
    for (int e = 0; e < kV; ++e) r.x[e] = fmaf(x[e], g, r.x[e] * f);
  }
}
template <int D>
__device__ __forceinline__ Joined<D> nothing_joined() {
  Joined<D> r;
  r.top = kFloor;
  r.sum = 0.0f;
#pragma unroll
  for (int e = 0; e < Joined<D>::kValues; ++e) r.x[e] = 0.0f;
  return r;
}
template <int D>
__device__ __forceinline__ void put_row(__half* dst, const Joined<D>& r, int lane) {
  const float inv = r.sum > 0.0f || r.sum != r.sum ? 1.0f / r.sum : 0.0f;
  if constexpr (D == 64) {
    *reinterpret_cast<uint32_t*>(dst + 2 * lane) = pack_half2(r.x[0] * inv, r.x[1] * inv);
  } else {
#pragma unroll
    for (int e = 0; e < D / 32; e += 4) put4(dst + lane * (D / 32) + e, r.x[e] * inv, r.x[e + 1] * inv, r.x[e + 2] * inv, r.x[e + 3] * inv);
  }
}
template <int D>
__device__ __forceinline__ void put_record(float* rec, const Joined<D>& r, int lane) {
  if constexpr (D == 64) {
    reinterpret_cast<float2*>(rec)[lane] = make_float2(r.x[0], r.x[1]);
  } else {
#pragma unroll
    for (int e = 0; e < D / 32; e += 4)
      *reinterpret_cast<float4*>(rec + lane * (D / 32) + e) = make_float4(r.x[e], r.x[e + 1], r.x[e + 2], r.x[e + 3]);
  }
  if (lane == 0) {
    rec[D] = r.top;
    rec[D + 1] = r.sum;
  }
}

// The first item of CTA i of n.
struct Shares {
  int each, rest, n;
  __device__ __forceinline__ Shares(int items, int n_) : each(items / n_), rest(items % n_), n(n_) {}
  __device__ __forceinline__ int begin(int i) const { return each * i + rest * i / n; }
  __device__ __forceinline__ int holder(int item) const {
    int i = min(n - 1, static_cast<int>(static_cast<float>(item) / (static_cast<float>(each) + static_cast<float>(rest) / n)));
    while (i > 0 && begin(i) > item) --i;
    while (i + 1 < n && begin(i + 1) <= item) ++i;
    return i;
  }
};

template <int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
  using S = Shape<D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* const ring_all = smem;                                                                 // [WARPS][kStages][kStageBytes]
  float* const slots = reinterpret_cast<float*>(smem + WARPS * S::kStages * S::kStageBytes);      // [WARPS][kRows][kRecord]
  uint64_t* const bars_all = reinterpret_cast<uint64_t*>(slots + WARPS * S::kRows * S::kRecord);  // [WARPS][kStages]
  Segment* const segs = reinterpret_cast<Segment*>(bars_all + WARPS * S::kStages);                // [WARPS][2]: segments of the slots
  int* const prefix = reinterpret_cast<int*>(segs + 2 * WARPS);                                   // [batch]
  __shared__ int warp_items[WARPS], warp_segs[WARPS];
  __shared__ int is_last[2];
  __shared__ uint64_t join_bar;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* const ring = ring_all + warp * S::kStages * S::kStageBytes;
  uint64_t* const bars = bars_all + warp * S::kStages;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < S::kStages; ++i) mbar_init(bars + i, 1);
    segs[2 * warp].start = segs[2 * warp + 1].start = -1;
    if (warp == 0) mbar_init(&join_bar, 1);
    fence_barrier_init();
  }
  pdl_wait();
  // ---- how many items lie ahead of each sequence
  int items = 0, segments = 0;
  bool deal;  // evenly over all CTAs
  {
    const int per = (a.batch + WARPS * 32 - 1) / (WARPS * 32);
    const int b0 = threadIdx.x * per, b1 = min(a.batch, b0 + per);
    int mine = 0, mine_segs = 0;
    bool mine_long = false;
    for (int b = b0; b < b1; ++b) {
      const Span s = span_of<D, NT>(a, b);
      if (blockIdx.x == 0 && !kv4_fits(a, b, {s.n, s.m, s.first_row_token})) atomicExch(a.error, kErrLength);
      mine += a.kv_heads * s.blocks * s.chunks;
      mine_segs += a.kv_heads * s.blocks;
      mine_long = mine_long || (s.blocks > 0 && s.chunks > 3 * WARPS);
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += v;
    }
    mine_segs = __reduce_add_sync(0xFFFFFFFFu, mine_segs);
    if (lane == 31) {
      warp_items[warp] = incl;
      warp_segs[warp] = mine_segs;
    }
    deal = __syncthreads_or(mine_long);
    int ahead = incl - mine;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i < warp) ahead += warp_items[i];
      items += warp_items[i];
      segments += warp_segs[i];
    }
    for (int b = b0; b < b1; ++b) {
      prefix[b] = ahead;
      if (per > 1) {
        const Span s = span_of<D, NT>(a, b);
        ahead += a.kv_heads * s.blocks * s.chunks;
      }
    }
    __syncthreads();
  }
  if (items == 0) return;
  // Where no segment has more than three chunks a warp, a CTA takes whole ones: joining parts through the workspace takes longer than
  // the chunks that are dealt out unevenly.  Whole / dealt, us, 8 heads of 128, one sequence of 36 chunks among 17 of one: 12.3 / 13.2,
  // of 48: 14.0 / 13.4, of 144: 27 / 15; 18 sequences of 25: 11.3 / 17.2; one alone of 36: 12.3 / 12.5.  Else a CTA's warps have a
  // chunk each at least.
  const bool snap = !deal && segments <= static_cast<int>(gridDim.x);
  const int ctas = min(static_cast<int>(gridDim.x), snap ? segments : (items + WARPS - 1) / WARPS);
  const int cta = blockIdx.x;
  if (cta >= ctas) return;
  const Shares shares(items, ctas);
  int lo = shares.begin(cta), hi = shares.begin(cta + 1);
  if (snap) {
    lo = locate<D, NT>(a, prefix, lo).start;
    if (hi < items) hi = locate<D, NT>(a, prefix, hi).start;
  }
  // warps without items are the last ones, so that the parts of a segment are neighbours
  const int base = (hi - lo) / WARPS, extra = (hi - lo) % WARPS;
  const int wlo = lo + warp * base + min(warp, extra), whi = wlo + base + (warp < extra ? 1 : 0);

  // ---- streaming
  if (wlo < whi) {
    Place pi;  // where copies are asked for
    pi.end = wlo;
    int ii = wlo, window = 0, run = 0;
    const uint8_t* src = nullptr;
    const LaneAt<D> at(lane);
    // Lane l looks up every 32nd tile of a segment and brings it when its chunk's turn comes, with the tiles of the chunk behind it
    // that lie in the same page.
    const auto look_up = [&]() {
      window = (pi.s.c0 + pi.c) * S::kTiles;
      const int tile = window + lane, tiles = (pi.s.n + kv4::kTile - 1) / kv4::kTile;
      run = 0;
      if (tile < tiles) {
        const int page = tile / a.page_tiles, in_page = tile - page * a.page_tiles, in_chunk = lane % S::kTiles;
        if (in_page == 0 || in_chunk == 0) {
          int pid = __ldg(a.table + static_cast<long long>(pi.b) * a.max_pages + page);
          if (pid < 0 || pid >= a.pages) {
            atomicExch(a.error, kErrPage);
            pid = 0;
          }
          run = min(min(a.page_tiles - in_page, S::kTiles - in_chunk), tiles - tile);
          src = a.pool + ((static_cast<long long>(pid) * a.kv_heads + pi.h) * a.page_tiles + in_page) * S::kTileBytes;
        }
      }
    };
    const auto next = [&]() {
      if (ii == pi.end) {
        pi = locate<D, NT>(a, prefix, ii);
        look_up();
      } else {
        ++pi.c;
        if ((pi.s.c0 + pi.c) * S::kTiles == window + 32) look_up();
      }
    };
    const auto ask = [&](int stage) {
      const int tile0 = (pi.s.c0 + pi.c) * S::kTiles, first = tile0 - window;
      const int there = min(S::kTiles, max(0, (pi.s.n + kv4::kTile - 1) / kv4::kTile - tile0));
      if (lane == 0) mbar_arrive_expect_tx(bars + stage, there * S::kTileBytes);
      __syncwarp();
      if (run > 0 && lane >= first && lane < first + S::kTiles)
        bulk_load_1d(ring + stage * S::kStageBytes + (lane - first) * S::kTileBytes, src, run * S::kTileBytes, bars + stage);
      if (++ii < whi) next();
    };
    next();
    Rows<D, NT> w;
    Place p;
    int stage = 0, phase = 0, asked = 0, sees[NT][2], whole_lo = 0, whole_hi = 0, first_lo = 0, sees_hi = 0, token = 0;
    bool alive = true;
    p.end = wlo;
    const auto ask_ahead = [&](int item) {
#pragma unroll 1
      while (alive && ii < whi && ii < item + S::kStages) {
        ask(asked);
        if (++asked == S::kStages) asked = 0;
      }
    };
    const auto release = [&]() {
      fence_proxy_async();  // the reads come ahead of the next copy's writes
      __syncwarp();
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
      token += S::kChunk;
    };
#pragma unroll 1
    for (int item = wlo; item < whi;) {
      ask_ahead(item);
      if (item == p.end) {
        p = locate<D, NT>(a, prefix, item);
        load_q<D, NT>(a, p, at, w);
        w.clear();
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int row = min(p.r * S::kRows + 8 * i + 2 * at.t + c, p.s.m * a.group - 1);
            sees[i][c] = p.s.n - p.s.m + row / a.group;
          }
        const int sees_lo = p.s.n - p.s.m + p.r * S::kRows / a.group;
        sees_hi = p.s.n - p.s.m + min(p.r * S::kRows + S::kRows - 1, p.s.m * a.group - 1) / a.group;
        // chunks that begin in [whole_lo, whole_hi] are seen by all rows; tokens in (first_lo, sees_hi] by any
        whole_lo = a.window > 0 ? sees_hi - a.window + 1 : 0;
        whole_hi = sees_lo - S::kChunk + 1;
        first_lo = a.window > 0 ? sees_lo - a.window + 1 : 0;
        token = (p.s.c0 + p.c) * S::kChunk;
      }
      const int end = min(p.end, whi);
      // A loop of its own for chunks that all rows see: one for both kinds moves the accumulators between registers where its
      // branches meet.
#pragma unroll 1
      while (item < end && token >= whole_lo && token <= whole_hi) {
        // the warp gives up together: what follows needs all of its lanes
        if (alive) alive = __all_sync(0xFFFFFFFFu, mbar_wait(bars + stage, phase));
        if (!alive) break;
#pragma unroll
        for (int k = 0; k < S::kTiles; k += S::kStep)
          step<D, NT, S::kStep, false>(ring + stage * S::kStageBytes + k * S::kTileBytes, at, w, sees, 0, 0, 0);
        release();
        ++item;
        ask_ahead(item);
      }
      if (item < end) {
        if (alive) alive = __all_sync(0xFFFFFFFFu, mbar_wait(bars + stage, phase));
#pragma unroll 1
        for (int k = 0; k < S::kTiles; k += S::kStep) {
          const int from = token + k * kv4::kTile;
          if (!alive || from > sees_hi || from + S::kStep * kv4::kTile <= first_lo) continue;
          step<D, NT, S::kStep, true>(ring + stage * S::kStageBytes + k * S::kTileBytes, at, w, sees, a.window, from, p.s.n);
        }
        release();
        ++item;
      }
      if (item < p.end && item < whi) continue;
      // a segment that ends here and began here is done; else its part goes to the warp's slot: the ring's place for one that
      // began here (nothing is asked for any more), a place of its own for one that began before
      const Segment seg = segment_of<D, NT>(a, p);
      const int which = p.start >= wlo ? 1 : 0;
      float* slot = nullptr;
      if (p.start < wlo || p.end > whi) {
        slot = which ? reinterpret_cast<float*>(ring) : slots + warp * S::kRows * S::kRecord;
        if (lane == 0) segs[2 * warp + which] = seg;
      }
      finish<D, NT>(a, seg, at, w, slot);
    }
    if (!alive && lane == 0) {
      atomicExch(a.error, kErrWait);
      const int n = ii - wlo;  // copies in flight end before the shared memory does
      for (int s = 0; s < S::kStages; ++s) mbar_wait(bars + s, ring_last_phase(s, n % S::kStages, n / S::kStages & 1));
    }
  }
  __syncthreads();

  // ---- segments that warps share: tasks (run of slots of one segment, row) dealt out to the warps
  // Lane l looks at slot l.  A run begins at a slot whose segment the warp before does not end with, and goes on over the [0] slots
  // of the following warps.
  const int my_start = lane < 2 * WARPS ? segs[lane].start : -1, my_end = lane < 2 * WARPS ? segs[lane].end : 0;
  const int one_before = __shfl_up_sync(0xFFFFFFFFu, my_start, 1), two_before = __shfl_up_sync(0xFFFFFFFFu, my_start, 2);
  const unsigned slots_used = __ballot_sync(0xFFFFFFFFu, my_start >= 0);
  const unsigned begins = __ballot_sync(0xFFFFFFFFu, my_start >= 0 && ((lane & 1) || lane < 2 || max(one_before, two_before) != my_start));
  const unsigned before = __ballot_sync(0xFFFFFFFFu, my_start >= 0 && my_start < lo);
  const unsigned beyond = __ballot_sync(0xFFFFFFFFu, my_start >= lo && my_end > hi);
  // the slots of the segments that other CTAs share: [0] began before, [1] begins here
  const int shared0 = before ? __ffs(before) - 1 : -1, shared1 = beyond ? __ffs(beyond) - 1 : -1;
  const int runs = __popc(begins);
#pragma unroll 1
  for (int task = warp; task < runs * S::kRows; task += WARPS) {
    const int slot = __fns(begins, 0, task / S::kRows + 1), row = task % S::kRows;
    const unsigned behind = slot == 31 ? 0u : begins >> (slot + 1) << (slot + 1);
    const unsigned until = behind ? (1u << (__ffs(behind) - 1)) - 1u : 0xFFFFFFFFu;
    const int parts = __popc(slots_used & until & ~((1u << slot) - 1u));
    const Segment p = segs[slot];
    // the first part may lie in a ring, the others are in the slots, one after the other
    const float* first = (slot & 1 ? reinterpret_cast<const float*>(ring_all + (slot / 2) * S::kStages * S::kStageBytes)
                                   : slots + (slot / 2) * S::kRows * S::kRecord) + row * S::kRecord;
    Joined<D> r = nothing_joined<D>();
    join<D>(r, first, slots + ((slot / 2 + 1) * S::kRows + row) * S::kRecord, S::kRows * S::kRecord, parts, lane);
    if (p.start >= lo && p.end <= hi) {
      __half* dst = out_row<D, NT>(a, p, row);
      if (dst != nullptr) put_row<D>(dst, r, lane);
    } else {
      put_record<D>(a.part + ((static_cast<long long>(cta) * 2 + (p.start >= lo ? 1 : 0)) * S::kRows + row) * S::kRecord, r, lane);
    }
  }
  if (shared0 < 0 && shared1 < 0) return;

  // ---- segments that CTAs share: the last of them joins
  __threadfence();
  __syncthreads();
  if (threadIdx.x < 2) {
    const int slot = threadIdx.x ? shared1 : shared0;
    int last = 0;
    if (slot >= 0) {
      const int c0 = shares.holder(segs[slot].start), c1 = shares.holder(segs[slot].end - 1);
      const int parts = c1 - c0 + 1;
      if (atomicAdd(a.tickets + c0, 1) == parts - 1) {
        a.tickets[c0] = 0;
        last = parts << 10 | (c0 + 1);
      }
    }
    is_last[threadIdx.x] = last;
  }
  __syncthreads();
  if (is_last[0] == 0 && is_last[1] == 0) return;
  // All parts come into the rings' place at once, by bulk copies: they lie far away (a trip takes a microsecond).
  __threadfence();
  asm volatile("fence.proxy.async;" ::: "memory");
  constexpr int kRoom = WARPS * S::kStages * S::kStageBytes / S::kSlotBytes < 32 ? WARPS * S::kStages * S::kStageBytes / S::kSlotBytes : 32;
  int phase = 0;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    if (is_last[which] == 0) continue;
    const int parts = is_last[which] >> 10, c0 = (is_last[which] & 1023) - 1;
    const Segment p = segs[which ? shared1 : shared0];
    static_assert(S::kRows <= 2 * WARPS, "two rows to a warp at most");
    Joined<D> r[2] = {nothing_joined<D>(), nothing_joined<D>()};
#pragma unroll 1
    for (int base = 0; base < parts; base += kRoom) {
      const int n = min(kRoom, parts - base);
      if (warp == 0) {
        if (lane == 0) mbar_arrive_expect_tx(&join_bar, n * S::kSlotBytes);
        __syncwarp();
        // the first part is a [1] record, the others are [0] records of the CTAs behind it
        const int part = base + lane;
        if (lane < n)
          bulk_load_1d(ring_all + lane * S::kSlotBytes,
                       a.part + (static_cast<long long>(c0 + part) * 2 + (part == 0 ? 1 : 0)) * S::kRows * S::kRecord, S::kSlotBytes, &join_bar);
      }
      const bool there = __all_sync(0xFFFFFFFFu, mbar_wait(&join_bar, phase));
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = warp + k * WARPS;
        if (row >= S::kRows || !there) break;
        const float* from = reinterpret_cast<const float*>(ring_all) + row * S::kRecord;
        join<D>(r[k], from, from + S::kRows * S::kRecord, S::kRows * S::kRecord, n, lane);
      }
      if (!__syncthreads_and(there)) {
        if (!there && lane == 0) atomicExch(a.error, kErrWait);
        mbar_wait(&join_bar, phase);  // copies in flight end before the shared memory does
        return;
      }
      phase ^= 1;
      asm volatile("fence.proxy.async;" ::: "memory");
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int row = warp + k * WARPS;
      if (row >= S::kRows) break;
      __half* dst = out_row<D, NT>(a, p, row);
      if (dst != nullptr) put_row<D>(dst, r[k], lane);
    }
  }
}

template <int D, int NT, int WARPS>
size_t attn_smem(int batch) {
  using S = Shape<D, NT>;
  return static_cast<size_t>(WARPS) * (S::kStages * S::kStageBytes + S::kSlotBytes + 8 * S::kStages + 2 * sizeof(Segment)) + 4 * static_cast<size_t>(batch);
}

template <int D, int NT, int WARPS>
int launch_attn_t(const Kv4AttnArgs& a, int grid, cudaStream_t stream) {
  static bool configured[kMaxDevices];
  int dev;
  const size_t most = attn_smem<D, NT, WARPS>(kKv4MaxBatch);
  static_assert(Shape<D, NT>::kSlotBytes <= Shape<D, NT>::kStages * Shape<D, NT>::kStageBytes, "a slot fits a ring");
  if (needs_configure(configured, &dev)) {
    MLD_CUDA_CHECK(cudaFuncSetAttribute(kv4_attn_kernel<D, NT, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)));
    if (dev >= 0) configured[dev] = true;
  }
  MLD_CUDA_CHECK(launch_overlapped(kv4_attn_kernel<D, NT, WARPS>, dim3(grid), dim3(WARPS * 32), attn_smem<D, NT, WARPS>(a.batch), stream, a));
  MLD_LAUNCH_CHECK();
  return MLD_OK;
}

// The pieces of work of a call are counted in 32 bits in this kernel, whatever row ranges the device holds: every sequence may have as
// many rows as any.
bool countable(const mld_kv4_attn_desc& d, const Kv4AttnArgs& a) {
  const double tiles = static_cast<double>(d.max_pages) * (d.cache.page_tokens / kv4::kTile);
  return tiles * a.batch * d.cache.kv_heads * div_up64(static_cast<int64_t>(a.max_queries) * a.group, 8) <= 2147483647.0;
}

// Whether a call's rows are worked on here or in blocks of 256 (128 for heads of 256) on the tensor cores.  64 tokens cost this
// kernel a time in proportion to `small`, heads x blocks of 16 rows (8 for heads of 256), spread over all SMs.
// The other kernel takes a time in proportion to `large`, heads x its blocks, and about 40 us for cutting and joining them, which
// are worth more or less of `small` with the tokens that a sequence has; the host does not know them, and 8192 are assumed.  Both
// sides, us, for 4608 and 16384 cached tokens: 8 heads of 128, 64 rows 24 / 44 and 42 / 65, 128 rows 34 / 45 and 69 / 66, 256 rows 47
// / 49 and 116 / 69, 512 rows 76 / 50 and 211 / 82; 32 heads of 128 (8 x 4 sequences), 64 rows 39 / 54 and 86 / 151, 128 rows 57 / 55
// and 152 / 151; 8 heads of 64, 256 rows 34 / 36 and 68 / 53, 512 rows 48 / 39 and 113 / 68; 2 heads of 256, 256 rows 36 / 52 and 84 /
// 83, 512 rows 54 / 55 and 151 / 88.
// Where sequences are too short to be cut, that kernel's time is a fixed one per wave of its blocks, of which one walks all tokens.
// Both sides, us, 4096 tokens: 8 heads of 128, 512 rows 70 / 85, 1024 rows 119 / 85; 32 heads, 128 rows 58 / 83, 256 rows 96 / 85; 64
// heads of 64, 128 rows 57 / 75, 256 rows 85 / 76; 8 heads of 256, 256 rows 67 / 127, 1024 rows 213 / 128.
bool few_rows(const mld_kv4_attn_desc& d, const Kv4AttnArgs& a, int sms, bool cut) {
  if (!countable(d, a)) return false;
  const int dim = d.cache.head_dim;
  const auto heads_blocks = [&](int rows) { return a.kv_heads * kv4_blocks(a.batch, a.max_queries, a.q_tokens, a.group, rows); };
  const int64_t small = heads_blocks(dim == 256 ? 8 : 16), large = heads_blocks(dim == 256 ? 128 : 256);
  if (cut) return dim == 64 ? small <= 4.5 * large + 150 : dim == 128 ? small <= 2.6 * large + 104 : small <= 2.7 * large + 75;
  return small <= (dim == 64 ? 1000 : dim == 128 ? 450 : 500) * div_up64(large, sms);
}

}  // namespace
}  // namespace mld

using namespace mld;

struct mld_kv4_attn_plan {
  mld_kv4_attn_desc d;
  int device, grid, slots;
  uint8_t* workspace;
  size_t bytes;
  float* part;
  int *tickets, *error;
  int4* pieces;  // null where no sequence can be long enough to be cut
};

extern "C" {

int mld_kv4_attn_plan_create(const mld_kv4_attn_desc* d, mld_kv4_attn_plan** out) {
  MLD_REQUIRE(d != nullptr && out != nullptr, "null argument");
  if (const int rc = check_kv4_desc(&d->cache); rc != MLD_OK) return rc;
  MLD_REQUIRE(d->heads >= 1 && d->heads % d->cache.kv_heads == 0, "heads must be a multiple of the cache's kv_heads");
  MLD_REQUIRE(d->heads <= 4096, "at most 4096 heads");
  MLD_REQUIRE(d->max_batch >= 1 && d->max_batch <= kKv4MaxBatch, "max_batch must be 1 to 1024");
  MLD_REQUIRE(d->max_pages >= 1 && static_cast<int64_t>(d->max_pages) * d->cache.page_tokens <= 0x7FFFFFFF,
              "a sequence holds 1 to 2^31 - 1 tokens in whole pages");
  MLD_REQUIRE(d->force_path >= MLD_KV4_PATH_AUTO && d->force_path <= MLD_KV4_PATH_MANY_ROWS, "bad force_path");
  MLD_REQUIRE(d->window >= 0, "window must not be negative (0: none)");
  MLD_REQUIRE(isfinite(d->scale) && d->scale >= 0.0f, "scale must be a finite positive number (0: 1 / sqrt(head_dim))");
  mld_kv4_attn_plan* p = new (std::nothrow) mld_kv4_attn_plan();
  MLD_REQUIRE(p != nullptr, "out of host memory");
  p->d = *d;
  p->device = d->device;
  if (p->device < 0 && cudaGetDevice(&p->device) != cudaSuccess) p->device = -1;
  const auto fail = [&](const char* what) {
    set_last_error(what, cudaGetLastError());
    mld_kv4_attn_plan_destroy(p);
    return MLD_CUDA_ERROR;
  };
  int before = -1;
  if (cudaGetDevice(&before) != cudaSuccess) return fail("cudaGetDevice");
  if (cudaSetDevice(p->device) != cudaSuccess) {
    cudaSetDevice(before);
    return fail("cudaSetDevice");
  }
  p->grid = sm_count(p->device);
  if (p->grid > kMaxGrid) p->grid = kMaxGrid;
  size_t part = static_cast<size_t>(p->grid) * 2 * 16 * (d->cache.head_dim + 4) * sizeof(float), pieces = 0;
  if (d->force_path != MLD_KV4_PATH_FEW_ROWS && kv4_can_cut(static_cast<int64_t>(d->max_pages) * d->cache.page_tokens)) {
    p->slots = p->grid * kKv4Slots;
    part = std::max(part, p->slots * kv4_slot_bytes(d->cache.head_dim));
    pieces = (kKv4MaxEntries + p->slots) * sizeof(int4);
  }
  const size_t words = (kTickets + 1) * sizeof(int);
  p->bytes = part + pieces + words;
  const bool made = cudaMalloc(&p->workspace, p->bytes) == cudaSuccess && zero_now(p->workspace + part + pieces, words) == cudaSuccess;
  cudaSetDevice(before);
  if (!made) return fail("workspace of the attention plan");
  p->part = reinterpret_cast<float*>(p->workspace);
  p->pieces = pieces > 0 ? reinterpret_cast<int4*>(p->workspace + part) : nullptr;
  p->tickets = reinterpret_cast<int*>(p->workspace + part + pieces);
  p->error = p->tickets + kTickets;
  *out = p;
  return MLD_OK;
}

int mld_kv4_attn_plan_destroy(mld_kv4_attn_plan* plan) {
  if (plan != nullptr && plan->workspace != nullptr) cudaFree(plan->workspace);
  delete plan;
  return MLD_OK;
}

size_t mld_kv4_attn_plan_workspace_bytes(const mld_kv4_attn_plan* plan) { return plan != nullptr ? plan->bytes : 0; }

int mld_kv4_attn_plan_device_status(mld_kv4_attn_plan* plan, int32_t* code) {
  MLD_REQUIRE(plan != nullptr && code != nullptr, "null argument");
  *code = 0;
  // The plan's device, which need not be the current one, is what has to be idle while its words are read and cleared.
  int before = -1;
  MLD_CUDA_CHECK(cudaGetDevice(&before));
  MLD_CUDA_CHECK(cudaSetDevice(plan->device));
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(code, plan->error, sizeof(int), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && *code != 0) e = zero_now(plan->tickets, (kTickets + 1) * sizeof(int));
  cudaSetDevice(before);
  MLD_CUDA_CHECK(e);
  if (*code == 0) return MLD_OK;
  if (*code == kErrPage) {
    set_last_error_text("a page table names a page that the pool does not have");
    return MLD_OUT_OF_RANGE;
  }
  if (*code == kErrLength) {
    set_last_error_text("a sequence is longer than its page table, or q_starts do not fit max_queries and q_tokens");
    return MLD_OUT_OF_RANGE;
  }
  set_last_error_text("a bounded device-side wait of the attention gave up");
  return MLD_TIMEOUT;
}

int mld_kv4_attn_run(mld_kv4_attn_plan* plan, const mld_kv4_attn_io* io, void* stream_v) {
  MLD_REQUIRE(plan != nullptr && io != nullptr, "null argument");
  const mld_kv4_attn_desc& d = plan->d;
  int device = -1;
  MLD_CUDA_CHECK(cudaGetDevice(&device));
  MLD_REQUIRE(device == plan->device, "the plan belongs to another device than the current one");
  MLD_REQUIRE(io->batch >= 0 && io->batch <= d.max_batch, "batch exceeds the plan's max_batch");
  MLD_REQUIRE(io->q_tokens >= 0 && io->max_queries >= 0, "bad query count");
  if (io->batch == 0 || io->q_tokens == 0 || io->max_queries == 0) return MLD_OK;
  MLD_REQUIRE(io->q != nullptr && io->out != nullptr && io->pool != nullptr && io->page_table != nullptr && io->lens != nullptr,
              "null tensor");
  MLD_REQUIRE(io->q_starts != nullptr || (io->q_tokens == io->batch && io->max_queries == 1),
              "without q_starts every sequence has one query token");
  MLD_REQUIRE(io->max_queries <= io->q_tokens, "max_queries exceeds q_tokens");
  const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  MLD_REQUIRE(aligned(io->q) && aligned(io->out) && aligned(io->pool), "tensors must be 16-byte aligned");
  const int64_t width = static_cast<int64_t>(d.heads) * d.cache.head_dim;
  MLD_REQUIRE(io->q_stride % 8 == 0 && io->out_stride % 8 == 0, "token strides must be multiples of 16 bytes");
  MLD_REQUIRE(io->q_tokens == 1 || (io->q_stride >= width && io->out_stride >= width),
              "token strides must not be shorter than a token");
  Kv4AttnArgs a = {};
  a.q = static_cast<const __half*>(io->q);
  a.out = static_cast<__half*>(io->out);
  a.q_stride = io->q_stride;
  a.out_stride = io->out_stride;
  a.pool = static_cast<const uint8_t*>(io->pool);
  a.table = io->page_table;
  a.lens = io->lens;
  a.starts = io->q_starts;
  a.batch = io->batch;
  a.max_pages = d.max_pages;
  a.q_tokens = io->q_tokens;
  a.max_queries = io->max_queries;
  a.heads = d.heads;
  a.kv_heads = d.cache.kv_heads;
  a.group = d.heads / d.cache.kv_heads;
  a.page_tiles = d.cache.page_tokens / kv4::kTile;
  a.pages = d.cache.pages;
  // A window that no sequence is longer than hides nothing; differences with the others stay within 32 bits.
  a.window = d.window < static_cast<int64_t>(d.max_pages) * d.cache.page_tokens ? d.window : 0;
  const float scale = d.scale > 0.0f ? d.scale : 1.0f / sqrtf(static_cast<float>(d.cache.head_dim));
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part = plan->part;
  a.tickets = plan->tickets;
  a.pieces = plan->pieces;
  a.slots = plan->slots;
  a.error = plan->error;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const bool cut = plan->pieces != nullptr && kv4_cuts(a, d.cache.head_dim);
  if (!cut) a.pieces = nullptr;
  if (d.force_path == MLD_KV4_PATH_MANY_ROWS || (d.force_path == MLD_KV4_PATH_AUTO && !few_rows(d, a, plan->grid, cut)))
    return launch_kv4_prefill(a, d.cache.head_dim, plan->grid, stream);
  if (!countable(d, a)) {
    set_last_error_text("more work than one call of this path can count: fewer sequences, or a narrower page table");
    return MLD_OUT_OF_RANGE;
  }
  const bool few = static_cast<int64_t>(io->max_queries) * a.group <= 8;
  switch (d.cache.head_dim) {
    case 64:
      return few ? launch_attn_t<64, 1, 12>(a, plan->grid, stream) : launch_attn_t<64, 2, 12>(a, plan->grid, stream);
    case 128:
      return few ? launch_attn_t<128, 1, 12>(a, plan->grid, stream) : launch_attn_t<128, 2, 8>(a, plan->grid, stream);
    default:
      return launch_attn_t<256, 1, 8>(a, plan->grid, stream);
  }
}

}  // extern "C"

// The 4-bit key/value cache: where a value lies, and how it is rounded.
//
// 32 neighbouring values of a head share a scale, the symmetric INT4 form of the weights (nibble q + 8, q in -7..7).  The
// scale is rounded to eight significant bits: times the three bits of a q that gives eleven, so every value of the cache is
// an fp16 number, and a matrix product may take the values as fp16 operands without a rounding of its own.
//
// 16 tokens of a head are a tile of 18 * D contiguous bytes (any run of tiles is one bulk copy, whatever the pages' size):
//   [0, 8 D)     codes of K, a row of D / 2 bytes per token
//   [8 D, 16 D)  codes of V, a row of D / 2 bytes per token, rows in the order of v_row()
//   [16 D, 17 D) scales of K, fp16 [16][D / 32];   [17 D, 18 D) scales of V
// A page is [kv_heads][page_tokens / 16] tiles.  A warp reads a tile's codes from shared memory as operands of m16n8k16 MMAs:
//   K (tokens are rows): lane (g, t) = (lane / 4, lane % 4) takes of rows g and g + 8 the eight values 8 t.. of each group, one
//     word; a row holds the four lanes' pieces one after the other.  In a word value 2 p + h is the nibble 4 h + p, so that
//     masks alone give the pairs (2 p, 2 p + 1) as two halves.
//   V (values are rows, tokens the depth): it takes of the tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 the four values 4 g.. of each
//     group, two bytes per group; a row holds the eight pieces of g = 0..7.
// Rows of V, and pieces within the rows (an exclusive or), are placed so that the lanes of one access hit distinct banks.
#pragma once
#include <stdint.h>

namespace mld {
namespace kv4 {

constexpr int kTile = 16;   // tokens
constexpr int kBlock = 32;  // values that share a scale

__host__ __device__ constexpr int tile_bytes(int d) { return 18 * d; }

// Byte offset of the word that holds values 32 j + 8 t .. + 7 of token tau in the codes of K.
template <int D>
__host__ __device__ __forceinline__ int k_word(int tau, int j, int t) {
  constexpr int kWords = D / 32 < 4 ? D / 32 : 4;
  const int unit = (j / kWords * 4 + t) ^ (D == 256 ? (tau & 1) * 4 : 0);
  return tau * (D / 2) + (unit * kWords + j % kWords) * 4;
}
// The row of token tau in the codes of V.
__host__ __device__ __forceinline__ int v_row(int tau) { return (tau & 8) | (tau & 7) >> 1 | (tau & 1) << 2; }
// Where in its row the piece of values 4 g .. + 3 of all groups lies.
template <int D>
__host__ __device__ __forceinline__ int v_piece(int row, int g) {
  return g ^ (D == 128 ? (row >> 1 & 1) * 4 : D == 256 ? (row & 3) * 2 : 0);
}
// Byte offset, from the start of the tile, of the two bytes that hold values 32 j + 4 g .. + 3 of token tau of V.
template <int D>
__host__ __device__ __forceinline__ int v_half(int tau, int j, int g) {
  const int row = v_row(tau);
  return 8 * D + row * (D / 2) + v_piece<D>(row, g) * (D / 16) + 2 * j;
}
template <int D>
__host__ __device__ __forceinline__ int scale_at(bool v, int tau, int j) {
  return (v ? 17 : 16) * D + (tau * (D / 32) + j) * 2;
}

}  // namespace kv4
}  // namespace mld

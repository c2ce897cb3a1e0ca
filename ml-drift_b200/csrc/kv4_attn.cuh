// Shared by the two attention kernels over the 4-bit cache: arguments and what a sequence has of them.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"
#include "kv4.cuh"
#include "ring_order.h"

namespace mld {

struct Kv4AttnArgs {
  const __half* q;
  __half* out;
  long long q_stride, out_stride;  // elements from token to token
  const uint8_t* pool;
  const int32_t* table;   // [batch][max_pages]
  const int32_t* lens;    // [batch]
  const int32_t* starts;  // [batch + 1], or null: one query token per sequence
  int batch, max_pages, q_tokens, max_queries;
  int heads, kv_heads, group;
  int page_tiles, pages;
  int window;
  float scale_log2;  // log2(e) times the scale of the scores
  float* part;       // few rows: [grid][2][rows][D + 4]; many: [slots][D / 4 + 1][rows of a block][4]
  int* tickets;      // few rows: [grid], many: [slots]; zero between launches
  int4* pieces;      // many rows: [kKv4MaxEntries + slots], or null
  int slots;
  int* error;
};

// Many rows: blocks of rows that may be cut along the cached tokens, in all sequences of a call.
constexpr int kKv4MaxEntries = 4096;
// Pieces of cut blocks that a call may have, for each SM (100 MB of workspace for heads of 128 on 148 SMs).  With 2 in place of 5: 8
// heads of 128, 2048 rows, 65536 tokens 768 us against 635, 4 sequences of 16384 583 against 454.
constexpr int kKv4Slots = 5;
size_t kv4_slot_bytes(int head_dim);
// Blocks of `rows` rows that the sequences of a call have at most, for each key/value head: none has more than `max_queries` tokens, all
// together have `q_tokens`.  (A chunk of a prompt beside single tokens: counted by its own rows, not by them times the batch.)
inline int64_t kv4_blocks(int64_t batch, int64_t max_queries, int64_t q_tokens, int64_t group, int64_t rows) {
  const int64_t alike = batch * div_up64(max_queries * group, rows), together = batch + q_tokens * group / rows;
  return alike < together ? alike : together;
}
// Whether sequences of so many tokens can be long enough for that; whether a call's blocks may be cut.
bool kv4_can_cut(int64_t tokens);
bool kv4_cuts(const Kv4AttnArgs& a, int head_dim);

int launch_kv4_prefill(const Kv4AttnArgs& a, int head_dim, int sms, cudaStream_t stream);

#ifdef __CUDACC__
namespace {

enum { kErrWait = 40, kErrPage = 41, kErrLength = 42 };

struct Kv4Sequence {
  int n, m, first_token;  // cached tokens, queries, the first query's row in q
};
__device__ __forceinline__ Kv4Sequence kv4_sequence(const Kv4AttnArgs& a, int b) {
  Kv4Sequence s;
  const long long most = static_cast<long long>(a.max_pages) * a.page_tiles * kv4::kTile;
  const int len = __ldg(a.lens + b);
  s.n = len < 0 ? 0 : len > most ? static_cast<int>(most) : len;
  s.m = 1;
  s.first_token = b;
  if (a.starts != nullptr) {
    int lo = __ldg(a.starts + b), hi = __ldg(a.starts + b + 1);
    lo = min(max(lo, 0), a.q_tokens);
    hi = min(max(hi, lo), a.q_tokens);
    s.m = min(hi - lo, a.max_queries);
    s.first_token = lo;
  }
  return s;
}
// Whether the sequence's length and queries were what the call allows (they are cut to that otherwise).
__device__ __forceinline__ bool kv4_fits(const Kv4AttnArgs& a, int b, const Kv4Sequence& s) {
  return a.lens[b] == s.n && (a.starts == nullptr || (a.starts[b] >= 0 && a.starts[b + 1] - a.starts[b] == s.m && a.starts[b + 1] <= a.q_tokens));
}

// Words from shared memory as one access.
template <int N>
__device__ __forceinline__ void kv4_lds(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    static_assert(N == 4, "");
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
}

}  // namespace
#endif

}  // namespace mld

// Pages of the 4-bit cache: who holds which (on the host), and their copies (on the GPU, all layers in one launch).
//
// A pager counts the holders of every page.  A fork shares all pages of a sequence; the first append to a shared page that is
// not full takes a page of its own and asks for one copy.  Compacting moves pages from the pool's end into holes before it.
// Both give lists of (from, to) pages in which no page is written twice or read after it is written, so that copies need no
// order among them and a launch takes them all.
#include <new>
#include <vector>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace mld {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kPairs = 480;  // in a launch's arguments, which are limited to 4 KB

struct CopyArgs {
  uint8_t* pool;
  long long layer_bytes, page_bytes;
  int pairs, pieces;  // pieces of a page
  int from[kPairs], to[kPairs];
};

// A block copies UNROLL * 4 KB: every thread has its 16-byte loads in flight before the first store.
// Bound by memory: 101 pages of 32 layers (238 MB read, as much written) 73.9 us, 0.98 of the plain copy's rate; one page of one
// layer 1.1 us, a launch's latency.
template <int UNROLL>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  pdl_wait();
  const int pair = blockIdx.x / a.pieces, piece = blockIdx.x - pair * a.pieces;
  uint8_t* const layer = a.pool + blockIdx.y * a.layer_bytes;
  const uint4* src = reinterpret_cast<const uint4*>(layer + a.from[pair] * a.page_bytes);
  uint4* dst = reinterpret_cast<uint4*>(layer + a.to[pair] * a.page_bytes);
  const long long words = a.page_bytes / 16, at = static_cast<long long>(piece) * UNROLL * kCopyThreads + threadIdx.x;
  uint4 v[UNROLL];
#pragma unroll
  for (int i = 0; i < UNROLL; ++i)
    if (at + i * kCopyThreads < words) v[i] = __ldcs(src + at + i * kCopyThreads);
#pragma unroll
  for (int i = 0; i < UNROLL; ++i)
    if (at + i * kCopyThreads < words) __stcs(dst + at + i * kCopyThreads, v[i]);
}

}  // namespace
}  // namespace mld

using namespace mld;

struct mld_kv4_pager {
  int pages, page_tokens, max_sequences;
  struct Sequence {
    bool open = false;
    int length = 0;
    std::vector<int32_t> table;
  };
  std::vector<int32_t> holders;  // per page
  std::vector<int32_t> spare;    // pages that nobody holds, the lowest last
  std::vector<Sequence> sequences;

  bool has(int32_t s) const { return s >= 0 && s < max_sequences && sequences[s].open; }
  void release(int32_t page) {
    if (--holders[page] == 0) spare.push_back(page);
  }
  int32_t take() {
    const int32_t p = spare.back();
    spare.pop_back();
    holders[p] = 1;
    return p;
  }
};

extern "C" {

int mld_kv4_copy_pages(const mld_kv4_desc* d, void* pool, int32_t layers, int64_t layer_bytes, const int32_t* from,
                       const int32_t* to, int32_t count, void* stream) {
  if (const int rc = check_kv4_desc(d); rc != MLD_OK) return rc;
  MLD_REQUIRE(count >= 0 && layers >= 0, "negative count");
  if (count == 0 || layers == 0) return MLD_OK;
  MLD_REQUIRE(pool != nullptr && from != nullptr && to != nullptr, "null argument");
  MLD_REQUIRE(layers <= 65535, "at most 65535 layers");
  MLD_REQUIRE((reinterpret_cast<uintptr_t>(pool) & 15) == 0, "the pool must be 16-byte aligned");
  const int64_t bytes = static_cast<int64_t>(mld_kv4_page_bytes(d));
  MLD_REQUIRE(layers == 1 || (layer_bytes % 16 == 0 && layer_bytes >= bytes * d->pages),
              "layer_bytes must be a multiple of 16 and no smaller than a layer's pool");
  try {
    std::vector<uint8_t> use(d->pages, 0);  // 1: read, 2: written
    for (int i = 0; i < count; ++i) {
      MLD_REQUIRE(from[i] >= 0 && from[i] < d->pages && to[i] >= 0 && to[i] < d->pages, "page outside the pool");
      MLD_REQUIRE((use[from[i]] & 2) == 0 && use[to[i]] == 0 && from[i] != to[i],
                  "a page that is written must not be read or written by another copy of the list");
      use[from[i]] |= 1;
      use[to[i]] |= 2;
    }
  } catch (const std::bad_alloc&) {
    set_last_error_text("out of host memory");
    return MLD_OUT_OF_RANGE;
  }
  for (int done = 0; done < count; done += kPairs) {
    CopyArgs a;
    a.pool = static_cast<uint8_t*>(pool);
    a.layer_bytes = layer_bytes;
    a.page_bytes = bytes;
    a.pairs = count - done < kPairs ? count - done : kPairs;
    for (int i = 0; i < a.pairs; ++i) {
      a.from[i] = from[done + i];
      a.to[i] = to[done + i];
    }
    constexpr int kUnroll = 4;
    const int64_t pieces = div_up64(bytes, 16 * kCopyThreads * kUnroll);
    MLD_REQUIRE(pieces * a.pairs <= 0x7FFFFFFF, "pages too large");
    a.pieces = static_cast<int>(pieces);
    MLD_CUDA_CHECK(launch_overlapped(copy_pages_kernel<kUnroll>, dim3(a.pairs * a.pieces, layers), dim3(kCopyThreads), 0,
                                     static_cast<cudaStream_t>(stream), a));
    MLD_LAUNCH_CHECK();
  }
  return MLD_OK;
}

int mld_kv4_pager_create(int32_t pages, int32_t page_tokens, int32_t max_sequences, mld_kv4_pager** out) {
  MLD_REQUIRE(out != nullptr, "null argument");
  MLD_REQUIRE(pages >= 1 && max_sequences >= 1 && page_tokens >= 16 && page_tokens % 16 == 0 &&
                  static_cast<int64_t>(pages) * page_tokens <= 0x7FFFFFFF,
              "bad pager size");
  mld_kv4_pager* p = new (std::nothrow) mld_kv4_pager();
  MLD_REQUIRE(p != nullptr, "out of host memory");
  p->pages = pages;
  p->page_tokens = page_tokens;
  p->max_sequences = max_sequences;
  try {
    p->holders.assign(pages, 0);
    p->spare.resize(pages);
    for (int i = 0; i < pages; ++i) p->spare[i] = pages - 1 - i;
    p->sequences.resize(max_sequences);
  } catch (const std::bad_alloc&) {
    delete p;
    set_last_error_text("out of host memory");
    return MLD_OUT_OF_RANGE;
  }
  *out = p;
  return MLD_OK;
}

int mld_kv4_pager_destroy(mld_kv4_pager* pager) {
  delete pager;
  return MLD_OK;
}

int mld_kv4_pager_free_pages(const mld_kv4_pager* pager) { return pager != nullptr ? static_cast<int>(pager->spare.size()) : 0; }

int mld_kv4_pager_open(mld_kv4_pager* pager, int32_t* sequence) {
  MLD_REQUIRE(pager != nullptr && sequence != nullptr, "null argument");
  for (int s = 0; s < pager->max_sequences; ++s) {
    if (pager->sequences[s].open) continue;
    pager->sequences[s].open = true;
    pager->sequences[s].length = 0;
    *sequence = s;
    return MLD_OK;
  }
  set_last_error_text("no sequence left");
  return MLD_OUT_OF_RANGE;
}

int mld_kv4_pager_length(const mld_kv4_pager* pager, int32_t sequence, int32_t* tokens) {
  MLD_REQUIRE(pager != nullptr && tokens != nullptr, "null argument");
  MLD_REQUIRE(pager->has(sequence), "no such sequence");
  *tokens = pager->sequences[sequence].length;
  return MLD_OK;
}

int mld_kv4_pager_table(const mld_kv4_pager* pager, int32_t sequence, int32_t* table, int32_t capacity, int32_t* count) {
  MLD_REQUIRE(pager != nullptr && count != nullptr, "null argument");
  MLD_REQUIRE(pager->has(sequence), "no such sequence");
  const std::vector<int32_t>& t = pager->sequences[sequence].table;
  *count = static_cast<int32_t>(t.size());
  MLD_REQUIRE(capacity >= *count && (table != nullptr || *count == 0), "the table does not fit");
  for (size_t i = 0; i < t.size(); ++i) table[i] = t[i];
  return MLD_OK;
}

int mld_kv4_pager_append(mld_kv4_pager* pager, int32_t sequence, int32_t tokens, int32_t* slots, int32_t* copy_from,
                         int32_t* copy_to, int32_t* copies) {
  MLD_REQUIRE(pager != nullptr && copy_from != nullptr && copy_to != nullptr && copies != nullptr, "null argument");
  MLD_REQUIRE(pager->has(sequence), "no such sequence");
  MLD_REQUIRE(tokens >= 0 && (tokens == 0 || slots != nullptr), "bad token count");
  *copies = 0;
  if (tokens == 0) return MLD_OK;
  mld_kv4_pager::Sequence& s = pager->sequences[sequence];
  const int64_t length = static_cast<int64_t>(s.length) + tokens;
  const int64_t need = (length + pager->page_tokens - 1) / pager->page_tokens;
  const int tail = s.length % pager->page_tokens;
  const bool own_copy = tail != 0 && pager->holders[s.table.back()] > 1;
  if (need - static_cast<int64_t>(s.table.size()) + (own_copy ? 1 : 0) > static_cast<int64_t>(pager->spare.size())) {
    set_last_error_text("no pages left");
    return MLD_OUT_OF_RANGE;
  }
  try {
    s.table.reserve(need);
  } catch (const std::bad_alloc&) {
    set_last_error_text("out of host memory");
    return MLD_OUT_OF_RANGE;
  }
  if (own_copy) {
    const int32_t old = s.table.back(), page = pager->take();
    --pager->holders[old];
    s.table.back() = page;
    *copy_from = old;
    *copy_to = page;
    *copies = 1;
  }
  while (static_cast<int64_t>(s.table.size()) < need) s.table.push_back(pager->take());
  for (int i = 0; i < tokens; ++i) {
    const int at = s.length + i;
    slots[i] = s.table[at / pager->page_tokens] * pager->page_tokens + at % pager->page_tokens;
  }
  s.length = static_cast<int>(length);
  return MLD_OK;
}

int mld_kv4_pager_fork(mld_kv4_pager* pager, int32_t sequence, int32_t* fork) {
  MLD_REQUIRE(pager != nullptr && fork != nullptr, "null argument");
  MLD_REQUIRE(pager->has(sequence), "no such sequence");
  int32_t n;
  if (const int rc = mld_kv4_pager_open(pager, &n); rc != MLD_OK) return rc;
  const mld_kv4_pager::Sequence& s = pager->sequences[sequence];
  try {
    pager->sequences[n].table = s.table;
  } catch (const std::bad_alloc&) {
    pager->sequences[n].open = false;
    set_last_error_text("out of host memory");
    return MLD_OUT_OF_RANGE;
  }
  pager->sequences[n].length = s.length;
  for (const int32_t p : s.table) ++pager->holders[p];
  *fork = n;
  return MLD_OK;
}

int mld_kv4_pager_truncate(mld_kv4_pager* pager, int32_t sequence, int32_t tokens) {
  MLD_REQUIRE(pager != nullptr, "null argument");
  MLD_REQUIRE(pager->has(sequence), "no such sequence");
  mld_kv4_pager::Sequence& s = pager->sequences[sequence];
  MLD_REQUIRE(tokens >= 0 && tokens <= s.length, "a sequence can only be cut to a length that it has");
  const size_t keep = (static_cast<size_t>(tokens) + pager->page_tokens - 1) / pager->page_tokens;
  while (s.table.size() > keep) {
    pager->release(s.table.back());
    s.table.pop_back();
  }
  s.length = tokens;
  return MLD_OK;
}

int mld_kv4_pager_close(mld_kv4_pager* pager, int32_t sequence) {
  if (const int rc = mld_kv4_pager_truncate(pager, sequence, 0); rc != MLD_OK) return rc;
  pager->sequences[sequence].open = false;
  return MLD_OK;
}

int mld_kv4_pager_compact(mld_kv4_pager* pager, int32_t* copy_from, int32_t* copy_to, int32_t capacity, int32_t* copies) {
  MLD_REQUIRE(pager != nullptr && copies != nullptr && capacity >= 0, "bad argument");
  MLD_REQUIRE(capacity == 0 || (copy_from != nullptr && copy_to != nullptr), "null argument");
  try {
    std::vector<int32_t> moved(pager->pages, -1), spare;
    int n = 0, hole = 0, last = pager->pages - 1;
    while (n < capacity) {
      while (hole < pager->pages && pager->holders[hole] > 0) ++hole;
      while (last >= 0 && pager->holders[last] == 0) --last;
      if (hole >= last) break;
      copy_from[n] = last;
      copy_to[n] = hole;
      moved[last] = hole;
      ++n;
      ++hole;
      --last;
    }
    spare.reserve(pager->pages);
    for (int i = 0; i < n; ++i) {
      pager->holders[copy_to[i]] = pager->holders[copy_from[i]];
      pager->holders[copy_from[i]] = 0;
    }
    for (auto& s : pager->sequences)
      for (int32_t& p : s.table)
        if (moved[p] >= 0) p = moved[p];
    for (int p = pager->pages - 1; p >= 0; --p)
      if (pager->holders[p] == 0) spare.push_back(p);
    pager->spare.swap(spare);
    *copies = n;
  } catch (const std::bad_alloc&) {
    set_last_error_text("out of host memory");
    return MLD_OUT_OF_RANGE;
  }
  return MLD_OK;
}

}  // extern "C"

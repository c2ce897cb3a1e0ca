// The block of the experts' products for few rows: its warps, its ring of boxes and what is kept of the items under way, as plain
// numbers, which the kernel and a model of its roles that runs on the host share.
#pragma once

#include <stddef.h>

namespace mld {

constexpr int kFewRows = 8;            // of a tile at most: the columns of a fragment
constexpr int kFewOutputs = 64;        // of an item
constexpr int kFewInputs = 128;        // of a box
constexpr int kFewCopyWarps = 4;
constexpr int kFewSumWarps = 4;
constexpr int kFewBoxBytes = kFewInputs / 4 * 128;  // 128 bytes of every input slice: 64 outputs in 4 bits, 32 in 8
// Items that something is kept for (where their rows are; barriers).  Of items of one box, the first copying warp may be a ring of boxes
// ahead of one that a multiplying warp has given back, which may have two parts that nobody has read and a third one in hand, while
// another one still reads the rows of an item before all of these; and it has a box in every fourth item only, and goes through
// those between without waiting.  Of items of more boxes that makes fewer.
constexpr int kFewItemBars = 128;
constexpr int kFewRoom = 226 * 1024;   // shared memory

// Places of the ring are a multiple of the multiplying warps, so that a place is always the same warp's, which then waits for
// each of the place's boxes in turn.  (A wait tells a box from the one before it and no more: a warp that took another one's
// place could take an old box for its own.)
template <int BITS>
struct FewShape {
  static constexpr int kWarps = 8;
  static constexpr int kThreads = 32 * (kFewCopyWarps + kWarps + kFewSumWarps);
  static constexpr int kWBytes = kFewBoxBytes * (BITS == 4 ? 1 : 2);
  static constexpr int kScaleBytes = 4 * kFewOutputs * 2;        // four rows at most
  static constexpr int kStage = kWBytes + kScaleBytes;
  static constexpr int kPart = 8 * 32;                           // float2s of a part
  static constexpr int kPlaces = 2;                              // for a warp's parts
  static constexpr int kPartBytes = kWarps * kPlaces * kPart * 8;
  static constexpr int kRowBytes = kFewItemBars * kFewRows * 8;  // where the rows of the items under way are
  static constexpr int kStages = (kFewRoom - 4 * 1024 - kPartBytes - kRowBytes) / kStage / kWarps * kWarps;
  static constexpr size_t kSmem =
      1024 + static_cast<size_t>(kStages) * kStage + kPartBytes + kRowBytes + (2 * kStages + 2 * kFewItemBars + kWarps * kPlaces) * 8;
  static_assert(kStages >= kWarps && kStages % kFewCopyWarps == 0 && kSmem <= 227 * 1024, "shared memory");
  static_assert(kStages + (kPlaces + 1) * kWarps + kFewCopyWarps <= kFewItemBars, "what is kept of the items under way");
};

}  // namespace mld

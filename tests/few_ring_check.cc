// The roles of the kernel for few rows go through the items of a block (warps that copy boxes, warps that multiply them, warps that
// sum their parts up), one of the multiplying warps, or the summing ones, held up at an item while all others run as far as they get.
// few_ring_check <bits> <boxes of an item>: 0 if what is kept for that item is not given to another meanwhile, 1 and the first
// fault otherwise.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "few_ring.h"

template <int BITS>
int check(int boxes) {
  using S = mld::FewShape<BITS>;
  constexpr int kWarps = S::kWarps, kCopy = mld::kFewCopyWarps, kBars = mld::kFewItemBars;
  const int sharing = std::min(boxes, kWarps);
  for (int held = 0; held <= kWarps; ++held) {  // the multiplying warp that is held up; kWarps: those that sum
    for (int at = 0; at < 3 * kBars; ++at) {    // the item that it is held up at
      struct Role {
        long item = 0;
        int box = 0;     // the next of the item's boxes for this role
        long boxes = 0;  // so far
        long parts = 0;  // handed over so far
        bool published = false;
      };
      std::vector<Role> copy(kCopy), product(kWarps);
      for (int c = 0; c < kCopy; ++c) copy[c].box = c;
      for (int w = 0; w < kWarps; ++w) product[w].box = w;
      std::vector<char> issued(1, 0), used(1, 0);  // boxes by number
      const auto has = [](std::vector<char>& v, long i) -> char& {
        if (i >= static_cast<long>(v.size())) v.resize(i + 1, 0);
        return v[i];
      };
      std::vector<long> read(kWarps, 0);  // parts of a warp that have been read
      std::vector<int> whole(1, 0);       // parts of an item that are there
      long summed = 0, published = -1;
      const long end = at + 40L * kBars;  // (nobody gets there past one that is held up)
      for (bool moved = true; moved;) {
        moved = false;
        for (int c = 0; c < kCopy; ++c)
          for (Role& r = copy[c]; r.item < end;) {
            if (c == 0 && !r.published) {
              published = r.item;
              r.published = moved = true;
            }
            if (r.box >= boxes) {
              r.box -= boxes;
              ++r.item;
              r.published = false;
              moved = true;
              continue;
            }
            const long b = r.item * boxes + r.box;
            if (b >= S::kStages && !has(used, b - S::kStages)) break;
            has(issued, b) = 1;
            r.box += kCopy;
            moved = true;
          }
        for (int w = 0; w < kWarps; ++w)
          for (Role& r = product[w]; r.item < end;) {
            if (r.box >= boxes && r.boxes == 0) {  // no box, or no further one, of this item
              r.box -= boxes;
              ++r.item;
              moved = true;
              continue;
            }
            if (r.box < boxes) {
              const long b = r.item * boxes + r.box;
              // (the item's rows are read behind the wait for a box)
              if (published < r.item || !has(issued, b) || (w == held && r.item >= at)) break;
              has(used, b) = 1;
              ++r.boxes;
              r.box += kWarps;
              moved = true;
              continue;
            }
            if (r.parts - read[w] >= S::kPlaces) break;
            ++r.parts;
            if (r.item >= static_cast<long>(whole.size())) whole.resize(r.item + 1, 0);
            ++whole[r.item];
            r.boxes = 0;
            r.box -= boxes;
            ++r.item;
            moved = true;
          }
        while (summed < static_cast<long>(whole.size()) && whole[summed] == sharing && !(held == kWarps && summed >= at)) {
          for (int p = 0; p < sharing; ++p) ++read[(summed * boxes + p) % kWarps];
          ++summed;
          moved = true;
        }
      }
      // what the one that is held up still reads, or waits for, of its item
      const long item = held < kWarps ? product[held].item : summed;
      const long handed = static_cast<long>(whole.size()) - 1;
      if (published >= end - 1) {
        std::printf("%d boxes, warp %d held up at %d: the others run away from it\n", boxes, held, at);
        return 1;
      }
      if (published >= item + kBars || handed >= item + kBars) {
        std::printf("%d boxes, warp %d held up at item %ld: rows known up to item %ld, parts of item %ld, %d kept\n", boxes, held, item,
                    published, handed, kBars);
        return 1;
      }
    }
  }
  return 0;
}

int main(int, char** argv) {
  const int bits = std::atoi(argv[1]), boxes = std::atoi(argv[2]);
  return bits == 4 ? check<4>(boxes) : check<8>(boxes);
}

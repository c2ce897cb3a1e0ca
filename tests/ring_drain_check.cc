// Copies go into the stages of a ring one after the other; what a kernel that gives up after any number of them waits for.
// ring_drain_check <stages>: 0 if every stage's last copy is waited for and nothing that never comes, 1 and the first fault otherwise.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "ring_order.h"

int main(int, char** argv) {
  const int stages = std::atoi(argv[1]);
  for (int copies = 0; copies <= 5 * stages; ++copies) {
    std::vector<int> into(stages, 0);  // copies asked for: a stage's phase 0, 1, 2 ... ends with its first, second ... copy
    int next = 0, phase = 0;
    for (int c = 0; c < copies; ++c) {
      ++into[next];
      if (++next == stages) {
        next = 0;
        phase ^= 1;
      }
    }
    for (int i = 0; i < stages; ++i) {
      const int parity = mld::ring_last_phase(i, next, phase);
      // a wait for a parity ends when the last phase that has ended has it; before the first, that is 1
      const int last = into[i] > 0 ? (into[i] - 1) & 1 : 1;
      if (parity != last) {
        std::printf("%d copies, stage %d: waits for %d, its last copy ends %d\n", copies, i, parity, last);
        return 1;
      }
    }
  }
  return 0;
}

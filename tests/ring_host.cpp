// A model of mbarriers behind bk_ring.h: copies are armed round a ring, land in any order, and a CTA that gave up waits for those on their way.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../bunker_b200/csrc/bk_ring.h"

struct Barrier {
  int phase = 0;       // completed phases
  bool armed = false;  // the present phase has its arrival, its bytes are on their way
  bool wait(unsigned parity) const { return ((unsigned)phase & 1) != parity; }   // the phase of this parity has completed
  void land() {
    phase++;
    armed = false;
  }
};

int main() {
  unsigned seed = 1;
  auto rnd = [&](int n) { return (int)((seed = seed * 1664525u + 1013904223u) >> 8) % n; };
  int wrong = 0;
  for (int stages : {1, 2, 5, 12})
    for (int armed = 0; armed < 4 * stages + 3; armed++)
      for (int trial = 0; trial < 40; trial++) {
        std::vector<Barrier> ring(stages);
        for (int i = 0; i < armed; i++) {
          Barrier& b = ring[i % stages];
          if (b.armed) b.land();   // (a stage is armed again when its copy has landed and was used)
          b.armed = true;
        }
        for (int s = 0; s < stages; s++)
          if (ring[s].armed && rnd(2)) ring[s].land();
        for (int s = 0; s < stages; s++) {
          const int last = bk_ring_last_parity(armed, s, stages);
          if (last < 0) wrong += armed > s;
          else wrong += ring[s].wait((unsigned)last) == ring[s].armed;   // a wait returns exactly when nothing is on its way
        }
      }
  printf("%d\n", wrong);
  return wrong != 0;
}

// What the attention kernels' rings of two stages do when a wait runs out: shared by the kernels and the tests (plain C++).
#pragma once

#include "kv4_layout.h"

namespace cb {

// A ring's steps have stages 0 and 1 in turn and, on the stage's mbarrier, the parity of the times it was filled before.  While a step is waited for,
// its own copies are under way and, if there is a step behind it (`more`), that one's: each is asked for two steps ahead, when its stage has been
// read.  When the wait ran out nothing is asked for any more, and land(stage, phase) waits for those: a copy that lands in the memory of
// a block that has ended, or has put its sums there, is in somebody else's.
template <class Land>
CB_HD void ring_land(int stage, unsigned phase, bool more, Land land) {
  land(stage, phase);
  if (more) land(stage ^ 1, phase ^ (unsigned)stage);
}

}  // namespace cb

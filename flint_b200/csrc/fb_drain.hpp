// In which order a launch that gives up waits for what it still has in flight, apart from the waiting itself: the kernels hand in their barriers, a host-side
// test a model of them. No CUDA here.
//
// A wait for parity p passes when the phase AHEAD of the one under way has that parity. So a wait for phase k says something only while phase k - 1 has ended and
// phase k + 1 has not: phase k - 1 still open, it passes at once, and with phase k + 1 over, not at all.
#pragma once
#include <stdint.h>

namespace fb {

// The last (up to) N of `issued` copies into a ring of N stages: wait(stage, parity). A copy into a stage is issued once the one before it there has ended. Only copies
// that were issued count: one more, and the oldest is passed over.
template <int N, class Wait>
constexpr void drain_ring_order(uint32_t issued, Wait wait) {
  const uint32_t n = issued < (uint32_t)N ? issued : (uint32_t)N;
  for (uint32_t k = 1; k <= n; k++) wait((issued - k) % N, ((issued - k) / N) & 1);
}

// Everything that was issued ahead of one more commit() on a barrier that `committed` commits have armed, the last of which may be under way: that one
// first, then the new one, which also ends what no commit was issued for.
template <class Wait, class Commit>
constexpr void drain_commit_order(uint32_t committed, Wait wait, Commit commit) {
  if (committed) wait((committed - 1) & 1);
  commit();
  wait(committed & 1);
}

}  // namespace fb

// The order in which a chunk's tile takes its steps (paged_tile.hpp), apart from what a step
// computes.  Plain C++ without HIP types, so it also compiles for the host.
#pragma once

#include "page_math.hpp"

namespace pa {

// Whether a step and the one after it have a live key.
struct LiveSteps {
  bool now, ahead;
};

// Steps 0 .. n - 1 (n >= 1), the scores of a step one iteration ahead of its sums and in two places
// in turn: `a` holds those of step 0 on entry and those of step n - 1, whose sums are left to the
// caller, at the end.  next(j) makes step j + 1's keys arrive and says which of steps j and j + 1 are live;
// body(j, live, x, y) takes step j's sums from its scores x and puts those of step j + 1 into y; turn()
// ends an iteration.  Where both steps are dead there is no body, and y keeps the scores of an earlier
// step: a later body finds them in x where its own step is dead (live false), and takes no sums of them.
template <typename Scores, typename Next, typename Body, typename Turn>
PA_HD void walk_steps(int n, Scores& a, Scores& b, Next& next, Body& body, Turn& turn) {
  auto iterate = [&](int j, const Scores& x, Scores& y) __attribute__((always_inline)) {
    const LiveSteps live = next(j);
    if (live.now || live.ahead) body(j, live.now, x, y);
    turn();
  };
  int j = 0;
#pragma unroll 1
  for (; j + 2 < n; j += 2) {
    iterate(j, a, b);
    iterate(j + 1, b, a);
  }
  if (j + 1 < n) {
    iterate(j, a, b);
    a = b;
  }
}

}  // namespace pa

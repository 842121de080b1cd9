// A wait on an mbarrier that ends whatever happens.
#pragma once

#include "pa_common.cuh"

namespace pa {

// False: gave up, after POLLS polls or, every LOOK polls, since another wait had.  g.marked() says whether one had, g.mark()
// leaves word of it and g.report() sets the status word: on both ways, so that a call that finds the mark of an earlier one
// does not fail in silence.  A kernel polls once by itself, which is enough for a phase that has completed, and
// calls this out of line (with one exit for both ways csrc/prefix_sm100.cu took 122 us for what takes 117).
template <int POLLS, int LOOK, class G>
__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity, const G& g) {
  static_assert(LOOK >= 1 && POLLS >= LOOK, "looks at the mark at least once");
  for (int i = 0; i < POLLS; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (i % LOOK == LOOK - 1 && g.marked()) {
      g.report();
      return false;
    }
  }
  g.mark();
  g.report();
  return false;
}

}  // namespace pa

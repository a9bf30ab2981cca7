// kg_pool_ring.h — the steps of the ring of stages between the warp that loads K
// and V and the warps that use them, in kg_pool_attend_dev's kernels. The barriers
// are `b`: the kernels' own, or those of a CPU test that runs the same steps.
#pragma once
#include "kg_pool_sched.h"

namespace kg {
namespace serve {

// Load `it` for the lanes of a warp that uses it: every lane calls. A wait may run out for one lane and not for another, so
// the lanes agree on what they saw before any of them goes on; a warp that has seen one run out takes nothing more.
template <typename B>
KG_HD bool ring_take(B &b, int stages, int it, bool alive) {
    return b.all(alive && b.wait_full(it % stages, (it / stages) & 1));
}

}  // namespace serve
}  // namespace kg

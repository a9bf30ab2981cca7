// kg_pool_ring.h — the steps of the ring of stages between the warp that loads K
// and V and the warps that use them, in kg_pool_attend_dev's kernels. The barriers
// are `b`: the kernels' own, or those of a CPU test that runs the same steps.
//   full[stage]   one arrival of the loader and the load's bytes
//   empty[stage]  an arrival of every warp that uses it
// When a wait runs out, the warp that saw it frees no stage any more: a load into that
// stage may still be under way. The loader then comes to a wait that does not end (or
// that ends at once, by the CTA's abort flag), issues nothing more, and leaves when what
// it has issued has landed, as it always does: a load must not outlive its CTA.
#pragma once
#include "kg_pool_sched.h"

namespace kg {
namespace serve {

// The loader, one thread: stage it % stages may be filled with load `it`; false when the wait ran out.
template <typename B>
KG_HD bool ring_claim(B &b, int stages, int it) {
    if (!b.wait_empty(it % stages, ((it / stages) & 1) ^ 1)) return false;
    b.arm(it % stages);
    return true;
}
// The loader at its end, `issued` loads after its start: the last ones have landed.
template <typename B>
KG_HD void ring_drain(B &b, int stages, int issued) {
    for (int it = issued > stages ? issued - stages : 0; it < issued; ++it) b.landed(it % stages, (it / stages) & 1);
}
// Load `it` for the lanes of a warp that uses it: every lane calls. A wait may run out for one lane and not for another, so
// the lanes agree on what they saw before any of them goes on; a warp that has seen one run out takes nothing more.
template <typename B>
KG_HD bool ring_take(B &b, int stages, int it, bool alive) {
    return b.all(alive && b.wait_full(it % stages, (it / stages) & 1));
}
// One lane of the warp, when it has used the stage.
template <typename B>
KG_HD void ring_free(B &b, int stages, int it, bool alive) {
    if (alive) b.free(it % stages);
}

}  // namespace serve
}  // namespace kg

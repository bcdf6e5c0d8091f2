// Barriers of the "looks" at V in the FP16 copies of paged_tensor.cu, without CUDA so that every
// order of events can be gone through on the host (tests/cpp/copy_ring_test.cpp).
//
// K and V tiles go through a ring of slots in turn.  A V tile that has to be looked through
// completes on a look barrier first: warp 9 arms it, all copying warps wait for it, look through
// their share and only then arrive on the slot's "full" barrier.  Waits go by a phase's parity, so
// a barrier may not be armed again before every warp has passed its last phase.  With one barrier
// to a slot the ring sees to that: warp 9 comes back to a slot when it is empty, for which the MMAs
// need the slot's full barrier, for which they need every copying warp behind its look.  (One
// barrier for all slots has no such chain: warp 9 can arm V of the next key tile as soon as the
// slot of this one's K is free.)
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define IB_RING_FN __host__ __device__ __forceinline__
#else
#define IB_RING_FN inline
#endif

namespace ib {

struct Looks {
    uint32_t parity = 0;  // of each barrier's next phase, a bit each
    static IB_RING_FN int bar(int slot) { return slot; }
    // The parity to wait for in this look at `slot`.
    IB_RING_FN int take(int slot) {
        const int p = (int)((parity >> bar(slot)) & 1u);
        parity ^= 1u << bar(slot);
        return p;
    }
};

}  // namespace ib

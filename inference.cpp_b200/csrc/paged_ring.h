// Bookkeeping of the copies in paged_tensor.cu, without CUDA so that every order of events can be
// gone through on the host (tests/cpp/copy_ring_test.cpp).
//
// Looks.  K and V tiles go through a ring of slots in turn.  A V tile that has to be looked through
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

// K and V tiles of a segment of n key tiles in the order in which they are used: the e-th is K (even) or V
// (odd) of key tile tile_order(e, n) / 2.  SPLIT (one query tile, two groups of softmax warps that take its
// key tiles in turn): K0 K1 V0 K2 V1 K3 ..; otherwise K0 V0 K1 V1 ..
template <bool SPLIT>
IB_RING_FN int tile_order(int e, int n) {
    if (!SPLIT) return e;
    if (e < 2) return e == 0 ? 0 : n > 1 ? 2 : 1;
    if (e >= 2 * n - 2) return 2 * (e - n) + 1;
    return e & 1 ? e + 1 : e - 1;  // K of e / 2 + 1/2, V of e / 2 - 1
}

// Which of the three copying warps sees to a tile by itself (SPLIT with TMA): the ring's tiles in turn.  A
// look is its warp's alone then, but the phases of all looks at a slot count: the others take them too.
IB_RING_FN int tile_owner(int half) { return half % 3; }

// The buffer of two in which the factors of a segment's rows lie (SPLIT, FP16 pages: the second group writes
// them with q, the first one reads them up to the segment's end).  Segments without key tiles are not counted:
// they stage no q and pass no barrier, so nothing would keep the second group from writing two ahead.
struct ScaleTurn {
    uint32_t n = 0;
    IB_RING_FN int buffer() const { return (int)(n & 1); }
    IB_RING_FN void next(int key_tiles) { n += key_tiles > 0; }
};

struct Looks {
    uint32_t parity = 0;  // of each barrier's next phase, a bit each
    static IB_RING_FN int bar(int slot) { return slot; }
    // The parity to wait for in this look at `slot`.
    IB_RING_FN int take(int slot) {
        const int p = (int)((parity >> bar(slot)) & 1u);
        parity ^= 1u << bar(slot);
        return p;
    }
    // The parity that the last look at `slot` waited for.
    IB_RING_FN int taken(int slot) const { return (int)(~(parity >> bar(slot)) & 1u); }
};

// Before a CTA ends no copy may still be landing in its shared memory, also where a wait has run
// out and the loops were left early.  The waits that the FP16 copies owe when they leave at tile
// `half` (not yet counted): full(slot, use) for the tiles before it, which a wait for an empty slot
// has not covered, and look(slot, parity) for its own where the look's wait ran out (looking).
template <int SLOTS, typename Full, typename Look>
IB_RING_FN void drain_copies(int half, bool looking, const Looks& looks, Full full, Look look) {
    if (looking) look(half % SLOTS, looks.taken(half % SLOTS));
    for (int h = half > SLOTS ? half - SLOTS : 0; h < half; ++h) full(h % SLOTS, h / SLOTS);
}

// The FP32 copies: how many K tiles (kv 0) and V tiles (kv 1) are on their way or there.
struct RawSent {
    int k = 0, v = 0;
    IB_RING_FN void add(int kv) { ++(kv ? v : k); }
    // full(kv, phase) for the last of each
    template <typename Full>
    IB_RING_FN void drain(Full full) const {
        if (k > 0) full(0, k - 1);
        if (v > 0) full(1, v - 1);
    }
};

}  // namespace ib

// mx_ring.cuh -- arithmetic of the few-row kernel's ring of k-blocks (mx_f4.cu),
// in plain C++ so that a host program can run the same rules.
#pragma once

#ifdef __CUDACC__
#define QMM_RING_FN __host__ __device__ __forceinline__
#else
#define QMM_RING_FN inline
#endif

namespace qmm {

// Slots in use by a block with nk k-blocks of each tile.  With a whole number of
// tiles in the ring a slot holds the same k-block of one tile after another:
// own planes made for an item's first tiles serve all of its tiles.
QMM_RING_FN int f4_ring_slots(bool own, int nk, int stages) {
    return own && nk <= stages ? stages - stages % nk : stages;
}
// An item's tiles that planes are made for.
QMM_RING_FN int f4_ring_fresh(bool own, int nk, int stages) {
    return own && nk <= stages ? f4_ring_slots(own, nk, stages) / nk : 0x7fffffff;
}

// A wait on a slot's parity tells two of its phases apart, not three.  Before
// k-block i is put into its slot, k-block i - L has to be consumed; the wait
// tells that from i - 2 L only once i - 2 L is known to be.  It is when i - L has
// begun, since the weights of i - L went into the slot after that: `begun`
// k-blocks have, counted from 0.
QMM_RING_FN bool f4_ring_may_wait(int begun, int i, int L) { return begun > i - L; }

}  // namespace qmm

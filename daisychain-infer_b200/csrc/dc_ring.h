// dc_ring.h -- which copies of a ring of buffers may still be in flight.
//
// Copy i of a ring of STAGES buffers goes to buffer i % STAGES and completes
// phase i / STAGES of that buffer's barrier.  A wait names a phase by its parity
// alone, so it tells a phase from the one before it and no further back: a wait
// for the parity of a phase that is over by an even number of phases returns at once.
//
// A block must not end, nor use its ring for something else, while copies into it
// are in flight.  Plain C++, so that a host program can check the bookkeeping.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define DC_RING __device__ __forceinline__
#else
#define DC_RING inline
#endif

namespace dcr {

// Waits for copies first .. end - 1, the newest ones (at most STAGES).
template <int STAGES, typename Wait>
DC_RING void await_copies(int first, int end, Wait wait) {
  for (int i = first; i < end; i++) wait(i % STAGES, (uint32_t)(i / STAGES) & 1);
}
// By the copier of a ring, once it issues no more: `issued` copies so far, for
// whatever reason.  (Others may have given up on copies that it had no cause to wait
// for, so it waits in any case; where all went well they are long met.)
template <int STAGES, typename Wait>
DC_RING void drain(int issued, Wait wait) {
  await_copies<STAGES>(issued > STAGES ? issued - STAGES : 0, issued, wait);
}
// By a warp that copies for itself, copy i + STAGES once it is done with tile i, of
// `n`: `next` is the tile that it gave up on (n: it is done with all of them).
template <int STAGES, typename Wait>
DC_RING void drain_own(int next, int n, Wait wait) {
  await_copies<STAGES>(next, next + STAGES < n ? next + STAGES : n, wait);
}

}  // namespace dcr

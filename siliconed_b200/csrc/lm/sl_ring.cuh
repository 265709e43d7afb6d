// The order of a warp's copies in a ring of slots, one mbarrier a slot: which slot the next copy fills, which copy is used
// next, and the parity of its barrier's phase.  Plain C++, so that it runs on the host too.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define SL_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define SL_HOST_DEVICE inline
#endif

namespace sl {

template <int kSlots>
struct Ring {
  static_assert(kSlots <= 32, "a parity bit a slot");
  uint32_t fill = 0, take = 0, phases = 0;  // the slot to fill, the slot to use, and the slots' parities

  SL_HOST_DEVICE uint32_t parity() const { return (phases >> take) & 1u; }
  // A copy into slot `fill` is on its way.
  SL_HOST_DEVICE void filled() { fill = fill + 1 == kSlots ? 0 : fill + 1; }
  // The copy into slot `take` has arrived.
  SL_HOST_DEVICE void taken() {
    phases ^= 1u << take;
    take = take + 1 == kSlots ? 0 : take + 1;
  }
  // After a wait that gave up: waits for every copy still on its way, the one that was waited for first.  That one was not
  // taken, so there is at least one (and take == fill means a full ring).
  template <typename Wait>
  SL_HOST_DEVICE void drain(Wait&& wait) {
    do {
      wait(take, parity());
      taken();
    } while (take != fill);
  }
};

}  // namespace sl

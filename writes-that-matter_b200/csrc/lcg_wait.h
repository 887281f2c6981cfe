// The bounded wait as control flow alone, so that it also compiles for the host.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define LCG_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define LCG_HOST_DEVICE inline
#endif

namespace lcg {

// Tries until `try_wait` (which may suspend the thread for a while) is met, `abort_flag` is set, or `limit_ns` of
// `now` have passed: then the flag is set and `give_up` called.
template <class TryWait, class Now, class GiveUp>
LCG_HOST_DEVICE void bounded_wait(volatile uint32_t* abort_flag, uint64_t limit_ns, TryWait try_wait, Now now,
                                  GiveUp give_up) {
  uint64_t t0 = 0;
  // the timer is read once in 64 tries: reading it takes longer than most waits
  for (uint32_t tries = 1; !try_wait(); ++tries) {
    if (*abort_flag) return;
    if ((tries & 63u) != 0) continue;
    const uint64_t t = now();
    if (t0 == 0) t0 = t;
    if (t - t0 > limit_ns) {
      *abort_flag = 1u;
      give_up();
      return;
    }
  }
}

// The end of a ring's producer, which stands at (stage, parity) behind its last fill and would wait there for the
// stage's release before the next: waits for the release of all stages.  They arrive in this CTA's barriers by
// themselves, so it must not end before the last has.  A stage never filled is not waited for.
template <class Wait>
LCG_HOST_DEVICE void drain_ring(uint32_t stages, uint32_t stage, uint32_t parity, Wait wait) {
  for (uint32_t i = 0; i < stages; ++i) {
    wait(stage, parity);
    if (++stage == stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
}

}  // namespace lcg

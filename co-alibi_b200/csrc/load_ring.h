// Cursors of a ring of load slots, each with an mbarrier that completes one phase per load.
// Plain C++, so that the host's tests run the same code as the kernel.
#pragma once

#ifdef __CUDACC__
#define COALIBI_HD __host__ __device__ __forceinline__
#else
#define COALIBI_HD inline
#endif

namespace coalibi {

template <int NBUF>
struct LoadRing {
  int fill = 0, drain = 0;              // slots of the next load and of the oldest one not yet awaited
  unsigned phase = 0;                   // parity of the latter's barrier
  unsigned issued = 0, awaited = 0;

  COALIBI_HD void issue() {
    fill = fill + 1 == NBUF ? 0 : fill + 1;
    ++issued;
  }
  // After a wait on the oldest load that succeeded, and on none other: what is still in flight
  // when a wait runs out has to land before the slots' memory may be given up.
  COALIBI_HD void landed() {
    drain = drain + 1 == NBUF ? 0 : drain + 1;
    if (drain == 0) phase ^= 1;
    ++awaited;
  }
  COALIBI_HD bool in_flight() const { return awaited != issued; }
};

}  // namespace coalibi

// The wait behind every spin of the tensor-core kernels, for device and host compilers alike.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define HA_ANY_INLINE __host__ __device__ __forceinline__
#else
#define HA_ANY_INLINE inline
#endif

namespace ha {

// Waits until done() is true: false once `limit` nanoseconds of now() have passed, which sets *stop, or if another thread has
// set it: at a look after every 256 tries that failed, and with EARLY after the first one.  EARLY is for kernels that go on
// after a lost arrival: a try may sleep for a millisecond, and a quarter of a second in each of their later waits adds up.
template <bool EARLY, class Done, class Now>
HA_ANY_INLINE bool bounded_wait(Done done, Now now, volatile uint32_t* stop, uint64_t limit) {
  if (done()) return true;
  if (EARLY && *stop) return false;
  const uint64_t t0 = now();
  for (;;) {
#ifdef __CUDACC__
#pragma unroll 1
#endif
    for (int i = 0; i < 256; ++i)
      if (done()) return true;
    if (*stop) return false;
    if (now() - t0 > limit) {
      *stop = 1;
      return false;
    }
  }
}

}  // namespace ha

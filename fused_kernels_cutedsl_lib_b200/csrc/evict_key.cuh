// Order-preserving keys of masses, and the range of the keys of a group of threads (cache_evict.cu).
// Plain C++, so that a host program can check it.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define FK_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FK_HOST_DEVICE inline
#endif

namespace fk {
namespace evict {

// The key of a place without a candidate, below every mass's: the key of -inf is 0x007FFFFF.
constexpr uint32_t kNoKey = 0u;

// From a float's bits, -0 already made +0: -inf < ... < 0 < ... < +inf < NaN.
FK_HOST_DEVICE uint32_t key_of_bits(uint32_t u) {
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Least and greatest key of any candidates. The least is held minus 1, so that kNoKey wraps to the greatest
// number and counts for nothing; the 1 is added when all ranges have been joined (added in a thread
// without a candidate it would give 0, a least key below every mass).
struct KeyRange {
  uint32_t below = 0xFFFFFFFFu;
  uint32_t greatest = 0u;
  FK_HOST_DEVICE void add(uint32_t key) { join(key - 1u, key); }
  FK_HOST_DEVICE void join(uint32_t other_below, uint32_t other_greatest) {
    if (other_below < below) below = other_below;
    if (other_greatest > greatest) greatest = other_greatest;
  }
  FK_HOST_DEVICE uint32_t least() const { return below + 1u; }
};

}  // namespace evict
}  // namespace fk

#pragma once
#include <cuda_runtime.h>

namespace fa_sm100 {

// Division of n < 2^31 by a number fixed at launch as one high product, an
// addition and a shift (Granlund and Montgomery).
struct FastDiv {
  unsigned d, mul, shift;
  FastDiv() = default;
  explicit FastDiv(unsigned divisor) : d(divisor), shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = (unsigned)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

}  // namespace fa_sm100

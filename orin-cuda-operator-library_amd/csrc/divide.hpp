#pragma once
// Division of non-negative ints by a divisor that is the same for a whole
// launch: a multiplication and a shift instead of some thirty instructions.

#include <hip/hip_runtime.h>

#include <cstdint>

namespace opl {

// n / divisor for 0 <= n < 2^31. With 2^(s - 1) < divisor <= 2^s,
// ceil(2^(31 + s) / divisor) fits 32 bits, and the product errs by less than one
// part in n.
struct Divider {
  unsigned mul = 0;
  int shift = 0;

  static Divider by(int divisor) {  // > 0
    Divider r;
    int s = 0;
    while ((std::uint64_t(1) << s) < static_cast<std::uint64_t>(divisor)) ++s;
    r.shift = 31 + s;
    r.mul = static_cast<unsigned>(((std::uint64_t(1) << r.shift) + divisor - 1) / divisor);
    return r;
  }

  __host__ __device__ int quotient(int n) const {
    return static_cast<int>(static_cast<std::uint64_t>(static_cast<unsigned>(n)) * mul >> shift);
  }
};

}  // namespace opl
